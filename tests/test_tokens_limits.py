"""Sizes at the ends of their types, without a GPU."""
import subprocess
import sys


def test_workspace_sizes_for_any_upper_bound_of_the_keys():
    """In a process of its own: an integer that runs over may end it."""
    code = ("from promptmoge_b200 import _lib\n"
            "f = _lib.load().pmg_attention_workspace_bytes\n"
            "for docs, hk, d in ((444, 8, 64), (296, 8, 128), (1, 1, 64), (65535, 64, 64), (7, 4, 128), (2**31 - 1, 65535, 64)):\n"
            "    for most in (2**31 - 1, 2**31 - 513, 2**30, 65536, 1, 0):\n"
            "        n = f(docs, hk, hk, d, 1, most)\n"
            "        assert 0 <= n < 1 << 30, (docs, hk, d, most, n)\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr[-2000:])


def test_one_status_word_for_all_threads(monkeypatch):
    """Threads on their first call: all get the word that check() reads."""
    import threading
    import time

    import torch

    from promptmoge_b200 import tokens
    made = []

    class Word:
        device = None

        def data_ptr(self):
            return id(self)

    def zeros(*_, **__):
        time.sleep(0.02)
        made.append(Word())
        return made[-1]

    class Stream:
        def synchronize(self):
            time.sleep(0.02)

    monkeypatch.setattr(tokens, "_status_words", {})
    monkeypatch.setattr(tokens, "_status_ptrs", {})
    monkeypatch.setattr(torch, "zeros", zeros)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *_: Stream())
    got, gate = [], threading.Barrier(8)

    def first():
        gate.wait()
        got.append(tokens._status(0))
    threads = [threading.Thread(target=first) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and set(got) == {tokens._status_words[0].data_ptr()}
