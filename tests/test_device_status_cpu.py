"""The device's status word on the host side: threads that ask for it at the same
time get the same one, and a device may be named by text or without its index.
(The word lies on the CPU here.)"""
import threading

import pytest
import torch

import tree_training_b200 as tt
from tree_training_b200 import attention


def test_threads_get_one_word(monkeypatch):
    monkeypatch.setattr(attention, "_status", {})
    zeros, inside = torch.zeros, threading.Barrier(2)

    def slow_zeros(*a, **kw):
        inside.wait(timeout=20)              # both threads have found no word
        return zeros(*a, **kw)
    monkeypatch.setattr(attention.torch, "zeros", slow_zeros)
    got = []
    threads = [threading.Thread(
        target=lambda: got.append(attention._status_word(torch.device("cpu")))) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 2 and got[0] is got[1]
    assert attention._status_word(torch.device("cpu")) is got[0]


@pytest.mark.parametrize("named", [torch.device("cuda"), "cuda", "cuda:1", torch.device("cuda", 1)])
def test_errors_of_a_device_without_an_index(monkeypatch, named):
    word = torch.tensor([4], dtype=torch.int32)
    monkeypatch.setattr(attention, "_status", {torch.device("cuda", 1): word})
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(tt.TTError):
        tt.check_device_status(named)
    assert int(word) == 0
