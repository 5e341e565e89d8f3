"""The layer operators from several host threads at once, each on a stream of its
own: calls of different widths share a kernel and its launch attributes."""
import threading

import pytest
import torch

import tree_training_b200 as tt

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def together(*jobs):
    """Runs every job in a thread of its own, on a stream of its own."""
    errors, start = [], threading.Barrier(len(jobs))

    def go(job):
        try:
            with torch.cuda.stream(torch.cuda.Stream(DEV)):
                start.wait()
                job()
                torch.cuda.current_stream(DEV).synchronize()
        except Exception as e:                       # noqa: BLE001  (told to the test)
            errors.append(e)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=go, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors[0]


def norms(D, gate, seed):
    """Forward and backward calls of one width, each compared with the first."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()
    x, res, w = (t.requires_grad_(True) for t in (r(9, D), r(9, D), r(D)))
    u = r(9, D).requires_grad_(True) if gate else None
    dy, dr = r(9, D), r(9, D)
    ins = [x, res, w] + ([u] if gate else [])

    def go():
        out = tt.residual_norm(x, res, w, gate=u)
        return [*out, *torch.autograd.grad(out, ins, [dy, dr])]
    first = go()

    def job():
        for _ in range(1500):
            last = go()
        assert all(torch.equal(a, b) for a, b in zip(first, last))
    return job


@pytest.mark.parametrize("gate", [False, True])
def test_widths_of_one_kernel(gate):
    together(*(norms(D, gate, D) for D in (8192, 528, 2048, 4096)))


def test_forward_calls_without_gradients():
    def job(D):
        x, w = torch.ones(4, D, device=DEV).bfloat16(), torch.ones(D, device=DEV).bfloat16()

        def go():
            for _ in range(8000):
                y, r = tt.residual_norm(x, x, w)
            assert (r == 2).all() and (y == 1).all()
        return go
    together(*(job(D) for D in (8192, 520, 8192, 1024)))
