"""The training operators called by two host threads at a time, under forward-mode
differentiation, and in inference mode."""
import threading

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import tree_training_b200 as tt

pytestmark = pytest.mark.gpu
DEV = "cuda"


def steps(seed):
    """A pass through every operator, forward and backward; what it gives."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()
    n, H = 100 + 37 * seed, 64 + 8 * seed
    table, wg, wu = r(500, H).requires_grad_(True), r(96, H), r(96, H)
    ids = torch.randint(0, 500, (n,), generator=g, device=DEV)
    x = tt.embedding(ids, table)
    h = tt.gated_linear(x, wg, wu)
    out = tt.linear_cross_entropy(x, table, ids)
    dt, = torch.autograd.grad([h.float().sum(), out.losses.sum()], [table])
    norm = tt.clip_grad_norm([dt], 1.0)
    return [x.detach(), h.detach(), out.losses.detach(), dt, norm]


def test_two_threads():
    want = [steps(i) for i in range(2)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(15):
                got = steps(i)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    tt.check_device_status()


def test_forward_mode_is_refused():
    x, w = torch.randn(4, 8, device=DEV), torch.randn(6, 8, device=DEV)
    ids = torch.zeros(4, dtype=torch.int64, device=DEV)
    with fwAD.dual_level():
        d = fwAD.make_dual(w, torch.ones_like(w))
        for f in (lambda: tt.embedding(ids, d), lambda: tt.gated_linear(x, d, w),
                  lambda: tt.gated_linear(x, w, d), lambda: tt.linear_cross_entropy(x, d, ids),
                  lambda: tt.grad_norm([d]), lambda: tt.clip_grad_norm([d], 1.0)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                f()


def test_inference_mode():
    with torch.inference_mode():
        w = torch.randn(6, 8, device=DEV)
        x = tt.embedding(torch.zeros(4, dtype=torch.int64, device=DEV), w)
        h = tt.gated_linear(x, w, w)
        assert tt.linear_cross_entropy(h.new_ones(3, 8), w, torch.zeros(
            3, dtype=torch.int64, device=DEV)).losses.shape == (3,)
        assert float(tt.clip_grad_norm([h], 1.0)) > 0
    before = h.clone()
    with pytest.raises(RuntimeError):
        tt.clip_grad_norm([h], 0.1)
    assert torch.equal(h, before)


def test_backward_into_leaves():
    table = torch.randn(50, 16, device=DEV, requires_grad=True)
    ids = torch.arange(50, device=DEV)
    for _ in range(2):
        x = tt.embedding(ids, table)
        tt.linear_cross_entropy(x, table, ids).losses.sum().backward()
    one = table.grad.clone()
    table.grad = None
    tt.linear_cross_entropy(tt.embedding(ids, table), table, ids).losses.sum().backward()
    assert torch.allclose(one, 2 * table.grad, rtol=1e-6)
