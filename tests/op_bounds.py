"""Error bounds shared by the tests of the layer operators.

A result that is computed in fp32 and rounded once to type T may differ from
the 64-bit value y by

    u(T) |y|  +  steps * 2^-24 * magnitude  +  tiny(T)

where u(T) is T's unit roundoff, ``magnitude`` the sum of the absolute values
of the terms that were added up, ``steps`` the most fp32 roundings a term goes
through, and tiny(T) half of T's smallest subnormal.
"""
import torch

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
EPS = 2.0 ** -24


def check(name, got, want, magnitude, steps):
    """got [T] against want and magnitude in 64 bits; infinities and NaN have
    to stand in the same places."""
    g, w = got.double().cpu(), want.double().cpu()
    assert g.shape == w.shape, f"{name}: {tuple(g.shape)} != {tuple(w.shape)}"
    fine = torch.isfinite(w)
    assert torch.equal(g.isnan(), w.isnan()), f"{name}: NaN in other places"
    assert torch.equal(g[~fine & ~w.isnan()], w[~fine & ~w.isnan()]), f"{name}: infinities differ"
    mag = torch.as_tensor(magnitude, dtype=torch.float64).cpu().expand_as(w)
    bound = UNIT[got.dtype] * w.abs() + steps * EPS * mag + TINY[got.dtype]
    over = ((g - w).abs() - bound)[fine]
    if over.numel():
        i = int(over.argmax())
        assert float(over.max()) <= 0, (
            f"{name}: {float(g[fine][i])!r} for {float(w[fine][i])!r}, over its bound "
            f"{float(bound[fine][i]):.3e} by {float(over[i]):.3e}")


def directional(f, xs, outs_grads, grads, steps, tol, seed=0):
    """<grads, d> against the central difference of sum <outs, outs_grads>
    along a random direction d of all inputs (everything fp32; sums in 64
    bits).  ``tol`` is relative to |grads| |d| / sqrt(n)."""
    g = torch.Generator(device=xs[0].device).manual_seed(seed)
    ds = [torch.randn(x.shape, generator=g, device=x.device) for x in xs]
    val = lambda s: sum(float((o.double() * w.double()).sum()) for o, w in
                        zip(f(*[(x + s * d).detach() for x, d in zip(xs, ds)]), outs_grads))
    fd = (val(steps) - val(-steps)) / (2 * steps)
    an = sum(float((gr.double() * d.double()).sum()) for gr, d in zip(grads, ds))
    size = sum(float((gr.double() ** 2).sum()) for gr in grads) ** 0.5
    assert abs(fd - an) <= tol * size, f"difference {fd}, gradient {an}, size {size}"
