"""Refusals of the layer operators' C ABI: bad sizes, pointers and types come back
as a status before anything touches a device (so they run without a GPU)."""
import pytest

from tree_training_b200 import _lib

F32, BF16, U8 = _lib.TT_F32, _lib.TT_BF16, _lib.TT_U8
P = 1 << 20            # a pointer that is never followed


def status(name, *args):
    return getattr(_lib.lib(), name)(*args)


def rotary(dtype=BF16, n=4, hq=2, hk=1, D=8, R=8, q=P, k=P, pos=P, table=P, qo=P, ko=P, n_pos=16):
    return status("tt_rotary", dtype, n, hq, hk, D, R, 0, 0, q, hq * D, D, k, hk * D, D, pos, 1,
                  table, n_pos, qo, ko, None, None)


@pytest.mark.parametrize("bad", [
    dict(n=-1), dict(hq=0, hk=0), dict(hq=-1), dict(hq=70000), dict(D=0), dict(D=1 << 20), dict(R=0),
    dict(R=7), dict(R=10), dict(n_pos=-1), dict(q=None), dict(k=None), dict(pos=None),
    dict(table=None), dict(qo=None), dict(ko=None)])
def test_rotary(bad):
    assert rotary(**bad) == _lib.TT_ERR_INVALID_ARG


def test_rotary_type_and_nothing_to_do():
    assert rotary(dtype=U8) == _lib.TT_ERR_UNSUPPORTED
    assert rotary(n=0, q=None, k=None, pos=None, table=None, qo=None, ko=None) == _lib.TT_OK


def norm(dtype=BF16, res_dtype=BF16, rows=4, D=16, x=P, res=P, w=P, mode=0, gate=None, y=P, r=P,
         stats=None):
    return status("tt_residual_norm_fwd", dtype, res_dtype, rows, D, x, D, res, D, w, None, 0, 0.0,
                  gate, D, mode, 1.0, 1e-6, y, r, stats, None, None)


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(D=0), dict(D=16385), dict(mode=4), dict(mode=-1), dict(mode=3), dict(x=None),
    dict(w=None), dict(y=None), dict(r=None), dict(stats=P + 4)])
def test_residual_norm(bad):
    assert norm(**bad) == _lib.TT_ERR_INVALID_ARG


def test_residual_norm_types_and_sizes():
    assert norm(dtype=U8, res_dtype=U8) == _lib.TT_ERR_UNSUPPORTED
    assert norm(res_dtype=_lib.TT_F16) == _lib.TT_ERR_UNSUPPORTED
    assert norm(rows=0, x=None, w=None, y=None, r=None) == _lib.TT_OK
    bwd = lambda blocks=4, **kw: status(
        "tt_residual_norm_bwd", BF16, BF16, kw.get("rows", 4), kw.get("D", 16), kw.get("x", P), 16,
        P, 16, P, None, 0, 0.0, None, 0, 0, 1.0, kw.get("stats", P), P, 16, P, 16, P, P, None, P,
        None, kw.get("part", P), blocks, None, None)
    for bad in (dict(blocks=0), dict(rows=-1), dict(D=0), dict(x=None), dict(stats=None),
                dict(part=None), dict(stats=P + 4)):
        assert bwd(**bad) == _lib.TT_ERR_INVALID_ARG
    assert bwd(rows=0) == _lib.TT_OK
    f = _lib.lib().tt_residual_norm_bwd_blocks
    assert f(0, 64) == 1 and f(5, 0) == 1 and 1 <= f(5, 64) <= 5 and f(1 << 40, 4096) > 100


def test_moe():
    plan = lambda ids=P, n=8, E=4, slots=P, entries=P, offsets=P, ws=None, size=0: status(
        "tt_moe_plan", ids, 1, n, E, slots, entries, offsets, ws, size, None)
    for bad in (dict(n=-1), dict(n=1 << 31), dict(E=0), dict(E=1025), dict(offsets=None),
                dict(ids=None), dict(slots=None), dict(entries=None)):
        assert plan(**bad) == _lib.TT_ERR_INVALID_ARG
    need = status("tt_moe_plan_workspace_size", 1 << 20, 64)
    assert need > 0 and status("tt_moe_plan_workspace_size", 8, 4) == 0
    assert status("tt_moe_plan_workspace_size", -1, 4) == -1
    assert plan(n=1 << 20, E=64) == _lib.TT_ERR_WORKSPACE
    assert plan(n=1 << 20, E=64, ws=P, size=need - 1) == _lib.TT_ERR_WORKSPACE
    rows = lambda name, T=4, k=2, H=8, E=4, slots=P, offsets=P, src=P, dst=P, dtype=BF16: status(
        name, dtype, T, k, H, E, slots, offsets, src, dst, None)
    for name in ("tt_moe_dispatch", "tt_moe_collect"):
        for bad in (dict(T=-1), dict(k=-1), dict(k=65), dict(H=0), dict(E=0), dict(T=1 << 30),
                    dict(slots=None), dict(offsets=None), dict(src=None), dict(dst=None)):
            assert rows(name, **bad) == _lib.TT_ERR_INVALID_ARG, (name, bad)
        assert rows(name, dtype=U8) == _lib.TT_ERR_UNSUPPORTED
        assert rows(name, T=0, src=None, dst=None) == _lib.TT_OK
    combine = lambda wd=F32, w=P: status("tt_moe_combine", BF16, wd, 4, 2, 8, 4, P, P, P, w, P, None)
    assert combine(w=None) == _lib.TT_ERR_INVALID_ARG
    assert combine(wd=U8) == _lib.TT_ERR_UNSUPPORTED
    spread = lambda ys=P, dw=P, wd=F32: status("tt_moe_spread", BF16, wd, 4, 2, 8, 4, P, P, P, ys, P,
                                               P, dw, None)
    assert spread(ys=None) == spread(dw=None) == _lib.TT_ERR_INVALID_ARG
    assert spread(wd=U8) == _lib.TT_ERR_UNSUPPORTED


def logprobs(dtype=BF16, T=4, V=32, x=P, ld=32, tok=P, M=1, temp=1.0, k=2, logp=P, ent=P, tl=P,
             tt=P):
    return status("tt_token_logprobs_fwd", dtype, T, V, x, ld, tok, M, temp, k, logp, ent, tl, tt,
                  None, None)


@pytest.mark.parametrize("bad", [
    dict(T=-1), dict(T=1 << 31), dict(V=0), dict(M=-1), dict(k=-1), dict(k=65), dict(V=1, ld=1),
    dict(ld=31), dict(temp=0.0), dict(temp=-1.0), dict(temp=float("nan")), dict(x=None),
    dict(tok=None), dict(logp=None), dict(ent=None), dict(tl=None), dict(tt=None)])
def test_token_logprobs(bad):
    assert logprobs(**bad) == _lib.TT_ERR_INVALID_ARG


def test_token_logprobs_type_and_backward():
    assert logprobs(dtype=U8) == _lib.TT_ERR_UNSUPPORTED
    assert logprobs(T=0, x=None, tok=None, logp=None, ent=None, tl=None, tt=None) == _lib.TT_OK
    bwd = lambda stats=P, dx=P, toks=P, x=P: status(
        "tt_token_logprobs_bwd", BF16, 4, 32, x, 32, P, 1, 1.0, 2, toks, P, P, P, stats, dx, None)
    for bad in (dict(stats=None), dict(dx=None), dict(toks=None), dict(x=None)):
        assert bwd(**bad) == _lib.TT_ERR_INVALID_ARG
