"""Refusals of the training operators' C ABI: bad sizes, pointers and types come back
as a status before anything touches a device (so they run without a GPU)."""
import ctypes
import math

import pytest

from tree_training_b200 import _lib

F32, BF16, F16, U8 = _lib.TT_F32, _lib.TT_BF16, _lib.TT_F16, _lib.TT_U8
INVALID, UNSUPPORTED, WORKSPACE = (_lib.TT_ERR_INVALID_ARG, _lib.TT_ERR_UNSUPPORTED,
                                   _lib.TT_ERR_WORKSPACE)
P = 1 << 20            # a pointer that is never followed
BIG = 1 << 60


def status(name, *args):
    return getattr(_lib.lib(), name)(*args)


def embed(dtype=BF16, n=4, V=10, H=8, ids=P, w=P, ld=8, y=P):
    return status("tt_embedding_fwd", dtype, n, V, H, ids, 1, w, ld, 1.0, y, None, None)


def embed_bwd(dtype=BF16, n=4, V=10, H=8, ids=P, dy=P, ld=8, dw=P, ws=P, size=BIG):
    return status("tt_embedding_bwd", dtype, n, V, H, ids, 1, dy, ld, 1.0, -1, dw, ws, size, None)


@pytest.mark.parametrize("bad", [dict(n=-1), dict(n=1 << 31), dict(V=0), dict(V=1 << 31), dict(H=0),
                                 dict(ld=7), dict(ids=None), dict(w=None), dict(y=None)])
def test_embedding(bad):
    assert embed(**bad) == INVALID


@pytest.mark.parametrize("bad", [dict(n=-1), dict(n=1 << 31), dict(V=0), dict(V=1 << 31), dict(H=0),
                                 dict(ld=7), dict(ids=None), dict(dy=None), dict(dw=None)])
def test_embedding_gradient(bad):
    assert embed_bwd(**bad) == INVALID


def test_embedding_types_and_workspace():
    assert embed(dtype=U8) == UNSUPPORTED and embed_bwd(dtype=U8) == UNSUPPORTED
    assert embed(n=0, ids=None, w=None, y=None) == _lib.TT_OK
    need = status("tt_embedding_bwd_workspace_size", 4, 10, 8)
    assert embed_bwd(size=need - 1) == WORKSPACE and embed_bwd(ws=None) == WORKSPACE
    assert status("tt_embedding_bwd_workspace_size", -1, 10, 8) == 0


def align(rows=4, cols=9, src=P, ld=9, dst=P, dst_ld=16):
    return status("tt_align_rows", rows, cols, src, ld, dst, dst_ld, None)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(cols=0), dict(ld=8), dict(dst_ld=8),
                                 dict(dst_ld=17), dict(src=None), dict(dst=None), dict(dst=P + 8),
                                 dict(src=P + 1)])
def test_align_rows(bad):
    assert align(**bad) == INVALID
    assert align(rows=0, src=None, dst=None) == _lib.TT_OK


def gated(dtype=BF16, T=4, H=16, F=8, x=P, x_ld=16, wg=P, wg_ld=16, wu=P, wu_ld=16, act=0, h=P,
          g=None, u=None, ld=8, ws=P, size=BIG):
    return status("tt_gated_linear_fwd", dtype, T, H, F, x, x_ld, wg, wg_ld, wu, wu_ld, act, h, g, u,
                  ld, ws, size, None, None)


def gated_bwd(dtype=BF16, T=4, H=16, F=8, x=P, x_ld=16, wg=P, wg_ld=16, wu=P, wu_ld=16, act=0, g=P,
              u=P, ld=8, dh=P, dh_ld=8, ws=P, size=BIG):
    return status("tt_gated_linear_bwd", dtype, T, H, F, x, x_ld, wg, wg_ld, wu, wu_ld, act, g, u,
                  ld, dh, dh_ld, P, P, P, ws, size, None, None)


BAD_GATED = [dict(T=-1), dict(T=1 << 31), dict(H=0), dict(F=0), dict(x_ld=15), dict(wg_ld=15),
             dict(wu_ld=15), dict(act=-1), dict(act=4), dict(x=None), dict(wg=None), dict(wu=None)]


@pytest.mark.parametrize("bad", BAD_GATED + [dict(h=None), dict(g=P), dict(u=P),
                                             dict(g=P, u=P, ld=7), dict(g=P, u=P, ld=10),
                                             dict(g=P + 8, u=P), dict(dtype=F32)])
def test_gated_linear(bad):
    assert gated(**bad) == INVALID


@pytest.mark.parametrize("bad", BAD_GATED + [dict(g=None), dict(u=None), dict(ld=7), dict(ld=10),
                                             dict(u=P + 4), dict(dh=None),
                                             dict(dh_ld=7)])
def test_gated_linear_gradient(bad):
    assert gated_bwd(**bad) == INVALID


def test_gated_linear_types_and_workspace():
    assert gated(dtype=U8) == UNSUPPORTED and gated_bwd(dtype=U8) == UNSUPPORTED
    assert gated(T=0, x=None, wg=None, wu=None, h=None) == _lib.TT_OK
    for dtype in (F32, BF16, F16):
        need = status("tt_gated_linear_bwd_workspace_size", dtype, 4, 16, 8)
        assert need > 0
        assert gated_bwd(dtype=dtype, size=need - 1) == WORKSPACE
        assert gated_bwd(dtype=dtype, ws=None) == WORKSPACE
    # a sum over k that is split has parts to keep
    need = status("tt_gated_linear_fwd_workspace_size", F32, 4, 4096, 8)
    assert need > 0
    big = dict(dtype=F32, H=4096, x_ld=4096, wg_ld=4096, wu_ld=4096, g=P, u=P)
    assert gated(size=need - 1, **big) == WORKSPACE


def ce(dtype=BF16, T=4, H=16, V=100, M=1, x=P, x_ld=16, w=P, w_ld=16, labels=P, losses=P, lse=P,
       kept=None, ws=P, size=BIG):
    return status("tt_linear_ce_fwd", dtype, T, H, V, M, x, x_ld, w, w_ld, labels, 1.0, losses, lse,
                  kept, ws, size, None, None)


def ce_bwd(dtype=BF16, T=4, H=16, V=100, M=1, x=P, x_ld=16, w=P, w_ld=16, labels=P, lse=P,
           kept=None, ws=P, size=BIG):
    return status("tt_linear_ce_bwd", dtype, T, H, V, M, x, x_ld, w, w_ld, labels, 1.0, lse, kept, P,
                  P, P, P, ws, size, None, None)


BAD_CE = [dict(T=-1), dict(T=1 << 31), dict(H=0), dict(V=0), dict(V=1 << 31), dict(M=-1),
          dict(M=1 << 31), dict(x_ld=15), dict(w_ld=15), dict(x=None), dict(w=None),
          dict(labels=None), dict(lse=None), dict(kept=P, T=100)]


@pytest.mark.parametrize("bad", BAD_CE + [dict(losses=None)])
def test_linear_ce(bad):
    assert ce(**bad) == INVALID


@pytest.mark.parametrize("bad", BAD_CE)
def test_linear_ce_gradient(bad):
    assert ce_bwd(**bad) == INVALID


def test_linear_ce_kept_logits():
    f = lambda *a: status("tt_linear_ce_kept_ld", *a)
    assert f(F32, 47, 64, 1001) == 1008 and f(F32, 0, 64, 1001) == 0 and f(U8, 47, 64, 1001) == 0
    assert f(F32, 1 << 20, 64, 4096) == 0
    assert f(F32, 4096, 64, 16384) == 16384 and f(F32, 4097, 64, 16384) == 0
    # 16 bits: where forming them again takes longer
    assert f(BF16, 47, 64, 1001) == 0 and f(BF16, 15, 64, 1001) == 1008
    assert f(F16, 400, 1024, 151936) == 151936 and f(BF16, 8192, 2560, 151936) == 0
    assert f(F32, -1, 64, 10) == 0 and f(F32, 10, 64, 0) == 0 and f(F32, 10, 0, 10) == 0


def test_linear_ce_types_and_workspace():
    assert ce(dtype=U8) == UNSUPPORTED and ce_bwd(dtype=U8) == UNSUPPORTED
    assert ce(T=0, x=None, w=None, labels=None) == _lib.TT_OK
    for dtype in (F32, BF16, F16):
        for name, call in (("fwd", ce), ("bwd", ce_bwd)):
            need = status(f"tt_linear_ce_{name}_workspace_size", dtype, 4, 16, 100, 1)
            assert need > 0
            assert call(dtype=dtype, size=need - 1) == WORKSPACE
            assert call(dtype=dtype, ws=None) == WORKSPACE


def arrays(n=2, dtype=BF16, size=10, at=P):
    return ((ctypes.c_int32 * n)(*[dtype] * n), (ctypes.c_int64 * n)(*[size] * n),
            (ctypes.c_void_p * n)(*[at] * n))


def norm(n=2, p=2.0, out=P, ws=P, size=BIG, tables=None):
    return status("tt_grad_norm", n, *(tables or arrays()), p, out, ws, size, None)


def clip(n=2, p=2.0, out=P, ws=P, size=BIG, tables=None, outs=None):
    t = tables or arrays()
    return status("tt_clip_grad_norm", n, *t, outs or t[2], p, None, 1.0, 1e-6, out, ws, size, None)


@pytest.mark.parametrize("call", [norm, clip])
def test_grad_norm(call):
    for bad in (dict(n=-1), dict(p=3.0), dict(p=-math.inf), dict(p=math.nan), dict(out=None),
                dict(tables=arrays(size=-1)), dict(tables=arrays(at=None)),
                dict(tables=arrays(at=P + 1)), dict(tables=arrays(dtype=F32, at=P + 2)),
                dict(tables=arrays(size=1 << 45))):
        assert call(**bad) == INVALID, bad
    assert call(tables=arrays(dtype=U8)) == UNSUPPORTED
    need = status("tt_grad_norm_workspace_size", 2)
    assert call(size=need - 1) == WORKSPACE and call(ws=None) == WORKSPACE
    assert status("tt_grad_norm_workspace_size", 5000) > need
    assert status("tt_grad_norm_workspace_size", -1) == 0


def test_clip_outputs():
    assert clip(outs=arrays(at=None)[2]) == INVALID
    assert clip(outs=arrays(at=P + 1)[2]) == INVALID


@pytest.mark.parametrize("call,wide", [
    (embed, dict(H=(1 << 22) + 1, ld=1 << 23)), (embed_bwd, dict(H=(1 << 22) + 1, ld=1 << 23)),
    (gated, dict(F=(1 << 30) - 255)), (gated_bwd, dict(F=(1 << 30) - 255, ld=1 << 30,
                                                      dh_ld=1 << 30)),
    (gated, dict(H=(1 << 31) - 257, x_ld=1 << 31, wg_ld=1 << 31, wu_ld=1 << 31)),
    (gated_bwd, dict(H=(1 << 31) - 257, x_ld=1 << 31, wg_ld=1 << 31, wu_ld=1 << 31)),
    (ce, dict(H=(1 << 31) - 257, x_ld=1 << 31, w_ld=1 << 31)),
    (ce_bwd, dict(H=(1 << 31) - 257, x_ld=1 << 31, w_ld=1 << 31))])
def test_widths_that_32_bits_do_not_count(call, wide):
    assert call(**wide) == INVALID


def test_the_largest_widths_have_a_workspace():
    size = lambda name, *a: status(f"tt_{name}_workspace_size", *a)
    assert size("embedding_bwd", 1, 1, 1 << 22) > 1 << 22
    assert size("gated_linear_bwd", BF16, 1, 1, (1 << 30) - 256) > 1 << 32
    assert size("linear_ce_fwd", BF16, 1, (1 << 31) - 258, 1, 1) > 0


@pytest.mark.parametrize("call", [embed_bwd, gated, gated_bwd, ce, ce_bwd, norm, clip])
def test_a_workspace_off_its_boundary(call):
    assert call(ws=P + 4) == INVALID


@pytest.mark.parametrize("call", [ce, ce_bwd])
def test_kept_logits_off_their_boundary(call):
    assert call(dtype=F32, kept=P + 16) == INVALID


def align_many(n=2, rows=4, cols=9, src=P, ld=9, dst=P, dst_ld=16, null=None):
    I, V = ctypes.c_int64 * max(n, 1), ctypes.c_void_p * max(n, 1)
    tables = [I(*[rows] * n), I(*[cols] * n), V(*[src] * n), I(*[ld] * n), V(*[dst] * n),
              I(*[dst_ld] * n)]
    return status("tt_align_rows_of", n, *[None if i == null else t for i, t in enumerate(tables)],
                  None)


@pytest.mark.parametrize("bad", [dict(n=-1), dict(n=5), dict(rows=-1), dict(cols=0), dict(ld=8),
                                 dict(dst_ld=8), dict(dst_ld=17), dict(src=None), dict(dst=None),
                                 dict(dst=P + 8), dict(src=P + 1), *[dict(null=i) for i in range(6)]])
def test_align_rows_of(bad):
    assert align_many(**bad) == INVALID
    assert align_many(n=0) == _lib.TT_OK
    assert align_many(rows=0, src=None, dst=None) == _lib.TT_OK
