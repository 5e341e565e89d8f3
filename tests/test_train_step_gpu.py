"""The training operators together, as a step uses them: a dense decoder on a
trajectory tree (embedding, rotary positions, tree attention, norms, the gated
feed-forward block, the loss of every successor, clipped gradients), against the
same model in plain torch in 64 bits, and the drivers with the blocks and losses
of an HF model routed through them.

Tolerance: fp32 products over up to 264 terms and two layers; a chain of about 20
such steps at 264 * 2^-24 each is 3e-4 of the largest value.
"""
import pytest
import torch
from torch import nn

import tree_training_b200 as tt
from tests.test_hybrid_gpu import DEV, _grads, max_rel, setup  # noqa: F401  (a fixture)
from tree_training_b200.hybrid import make_tree_loss_fn, tree_grad_hybrid
from tree_training_b200.synthetic import bfs_tree

pytestmark = pytest.mark.gpu
HEADS, KV, D, H, F, V, LAYERS = 4, 2, 64, 96, 264, 300, 2


def parameters(seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = lambda *s: nn.Parameter(torch.randn(*s, generator=g, device=DEV) * s[-1] ** -0.5)
    one = lambda: nn.Parameter(1 + 0.1 * torch.randn(H, generator=g, device=DEV))
    p = {"table": w(V, H), "head": w(V, H), "first": one(), "last": one()}
    for i in range(LAYERS):
        p.update({f"qkv{i}": w((HEADS + 2 * KV) * D, H), f"out{i}": w(H, HEADS * D),
                  f"ffn{i}": one(), f"gate{i}": w(F, H), f"up{i}": w(F, H), f"down{i}": w(H, F)})
        if i + 1 < LAYERS:
            p[f"next{i}"] = one()
    return p


def losses(p, ids, pos, rotary, meta, successors):
    """The package's operators: losses [N, M]."""
    x = tt.embedding(ids, p["table"], scale=H ** 0.5)
    y, stream = tt.residual_norm(x, None, p["first"])
    for i in range(LAYERS):
        q, k, v = (y @ p[f"qkv{i}"].t()).split([HEADS * D, KV * D, KV * D], 1)
        q, k = tt.apply_rotary(q.view(-1, HEADS, D), k.view(-1, KV, D), pos, rotary)
        a = tt.tree_attention(q, k, v.view(-1, KV, D), meta).flatten(1) @ p[f"out{i}"].t()
        y, stream = tt.residual_norm(a, stream, p[f"ffn{i}"])
        m = tt.gated_linear(y, p[f"gate{i}"], p[f"up{i}"]) @ p[f"down{i}"].t()
        y, stream = tt.residual_norm(m, stream, p.get(f"next{i}", p["last"]))
    return tt.linear_cross_entropy(y, p["head"], successors).losses


def plain_losses(p, ids, pos, rotary, allowed, successors):
    rms = lambda t, w: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w
    c, s = rotary[pos][:, None].chunk(2, -1)
    turn = lambda t: torch.cat([t[..., :D // 2] * c - t[..., D // 2:] * s,
                                t[..., D // 2:] * c + t[..., :D // 2] * s], -1)
    stream = p["table"][ids] * H ** 0.5
    y = rms(stream, p["first"])
    for i in range(LAYERS):
        q, k, v = (y @ p[f"qkv{i}"].t()).split([HEADS * D, KV * D, KV * D], 1)
        q, k, v = turn(q.view(-1, HEADS, D)), turn(k.view(-1, KV, D)), v.view(-1, KV, D)
        k, v = k.repeat_interleave(HEADS // KV, 1), v.repeat_interleave(HEADS // KV, 1)
        sc = torch.einsum("qhd,khd->hqk", q, k) * D ** -0.5
        a = torch.softmax(sc.masked_fill(~allowed, float("-inf")), -1)
        stream = stream + torch.einsum("hqk,khd->qhd", a, v).flatten(1) @ p[f"out{i}"].t()
        y = rms(stream, p[f"ffn{i}"])
        m = nn.functional.silu(y @ p[f"gate{i}"].t()) * (y @ p[f"up{i}"].t())
        stream = stream + m @ p[f"down{i}"].t()
        y = rms(stream, p.get(f"next{i}", p["last"]))
    lp = torch.log_softmax(y @ p["head"].t(), -1)
    taken = (successors >= 0) & (successors < V)
    return -torch.where(taken, lp.gather(1, successors.clamp(0, V - 1)), 0.0)


def test_step_matches_plain_torch():
    roots = bfs_tree(5, 300, 8, 40, 30, vocab=V)
    info = tt.build_dfs_tree_info(roots)
    on = lambda a: torch.as_tensor(a, dtype=torch.int64, device=DEV)
    ids, pos, meta = on(info.dfs_token_ids_np), on(info.dfs_pos_ids_np), info.attn_meta()
    succ = on(tt.tree_next_tokens(roots))
    assert int((succ >= 0).sum(1).max()) > 1                 # the tree branches
    rotary = tt.rotary_table(512, D, 1e4, device=DEV)
    p = parameters()
    weights = torch.rand(succ.shape, device=DEV) / succ.shape[0]
    loss = (losses(p, ids, pos, rotary, meta, succ) * weights).sum()
    loss.backward()
    tt.check_device_status(DEV)

    P = {n: t.detach().double().requires_grad_(True) for n, t in p.items()}
    allowed = torch.as_tensor(meta.dense_mask(), device=DEV)
    want = (plain_losses(P, ids, pos, rotary.double(), allowed, succ) * weights).sum()
    want.backward()
    assert abs(float(loss) - float(want)) < 3e-4 * float(want)
    for n, t in p.items():
        err = float((t.grad.double() - P[n].grad).abs().max() / P[n].grad.abs().max())
        assert err < 3e-4, f"{n}: {err:.2e}"
    grads = [t.grad for t in p.values()]
    size = torch.cat([t.grad.flatten() for t in P.values()]).norm()
    norm = tt.clip_grad_norm(grads, 0.5 * float(size))
    assert abs(float(norm) - float(size)) < 3e-4 * float(size)
    assert abs(float(tt.grad_norm(grads)) - 0.5 * float(size)) < 6e-4 * float(size)
    for n, t in p.items():
        err = float((t.grad.double() - 0.5 * P[n].grad).abs().max() / P[n].grad.abs().max())
        assert err < 6e-4, f"{n}: {err:.2e}"


@pytest.mark.parametrize("max_tokens", [1000, 10])
def test_driver_with_fused_blocks_and_pieces(setup, max_tokens):  # noqa: F811
    model, roots, ref, leaves, labels = setup
    mlps = [l.mlp for l in model.model.layers]
    own = [m.forward for m in mlps]
    assert tt.fuse_gated_mlps(model) == len(mlps)
    try:
        model.zero_grad(set_to_none=True)
        tree_grad_hybrid(model, roots, make_tree_loss_fn(labels, leaves, len(leaves)), max_tokens,
                         fused_ce="pieces")
        tt.check_device_status(DEV)
        assert max_rel(ref, _grads(model)) < 1e-4
    finally:
        for m, f in zip(mlps, own):
            m.forward = f


def test_driver_refuses_other_losses(setup):  # noqa: F811
    model, roots, _, leaves, labels = setup
    with pytest.raises(ValueError):
        tree_grad_hybrid(model, roots, make_tree_loss_fn(labels, leaves, len(leaves)), 1000,
                         fused_ce="chunks")
    with pytest.raises(ValueError):
        tree_grad_hybrid(model, roots, lambda z, n: z.sum(), 1000, fused_ce="pieces")
