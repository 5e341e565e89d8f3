"""The example's policy step (``examples/tree_policy_step.py``) in fp32 against
the same model written in plain torch in 64 bits, token by token over dense
masks: loss and every parameter's gradient.

Tolerance: fp32 products over up to 256 terms and two layers; a chain of about
20 such steps at 256 * 2^-24 each is 3e-4 of the largest value.  The routers'
choices agree unless two scores are that close, which the seed's are not.
"""
import importlib.util
import os

import pytest
import torch

import tree_training_b200 as tt
from tree_training_b200.synthetic import bfs_tree

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
HERE = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location(
        "tree_policy_step", os.path.join(HERE, "examples", "tree_policy_step.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def plain_logits(m, P, ids, positions, allowed):
    """The model's forward with parameters P (64 bits), in plain torch."""
    rms = lambda t, w: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w
    table = m.table.double()[positions][:, None]
    half = table.shape[-1] // 2
    c, s = table[..., :half], table[..., half:]

    def turn(t):
        a, b, rest = t[..., :half], t[..., half:2 * half], t[..., 2 * half:]
        return torch.cat([a * c - b * s, b * c + a * s, rest], -1)

    stream = P["embed"][ids]
    y = rms(stream, P["first"])
    for i, layer in enumerate(m.layers):
        L = lambda n: P[f"layers.{i}.{n}"]
        h, kv, d = layer.heads, layer.kv_heads, layer.head_dim
        q, k, v = (y @ L("qkv").t()).split([h * d, kv * d, kv * d], 1)
        q, k, v = turn(q.view(-1, h, d)), turn(k.view(-1, kv, d)), v.view(-1, kv, d)
        k, v = k.repeat_interleave(h // kv, 1), v.repeat_interleave(h // kv, 1)
        sc = torch.einsum("qhd,khd->hqk", q, k) * d ** -0.5
        p = torch.softmax(sc.masked_fill(~allowed, float("-inf")), -1)
        a = torch.einsum("hqk,khd->qhd", p, v).flatten(1) @ L("out").t()
        gate = torch.sigmoid(y @ L("gate").t())
        stream = stream + gate * rms(a, L("after_attention"))
        y = rms(stream, L("before_experts"))
        score, choice = torch.softmax(y @ L("router").t(), -1).topk(m.choices, dim=-1)
        score = score / score.sum(-1, keepdim=True)
        mix = torch.zeros_like(y)
        for e in range(layer.router.shape[0]):
            u, g = (y @ L("up")[e].t()).chunk(2, 1)
            out = (torch.nn.functional.silu(g) * u) @ L("down")[e].t()
            mix = mix + out * (score * (choice == e)).sum(-1, keepdim=True)
        stream = stream + 0.5 * rms(mix, L("after_experts"))
        y = rms(stream, P[f"before.{i}"] if i + 1 < len(m.layers) else P["last"])
    return y @ P["head"].t()


def test_policy_step_matches_plain_torch():
    ex = example()
    torch.manual_seed(0)
    roots = bfs_tree(5, 300, 8, 40, 30, vocab=100)
    m = ex.TreePolicy(vocab=100, hidden=96, experts=5, expert_dim=48, max_positions=512).to(DEV)
    ids, positions, meta, successors = ex.pack(roots, DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    adv = torch.randn(successors.shape, generator=g, device=DEV)
    old = torch.full(successors.shape, -4.5, device=DEV)
    loss = ex.policy_loss(m(ids, positions, meta), successors, old, adv)
    loss.backward()
    tt.check_device_status(DEV)

    P = {n: p.detach().double().requires_grad_(True) for n, p in m.named_parameters()}
    allowed = torch.as_tensor(meta.dense_mask(), device=DEV)
    logits = plain_logits(m, P, ids, positions, allowed)
    lp = torch.log_softmax(logits, -1)
    taken = successors >= 0
    assert int(taken.sum(1).max()) > 1              # the tree branches
    logp = torch.where(taken, lp.gather(1, successors.clamp(min=0)), torch.zeros((), device=DEV))
    ratio = torch.exp(logp - old.double())
    gain = torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv)
    ent = -(lp.exp() * lp).sum(-1).mean()
    want = -(gain * taken).sum() / taken.sum() - 0.01 * ent
    want.backward()
    assert abs(float(loss) - float(want)) < 3e-4 * max(1.0, abs(float(want)))
    for n, p in m.named_parameters():
        err = float((p.grad.double() - P[n].grad).abs().max() / P[n].grad.abs().max())
        assert err < 3e-4, f"{n}: {err:.2e}"


def test_example_runs_in_bf16():
    import subprocess
    import sys
    r = subprocess.run([sys.executable, os.path.join(HERE, "examples", "tree_policy_step.py"),
                        "--tokens", "700", "--steps", "2"], capture_output=True, text=True,
                       timeout=300, cwd=HERE)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "step 1: loss" in r.stdout and "nan" not in r.stdout.lower()
