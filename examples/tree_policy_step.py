"""Policy-gradient steps of a small mixture decoder on a trajectory tree.

    python examples/tree_policy_step.py --tokens 2048 --steps 5

Everything between the matrix products runs on the package's operators: rotary
positions at the tree's depths, tree attention, the norms around each block with
the residual sum, tokens sorted by expert and back, and at the head the log
probabilities of every successor of a token (several at a branch) with their
entropy.  A shared prefix is computed once for all of its continuations.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import tree_training_b200 as tt  # noqa: E402


class Layer(nn.Module):
    def __init__(self, hidden, heads, kv_heads, head_dim, experts, expert_dim):
        super().__init__()
        w = lambda *s: nn.Parameter(torch.randn(*s) * s[-1] ** -0.5)
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.qkv = w((heads + 2 * kv_heads) * head_dim, hidden)
        self.out = w(hidden, heads * head_dim)
        self.gate = w(hidden, hidden)
        self.after_attention = nn.Parameter(torch.ones(hidden))
        self.before_experts = nn.Parameter(torch.ones(hidden))
        self.after_experts = nn.Parameter(torch.ones(hidden))
        self.router = w(experts, hidden)
        self.up, self.down = w(experts, 2 * expert_dim, hidden), w(experts, hidden, expert_dim)

    def attention(self, y, positions, table, meta):
        """The block's output and the gate of its way into the stream."""
        q, k, v = (y @ self.qkv.t()).split(
            [self.heads * self.head_dim, self.kv_heads * self.head_dim,
             self.kv_heads * self.head_dim], dim=1)
        heads = lambda t: t.unflatten(1, (-1, self.head_dim))
        q, k = tt.apply_rotary(heads(q), heads(k), positions, table)
        a = tt.tree_attention(q, k, heads(v), meta)
        return a.flatten(1) @ self.out.t(), torch.sigmoid(y @ self.gate.t())

    def mixture(self, y, k):
        score, ids = torch.softmax((y @ self.router.t()).float(), -1).topk(k, dim=-1)
        plan = tt.expert_plan(ids, self.router.shape[0])
        xs = tt.expert_dispatch(y, plan)
        # the experts' products, one after another: the first row of each comes
        # from the device
        rows = plan.offsets.tolist()
        parts = []
        for e, (b, n) in enumerate(zip(rows, rows[1:])):
            u, g = (xs[b:n] @ self.up[e].t()).chunk(2, dim=1)
            parts.append((nn.functional.silu(g) * u) @ self.down[e].t())
        ys = torch.cat(parts)
        return tt.expert_combine(ys, score / score.sum(-1, keepdim=True), plan)


class TreePolicy(nn.Module):
    def __init__(self, vocab=512, hidden=256, layers=2, heads=4, kv_heads=2, head_dim=64,
                 experts=8, choices=2, expert_dim=128, rotary_dim=32, max_positions=4096):
        super().__init__()
        self.choices = choices
        self.embed = nn.Parameter(torch.randn(vocab, hidden))
        self.layers = nn.ModuleList(
            Layer(hidden, heads, kv_heads, head_dim, experts, expert_dim) for _ in range(layers))
        self.first = nn.Parameter(torch.ones(hidden))
        self.before = nn.ParameterList(torch.ones(hidden) for _ in range(layers - 1))
        self.last = nn.Parameter(torch.ones(hidden))
        self.head = nn.Parameter(torch.randn(vocab, hidden) * hidden ** -0.5)
        self.register_buffer("table", tt.rotary_table(
            max_positions, rotary_dim, 1e4,
            {"rope_type": "yarn", "factor": 4.0,
             "original_max_position_embeddings": max_positions // 4}))

    def forward(self, ids, positions, meta):
        """Logits [N, vocab] of a packed tree's tokens."""
        y, stream = tt.residual_norm(self.embed[ids], None, self.first)
        for i, layer in enumerate(self.layers):
            a, gate = layer.attention(y, positions, self.table, meta)
            y, stream = tt.residual_norm(a, stream, layer.before_experts,
                                         post_weight=layer.after_attention, gate=gate)
            m = layer.mixture(y, self.choices)
            following = self.before[i] if i + 1 < len(self.layers) else self.last
            y, stream = tt.residual_norm(m, stream, following, post_weight=layer.after_experts,
                                         scale=0.5)
        return y @ self.head.t()


def pack(roots, device):
    """What a step needs of a forest: ids, depths, attention metadata and the
    successors of every token."""
    info = tt.build_dfs_tree_info(roots)
    on = lambda a: torch.as_tensor(a, dtype=torch.int64, device=device)
    return (on(info.dfs_token_ids_np), on(info.dfs_pos_ids_np), info.attn_meta(),
            on(tt.tree_next_tokens(roots)))


def policy_loss(logits, successors, old_logprobs, advantages, clip=0.2, entropy_bonus=0.01):
    """The clipped policy-gradient loss over every edge of the tree."""
    r = tt.token_logprobs(logits, successors)
    taken = (successors >= 0).float()
    ratio = torch.exp(r.logprobs - old_logprobs)
    gain = torch.minimum(ratio * advantages, ratio.clamp(1 - clip, 1 + clip) * advantages)
    return -(gain * taken).sum() / taken.sum() - entropy_bonus * r.entropy.mean()


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=5)
    ap.add_argument("--dtype", choices=["float32", "bfloat16"], default="bfloat16")
    a = ap.parse_args()
    from tree_training_b200.synthetic import bfs_tree
    torch.manual_seed(0)
    dev = torch.device("cuda")
    vocab = 512
    roots = bfs_tree(0, a.tokens, 16, 200, 150, vocab=vocab)
    # (the tree attention's tensor-core path takes heads of 128)
    model = TreePolicy(vocab, head_dim=128, max_positions=1 << 14).to(dev, getattr(torch, a.dtype))
    model.table = model.table.float()
    ids, positions, meta, successors = pack(roots, dev)
    advantages = torch.randn(successors.shape, device=dev)
    with torch.no_grad():
        old = tt.token_logprobs(model(ids, positions, meta), successors, top_k=4)
    print("most likely after the first token:", old.top_tokens[0].tolist(),
          [round(v, 3) for v in old.top_logprobs[0].tolist()])
    opt = torch.optim.SGD(model.parameters(), lr=0.05)
    for step in range(a.steps):
        opt.zero_grad()
        loss = policy_loss(model(ids, positions, meta), successors, old.logprobs, advantages)
        loss.backward()
        opt.step()
        print(f"step {step}: loss {loss.item():.4f}")
    tt.check_device_status(dev)


if __name__ == "__main__":
    main()
