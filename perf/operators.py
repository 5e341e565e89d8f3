"""Cases for the operators of a decoder layer and its head: token log
probabilities, rotary positions, residual norms, and tokens sorted by expert.

``run`` computes one pass through an operator: in elementary torch operations
(32-bit arithmetic, one rounding at the end) while ``own`` is false, through
the package's public entry points while it is true.  ``exact`` computes the
same from the definitions in 64 bits.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# -----------------------------------------------------------------------------
# cases
# -----------------------------------------------------------------------------

def _logprob_case(T, V, M, k, dtype, bwd, temperature=1.0, masked=False):
    return {"op": "logprob", "T": T, "V": V, "M": M, "k": k, "dtype": dtype, "bwd": bwd,
            "temperature": temperature, "masked": masked}


def _rotary_case(N, hq, hk, D, R, dtype, bwd, interleaved=False, packed=False, factor=1.0):
    return {"op": "rotary", "N": N, "hq": hq, "hk": hk, "D": D, "R": R, "dtype": dtype, "bwd": bwd,
            "interleaved": interleaved, "packed": packed, "factor": factor}


def _norm_case(T, D, dtype, bwd, res="same", post=False, gate="none", scale=1.0, offset=0.0):
    return {"op": "norm", "T": T, "D": D, "dtype": dtype, "bwd": bwd, "res": res, "post": post,
            "gate": gate, "scale": scale, "offset": offset}


def _moe_case(T, H, E, K, dtype, bwd, dropped=False):
    return {"op": "moe", "T": T, "H": H, "E": E, "K": K, "dtype": dtype, "bwd": bwd,
            "dropped": dropped}


def listed():
    return [
        # one 47-token forest scored against a 32,000-word vocabulary, eight
        # alternatives each: a call whose latency counts
        dict(_logprob_case(47, 32000, 1, 8, "f32", False, masked=True), name="logprob_small"),
        # a policy step's head: 2,047 tokens of a tree, up to two successors at
        # a branch, entropy bonus, gradient back to 151,936 logits
        dict(_logprob_case(2047, 151936, 2, 0, "bf16", True), name="logprob_train"),
        # scoring a batch of sampled tokens with sixteen alternatives each
        dict(_logprob_case(4096, 151936, 1, 16, "bf16", False, temperature=0.7),
             name="logprob_score"),
        # the 47-token forest through a layer of the two-layer test model
        dict(_rotary_case(47, 4, 2, 64, 64, "f32", False), name="rotary_small"),
        # one 32,768-token tree, 32 query and 8 key heads of 128, forward and backward
        dict(_rotary_case(32768, 32, 8, 128, 128, "bf16", True), name="rotary_train"),
        # a quarter of each 256-wide head rotated, interleaved, positions scaled
        # by four, q and k being views of one projection's output
        dict(_rotary_case(8191, 16, 2, 256, 64, "bf16", True, interleaved=True, packed=True,
                          factor=4.0), name="rotary_partial"),
        # the 47-token forest, hidden size 256
        dict(_norm_case(47, 256, "f32", False), name="norm_small"),
        # one 32,768-token tree, hidden size 2,560, residual sum and norm of the
        # next block, forward and backward
        dict(_norm_case(32768, 2560, "bf16", True), name="norm_train"),
        # norms on both sides of a gated block, residual kept in 32 bits
        dict(_norm_case(8191, 4096, "bf16", True, res="f32", post=True, gate="full", scale=0.5,
                        offset=1.0), name="norm_gated"),
        # the 47-token forest through four experts, two a token
        dict(_moe_case(47, 128, 4, 2, "f32", False), name="moe_small"),
        # a training step of 8,191 tokens over 128 experts, eight a token
        dict(_moe_case(8191, 2048, 128, 8, "bf16", True), name="moe_train"),
        # one 32,768-token tree over 64 experts, four a token, some dropped
        dict(_moe_case(32768, 2560, 64, 4, "bf16", False, dropped=True), name="moe_tree"),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprob", "rotary", "norm", "moe"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    bwd = rng.random() < 0.5
    b = _SIZE[dtype]
    if op == "logprob":
        V = _log_int(rng, 128, 151936)
        cap = 4096 * 151936 if not bwd else 2047 * 151936
        T = _log_int(rng, 1, max(1, min(32768, cap * 2 // b // V)))
        return _logprob_case(T, V, rng.randint(1, 4), rng.choice([0, 1, 5, 8, 20, 64]), dtype, bwd,
                             rng.choice([1.0, 0.7, 1.3]), rng.random() < 0.4)
    if op == "rotary":
        hk = rng.choice([1, 2, 4, 8])
        hq = hk * rng.choice([1, 2, 4, 7])
        D = rng.choice([64, 80, 128, 192, 256])
        R = max(2, int(D * rng.choice([1.0, 1.0, 0.5, 0.25])) // 2 * 2)
        cap = 32768 * 40 * 128
        N = _log_int(rng, 1, max(1, min(32768, cap * 2 // b // ((hq + hk) * D))))
        return _rotary_case(N, hq, hk, D, R, dtype, bwd, rng.random() < 0.5, rng.random() < 0.5,
                            rng.choice([1.0, 4.0]))
    if op == "norm":
        D = _log_int(rng, 64, 8192)
        D = D if rng.random() < 0.25 else max(64, D // 64 * 64)
        cap = 32768 * 2560
        T = _log_int(rng, 1, max(1, min(32768, cap * 2 // b // (2 * D))))
        return _norm_case(T, D, dtype, bwd, rng.choice(["same", "same", "f32"]),
                          rng.random() < 0.5, rng.choice(["none", "channel", "token", "full"]),
                          rng.choice([1.0, 0.5]), rng.choice([0.0, 1.0]))
    H = _log_int(rng, 64, 8192)
    H = H if rng.random() < 0.25 else max(64, H // 64 * 64)
    E = _log_int(rng, 2, 256)
    K = rng.randint(1, min(8, E))
    cap = 8191 * 8 * 2048
    T = _log_int(rng, 1, max(1, min(32768, cap * 2 // b // (K * H))))
    return _moe_case(T, H, E, K, dtype, bwd, rng.random() < 0.4)


# -----------------------------------------------------------------------------
# inputs
# -----------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, shape, dtype, scale=1.0):
    # made in slices, so that a large tensor needs no 32-bit copy of its own size
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    step = 1 << 27
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device="cuda") * scale
    return out


def prepare(case, seed):
    g = _gen(seed)
    dt = _DTYPES[case["dtype"]]
    bwd = bool(case["bwd"])
    s = {"op": case["op"], "bwd": bwd}
    if case["op"] == "logprob":
        T, V, M, k = case["T"], case["V"], case["M"], min(case["k"], case["V"])
        x = _randn(g, (T, V), dt, 2.5)
        # as a trained head gives them: some words of each row stand out
        hot = torch.randint(0, V, (T, 4), generator=g, device="cuda")
        x.scatter_add_(1, hot, (torch.rand(T, 4, generator=g, device="cuda") * 12).to(dt))
        tokens = torch.where(torch.rand(T, M, generator=g, device="cuda") < 0.5, hot[:, :1],
                             torch.randint(0, V, (T, M), generator=g, device="cuda"))
        # rows with one successor only, and rows without any
        tokens[:, 1:][torch.rand(T, M - 1, generator=g, device="cuda") < 0.7] = -100
        tokens[::9] = -100
        if case["masked"]:
            # constrained answers: words ruled out in some rows, every word in one
            x[1::3, V // 3:] = float("-inf")
            x[2::5, ::2] = torch.finfo(dt).min
            tokens[2::5] |= 1
            if T > 4:
                x[4] = float("-inf")
        s.update(x=x.requires_grad_(bwd), tokens=tokens, k=k, temperature=case["temperature"])
        if bwd:
            s.update(g_logp=torch.randn(T, M, generator=g, device="cuda") / T,
                     g_ent=torch.full((T,), 0.01 / T, device="cuda"),
                     g_top=torch.randn(T, k, generator=g, device="cuda") / T)
        return s
    if case["op"] == "rotary":
        N, hq, hk, D, R = case["N"], case["hq"], case["hk"], case["D"], case["R"]
        if case["packed"]:
            qkv = _randn(g, (N, (hq + 2 * hk) * D), dt)
            q = qkv[:, :hq * D].view(N, hq, D).detach()
            k = qkv[:, hq * D:(hq + hk) * D].view(N, hk, D).detach()
        else:
            q, k = _randn(g, (N, hq, D), dt), _randn(g, (N, hk, D), dt)
        P = 40960
        inv = 1e6 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
        ang = torch.arange(P, dtype=torch.float64, device="cuda")[:, None] / case["factor"] * inv
        table = torch.cat([ang.cos(), ang.sin()], 1).float()
        pos = torch.randint(0, P, (N,), generator=g, device="cuda")
        # depths of a tree: runs that go on, and siblings that start at the same place
        run_of = torch.arange(N, device="cuda") // 64
        pos = (pos[run_of * 64 % max(N, 1)] + torch.arange(N, device="cuda") % 64) % P
        s.update(q=q.requires_grad_(bwd), k=k.requires_grad_(bwd), pos=pos, table=table,
                 interleaved=bool(case["interleaved"]))
        if bwd:
            s.update(dq=_randn(g, (N, hq, D), dt), dk=_randn(g, (N, hk, D), dt))
        return s
    if case["op"] == "norm":
        T, D = case["T"], case["D"]
        rt = dt if case["res"] == "same" else torch.float32
        o = case["offset"]
        x, r = _randn(g, (T, D), dt, 0.7), _randn(g, (T, D), rt, 2.0)
        w = ((1.0 - o) + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dt)
        post = ((1.0 - o) + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dt)
        shape = {"none": None, "channel": (D,), "token": (T, 1), "full": (T, D)}[case["gate"]]
        gate = None if shape is None else torch.sigmoid(_randn(g, shape, dt).float()).to(dt)
        s.update(x=x.requires_grad_(bwd), r=r.requires_grad_(bwd), w=w.requires_grad_(bwd),
                 post=post.requires_grad_(bwd) if case["post"] else None,
                 gate=None if gate is None else gate.requires_grad_(bwd),
                 scale=case["scale"], offset=o, eps=1e-6)
        if bwd:
            s.update(dy=_randn(g, (T, D), dt), dr=_randn(g, (T, D), rt))
        return s
    T, H, E, K = case["T"], case["H"], case["E"], case["K"]
    # a router's choice: K different experts a token, some experts far more often
    liking = torch.randn(E, generator=g, device="cuda")
    score = torch.randn(T, E, generator=g, device="cuda") + liking
    top, ids = score.topk(K, dim=1)
    if case["dropped"]:
        ids[torch.rand(T, K, generator=g, device="cuda") < 0.1] = -1
    s.update(x=_randn(g, (T, H), dt).requires_grad_(bwd), ids=ids, E=E,
             w=torch.softmax(top, 1).requires_grad_(bwd),
             ys=_randn(g, (T * K, H), dt).requires_grad_(bwd))
    if bwd:
        s.update(dxs=_randn(g, (T * K, H), dt), dy=_randn(g, (T, H), dt))
    return s


# -----------------------------------------------------------------------------
# the plain forms
# -----------------------------------------------------------------------------

def _plain_logprob(s):
    x, tokens, k, temp = s["x"].detach(), s["tokens"], s["k"], s["temperature"]
    T, V = x.shape
    z = x.float() / temp
    m = z.amax(1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    z -= m
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    empty = total == 0                            # every word ruled out
    log_total = torch.where(empty, torch.zeros_like(total), total.log())
    p = e / torch.where(empty, torch.ones_like(total), total)
    logp = z - log_total
    plogp = torch.where(p == 0, torch.zeros_like(p), p * logp)
    entropy = -plogp.sum(1)
    valid = (tokens >= 0) & (tokens < V)
    at = torch.where(valid, tokens, torch.zeros_like(tokens))
    out = {"logprobs": torch.where(valid, logp.gather(1, at), torch.zeros_like(entropy[:, None])),
           "entropy": entropy}
    if k:
        # value first, then the lowest index: one whole number that orders both
        bits = (x.float() + 0.0).view(torch.int32).long()
        bits = torch.where(bits < 0, ~bits & 0xFFFFFFFF, bits + (1 << 31))
        key = (bits << 20) + (V - torch.arange(V, device=x.device))
        top = V - (key.topk(k, dim=1).values & ((1 << 20) - 1))
        out["top_tokens"] = top
        out["top_logprobs"] = logp.gather(1, top)
    if s["bwd"]:
        live = (~empty).float()
        g = torch.where(valid, s["g_logp"], torch.zeros_like(s["g_logp"])) * live
        d = g.sum(1, keepdim=True)
        if k:
            d = d + s["g_top"].sum(1, keepdim=True) * live
        dx = -p * d - s["g_ent"][:, None] * (plogp + p * entropy[:, None])
        dx.scatter_add_(1, at, g)
        if k:
            dx.scatter_add_(1, top, s["g_top"] * live)
        out["dx"] = (dx / temp).to(x.dtype)
    return out


def _rotate(x, c, sn, R, interleaved):
    half = R // 2
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        y = torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:R]
        y = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    return torch.cat([y, x[..., R:]], -1)


def _plain_rotary(s):
    table, pos, il = s["table"], s["pos"], s["interleaved"]
    R = table.shape[1]
    row = table[pos]
    c, sn = row[:, None, :R // 2], row[:, None, R // 2:]
    one = lambda x, sg: _rotate(x.detach().float(), c, sg * sn, R, il).to(x.dtype)
    out = {"q": one(s["q"], 1.0), "k": one(s["k"], 1.0)}
    if s["bwd"]:
        out["dq"], out["dk"] = one(s["dq"], -1.0), one(s["dk"], -1.0)
    return out


def _plain_norm(s):
    x, r0, o, eps, scale = s["x"].detach(), s["r"].detach(), s["offset"], s["eps"], s["scale"]
    xf, w = x.float(), s["w"].detach().float() + o
    if s["post"] is not None:
        w1 = s["post"].detach().float() + o
        i1 = torch.rsqrt(xf.square().mean(1, keepdim=True) + eps)
        h = xf * i1 * w1
    else:
        h = xf
    gate = None if s["gate"] is None else s["gate"].detach().float()
    b = h if gate is None else h * gate
    r = r0.float() + scale * b
    i2 = torch.rsqrt(r.square().mean(1, keepdim=True) + eps)
    n = r * i2
    out = {"y": (n * w).to(x.dtype), "r": r.to(r0.dtype)}
    if s["bwd"]:
        dy, dr = s["dy"].float(), s["dr"].float()
        gn = dy * w
        d = dr + i2 * (gn - n * (gn * n).mean(1, keepdim=True))
        out["dr"] = d.to(r0.dtype)
        out["dw"] = (dy * n).sum(0).to(s["w"].dtype)
        dh = scale * d
        if gate is not None:
            dg = dh * h
            if gate.dim() == 1:
                dg = dg.sum(0)
            elif gate.shape[1] == 1 and x.shape[1] != 1:
                dg = dg.sum(1, keepdim=True)
            out["dgate"] = dg.to(s["gate"].dtype)
            dh = dh * gate
        if s["post"] is not None:
            n1 = xf * i1
            out["dpost"] = (dh * n1).sum(0).to(s["post"].dtype)
            gh = dh * w1
            dh = i1 * (gh - n1 * (gh * n1).mean(1, keepdim=True))
        out["dx"] = dh.to(x.dtype)
    return out


def _plain_moe(s):
    x, ids, w, ys, E = s["x"].detach(), s["ids"], s["w"].detach(), s["ys"].detach(), s["E"]
    T, K = ids.shape
    flat = ids.reshape(-1)
    kept = (flat >= 0) & (flat < E)
    key = torch.where(kept, flat, torch.full_like(flat, E))
    order = torch.argsort(key, stable=True)
    rows = torch.arange(T * K, device=x.device)
    counts = (key[:, None] == torch.arange(E, device=x.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    slot = torch.empty_like(rows)
    slot[order] = rows
    slot = torch.where(kept, slot, torch.full_like(slot, -1)).view(T, K)
    used = (rows < offsets[-1])[:, None]
    xs = torch.where(used, x[order // K], torch.zeros((), dtype=x.dtype, device=x.device))
    there = (slot >= 0)
    at = slot.clamp(min=0)
    wk = torch.where(there, w.float(), torch.zeros_like(w, dtype=torch.float32))
    picked = ys.float()[at]
    out = {"slots": slot.int(), "offsets": offsets.int(), "xs": xs,
           "y": (wk[..., None] * picked).sum(1).to(ys.dtype)}
    if s["bwd"]:
        dy = s["dy"].float()
        mask = there[..., None].float()
        out["dx"] = (s["dxs"].float()[at] * mask).sum(1).to(x.dtype)
        out["dw"] = torch.where(there, (picked * dy[:, None]).sum(-1),
                                torch.zeros_like(wk)).to(w.dtype)
        dys = (wk.reshape(-1)[order][:, None] * dy[order // K]).to(ys.dtype)
        out["dys"] = torch.where(used, dys, torch.zeros((), dtype=ys.dtype, device=x.device))
    return out


# -----------------------------------------------------------------------------
# the framework's operators
# -----------------------------------------------------------------------------

def _own_logprob(s):
    import tree_training_b200 as tt
    r = tt.token_logprobs(s["x"], s["tokens"], top_k=s["k"], temperature=s["temperature"])
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    if s["k"]:
        out["top_tokens"], out["top_logprobs"] = r.top_tokens, r.top_logprobs
    if s["bwd"]:
        outs, grads = [r.logprobs, r.entropy], [s["g_logp"], s["g_ent"]]
        if s["k"]:
            outs, grads = outs + [r.top_logprobs], grads + [s["g_top"]]
        out["dx"], = torch.autograd.grad(outs, [s["x"]], grads)
    return out


def _own_rotary(s):
    import tree_training_b200 as tt
    q, k = tt.apply_rotary(s["q"], s["k"], s["pos"], s["table"], interleaved=s["interleaved"])
    out = {"q": q, "k": k}
    if s["bwd"]:
        out["dq"], out["dk"] = torch.autograd.grad([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]])
    return out


def _own_norm(s):
    import tree_training_b200 as tt
    y, r = tt.residual_norm(s["x"], s["r"], s["w"], post_weight=s["post"], gate=s["gate"],
                            scale=s["scale"], eps=s["eps"], weight_offset=s["offset"])
    out = {"y": y, "r": r}
    if s["bwd"]:
        names = ["dx", "dr", "dw"] + ["dpost"] * (s["post"] is not None) \
            + ["dgate"] * (s["gate"] is not None)
        ins = [s[n] for n in ("x", "r", "w", "post", "gate") if s[n] is not None]
        out.update(zip(names, torch.autograd.grad([y, r], ins, [s["dy"], s["dr"]])))
    return out


def _own_moe(s):
    import tree_training_b200 as tt
    plan = tt.expert_plan(s["ids"], s["E"])
    xs = tt.expert_dispatch(s["x"], plan)
    y = tt.expert_combine(s["ys"], s["w"], plan)
    out = {"slots": plan.slots, "offsets": plan.offsets, "xs": xs, "y": y}
    if s["bwd"]:
        out["dx"], out["dw"], out["dys"] = torch.autograd.grad(
            [xs, y], [s["x"], s["w"], s["ys"]], [s["dxs"], s["dy"]])
    return out


_PLAIN = {"logprob": _plain_logprob, "rotary": _plain_rotary, "norm": _plain_norm,
          "moe": _plain_moe}
_OWN = {"logprob": _own_logprob, "rotary": _own_rotary, "norm": _own_norm, "moe": _own_moe}


def run(state):
    if own:
        return _OWN[state["op"]](state)
    with torch.no_grad():
        return _PLAIN[state["op"]](state)


# -----------------------------------------------------------------------------
# what a pass cannot do without
# -----------------------------------------------------------------------------

def work(case):
    """Bytes and operations of the forward call and, for a training pass, of
    the backward call, each of which reads its inputs once and writes its
    outputs once: between the two the rest of the model runs, so nothing of
    the first is still on the chip when the second begins."""
    b = _SIZE[case["dtype"]]
    bwd = bool(case["bwd"])
    if case["op"] == "logprob":
        n = case["T"] * case["V"]
        small = case["T"] * (12 * case["M"] + 4 + 12 * case["k"])
        return {"bytes": n * b * (3 if bwd else 1) + small * (2 if bwd else 1),
                "flops": n * (14 if bwd else 8)}
    if case["op"] == "rotary":
        n = case["N"] * (case["hq"] + case["hk"]) * case["D"]
        side = case["N"] * 8 + min(case["N"], 40960) * case["R"] * 4
        turned = case["N"] * (case["hq"] + case["hk"]) * case["R"]
        return {"bytes": (2 * n * b + side) * (2 if bwd else 1),
                "flops": 3 * turned * (2 if bwd else 1)}
    if case["op"] == "norm":
        n = case["T"] * case["D"]
        rb = 4 if case["res"] == "f32" else b
        gate = {"none": 0, "channel": case["D"], "token": case["T"], "full": n}[case["gate"]] * b
        vec = case["D"] * b * (2 if case["post"] else 1)
        total = n * (2 * b + 2 * rb) + gate + vec
        if bwd:
            total += n * (2 * b + 2 * rb) + 2 * gate + 2 * vec       # x, r, dy, dr, gate; dgate, dw
            # dx and dr are one array where nothing stands between them
            same = not case["post"] and not gate and case["scale"] == 1.0 and rb == b
            total += n * (rb if same else b + rb)
        return {"bytes": total, "flops": n * (30 if bwd else 10)}
    tk, H = case["T"] * case["K"], case["H"]
    side = tk * 8 + tk * 4 + case["E"] * 4
    total = (case["T"] + tk) * H * b * 2 + side + tk * 4
    if bwd:
        total += (tk + case["T"]) * H * b + (case["T"] + 2 * tk) * H * b + tk * 8
    return {"bytes": total, "flops": tk * H * (6 if bwd else 2)}


# -----------------------------------------------------------------------------
# 64 bits
# -----------------------------------------------------------------------------

def _exact_logprob(s):
    x = s["x"].detach().double() / s["temperature"]
    T, V = x.shape
    n_ok = (x > float("-inf")).any(1)
    x[~n_ok] = 0.0
    lp = x - torch.logsumexp(x, 1, keepdim=True)
    del x
    p = lp.exp()
    ent = -(p * lp.clamp(min=-1e300)).sum(1) * n_ok
    tok = s["tokens"]
    valid = (tok >= 0) & (tok < V)
    at = tok.clamp(0, V - 1)
    lo = torch.full((), float("-inf"), dtype=torch.float64, device=lp.device)
    pick = torch.where(n_ok[:, None], lp.gather(1, at), lo)
    out = {"logprobs": torch.where(valid, pick, torch.zeros_like(pick)), "entropy": ent}
    k = s["k"]
    if k:
        xx = s["x"].detach().double()
        key, idx = torch.sort(xx, dim=1, descending=True, stable=True)
        idx = idx[:, :k].contiguous()
        del key, xx
        out["top_tokens"] = None
        out["top_logprobs"] = torch.where(n_ok[:, None], lp.gather(1, idx), lo)
    if s["bwd"]:
        gl = s["g_logp"].double() * valid * n_ok[:, None]
        total = gl.sum(1)
        if k:
            gt = s["g_top"].double() * n_ok[:, None]
            total = total + gt.sum(1)
        dx = p * (-total[:, None] - s["g_ent"].double()[:, None]
                  * (lp.clamp(min=-1e300) + ent[:, None])) * n_ok[:, None]
        dx.scatter_add_(1, at, gl)
        if k:
            dx.scatter_add_(1, idx, gt)
        out["dx"] = dx / s["temperature"]
    return out


def _exact_rotary(s):
    t = s["table"].double()[s["pos"]]
    half = t.shape[1] // 2
    u = torch.complex(t[:, :half], t[:, half:])[:, None]

    def turn(x, u):
        x = x.detach().double()
        y = x.clone()
        if s["interleaved"]:
            first, second = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
        else:
            first, second = slice(0, half), slice(half, 2 * half)
        v = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * u
        y[..., first], y[..., second] = v.real, v.imag
        return y

    out = {"q": turn(s["q"], u), "k": turn(s["k"], u)}
    if s["bwd"]:
        out["dq"], out["dk"] = turn(s["dq"], u.conj()), turn(s["dk"], u.conj())
    return out


def _exact_norm(s):
    # from the forward's definition; the gradients by differentiation in 64 bits
    names = [n for n in ("x", "r", "w", "post", "gate") if s[n] is not None]
    v = {n: s[n].detach().double().requires_grad_(s["bwd"]) for n in names}
    norm = lambda t, w: t / torch.sqrt((t * t).sum(1, keepdim=True) / t.shape[1] + s["eps"]) \
        * (w + s["offset"])
    b = norm(v["x"], v["post"]) if "post" in v else v["x"]
    b = b * v["gate"] if "gate" in v else b
    r = v["r"] + b * s["scale"]
    y = norm(r, v["w"])
    out = {"y": y.detach(), "r": r.detach()}
    if s["bwd"]:
        gs = torch.autograd.grad([y, r], [v[n] for n in names],
                                 [s["dy"].double(), s["dr"].double()])
        out.update(zip(["d" + n for n in names], gs))
    return out


def _exact_moe(s):
    ids, E = s["ids"], s["E"]
    T, K = ids.shape
    H = s["x"].shape[1]
    # each expert's entries in order, one expert after another
    there = [torch.nonzero(ids.reshape(-1) == e).view(-1) for e in range(E)]
    entry = torch.cat(there)
    n = entry.numel()
    dev = ids.device
    f64 = torch.float64
    xs = torch.zeros(T * K, H, dtype=f64, device=dev)
    xs[:n] = s["x"].detach().double()[entry // K]
    wr = s["w"].detach().double().reshape(-1)[entry]
    ys = s["ys"].detach().double()[:n]
    y = torch.zeros(T, H, dtype=f64, device=dev).index_add_(0, entry // K, ys * wr[:, None])
    out = {"slots": None, "offsets": None, "xs": xs, "y": y}
    if s["bwd"]:
        dy = s["dy"].double()[entry // K]
        out["dx"] = torch.zeros(T, H, dtype=f64, device=dev).index_add_(
            0, entry // K, s["dxs"].double()[:n])
        dw = torch.zeros(T * K, dtype=f64, device=dev)
        dw[entry] = (dy * ys).sum(1)
        out["dw"] = dw.view(T, K)
        dys = torch.zeros(T * K, H, dtype=f64, device=dev)
        dys[:n] = dy * wr[:, None]
        out["dys"] = dys
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.set_grad_enabled(case["op"] == "norm"):
        return {"logprob": _exact_logprob, "rotary": _exact_rotary, "norm": _exact_norm,
                "moe": _exact_moe}[case["op"]](s)
