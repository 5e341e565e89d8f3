"""Cases for the operators at the ends and in the middle of a training step:
embedding rows and their gradient, the gated feed-forward product, the loss of
an LM head without its logits, and the norm and clipping of all gradients.

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

def _embed_case(T, V, H, dtype, bwd, scale=1.0, padded=False):
    return {"op": "embed", "T": T, "V": V, "H": H, "dtype": dtype, "bwd": bwd, "scale": scale,
            "padded": padded}


def _ffn_case(T, H, F, dtype, bwd, act="silu"):
    return {"op": "ffn", "T": T, "H": H, "F": F, "dtype": dtype, "bwd": bwd, "act": act}


def _ce_case(T, H, V, M, dtype, bwd, scale=1.0):
    return {"op": "ce", "T": T, "H": H, "V": V, "M": M, "dtype": dtype, "bwd": bwd, "scale": scale}


def _clip_case(tensors, elements, dtype, model=False, norm_type=2.0, clipped=True):
    """``model``: the tensors of a decoder with ``tensors`` layers of hidden size
    ``elements`` (the other sizes follow); else ``tensors`` tensors of up to
    ``elements`` elements."""
    return {"op": "clip", "tensors": tensors, "elements": elements, "dtype": dtype,
            "model": model, "norm_type": norm_type, "clipped": clipped}


def listed():
    return [
        # the 47-token forest's tokens through the test model's table: latency
        dict(_embed_case(47, 32000, 256, "f32", False), name="embed_small"),
        # one 32,768-token tree, 151,936 words of 2,560, and the table's gradient
        dict(_embed_case(32768, 151936, 2560, "bf16", True), name="embed_train"),
        # rows of an odd width, scaled, with padding between the sequences
        dict(_embed_case(8191, 32003, 1001, "f16", True, scale=31.6, padded=True),
             name="embed_odd"),
        # one token of a rollout: both weights are read for a single row
        dict(_ffn_case(1, 2560, 9728, "bf16", False), name="ffn_token"),
        # the 47-token forest through the test model's block, with gradients
        dict(_ffn_case(47, 256, 688, "f32", True), name="ffn_small"),
        # a partition of 8,192 tokens through a block of 2,560 and 9,728
        dict(_ffn_case(8192, 2560, 9728, "bf16", True), name="ffn_train"),
        # odd sizes everywhere
        dict(_ffn_case(2047, 1001, 2735, "f16", True, act="gelu_tanh"), name="ffn_odd"),
        # the 47-token forest's loss over a 32,000-word vocabulary
        dict(_ce_case(47, 256, 32000, 1, "f32", True), name="ce_small"),
        # a partition's loss and gradients over 151,936 words, one successor a token
        dict(_ce_case(8192, 2560, 151936, 1, "bf16", True), name="ce_train"),
        # scoring a tree's tokens, up to two successors at a branch
        dict(_ce_case(2047, 2560, 151936, 2, "bf16", False, scale=0.7), name="ce_score"),
        # gradients of the two-layer test model
        dict(_clip_case(2, 256, "f32", model=True), name="clip_small"),
        # gradients of eight layers of 2,560 and the tied table
        dict(_clip_case(8, 2560, "bf16", model=True), name="clip_train"),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """Three in four a multiple of 64, as models have them."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.25 else max(lo, n // 64 * 64)


def draw(rng):
    op = rng.choice(["embed", "ffn", "ce", "clip"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    bwd = rng.random() < 0.6
    wide = 2 if dtype == "f32" else 1
    if op == "embed":
        H, V = _width(rng, 64, 8192), _log_int(rng, 128, 151936)
        if bwd:
            V = min(V, 151936 * 2560 // wide // H)
        T = _log_int(rng, 1, min(32768, 32768 * 2560 // wide // H))
        return _embed_case(T, V, H, dtype, bwd, rng.choice([1.0, 0.5, 31.6]), rng.random() < 0.4)
    if op == "ffn":
        # 32-bit products take longer: an eighth of the work
        cap = 8192 * 2560 * 9728 // (8 if wide == 2 else 1)
        H, F = _width(rng, 64, 8192), _width(rng, 64, 16384)
        T = _log_int(rng, 1, max(1, min(32768, cap // (H * F))))
        return _ffn_case(T, H, F, dtype, bwd, rng.choice(["silu", "silu", "gelu_tanh", "gelu",
                                                          "relu"]))
    if op == "ce":
        cap = 8192 * 2560 * 151936 // (32 if wide == 2 else 1)
        H = _width(rng, 64, 5120)
        V = _log_int(rng, 128, min(151936, 151936 * 2560 // wide // H))
        T = _log_int(rng, 1, max(1, min(16384, cap // (H * V))))
        return _ce_case(T, H, V, rng.choice([1, 1, 2, 4]), dtype, bwd, rng.choice([1.0, 1.0, 0.7]))
    elements = _log_int(rng, 1, 1 << 26)
    n = _log_int(rng, 1, max(1, min(600, (1 << 30) // elements)))
    return _clip_case(n, elements, rng.choice(["bf16", "f32", "f16", "mixed"]), False,
                      rng.choice([2.0, 2.0, math.inf, 1.0]), rng.random() < 0.7)


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


def _words(g, n, V):
    """Tokens as texts have them: few words make up much of a text."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(V)) - 1).long().clamp(0, V - 1)


def _model_shapes(layers, H):
    """A decoder's weights, as the test model and the benchmark's have them."""
    F, V, q, kv = (688, 32000, 256, 128) if H == 256 else (9728, 151936, 4096, 1024)
    layer = [(q, H), (kv, H), (kv, H), (H, q), (H,), (H,), (F, H), (F, H), (H, F)]
    return [(V, H)] + layer * layers + [(H,)]


def _clip_shapes(case):
    if case["model"]:
        return [(s, case["dtype"]) for s in _model_shapes(case["tensors"], case["elements"])]
    # sizes between 1 and the largest, the same for every seed
    out = []
    for i in range(case["tensors"]):
        n = case["elements"] if i == 0 else max(1, int(case["elements"] ** (((i * 37) % 64) / 64)))
        kind = ("bf16", "f32", "f16")[i % 3] if case["dtype"] == "mixed" else case["dtype"]
        out.append(((n,), kind))
    return out


def _flat_like(tensors):
    """Views of one buffer a type, each on a 256-byte boundary, as an optimiser
    with flat buffers holds its gradients."""
    flat, views = {}, []
    for dt in sorted({t.dtype for t in tensors}, key=str):
        step = 256 // dt.itemsize
        n = sum((t.numel() + step - 1) // step * step for t in tensors if t.dtype == dt)
        flat[str(dt).split(".")[1]] = torch.zeros(n, dtype=dt, device="cuda")
    used = dict.fromkeys(flat, 0)
    for t in tensors:
        kind, step = str(t.dtype).split(".")[1], 256 // t.dtype.itemsize
        views.append(flat[kind][used[kind]:used[kind] + t.numel()].view(t.shape))
        used[kind] += (t.numel() + step - 1) // step * step
    return {"flat": flat, "out": views}


def prepare(case, seed):
    g = _gen(seed)
    s = {"op": case["op"]}
    if case["op"] == "clip":
        s["grads"] = [_randn(g, shape, _DTYPES[kind], 1e-2) for shape, kind in _clip_shapes(case)]
        n = sum(t.numel() for t in s["grads"])
        # what the norm is expected to be: clipped to a third of it, or not at all
        size = {2.0: 1e-2 * math.sqrt(n), 1.0: 1e-2 * n * 0.8, math.inf: 1e-2}[case["norm_type"]]
        s.update(norm_type=case["norm_type"], max_norm=size * (0.33 if case["clipped"] else 100.0),
                 **_flat_like(s["grads"]))
        return s
    dt = _DTYPES[case["dtype"]]
    bwd = bool(case["bwd"])
    s["bwd"] = bwd
    if case["op"] == "embed":
        T, V, H = case["T"], case["V"], case["H"]
        ids = _words(g, T, V)
        if case["padded"]:
            at = torch.arange(T, device="cuda")
            ids[(at // 61) % 5 == 4] = V - 1
        s.update(ids=ids, w=_randn(g, (V, H), dt, 0.02 if case["scale"] == 1.0 else 1.0)
                 .requires_grad_(bwd), scale=case["scale"],
                 padding=V - 1 if case["padded"] else None)
        if bwd:
            s["dy"] = _randn(g, (T, H), dt)
        return s
    if case["op"] == "ffn":
        T, H, F = case["T"], case["H"], case["F"]
        s.update(x=_randn(g, (T, H), dt).requires_grad_(bwd), act=case["act"],
                 wg=_randn(g, (F, H), dt, H ** -0.5).requires_grad_(bwd),
                 wu=_randn(g, (F, H), dt, H ** -0.5).requires_grad_(bwd))
        if bwd:
            s["dh"] = _randn(g, (T, F), dt)
        return s
    T, H, V, M = case["T"], case["H"], case["V"], case["M"]
    w = _randn(g, (V, H), dt, H ** -0.5)
    x = _randn(g, (T, H), dt, 1.5)
    labels = torch.randint(0, V, (T, M), generator=g, device="cuda")
    # as a trained head gives them: half of the first successors stand out
    sure = (torch.rand(T, 1, generator=g, device="cuda") < 0.5) * 9.0
    x += (sure * w[labels[:, 0]].float()).to(dt)
    labels[:, 1:][torch.rand(T, M - 1, generator=g, device="cuda") < 0.7] = -100
    labels[5::9] = -100
    s.update(x=x.requires_grad_(bwd), w=w.requires_grad_(bwd),
             labels=labels[:, 0].contiguous() if M == 1 else labels, scale=case["scale"])
    if bwd:
        s.update(g_loss=torch.rand(s["labels"].shape, generator=g, device="cuda") / T,
                 g_lse=torch.randn(T, generator=g, device="cuda") * 1e-4 / T)
    return s


# -----------------------------------------------------------------------------
# the plain forms
# -----------------------------------------------------------------------------

def _plain_embed(s):
    ids, w = s["ids"], s["w"].detach()
    out = {"y": (w[ids].float() * s["scale"]).to(w.dtype)}
    if s["bwd"]:
        dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
        dw.index_add_(0, ids, s["dy"].float())
        if s["padding"] is not None:
            dw[s["padding"]] = 0
        out["dw"] = (dw * s["scale"]).to(w.dtype)
    return out


def _activation(g, act):
    """The activation and its derivative."""
    if act == "silu":
        q = 1 / (1 + torch.exp(-g))
        return g * q, q * (1 + g * (1 - q))
    if act == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        t = torch.tanh(a * (g + 0.044715 * g * g * g))
        return (0.5 * g * (1 + t),
                0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 0.134145 * g * g))
    if act == "gelu":
        c = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * c, c + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    on = (g > 0).float()
    return g * on, on


def _plain_ffn(s):
    x, wg, wu = (s[n].detach().float() for n in ("x", "wg", "wu"))
    dt = s["x"].dtype
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _activation(g, s["act"])
    out = {"h": (a * u).to(dt)}
    if s["bwd"]:
        dh = s["dh"].float()
        dg, du = dh * u * da, dh * a
        out["dx"] = (dg @ wg + du @ wu).to(dt)
        out["dwg"], out["dwu"] = (dg.t() @ x).to(dt), (du.t() @ x).to(dt)
    return out


def _plain_ce(s):
    x, w = s["x"].detach().float(), s["w"].detach().float()
    T, V = x.shape[0], w.shape[0]
    labels = s["labels"].view(T, -1)
    valid = (labels >= 0) & (labels < V)
    at = torch.where(valid, labels, torch.zeros_like(labels))
    loss = torch.empty(labels.shape, dtype=torch.float32, device=x.device)
    lse = torch.empty(T, dtype=torch.float32, device=x.device)
    if s["bwd"]:
        dx, dw = torch.empty_like(x), torch.zeros_like(w)
        g = torch.where(valid, s["g_loss"].view(T, -1), torch.zeros_like(loss))
    rows = max(1, (1 << 29) // V)
    for r in range(0, T, rows):
        part = slice(r, min(T, r + rows))
        z = (x[part] @ w.t()) * s["scale"]
        m = z.amax(1, keepdim=True)
        total = torch.exp(z - m).sum(1, keepdim=True)
        l = m + total.log()
        lse[part] = l[:, 0]
        loss[part] = torch.where(valid[part], l - z.gather(1, at[part]), torch.zeros_like(z[:, :1]))
        if s["bwd"]:
            d = torch.exp(z - l) * (g[part].sum(1, keepdim=True) + s["g_lse"][part, None])
            d.scatter_add_(1, at[part], -g[part])
            d *= s["scale"]
            dx[part] = d @ w
            dw += d.t() @ x[part]
    out = {"loss": loss.view(s["labels"].shape), "lse": lse}
    if s["bwd"]:
        out["dx"], out["dw"] = dx.to(s["x"].dtype), dw.to(s["w"].dtype)
    return out


def _plain_clip(s):
    p = s["norm_type"]
    if p == math.inf:
        norm = torch.stack([t.float().abs().amax() for t in s["grads"]]).amax()
    elif p == 1.0:
        norm = sum(t.float().abs().sum(dtype=torch.float64) for t in s["grads"]).float()
    else:
        norm = sum(t.float().square().sum(dtype=torch.float64) for t in s["grads"]).sqrt().float()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    for o, t in zip(s["out"], s["grads"]):
        o.copy_(t.float() * coef)
    return {"norm": norm, "grads": s["flat"]}


# -----------------------------------------------------------------------------
# the framework's operators
# -----------------------------------------------------------------------------

def _own_embed(s):
    import tree_training_b200 as tt
    y = tt.embedding(s["ids"], s["w"], scale=s["scale"], padding_idx=s["padding"])
    out = {"y": y}
    if s["bwd"]:
        out["dw"], = torch.autograd.grad([y], [s["w"]], [s["dy"]])
    return out


def _own_ffn(s):
    import tree_training_b200 as tt
    h = tt.gated_linear(s["x"], s["wg"], s["wu"], activation=s["act"])
    out = {"h": h}
    if s["bwd"]:
        out["dx"], out["dwg"], out["dwu"] = torch.autograd.grad(
            [h], [s["x"], s["wg"], s["wu"]], [s["dh"]])
    return out


def _own_ce(s):
    import tree_training_b200 as tt
    r = tt.linear_cross_entropy(s["x"], s["w"], s["labels"], scale=s["scale"])
    out = {"loss": r.losses, "lse": r.lse}
    if s["bwd"]:
        out["dx"], out["dw"] = torch.autograd.grad([r.losses, r.lse], [s["x"], s["w"]],
                                                   [s["g_loss"], s["g_lse"]])
    return out


def _own_clip(s):
    import tree_training_b200 as tt
    norm = tt.clip_grad_norm(s["grads"], s["max_norm"], norm_type=s["norm_type"], out=s["out"])
    return {"norm": norm, "grads": s["flat"]}


_PLAIN = {"embed": _plain_embed, "ffn": _plain_ffn, "ce": _plain_ce, "clip": _plain_clip}
_OWN = {"embed": _own_embed, "ffn": _own_ffn, "ce": _own_ce, "clip": _own_clip}


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
    if case["op"] == "clip":
        n = b = 0
        for shape, kind in _clip_shapes(case):
            n += math.prod(shape)
            b += math.prod(shape) * _SIZE[kind]
        return {"bytes": 2 * b, "flops": 3 * n}
    b, bwd = _SIZE[case["dtype"]], bool(case["bwd"])
    if case["op"] == "embed":
        T, V, H = case["T"], case["V"], case["H"]
        # every row of the table that the tokens name once, every row of its gradient
        named = min(T, V) * H * b
        total = T * 8 + named + T * H * b
        if bwd:
            total += T * 8 + T * H * b + V * H * b
        return {"bytes": total, "flops": T * H * (2 if bwd else 1)}
    if case["op"] == "ffn":
        T, H, F = case["T"], case["H"], case["F"]
        total = (T * H + 2 * F * H + T * F) * b
        flops = 4 * T * H * F
        if bwd:
            total += (T * H + 2 * F * H + T * F) * b + (T * H + 2 * F * H) * b
            flops += 8 * T * H * F
        return {"bytes": total, "flops": flops}
    T, H, V, M = case["T"], case["H"], case["V"], case["M"]
    total = (T * H + V * H) * b + T * (12 * M + 4)
    flops = 2 * T * H * V
    if bwd:
        total += 2 * (T * H + V * H) * b + T * (12 * M + 8)
        flops += 4 * T * H * V
    return {"bytes": total, "flops": flops}


# -----------------------------------------------------------------------------
# 64 bits
# -----------------------------------------------------------------------------

def _exact_embed(s):
    w = s["w"].detach()
    out = {"y": w[s["ids"]].double() * s["scale"]}
    if s["bwd"]:
        ids, dy = s["ids"], s["dy"]
        if s["padding"] is not None:
            keep = (ids != s["padding"]).nonzero().view(-1)
            ids, dy = ids[keep], dy[keep]
        # by words: the rows of equal tokens next to one another, sums by differences
        # of positions would cancel, so every word's rows are added on their own
        order = torch.argsort(ids, stable=True)
        dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
        dw.index_put_((ids[order],), dy[order].double() * s["scale"], accumulate=True)
        out["dw"] = dw
    return out


def _exact_ffn(s):
    names = ("x", "wg", "wu")
    v = {n: s[n].detach().double().requires_grad_(s["bwd"]) for n in names}
    g, u = v["x"] @ v["wg"].t(), v["x"] @ v["wu"].t()
    act = s["act"]
    if act == "silu":
        a = g * torch.sigmoid(g)
    elif act == "gelu_tanh":
        a = g / 2 * (1 + torch.tanh((2 / math.pi) ** 0.5 * (g + 0.044715 * g ** 3)))
    elif act == "gelu":
        a = g / 2 * torch.erfc(-g / 2 ** 0.5)
    else:
        a = g.clamp(min=0)
    h = a * u
    out = {"h": h.detach()}
    if s["bwd"]:
        # the gradients by differentiation in 64 bits
        gs = torch.autograd.grad(h, [v[n] for n in names], s["dh"].double())
        out.update(zip(["d" + n for n in names], gs))
    return out


def _exact_ce(s):
    x, w = s["x"].detach().double(), s["w"].detach().double()
    T, V = x.shape[0], w.shape[0]
    labels = s["labels"].view(T, -1)
    losses, lses = [], []
    dx, dw = [], None
    if s["bwd"]:
        w.requires_grad_(True)
    rows = max(1, (1 << 28) // V)
    for r in range(0, T, rows):
        xr = x[r:r + rows].detach().requires_grad_(s["bwd"])
        lab = labels[r:r + rows]
        z = xr @ w.t() * s["scale"]
        lse = torch.logsumexp(z, 1)
        ok = (lab >= 0) & (lab < V)
        loss = torch.where(ok, lse[:, None] - z.gather(1, lab.clamp(0, V - 1)), 0.0)
        if s["bwd"]:
            gx, gw = torch.autograd.grad(
                [loss, lse], [xr, w], [s["g_loss"].view(T, -1)[r:r + rows].double(),
                                       s["g_lse"][r:r + rows].double()])
            dx.append(gx)
            dw = gw if dw is None else dw.add_(gw)
        losses.append(loss.detach())
        lses.append(lse.detach())
        del z, loss, lse
    out = {"loss": torch.cat(losses).view(s["labels"].shape), "lse": torch.cat(lses)}
    if s["bwd"]:
        out["dx"], out["dw"] = torch.cat(dx), dw
    return out


def _exact_clip(s):
    p = s["norm_type"]
    each = torch.stack([torch.linalg.vector_norm(t.double(), p) for t in s["grads"]])
    norm = torch.linalg.vector_norm(each, p)
    coef = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    flat = {}
    for kind in s["flat"]:
        parts = []
        for t in s["grads"]:
            if str(t.dtype) == "torch." + kind:
                parts += [t.double().view(-1) * coef,
                          t.new_zeros(-t.numel() % (256 // t.dtype.itemsize)).double()]
        flat[kind] = torch.cat(parts)
    return {"norm": norm, "grads": flat}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.set_grad_enabled(case["op"] in ("ffn", "ce") and bool(case.get("bwd"))):
        return {"embed": _exact_embed, "ffn": _exact_ffn, "ce": _exact_ce,
                "clip": _exact_clip}[case["op"]](s)
