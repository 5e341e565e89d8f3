"""The gated feed-forward product and its gradients against the formulas in 64 bits.

Bounds.  A sum of n products on the tensor cores or by fma is off by at most
2 n 2^-24 of the sum of its terms' magnitudes (the tensor cores cut off instead of
rounding: twice the step).  dg and du are rounded to the inputs' type on their way
into the products: u(T) of each, through the product with the weights' magnitudes.
"""
import pytest
import torch

import tree_training_b200 as tt
from tests.op_bounds import EPS, TINY, UNIT, directional

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16
ACTS = ["silu", "gelu", "gelu_tanh", "relu"]
SLOPE = 1.14              # no activation here is steeper (nor curves more, bar relu)


def act64(g, name):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return g * torch.special.ndtr(g)
    if name == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3)))
    return g.clamp(min=0)


def make(T, H, F, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    return (r(T, H).to(dtype), (r(F, H) * H ** -0.5).to(dtype), (r(F, H) * H ** -0.5).to(dtype),
            r(T, F).to(dtype))


def within(name, got, want, extra):
    t = got.dtype
    bound = UNIT[t] * want.abs() + extra + TINY[t]
    over = (got.double() - want).abs() - bound
    assert over.max() <= 0, f"{name}: over its bound {bound.flatten()[over.argmax()]:.3e} by " \
                            f"{over.max():.3e}"


def compare(x, wg, wu, dh, act="silu"):
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu)]
    h = tt.gated_linear(*leaves, activation=act)
    got = torch.autograd.grad(h, leaves, dh)
    tt.check_device_status()
    x, wg, wu, dh = (t.detach().double() for t in (x, wg, wu, dh))
    T, (F, H), u16 = x.shape[0], wg.shape, UNIT[got[0].dtype] if got[0].dtype != F32 else EPS
    g = (x @ wg.t()).requires_grad_(True)
    u = x @ wu.t()
    a = act64(g, act)
    da, = torch.autograd.grad(a.sum(), g)
    g, a = g.detach(), a.detach()
    ag, au = x.abs() @ wg.abs().t(), x.abs() @ wu.abs().t()      # the sums' magnitudes
    eg, eu = 2 * H * EPS * ag, 2 * H * EPS * au                  # what g and u may be off
    # (the activations' own roundings: tanh's argument and the exponential's go in
    # with their size, a few units of fp32)
    few = 32 * EPS * (1 + g.abs())
    within("h", h.detach(), a * u, SLOPE * eg * u.abs() + a.abs() * eu + few * u.abs())
    dg, du = dh * u * da, dh * a
    curve = SLOPE * eg                                           # what act' may be off by g's
    if act == "relu":                                            # it jumps: where g's sign is open
        curve = (g.abs() <= eg).double()
    edg = dh.abs() * (da.abs() * eu + u.abs() * (curve + few)) + u16 * dg.abs()
    edu = dh.abs() * (SLOPE * eg + few) + u16 * du.abs()
    if got[0].dtype == F16:                                      # subnormal dg, du
        edg, edu = edg + 2.0 ** -25, edu + 2.0 ** -25
    within("dx", got[0], dg @ wg + du @ wu,
           edg @ wg.abs() + edu @ wu.abs()
           + 4 * F * EPS * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()))
    within("dwg", got[1], dg.t() @ x, edg.t() @ x.abs() + 2 * T * EPS * (dg.abs().t() @ x.abs()))
    within("dwu", got[2], du.t() @ x, edu.t() @ x.abs() + 2 * T * EPS * (du.abs().t() @ x.abs()))
    return h, got


SIZES = [(1, 1, 1), (1, 64, 64), (3, 8, 5), (47, 256, 688), (127, 72, 130), (128, 64, 128),
         (129, 200, 257), (300, 1001, 735), (257, 520, 1000), (700, 136, 2048), (2049, 64, 72)]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("T,H,F", SIZES)
def test_forward_and_gradients(T, H, F, dtype):
    compare(*make(T, H, F, dtype, T))


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("act", ACTS)
def test_activations(act, dtype):
    x, wg, wu, dh = make(150, 96, 168, dtype, 1)
    compare(x * 3, wg, wu, dh, act)


@pytest.mark.parametrize("T,H,F", [(1, 2560, 9728), (16, 1024, 4000), (1500, 2560, 1024),
                                   (64, 64, 30000), (20000, 64, 64), (40, 8192, 512)])
def test_long_sides(T, H, F):
    compare(*make(T, H, F, BF, 2))


def test_single_rows_equal_the_batch():
    # a token's result does not depend on which others are in the call, as far as
    # the sum over H has the same order: within the bounds of two roundings
    x, wg, wu, _ = make(300, 520, 640, BF, 3)
    whole = tt.gated_linear(x, wg, wu).double()
    one = torch.cat([tt.gated_linear(x[i:i + 1], wg, wu) for i in (0, 150, 299)]).double()
    assert ((whole[[0, 150, 299]] - one).abs() <= 2 * UNIT[BF] * one.abs() + 1e-5).all()


def test_strides_and_shapes():
    x, wg, wu, dh = make(96, 64, 80, BF, 4)
    both = torch.cat([wg, wu])
    compare(x, both[:80], both[80:], dh)
    wide = torch.randn(96, 200, device=DEV).to(BF)
    compare(wide[:, 8:72], wg, wu, dh)                       # on 16-byte boundaries
    compare(wide[:, 3:67], wg, wu, dh)                       # off them: copied
    compare(x, wide[:80, 1:65], wide[:80, 100:164], dh)
    compare(torch.randn(64, 96, device=DEV).to(BF).t(), wg, wu, dh)
    compare(x, wg, wu, dh[:, :1].expand(96, 80))
    compare(x, wg, wu, torch.randn(80, 96, device=DEV).to(BF).t())
    h = tt.gated_linear(x.view(4, 24, 64), wg, wu)
    assert h.shape == (4, 24, 80) and torch.equal(h.view(96, 80), tt.gated_linear(x, wg, wu))
    assert torch.equal(tt.gated_linear(x[0], wg, wu), tt.gated_linear(x[:1], wg, wu)[0])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_no_rows(dtype):
    x, wg, wu, _ = make(1, 16, 24, dtype)
    leaves = [x[:0].requires_grad_(True), wg.requires_grad_(True), wu.requires_grad_(True)]
    h = tt.gated_linear(*leaves)
    assert h.shape == (0, 24)
    grads = torch.autograd.grad(h.sum(), leaves)
    assert [tuple(g.shape) for g in grads] == [(0, 16), (24, 16), (24, 16)]
    assert not any(g.any() for g in grads)


def test_only_the_gradients_that_are_asked_for():
    x, wg, wu, dh = make(200, 128, 264, BF, 5)
    _, want = compare(x, wg, wu, dh)
    for i in range(3):
        leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, wg, wu))]
        g, = torch.autograd.grad(tt.gated_linear(*leaves), leaves[i], dh)
        assert torch.equal(g, want[i])


def test_differences():
    x, wg, wu, dh = make(20, 33, 41, F32, 6)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu)]
    f = lambda *a: [tt.gated_linear(*a)]
    grads = torch.autograd.grad(f(*leaves), leaves, dh)
    # central differences of step s: s^2 / 6 of the third derivative and 2^-24 of the
    # values over s, with s = 2^-7 both under 1e-3 of the gradients' norm
    directional(f, leaves, [dh], grads, 2.0 ** -7, 1e-3)


def test_nan_and_infinity_stay_in_their_rows():
    x, wg, wu, _ = make(140, 64, 96, BF, 7)
    clean = tt.gated_linear(x, wg, wu)
    y = x.clone()
    y[5, 3], y[131, 60] = float("nan"), float("inf")
    h = tt.gated_linear(y, wg, wu)
    assert h[5].isnan().all() and not h[131].isfinite().any()
    rest = [i for i in range(140) if i not in (5, 131)]
    assert torch.equal(h[rest], clean[rest])


def test_same_bits_another_stream_and_replay():
    x, wg, wu, dh = make(333, 256, 512, BF, 8)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu)]

    def step():
        h = tt.gated_linear(*leaves)
        return [h.detach(), *torch.autograd.grad(h, leaves, dh)]
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(want, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        x.copy_(x.flip(0))
    dh.copy_(dh.flip(0))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(step(), got))
    tt.check_device_status()


def test_refusals():
    x, wg, wu, _ = make(4, 16, 24, BF)
    with pytest.raises(ValueError):
        tt.gated_linear(x, wg, wu, activation="tanh")
    with pytest.raises(ValueError):
        tt.gated_linear(x, wg[:, :8], wu)
    with pytest.raises(ValueError):
        tt.gated_linear(x, wg, wu[:8])
    with pytest.raises(TypeError):
        tt.gated_linear(x, wg, wu.half())
    with pytest.raises(TypeError):
        tt.gated_linear(x.double(), wg.double(), wu.double())
    with pytest.raises(RuntimeError):
        tt.gated_linear(x, wg.cpu(), wu)
    x.requires_grad_(True)
    g, = torch.autograd.grad(tt.gated_linear(x, wg, wu).float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_hf_modules():
    transformers = pytest.importorskip("transformers")
    from transformers.models.qwen3.modeling_qwen3 import Qwen3MLP
    cfg = transformers.Qwen3Config(hidden_size=128, intermediate_size=264, num_hidden_layers=1)
    torch.manual_seed(0)
    mlp = torch.nn.ModuleList([Qwen3MLP(cfg), torch.nn.Linear(4, 4)]).to(DEV)
    x = torch.randn(2, 37, 128, device=DEV, requires_grad=True)
    dy = torch.randn(2, 37, 128, device=DEV)
    ps = list(mlp[0].parameters())
    want = [mlp[0](x), *torch.autograd.grad(mlp[0](x), [x, *ps], dy)]
    assert tt.fuse_gated_mlps(mlp) == 1
    got = [mlp[0](x), *torch.autograd.grad(mlp[0](x), [x, *ps], dy)]
    for a, b in zip(got, want):          # fp32 on both sides: sums of up to 264 terms
        assert float((a - b).norm() / b.norm()) < 264 * EPS


def test_modules_that_do_more_keep_their_forward():
    class Block(torch.nn.Module):
        def __init__(self, act, limit=None, bias=False):
            super().__init__()
            self.gate_proj = torch.nn.Linear(32, 48, bias=bias)
            self.up_proj = torch.nn.Linear(32, 48, bias=False)
            self.down_proj = torch.nn.Linear(48, 32)
            self.act_fn, self.limit = act, limit

        def forward(self, x):
            h = self.act_fn(self.gate_proj(x)) * self.up_proj(x)
            return self.down_proj(h if self.limit is None else h.clamp(max=self.limit))
    torch.manual_seed(1)
    m = torch.nn.ModuleList([Block(torch.nn.SiLU()), Block(torch.nn.SiLU(), 0.01),
                             Block(torch.nn.Tanh()), Block(torch.nn.SiLU(), bias=True),
                             Block(torch.nn.GELU(approximate="tanh")), Block(torch.nn.GELU()),
                             Block(torch.nn.ReLU())]).to(DEV)
    x = torch.randn(5, 32, device=DEV)
    want = [b(x) for b in m]
    assert tt.fuse_gated_mlps(m) == 4
    for b, w in zip(m, want):
        assert float((b(x) - w).norm() / w.norm()) < 100 * EPS


@pytest.mark.parametrize("dtype,largest", [(BF, 1e18), (F16, 6e4 * 6e4)])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_gradients_far_below_zero(act, dtype, largest):
    """Where the activation is nothing its slope is, however large the product: dg and
    du are 0 there (the cube in tanh's argument reaches 1e54, past fp32)."""
    sizes = torch.logspace(1, torch.tensor(largest).log10().item() / 2, 24, device=DEV)
    for r in sizes.tolist():                # feature 0: g = -r^2, u = 1
        x = torch.zeros(1, 16, device=DEV, dtype=dtype)
        wg, wu = (torch.zeros(8, 16, device=DEV, dtype=dtype) for _ in range(2))
        x[0, 0], wg[0, 0] = r, -r
        x[0, 1] = wu[:, 1] = 1
        leaves = [t.requires_grad_(True) for t in (x, wg, wu)]
        h = tt.gated_linear(*leaves, activation=act)
        dx, dwg, dwu = torch.autograd.grad(h, leaves, torch.ones_like(h))
        for got in (h[0, 0], dx[0, 0], dwg[0], dwu[0]):
            assert float(got.abs().max()) == 0, (r, got)
    tt.check_device_status()


def test_widths_that_32_bits_do_not_count():
    one = torch.ones(1, 1, device=DEV, dtype=BF)
    with pytest.raises(ValueError):
        tt.gated_linear(one, *[one.expand((1 << 30) - 255, 1)] * 2)
    wide = one.expand(1, (1 << 31) - 257)
    with pytest.raises(ValueError):
        tt.gated_linear(wide, wide, wide)


def test_modules_that_are_wrapped_or_watched_keep_their_forward():
    transformers = pytest.importorskip("transformers")
    from transformers.models.qwen3.modeling_qwen3 import Qwen3MLP
    cfg = transformers.Qwen3Config(hidden_size=64, intermediate_size=96, num_hidden_layers=1)

    class Dropping(Qwen3MLP):
        def forward(self, x):
            return torch.nn.functional.dropout(super().forward(x), 0.5, self.training)

    class Normed(Qwen3MLP):
        def __init__(self, cfg):
            super().__init__(cfg)
            self.norm = torch.nn.LayerNorm(64)
    seen = []
    wrapped, hooked, double, plain = (Qwen3MLP(cfg) for _ in range(4))
    forward = wrapped.forward
    wrapped.forward = lambda x: (seen.append(1), forward(x))[1]
    hooked.up_proj.register_forward_hook(lambda *a: seen.append(2))
    m = torch.nn.ModuleList([wrapped, hooked, double.double(), Dropping(cfg), Normed(cfg)]).to(DEV)
    m.eval()
    state = torch.cuda.get_rng_state(), torch.get_rng_state()
    assert tt.fuse_gated_mlps(m) == 0
    assert torch.equal(torch.cuda.get_rng_state(), state[0])
    assert torch.equal(torch.get_rng_state(), state[1])
    assert not any(b.training for b in m)
    seen.clear()
    x = torch.randn(3, 64, device=DEV)
    wrapped(x), hooked(x)
    assert seen == [1, 2]
    plain = torch.nn.ModuleList([plain]).to(DEV)
    assert tt.fuse_gated_mlps(plain) == 1 and tt.fuse_gated_mlps(plain) == 0


def test_fused_and_then_checkpointed():
    from types import SimpleNamespace
    transformers = pytest.importorskip("transformers")
    from transformers.models.qwen3.modeling_qwen3 import Qwen3MLP
    from tree_training_b200.hybrid import checkpoint_mlps
    cfg = transformers.Qwen3Config(hidden_size=64, intermediate_size=96, num_hidden_layers=1)
    mlp = Qwen3MLP(cfg).to(DEV)
    x = torch.randn(5, 64, device=DEV, requires_grad=True)
    ps = [x, *mlp.parameters()]
    assert tt.fuse_gated_mlps(torch.nn.ModuleList([mlp])) == 1
    want = torch.autograd.grad(mlp(x).sum(), ps)
    layer = SimpleNamespace(mlp=mlp)
    assert checkpoint_mlps(SimpleNamespace(model=SimpleNamespace(layers=[layer]))) == 1
    got = torch.autograd.grad(mlp(x).sum(), ps)
    assert all(torch.equal(a, b) for a, b in zip(got, want))     # the same kernels, run again
    assert tt.fuse_gated_mlps(torch.nn.ModuleList([mlp])) == 0   # (and the wrapper stays)


@pytest.mark.parametrize("T,H,F", [(208, 4288, 4544), (1024, 2560, 4864), (300, 8192, 4096),
                                   (130, 1001, 2735)])
def test_signs_of_products_near_zero(T, H, F):
    """relu is open where the product is above 0, whatever the sums' own error: a sum in
    64 bits of products of bf16 (exact) errs by H 2^-53 of its terms' magnitudes."""
    x, wg, wu, _ = make(T, H, F, BF, seed=7)
    g = torch.cat([x.double() @ w.double().t() for w in wg.split(1024)], 1)
    size = torch.cat([x.abs().double() @ w.abs().double().t() for w in wg.split(1024)], 1)
    h = tt.gated_linear(x, wg, wu, activation="relu")
    tt.check_device_status()
    u = torch.cat([x.double() @ w.double().t() for w in wu.split(1024)], 1)
    sure = (g.abs() > H * 2.0 ** -53 * size) & (u.abs() > 1e-3) & (g.abs() > 1e-30)
    wrong = sure & ((h != 0) != (g > 0))
    assert int(wrong.sum()) == 0, g[wrong]


def test_rows_of_zeros_and_of_very_different_sizes():
    """Products of exactly 0, and rows in which nearly all are small beside one: as every
    other activation's (no sum is formed again for them, or few are)."""
    x, wg, wu, dh = make(300, 512, 1000, BF, seed=8)
    wg[::3] = 0
    wg[1::64] *= 2.0 ** 20
    x[::7] = 0
    compare(x, wg, wu, dh, "relu")


@pytest.mark.parametrize("T", [1, 2, 3, 4, 7, 8, 13, 16, 17])
@pytest.mark.parametrize("H,F", [(1001, 735), (4096, 520), (256, 9001)])
def test_few_rows_of_fp32(T, H, F):
    compare(*make(T, H, F, F32, seed=T))


@pytest.mark.parametrize("autocast", [BF, F16])
@pytest.mark.parametrize("given", [F32, BF])
def test_hf_modules_under_autocast(given, autocast):
    """Patched modules run in autocast's type: h and its gradients within a few of its
    roundings (five on the way: both factors, the activation, the product, the result)."""
    transformers = pytest.importorskip("transformers")
    from transformers.models.qwen3.modeling_qwen3 import Qwen3MLP
    cfg = transformers.Qwen3Config(hidden_size=128, intermediate_size=264, num_hidden_layers=1)
    torch.manual_seed(0)
    mlp = torch.nn.ModuleList([Qwen3MLP(cfg)]).to(DEV)
    x = torch.randn(2, 37, 128, device=DEV).to(given)
    dy = torch.randn(2, 37, 128, device=DEV).to(autocast)
    got = []
    for fuse in (0, 1):
        assert tt.fuse_gated_mlps(mlp) == 1 if fuse else True
        leaf = x.clone().requires_grad_(True)
        with torch.autocast("cuda", autocast):
            y = mlp[0](leaf)
        assert y.dtype == autocast
        got.append([y, *torch.autograd.grad(y, [leaf, *mlp.parameters()], dy)])
    for a, b in zip(*got):
        assert a.dtype == b.dtype
        assert float((a - b).norm() / b.norm()) < 5 * max(UNIT[autocast], UNIT[b.dtype])
