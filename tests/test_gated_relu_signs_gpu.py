"""relu's sign where a product nearly cancels: features whose weights take back over the
second half of x what they give over the first, but for one small term.  Tensor-core sums
miss such a term by far and the sign with it; the epilogue forms them again in 64 bits.

Bounds.  A sum formed again is off by its rounding to fp32 and 2^-12 of a term of 2^-34;
u = x wu errs by at most H 2^-23 of its terms' magnitudes: where |u| is at least 2^-5 of
their root, under 2^-9 of itself for these sizes; and h rounds once more (2^-8).
"""
import pytest
import torch

import tree_training_b200 as tt

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


def small_of(pairs):
    # (beside products of 2^-8 a step of the tensor cores does not hold the second at all)
    return 2.0 ** -34 if pairs else 2.0 ** -24


def planted(T, H, F, features, up=1.0, pairs=False, seed=0):
    """x, wg, wu [.., H + 8]: g of ``features`` is +-small_of(pairs).  pairs: what cancels
    stands side by side (within one step of the tensor cores), else half of H apart."""
    small = small_of(pairs)
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x, wg, wu = r(T, H + 8), r(F, H + 8) * H ** -0.5, r(F, H + 8) * H ** -0.5 * up
    x[:, H:], wg[:, H:], wu[:, H:] = 0, 0, 0
    half = r(len(features), H // 2) * H ** -0.5 / 4
    if pairs:
        x[:, 1:H:2] = x[:, 0:H:2]
        both = torch.stack([half, -half], 2).flatten(1)
    else:
        x[:, H // 2:H] = x[:, :H // 2]
        both = torch.cat([half, -half], 1)
    wg[features, :H] = both
    # (pairs: in the last whole step of 16, beside larger terms)
    at = H - 16 if pairs else H
    if pairs:
        x[:, at:at + 2], wg[features, at:at + 2] = 0, 0
    x[:, at] = 1
    wg[features, at] = small * (2.0 * torch.randint(0, 2, (len(features),), generator=g,
                                                    device=DEV) - 1)
    return x.to(BF), wg.to(BF), wu.to(BF)


def check(x, wg, wu, features, up, pairs=False):
    h = tt.gated_linear(x, wg, wu, activation="relu")
    tt.check_device_status()
    by = lambda w: torch.cat([x.double() @ v.double().t() for v in w.split(512)], 1)
    g, u = by(wg), by(wu)
    assert ((g[:, features].abs() / small_of(pairs) - 1).abs() < 2.0 ** -12).all()
    size = torch.cat([x.abs().double() @ w.abs().double().t() for w in wg.split(512)], 1)
    seen = u.abs() > 2.0 ** -5 * up
    wrong = seen & (g.abs() > x.shape[1] * 2.0 ** -53 * size) & ((h != 0) != (g > 0))
    assert int(wrong.sum()) == 0, (int(wrong.sum()), wrong.nonzero()[:8].tolist())
    want = (g.clamp(min=0) * u)[:, features]
    off = (h[:, features].double() - want).abs()[seen[:, features]]
    assert (off <= (2.0 ** -8 + 2.0 ** -9) * want.abs()[seen[:, features]]).all()


@pytest.mark.parametrize("up", [2.0 ** -10, 1.0, 2.0 ** 16])
@pytest.mark.parametrize("T,H,F", [(64, 4096, 1024), (100, 1024, 688), (600, 4096, 3840),
                                   (1024, 2560, 4864)])
def test_whatever_the_other_factors_size(T, H, F, up):
    features = list(range(5, F, 16))
    check(*planted(T, H, F, features, up), features, up)


@pytest.mark.parametrize("T,H,F,features", [
    (64, 4096, 1025, [1024]), (600, 4096, 3841, [3840]), (2048, 2560, 2561, [2560]),
    (2048, 2560, 2564, [2561, 2563]), (2048, 2560, 2567, [2560, 2566]), (16, 4096, 1, [0]),
    (40, 4096, 3, [1]), (40, 4096, 5, [0, 4]), (300, 4096, 9, [8]), (1000, 2560, 2049, [2048])])
def test_the_last_few_features(T, H, F, features):
    check(*planted(T, H, F, features), features, 1.0)


@pytest.mark.parametrize("T,H,F,features", [
    (600, 4096, 3840, range(5, 3840, 32)), (1024, 2560, 4864, range(0, 4864, 31)),
    (2048, 1024, 2048, range(7, 2048, 64)), (64, 4096, 1024, range(3, 1024, 16)),
    (64, 4096, 1025, [1024]), (16, 1024, 3, [0, 2])])
def test_terms_that_are_cut_off_altogether(T, H, F, features):
    features = list(features)
    check(*planted(T, H, F, features, pairs=True), features, 1.0, pairs=True)


def test_terms_within_the_sums_error():
    features = list(range(5, 4864, 16))
    check(*planted(1024, 2560, 4864, features), features, 1.0)


def test_features_without_weights():
    features = list(range(3, 2048, 64))
    x, wg, wu = planted(700, 1024, 2048, features, pairs=True)
    wg[9::64] = 0
    wg[500:600] = 0
    features = [f for f in features if not 500 <= f < 600]
    check(x, wg, wu, features, 1.0, pairs=True)
