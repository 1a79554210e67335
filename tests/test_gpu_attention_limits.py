"""Attention at the ends of its ranges: keys and queries so small that their products leave FP32, scores so
large that a unit in their last place is more than a weight's range, values that dwarf all others where a
row does not see them or gives them no weight, and infinities and NaN."""
import numpy as np
import pytest

import layer_util as L
from test_gpu_attention import Setup, check, inputs, queries
from test_gpu_layer_cache import tensor

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def attend(s, q, q_heads, kv_len, dtype, **kw):
    qt = tensor(q, dtype)
    out = torch.empty_like(qt)
    s.cache.attend(inputs(s, qt, out, q_heads, kv_len, dtype=dtype, **kw))
    torch.cuda.synchronize()
    return out


# keys' size, queries' size: a record's largest key times a query's largest value is below FP32's range
@pytest.mark.parametrize("k_size,q_size", [(0.0, 1e-6), (0.0, 1e-30), (1e-30, 1e-11), (1e-37, 1e-3)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scores_below_the_types_range_are_even_weights(dtype, k_size, q_size):
    rng = np.random.default_rng(1)
    s = Setup(rng, 2, 256, 8, 32, 45, [40, 3], k_size=k_size)
    q = queries(rng, 2, 4, 256, dtype) * np.float32(q_size)
    q = L.bf16(q) if dtype == "bf16" else q
    out = attend(s, q, 4, [85, 48], dtype)
    check(s, q, out, [85, 48], 1, 0, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_scale_that_overflows_against_zero_keys(dtype):
    """Scores are exactly 0 however large the factor before them is. The mean of values with weights of 11 bits, BF16
    rounded by half a step."""
    rng = np.random.default_rng(2)
    s = Setup(rng, 1, 64, 8, 32, 0, [40], k_size=0.0)
    q = queries(rng, 1, 2, 64, dtype) * np.float32(2.0**120)
    want, size = (x.mean(axis=0) for x in s.stored(s.v))
    got = attend(s, q, 2, [40], dtype, scale=1e30)[0].float().cpu().numpy()
    assert np.all(np.abs(got - want) <= 2.0**-8 * np.abs(want) + 2.0**-10 * size), got


@pytest.mark.parametrize("size", [2.0**18, 2.0**25, 2.0**26, 2.0**27, 2.0**28, 2.0**30, 2.0**34])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scores_whose_last_place_is_more_than_one(dtype, size):
    """Scores of `size` (log2 units), in a later record of the same wave higher by 8, or by a unit in the
    last place where that is more. Keys are constant in each group of 64 values, so every score is exact."""
    rng = np.random.default_rng(3)
    s = Setup(rng, 1, 128, 8, 32, 0, [256])
    step = max(8.0, size * 2.0**-23)
    s.k[:] = 0.0
    s.k[:32, 0, :64] = s.k[128:160, 0, :64] = size / 2**16
    s.k[128:160, 0, 64:] = step / 2**8
    s.write(np.arange(256))
    q = np.zeros((1, 2, 128), np.float32)
    q[..., :64], q[..., 64:] = 2.0**10, 2.0**2
    scale = 0.69314718  # its product with log2(e) rounds to 1 in FP32
    assert np.float32(np.float64(np.float32(scale)) * 1.4426950408889634) == np.float32(1)
    out = attend(s, q, 2, [256], dtype, scale=scale, max_kv_len=1)  # one workgroup: wave 0 has records 0 and 4
    v = s.stored(s.v)[0][:, 0]
    later = 2.0 ** min(step, 1000.0)
    want = (v[:32].sum(0) + later * v[128:160].sum(0)) / (32 * (1 + later))
    got = out[0].float().cpu().numpy().astype(np.float64)
    # weights of 11 bits (FP32: 22) and 32 equal ones; BF16 rounds the result by half a step
    w = (2.0**-12 if dtype == "bf16" else 2.0**-22) + 80 * 2.0**-24
    size_v = s.stored(s.v)[1][:, 0]
    bound = w * np.maximum(size_v[:32].mean(0), size_v[128:160].mean(0))
    bound += 2.0**-8 * (np.abs(want) + bound) if dtype == "bf16" else 0.0
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) / bound).max())


def seen(s, q, b, q_len, kv_len, window, scale, dtype):
    """Sequence b's outputs and a bound that knows of a row only the tokens that it sees. With a value as
    (code - middle) * scale + centre, K the sum of both addends' sizes and S the larger of 128 scale and
    |centre| over the head:
      a score is off by scale * sum |q| K (2^-22 + 80 * 2^-24) (queries keep 22 bits; 64 products, the groups
      and the centres add in FP32) and (2 |s| log2(e) + 2) 2^-23 of the weight (factor, difference, exponential);
      a weight is rounded to 2^-12 (BF16) or 2^-22 of itself, or, where that is coarser, a weighted value to 2^-32
      of the row's largest weighted S, known to a factor of 4;
      40 + keys / 32 roundings of the sums."""
    t = s.tokens(b)[:kv_len]
    mid = 128.0 if s.bits == 8 else 8.0

    def parts(x):
        c, sc, bi = (a.astype(np.float64) for a in L.quantise(x[t], s.bits))
        centre = bi + mid * sc
        size = np.maximum(128 * sc, np.abs(centre)).max(-1)
        add = np.abs(c - mid) * sc[..., None] + np.abs(centre)[..., None]
        return (c * sc[..., None] + bi[..., None]).reshape(x[t].shape), add.reshape(x[t].shape), size

    (k, kk, _), (v, vv, vs) = parts(s.k), parts(s.v)
    q = q.astype(np.float64)
    g = q.shape[1] // s.heads
    out, bound = np.zeros_like(q), np.zeros_like(q)
    for i in range(q_len):
        p = kv_len - q_len + i
        lo, hi = (max(0, p - window + 1) if window else 0), p + 1
        if hi <= lo:
            continue
        for h in range(q.shape[1]):
            at = (slice(lo, hi), h // g)
            sc = k[at] @ q[i, h] * scale
            w = np.exp(sc - sc.max())
            w /= w.sum()
            out[i, h] = w @ v[at]
            e = abs(scale) * (kk[at] @ np.abs(q[i, h])) * (2.0**-22 + 80 * 2.0**-24) + (2 * np.abs(sc) * 1.4427 + 2) * 2.0**-23
            rel = (2.0**-22 if dtype == "f32" else 2.0**-12) + (40 + (hi - lo) / 32) * 2.0**-24
            bound[i, h] = (2 * e.max() + rel) * (w @ vv[at]) + (hi - lo) * 2.0**-30 * (w * vs[at]).max()
    if dtype == "bf16":
        bound += 2.0**-8 * (np.abs(out) + bound)
    return out, bound + 1e-37


def hold(s, q, out, kv_len, q_len, window, dtype, scale):
    got = out.float().cpu().numpy().astype(np.float64)
    for b, n in enumerate(kv_len):
        rows = slice(b * q_len, (b + 1) * q_len)
        want, bound = seen(s, q[rows], b, q_len, n, window, scale, dtype)
        off = np.abs(got[rows] - want)
        assert np.all(off <= bound), (b, n, float((off / bound).max()))


@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4), (256, 8), (512, 8)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_scores_of_nearly_equal_keys(dtype, dim, bits):
    """Pairs of keys whose large scores are close: their weights are as exact as the scores, to which a code
    enters as it is."""
    rng = np.random.default_rng(6)
    s = Setup(rng, 1, dim, bits, 32, 64, [64])
    near = rng.standard_normal((1, 1, dim)).astype(np.float32)
    s.k = L.bf16((near * (1 + 0.01 * rng.standard_normal(s.k.shape))).astype(np.float32))
    s.write(np.arange(128))
    q = L.bf16(40.0 * queries(rng, 1, 16, dim, "f32"))
    out = attend(s, q, 16, [128], dtype)
    hold(s, q, out, [128], 1, 0, dtype, dim**-0.5)


OUTLIERS = {  # prefix, own tokens, q_len, window, the token that dwarfs all others, group, max_kv_len
    "later_queries_see_it": (0, [200], 64, 0, 170, 1, None),
    "left_behind_by_the_window": (0, [900], 24, 400, 484, 2, 1),
    "in_the_window_of_the_first_query": (0, [900], 24, 400, 477, 3, 1),
    "in_a_prefix_part_of_the_batch_reaches": (300, [10, 0, 0, 40], 1, 0, 130, 4, None),
    "first_of_all_and_weightless": (0, [600], 3, 0, 0, 2, 1),
    "weightless_in_a_prefix": (500, [1, 90, 7], 2, 0, 41, 2, None),
}


@pytest.mark.parametrize("case", list(OUTLIERS))
@pytest.mark.parametrize("ratio", [2.0**14, 2.0**20, 2.0**30, 2.0**70])
@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4), (256, 8), (512, 4)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_value_that_a_row_does_not_weight_costs_it_nothing(dtype, dim, bits, ratio, case):
    prefix, own, q_len, window, at, group, most = OUTLIERS[case]
    rng = np.random.default_rng(dim + len(case))
    s = Setup(rng, 1, dim, bits, 32, prefix, own)
    kv_len = [prefix + n for n in own] if "part" not in case else [310, 120, 60, 340]
    base = rng.standard_normal(dim).astype(np.float32)
    rows = len(kv_len) * q_len
    q = 0.5 * queries(rng, rows, group, dim, "f32") + base
    q = L.bf16(q)
    scale = dim**-0.5
    s.v[at] *= np.float32(ratio)
    if "weightless" in case:
        s.k[at] = -20.0 * base * 16.0 / np.sqrt(dim)
    s.write(np.array([at]))
    out = attend(s, q, group, kv_len, dtype, q_len=q_len, window=window, max_kv_len=most)
    hold(s, q, out, kv_len, q_len, window, dtype, scale)


@pytest.mark.parametrize("dim,bits", [(64, 4), (128, 8), (256, 4), (512, 8)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_small_groups_beside_large_ones(dtype, dim, bits):
    """Groups of 64 whose keys and values differ by up to 2^8 inside a token, tokens by 2^20."""
    rng = np.random.default_rng(5)
    s = Setup(rng, 2, dim, bits, 64, 100, [90, 33])
    by = 2.0 ** rng.uniform(-4, 4, (1, 1, dim // 64)).repeat(64, axis=2) * 2.0 ** rng.uniform(-10, 10, (223, 1, 1))
    s.v = (s.v * by).astype(np.float32)
    s.write(np.arange(223))
    q = L.bf16(queries(rng, 2, 6, dim, "f32"))
    out = attend(s, q, 6, [190, 133], dtype)
    hold(s, q, out, [190, 133], 1, 0, dtype, dim**-0.5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_nan_with_a_weight_of_zero_is_nan(dtype):
    """Wherever the token lies: in the record of the row's largest scores or far from them."""
    rng = np.random.default_rng(8)
    for own in (64, 600):
        s = Setup(rng, 1, 64, 8, 32, 0, [own])
        base = rng.standard_normal(64).astype(np.float32)
        base *= np.float32(20.0 / np.linalg.norm(base))
        s.k[:] = L.bf16(base)
        s.k[32:64] = L.bf16(-base)
        s.v[40] = np.nan
        s.write(np.arange(own))
        q = L.bf16(np.tile(base, (1, 2, 1)).astype(np.float32))
        out = attend(s, q, 2, [own], dtype, scale=1.0)
        assert torch.isnan(out).all(), own


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_query_with_an_infinity_gives_nan(dtype, sign):
    """Also where every key makes its score -inf, and in no other row."""
    rng = np.random.default_rng(7)
    s = Setup(rng, 1, 64, 8, 32, 0, [70])
    s.k[:, 0, 5] = -np.abs(s.k[:, 0, 5]) - 2.0
    s.write(np.arange(70))
    q = queries(rng, 3, 2, 64, dtype)
    q[1, 1, 5] = sign * np.inf
    out = attend(s, q, 2, [70], dtype, q_len=3).float().cpu().numpy()
    assert np.isnan(out[1, 1]).all()
    out[1, 1] = 0.0
    assert np.isfinite(out).all()


@pytest.mark.parametrize("scale,q_size", [(3e38, 2.0**-126), (-3e38, 2.0**-126), (2.0**-126, 2.0**126), (2.0**-140, 2.0**127)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scales_at_the_ends_of_the_type(dtype, scale, q_size):
    """scale * log2(e) may be above FP32's largest number, or below its smallest normal one."""
    rng = np.random.default_rng(9)
    s = Setup(rng, 1, 64, 8, 32, 0, [70], k_size=2.0**10 if scale == 2.0**-140 else 1.0)
    q = (np.clip(queries(rng, 1, 2, 64, "f32"), -1.9, 1.9) * np.float32(q_size)).astype(np.float32)
    q = L.bf16(q) if dtype == "bf16" else q
    out = attend(s, q, 2, [70], dtype, scale=scale)
    want, bound = seen(s, q, 0, 1, 70, 0, float(np.float32(scale)), dtype)
    assert np.all(np.abs(out.float().cpu().numpy() - want) <= bound)
