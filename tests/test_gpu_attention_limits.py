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
    if dtype == "bf16":  # one running sum over the head: the small difference may be lost, the weights stay finite
        ends = np.concatenate([v[:32], v[128:160]])
        assert np.all(got <= ends.max(0) + bound) and np.all(got >= ends.min(0) - bound)
        return
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) / bound).max())
