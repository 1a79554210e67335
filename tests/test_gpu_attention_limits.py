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
