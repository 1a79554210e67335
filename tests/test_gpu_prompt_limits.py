"""Causal attention over packed prompts (turbo_prompt_attention) at the ends of its numbers' ranges, against the formula in 64
bits."""
import pytest

torch = pytest.importorskip("torch")
import turbo_decode_tail as T
from test_gpu_prompt_attention import BF16, F32, call, check, inputs

pytestmark = pytest.mark.gpu
# lengths and heads of the forms: few tiles and many
FORMS = [([150, 50], 4, 2), ([700] * 8, 16, 8)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("lengths,hq,hk", FORMS)
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-39, -3e-39])
def test_the_smallest_scales(lengths, hq, hk, d, dtype, scale):
    """Products of 2^126 with a scale that is 0, or below the normal numbers: all keys weigh the same, or nearly."""
    q, k, v = inputs(lengths, hq, hk, d, dtype, 21)
    q[:] = 2.0**62
    k[:] = torch.where(k[..., :1] > 0, 2.0**64, -(2.0**64)) / d
    check(q, k, v, call(q, k, v, lengths, dtype, scale=scale), lengths, dtype, scale=scale)
