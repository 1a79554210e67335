"""Causal attention over packed prompts (turbo_prompt_attention) at the ends of its numbers' ranges, against the formula in 64
bits."""
import math

import pytest

torch = pytest.importorskip("torch")
import step_util as S
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


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("lengths,hq,hk", FORMS)
@pytest.mark.parametrize("flip", [1, -1])
def test_a_score_of_minus_infinity_weighs_nothing(lengths, hq, hk, d, dtype, flip):
    """An infinity in a key: -infinity as a score takes the key out, +infinity gives NaN."""
    q, k, v = inputs(lengths, hq, hk, d, dtype, 22)
    q[..., 3] = q[..., 3].abs() + 0.25
    at = 37
    k[at, 0, 3] = -math.inf * flip
    out = call(q, k, v, lengths, dtype, scale=flip * d**-0.5)
    n, g = lengths[0], hq // hk
    seen = S.causal(n, 0)
    seen[:, at] = False
    kk = k[:n].clone()
    kk[at, 0, 3] = 0.0
    want, mean, size = S.softmax_rows(q[:n, :g], kk[:, :1], v[:n, :1], seen, flip * d**-0.5)
    bound = S.prompt_bound(want, mean, size, d**-0.5, d, n, dtype == BF16)
    far = (out[:n, :g].double() - want).abs()
    assert bool((far <= bound).all())
    out = call(q, k, v, lengths, dtype, scale=-flip * d**-0.5)
    assert bool(out[at:n, :g].isnan().all()) and bool(out[:at].isfinite().all()) and bool(out[n:].isfinite().all())
    # nothing but such keys: no weight is left
    k[:n, 0, 3] = -math.inf * flip
    v[at, 0, 7] = math.inf
    assert bool(call(q, k, v, lengths, dtype, scale=flip * d**-0.5)[:n, :g].isnan().all())


@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("lengths,hq,hk", FORMS)
@pytest.mark.parametrize("power", [8, 18, 26])
@pytest.mark.parametrize("strong", ["q", "k"])
def test_strong_channels_of_one_operand(lengths, hq, hk, d, power, strong):
    """FP32: channels of 2^power in queries where keys hold next to nothing (or the other way round), as trained ones do."""
    q, k, v = inputs(lengths, hq, hk, d, F32, 23)
    x, y = (q, k) if strong == "q" else (k, q)
    x[..., 5::29] *= 2.0**power
    y[..., 5::29] *= 2.0**-(power + 8)
    out = call(q, k, v, lengths, F32)
    scale, at = d**-0.5, 0
    for n in lengths[:3]:
        rows = slice(at, at + n)
        at += n
        seen = S.causal(n, 0)
        want, mean, size = S.softmax_rows(q[rows], k[rows], v[rows], seen, scale)
        # Queries and keys keep 2^-22 of each number and 2^-39 of their row's largest (fp16's least step, 2^-24, of numbers
        # whose largest lies at 2^14), and the product of what their first parts leave is left out: three times 2^-22 of
        # sum |q k|, 2^-39 of sum |q| max |k| + max |q| |k|.
        g = hq // hk
        qq, kk = q[rows].double().abs(), k[rows].double().abs().repeat_interleave(g, dim=1)
        cross = torch.einsum("qh,kh->hqk", qq.sum(dim=2), kk.amax(dim=2)) + torch.einsum("qh,kh->hqk", qq.amax(dim=2), kk.sum(dim=2))
        cross = (cross * seen).amax(dim=2).T[..., None]
        score = scale * ((d + 28) * 2.0**-24 * size[..., None] + 2.0**-39 * cross) + 2.0**-21
        bound = mean * (2 * score + (n + 16) * 2.0**-24) * 1.01 + want.abs() * 2.0**-23 + 1e-30
        far = (out[rows].double() - want).abs()
        assert bool((far <= bound).all()), (n, (far / bound).max().item())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("lengths,hq,hk", FORMS)
@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("first,second", [(0, 77), (40, 41), (77, 60)])
def test_columns_that_are_not_finite_by_different_keys(lengths, hq, hk, d, dtype, window, first, second):
    """NaN in one column and an infinity in another, each met by the rows that see it, whichever of both they see."""
    q, k, v = inputs(lengths, hq, hk, d, dtype, 24)
    clean = v.clone()
    n, g = lengths[0], hq // hk
    v[first, 0, 5], v[second, 0, d - 1] = math.nan, math.inf
    out = call(q, k, v, lengths, dtype, window=window)
    seen = S.causal(n, window)
    bad = torch.zeros((n, g, d), dtype=torch.bool, device="cuda")
    bad[seen[:, first], :, 5] = True
    bad[seen[:, second], :, d - 1] = True
    assert torch.equal(~out[:n, :g].isfinite(), bad) and bool(out[n:].isfinite().all()) and bool(out[:n, g:].isfinite().all())
    want, mean, size = S.softmax_rows(q[:n], k[:n], clean[:n], seen, d**-0.5)
    bound = S.prompt_bound(want, mean, size, d**-0.5, d, n, dtype == BF16)
    far = (out[:n].double() - want).abs()
    far[:, :g][bad] = 0.0
    assert bool((far <= bound).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 256, 512])
@pytest.mark.parametrize("lengths,hq,hk", FORMS)
def test_values_near_the_largest_number(lengths, hq, hk, d, dtype):
    """A value that a weight above 1 would take out of FP32 before the sum is divided."""
    q, k, v = inputs(lengths, hq, hk, d, dtype, 25, size=3.0)
    v[20, 0, 7] = 3e38
    check(q, k, v, call(q, k, v, lengths, dtype), lengths, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d,hq,hk", [(128, 8, 2), (256, 4, 2), (512, 4, 1)])
@pytest.mark.parametrize("what", ["k", "v"])
def test_one_bad_token_does_not_hold_the_call(d, hq, hk, dtype, what):
    """NaN in the first token of a long prompt, which every row of its heads sees."""
    q, k, v = inputs([6000], hq, hk, d, dtype, 26)
    out, st = torch.empty_like(q), S.ids([0, 6000])
    inp = T.make_prompt_inputs(1, 6000, dtype=dtype, q=q, k=k, v=v, out=out, q_heads=hq, kv_heads=hk, head_dim=d, starts=st, scale=d**-0.5)

    def ms():
        times = []
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            T.prompt_attention(inp)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    before = ms()
    (k if what == "k" else v)[0, 0, 3] = math.nan
    after = ms()
    print(f"{what} d {d} dtype {dtype}: {before:.3f} ms, with NaN {after:.3f}")
    assert bool(out[:, :hq // hk, 3].isnan().all())
    assert after < 4 * before + 1.0
