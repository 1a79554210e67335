"""Causal attention over packed prompts (turbo_prompt_attention) against the formula in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")
import step_util as S
import turbo_decode_tail as T

pytestmark = pytest.mark.gpu
F32, BF16 = T.TURBO_HIDDEN_F32, T.TURBO_HIDDEN_BF16
TYPES = {F32: torch.float32, BF16: torch.bfloat16}


def inputs(lengths, hq, hk, d, dtype, seed, spare=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = sum(lengths) + spare
    rand = lambda h: torch.randn((n, h, d), generator=g, device="cuda")  # noqa: E731
    return [x.to(TYPES[dtype]) for x in (rand(hq) * size, rand(hk), rand(hk))]


def starts_of(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def call(q, k, v, lengths, dtype, *, window=0, scale=None, out=None, starts=None, stream=None):
    d = q.shape[2]
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda") if out is None else out
    st = S.ids(starts_of(lengths) if starts is None else starts)
    inp = T.make_prompt_inputs(len(lengths), q.shape[0], dtype=dtype, q=q, k=k, v=v, out=out, q_heads=q.shape[1], kv_heads=k.shape[1],
                               head_dim=d, starts=st, window=window, scale=d**-0.5 if scale is None else scale)
    T.prompt_attention(inp, stream)
    torch.cuda.synchronize()
    return out


def check(q, k, v, out, lengths, dtype, window=0, scale=None):
    d = q.shape[2]
    scale = d**-0.5 if scale is None else scale
    at = 0
    for n in lengths:
        rows = slice(at, at + n)
        at += n
        if n == 0:
            continue
        want, mean, size = S.softmax_rows(q[rows], k[rows], v[rows], S.causal(n, window), scale)
        far = (out[rows].double() - want).abs()
        bound = S.prompt_bound(want, mean, size, scale, d, n, dtype == BF16)
        assert bool((far <= bound).all()), (n, (far / bound).max().item())


LENGTHS = [[1], [2, 1], [31, 32, 33], [0, 5, 0, 64, 1, 0], [130, 3, 257], [700]]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d,hq,hk", [(64, 4, 4), (64, 6, 2), (128, 8, 1), (128, 3, 3), (256, 4, 2), (256, 5, 1), (512, 8, 2), (512, 1, 1)])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_ragged(d, hq, hk, lengths, dtype):
    q, k, v = inputs(lengths, hq, hk, d, dtype, 1, spare=3, size=2.0)
    out = call(q, k, v, lengths, dtype)
    check(q, k, v, out, lengths, dtype)
    assert bool((out[sum(lengths):] == 7.0).all())  # rows of nobody


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 64, 100, 1000])
def test_windows(d, window, dtype):
    lengths = [1, 40, 333]
    q, k, v = inputs(lengths, 6, 2, d, dtype, 2)
    check(q, k, v, call(q, k, v, lengths, dtype, window=window), lengths, dtype, window)


@pytest.mark.parametrize("d,hq,hk", [(64, 32, 16), (128, 24, 8), (256, 16, 8), (512, 16, 8)])
@pytest.mark.parametrize("window", [0, 77])
def test_many_rows(d, hq, hk, window):
    """As many tiles as the card has compute units, and more, of unequal length."""
    lengths = [5, 900, 64, 1, 0, 1300, 333, 128, 129, 512]
    q, k, v = inputs(lengths, hq, hk, d, BF16, 3)
    check(q, k, v, call(q, k, v, lengths, BF16, window=window), lengths, BF16, window)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d,n", [(64, 65), (256, 200), (512, 129), (64, 5000)])
def test_many_sequences(d, n, dtype):
    lengths = [(7 * i) % 23 + (150 if i % 97 == 3 else 0) for i in range(n)]
    q, k, v = inputs(lengths, 4, 2, d, dtype, 4, spare=2)
    out = call(q, k, v, lengths, dtype)
    last = slice(sum(lengths[:-100]), None)  # the sequences at both ends, all of up to 200
    if n > 1000:
        check(q, k, v, out, lengths[:100], dtype)
        check(q[last], k[last], v[last], out[last], lengths[-100:], dtype)
    else:
        check(q, k, v, out, lengths, dtype)
    assert bool((out[sum(lengths):] == 7.0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d,n", [(64, 2500), (128, 1800), (256, 1100), (256, 2300), (512, 700)])
def test_one_long_sequence(d, n, dtype):
    q, k, v = inputs([n], 8, 4, d, dtype, 14)
    check(q, k, v, call(q, k, v, [n], dtype), [n], dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0])
def test_scales(d, scale, dtype):
    lengths = [150, 50]
    q, k, v = inputs(lengths, 4, 2, d, dtype, 5, size=0.3)
    check(q, k, v, call(q, k, v, lengths, dtype, scale=scale), lengths, dtype, scale=scale)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads", [(4, 2), (48, 24)])
def test_slices_of_one_projection(heads, dtype):
    hq, hk = heads
    lengths, d = [300, 41, 700], 128
    q, k, v = inputs(lengths, hq, hk, d, dtype, 6)
    rows = torch.cat([q, k, v, q], dim=1)
    qs, ks, vs, os = rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:hq + 2 * hk], rows[:, hq + 2 * hk:]
    before = rows[:, :hq + 2 * hk].clone()
    call(qs, ks, vs, lengths, dtype, out=os)
    check(q, k, v, os, lengths, dtype)
    assert torch.equal(rows[:, :hq + 2 * hk], before)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d,hq,hk,copies", [(64, 2, 1, 1), (128, 2, 1, 1), (256, 2, 1, 1), (512, 2, 1, 1), (64, 32, 16, 6),
                                            (128, 24, 8, 6), (256, 16, 8, 6), (512, 16, 8, 3)])
@pytest.mark.parametrize("what", ["v", "k", "both"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_what_is_hidden_has_no_part(d, hq, hk, copies, what, bad, dtype):
    """An infinity or NaN in a key or value is met by the rows that see it, and by no other, in its own head alone."""
    n, at, window = 200, 101, 40
    lengths = [n] * copies
    q, k, v = inputs(lengths, hq, hk, d, dtype, 7)
    clean = [x.clone() for x in (q, k, v)]
    for c in range(copies):
        if what != "k":
            v[c * n + at, 0, 5] = bad
        if what != "v":
            k[c * n + at, 0, 3] = bad
    out = call(q, k, v, lengths, dtype, window=window)
    sees = torch.zeros(sum(lengths), dtype=torch.bool, device="cuda")
    for c in range(copies):
        sees[c * n + at:c * n + at + window] = True
    g = hq // hk
    hit = out[sees][:, :g]
    if what == "v":  # its column; an infinity may be one or NaN
        assert bool((~hit[..., 5].isfinite()).all()) and bool(hit[..., 6:].isfinite().all())
        if math.isnan(bad):
            assert bool(hit[..., 5].isnan().all())
    elif not math.isnan(bad):  # a score of -infinity has a weight of 0, one of +infinity gives NaN
        assert bool((~hit.isfinite()).any())
    else:
        assert bool(hit.isnan().all())
    # all other rows and heads are as without it
    out[sees, :g] = 0
    assert bool(out.isfinite().all())
    for c in range(copies):
        rows = slice(c * n, (c + 1) * n)
        want, mean, size = S.softmax_rows(*(x[rows] for x in clean), S.causal(n, window), d**-0.5)
        bound = S.prompt_bound(want, mean, size, d**-0.5, d, n, dtype == BF16)
        hits = torch.zeros_like(want, dtype=torch.bool)
        hits[at:at + window, :g] = True
        assert bool((((out[rows].double() - want).abs() <= bound) | hits).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_query_that_is_not_finite(dtype):
    q, k, v = inputs([90], 4, 2, 128, dtype, 8)
    q[50, 1, 9] = math.nan
    q[60, 2, 0] = math.inf
    out = call(q, k, v, [90], dtype)
    assert bool(out[50, 1].isnan().all()) and bool(out[60, 2].isnan().all())
    out[50, 1] = out[60, 2] = 0
    assert bool(out.isfinite().all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 256])
def test_large_scores(d, dtype):
    """Scores of thousands: the maximum moves often, and one key takes nearly all of the weight."""
    lengths = [500]
    q, k, v = inputs(lengths, 2, 2, d, dtype, 9, size=300.0)
    k *= torch.linspace(0.1, 3.0, 500, device="cuda")[:, None, None].to(k.dtype)
    check(q, k, v, call(q, k, v, lengths, dtype), lengths, dtype)


def test_offsets_past_32_bits():
    n, stride = 70000, 32768
    wide = torch.empty(n * stride, dtype=torch.bfloat16, device="cuda")  # 4.6 GB
    k = wide.as_strided((n, 1, 64), (stride, 64, 1))
    g = torch.Generator(device="cuda").manual_seed(10)
    k.copy_(torch.randn((n, 1, 64), generator=g, device="cuda"))
    q, v = (torch.randn((n, 1, 64), generator=g, device="cuda").bfloat16() for _ in range(2))
    out = call(q, k, v, [n], BF16, window=96)
    lo = n - 600
    rows = torch.arange(lo, n, device="cuda")
    seen = (torch.arange(lo - 100, n, device="cuda")[None] <= rows[:, None]) & (torch.arange(lo - 100, n, device="cuda")[None] > rows[:, None] - 96)
    want, mean, size = S.softmax_rows(q[lo:], k[lo - 100:], v[lo - 100:], seen, 0.125)
    bound = S.prompt_bound(want, mean, size, 0.125, 64, 96, True)
    assert bool(((out[lo:].double() - want).abs() <= bound).all())


def test_starts_past_the_rows_and_gaps():
    """Sequences end at the buffers' end, and rows in front of the first one are left alone."""
    q, k, v = inputs([100], 2, 1, 64, BF16, 11)
    out = call(q, k, v, [0, 0], BF16, starts=[10, 60, 250])
    assert bool((out[:10] == 7.0).all())
    for lo, hi in ((10, 60), (60, 100)):
        check(q[lo:hi], k[lo:hi], v[lo:hi], out[lo:hi], [hi - lo], BF16)
    out = call(q, k, v, [0, 0], BF16, starts=[100, 100, 100])
    assert bool((out == 7.0).all())


@pytest.mark.parametrize("lengths", [[40, 7], [800, 300, 900]], ids=str)
def test_graph_and_stream(lengths):
    q, k, v = inputs(lengths, 16, 8, 256, BF16, 12)
    want = call(q, k, v, lengths, BF16)
    assert torch.equal(want, call(q, k, v, lengths, BF16))
    out, st = torch.zeros_like(want), S.ids(starts_of(lengths))
    inp = T.make_prompt_inputs(len(lengths), q.shape[0], dtype=BF16, q=q, k=k, v=v, out=out, q_heads=16, kv_heads=8, head_dim=256,
                               starts=st, scale=256**-0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        T.prompt_attention(inp, side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        T.prompt_attention(inp, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    # other lengths in the same buffers
    q2, k2, v2 = inputs(lengths, 16, 8, 256, BF16, 13)
    for x, y in ((q, q2), (k, k2), (v, v2)):
        x.copy_(y)
    graph.replay()
    torch.cuda.synchronize()
    check(q, k, v, out, lengths, BF16)
