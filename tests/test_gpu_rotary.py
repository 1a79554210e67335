"""Norms of the heads with the position rotation in one pass, alone and straight into the cache,
against the formulas in 64 bits (angles in 80).

Tolerance, relative to a pair's size |(a, b)| after the norm: the mean square sums E = 4 or 8 products in
a row and 6 levels of a tree, so its relative error is at most (8 + 6) 2^-24 and half of that after
the root; root, division, eps and the two products add 5 roundings; cosine and sine are off by at most
4 * 2^-24 each (argument, polynomial, last term), together 4 sqrt(2); products and sum of the rotation
add 2: under 21 * 2^-24. BF16 outputs add half a step, 2^-8 of the value."""
import numpy as np
import pytest

import layer_util as L
import turbo_decode_tail as T
from test_gpu_layer_cache import code, ids, same, tensor

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TOL = 21 * 2.0**-24


def freqs(theta, r):
    return [theta ** (-2.0 * i / r) for i in range(r // 2)]


def plain(x, w, normed, positions, inv_freq, pairs, eps=1e-6):
    """(values, the size that the tolerance is relative to)"""
    y = L.norm(x, eps, w) if normed else np.asarray(x, np.float64)
    return L.rotate(y, positions, inv_freq, pairs), L.pair_size(y, 2 * len(inv_freq), pairs)


def close(got, want, size, dtype):
    got = got.float().cpu().numpy().astype(np.float64)
    bound = TOL * size + (2.0**-8 * (np.abs(want) + TOL * size) if dtype == "bf16" else 0.0) + 1e-37
    off = np.abs(got - want)
    assert np.all(off <= bound), float((off / bound).max())


def heads_of(rng, n, heads, dim, dtype):
    x = (rng.standard_normal((n, heads, dim)) * np.exp(rng.uniform(-3, 3, (n, heads, 1)))).astype(np.float32)
    return L.bf16(x) if dtype == "bf16" else x


@pytest.mark.parametrize("dim,rotary,pairs", [(64, 64, False), (64, 16, False), (128, 128, True), (128, 2, True), (256, 256, False),
                                              (256, 64, False), (256, 0, False), (512, 512, True), (512, 128, False)])
@pytest.mark.parametrize("tokens,q_heads,kv_heads", [(1, 16, 8), (3, 5, 1), (67, 12, 4), (130, 9, 9)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_and_rotation(dim, rotary, pairs, tokens, q_heads, kv_heads, dtype):
    rng = np.random.default_rng(dim + rotary + tokens)
    q, k = heads_of(rng, tokens, q_heads, dim, dtype), heads_of(rng, tokens, kv_heads, dim, dtype)
    wq, wk = (L.bf16(rng.uniform(0.5, 1.5, dim).astype(np.float32)) for _ in range(2))
    pos = rng.integers(0, 2**32, tokens, dtype=np.uint64).astype(np.uint32)
    pos[0] = 0 if tokens > 1 else 2**32 - 1
    r = T.Rotary(dim, rotary_dim=rotary, theta=1e6, layout=T.TURBO_ROPE_PAIRS if pairs else T.TURBO_ROPE_HALVES,
                 q_norm=L.bf16_bits(wq), k_norm=L.bf16_bits(wk))
    qt, kt, pt = tensor(q, dtype), tensor(k, dtype), ids(pos)
    qo, ko = torch.full_like(qt, float("nan")), torch.full_like(kt, float("nan"))
    inp = r.make_inputs(tokens, dtype=code(dtype), q=qt, k=kt, q_heads=q_heads, kv_heads=kv_heads, positions=pt, q_out=qo,
                        k_out=ko)
    r.apply(inp)
    f = freqs(1e6, rotary) if rotary else []
    close(qo, *plain(q, wq, True, pos, f, pairs), dtype)
    close(ko, *plain(k, wk, True, pos, f, pairs), dtype)
    # in place, and each alone: the same bits
    q2, k2 = qt.clone(), kt.clone()
    r.apply(r.make_inputs(tokens, dtype=code(dtype), q=q2, q_heads=q_heads, positions=pt, q_out=q2))
    r.apply(r.make_inputs(tokens, dtype=code(dtype), k=k2, kv_heads=kv_heads, positions=pt, k_out=k2))
    assert torch.equal(q2, qo) and torch.equal(k2, ko)


@pytest.mark.parametrize("norms", [0, T.TURBO_NORM_Q, T.TURBO_NORM_K, T.TURBO_NORM_Q | T.TURBO_NORM_K])
def test_each_norm_may_be_off_and_frequencies_may_be_given(norms):
    rng = np.random.default_rng(norms)
    n, dim = 19, 128
    f = rng.uniform(-2, 2, dim // 2)
    f[::3] = 0.0  # these pairs stay as they are
    q, k = heads_of(rng, n, 4, dim, "f32"), heads_of(rng, n, 2, dim, "f32")
    pos = rng.integers(0, 10**6, n).astype(np.uint32)
    r = T.Rotary(dim, inv_freq=f, norms=norms, eps=1e-3)
    qt, kt, pt = tensor(q, "f32"), tensor(k, "f32"), ids(pos)
    qo, ko = torch.empty_like(qt), torch.empty_like(kt)
    r.apply(r.make_inputs(n, q=qt, k=kt, q_heads=4, kv_heads=2, positions=pt, q_out=qo, k_out=ko))
    close(qo, *plain(q, None, norms & 1, pos, f, False, 1e-3), "f32")
    close(ko, *plain(k, None, norms & 2, pos, f, False, 1e-3), "f32")
    if not norms:
        still = np.concatenate([np.arange(0, 64, 3), 64 + np.arange(0, 64, 3)])
        assert torch.equal(qo[..., still], qt[..., still])


def test_rows_of_zeros_and_of_values_that_are_not_finite():
    """A row of zeros stays zeros; NaN or infinity in one head reaches no other."""
    dim, n = 256, 6
    rng = np.random.default_rng(2)
    q = heads_of(rng, n, 3, dim, "f32")
    q[1, 0], q[2, 1, 5], q[3, 2, 200] = 0.0, np.nan, np.inf
    r = T.Rotary(dim)
    qt, pt = tensor(q, "f32"), ids(np.arange(n))
    qo = torch.empty_like(qt)
    r.apply(r.make_inputs(n, q=qt, q_heads=3, positions=pt, q_out=qo))
    out = qo.cpu().numpy()
    assert np.all(out[1, 0] == 0.0) and np.isnan(out[2, 1]).all() and np.isnan(out[3, 2]).any()
    good = np.ones((n, 3), bool)
    good[2, 1] = good[3, 2] = False
    want, size = plain(q, None, True, np.arange(n), freqs(10000.0, dim), False)
    close(qo[torch.from_numpy(good).cuda()], want[good], size[good], "f32")


@pytest.mark.parametrize("dim,rotary,pairs,bits", [(64, 32, False, 8), (128, 128, True, 4), (256, 256, False, 8), (512, 256, False, 4)])
@pytest.mark.parametrize("tokens", [1, 5, 150])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_straight_into_the_cache(dim, rotary, pairs, bits, tokens, dtype):
    """Queries, keys and values as slices of one projection; the cache takes the turned keys and the normed
    values from FP32. What it holds is within half a step of the exact value and its rounding; k_out, asked
    for as well, has the bits of the pass without a cache."""
    rng = np.random.default_rng(dim + tokens)
    hq, hk = 6, 3
    x = heads_of(rng, tokens, hq + 2 * hk, dim, dtype)
    row = tensor(x, dtype)
    wq, wk = (L.bf16(rng.uniform(0.5, 1.5, dim).astype(np.float32)) for _ in range(2))
    pos = rng.integers(0, 10**7, tokens).astype(np.uint32)
    r = T.Rotary(dim, rotary_dim=rotary, theta=5e5, layout=int(pairs), norms=7,
                 q_norm=torch.from_numpy(wq).cuda().bfloat16(), k_norm=torch.from_numpy(wk).cuda().bfloat16())
    pages = tokens // 32 + 2
    cache = T.KvCache(pages, 32, hk, dim, bits=bits)
    slots = np.arange(7, 7 + tokens, dtype=np.uint32)
    if tokens > 4:
        slots[[1, 4]] = L.NO_SLOT
    sl, pt = ids(slots), ids(pos)
    qo = torch.empty((tokens, hq, dim), device="cuda", dtype=row.dtype)
    ko = torch.empty((tokens, hk, dim), device="cuda", dtype=row.dtype)
    q, k, v = row[:, :hq], row[:, hq:hq + hk], row[:, hq + hk:]
    r.apply(r.make_inputs(tokens, dtype=code(dtype), q=q, k=k, v=v, q_heads=hq, kv_heads=hk, positions=pt, q_out=qo, k_out=ko,
                          cache=cache, slots=sl))
    f = freqs(5e5, rotary)
    close(qo, *plain(x[:, :hq], wq, True, pos, f, pairs), dtype)
    k2 = torch.empty_like(ko)
    r.apply(r.make_inputs(tokens, dtype=code(dtype), k=k, kv_heads=hk, positions=pt, k_out=k2))
    assert torch.equal(k2, ko)
    kr, vr = torch.empty((tokens, hk, dim), device="cuda"), torch.empty((tokens, hk, dim), device="cuda")
    cache.read(sl, tokens, kr, vr)
    there = slots != L.NO_SLOT
    assert bool(torch.isnan(kr[torch.from_numpy(~there).cuda()]).all())
    for got, (want, size) in ((kr, plain(x[:, hq:hq + hk], wk, True, pos, f, pairs)), (vr, plain(x[:, hq + hk:], None, True, pos, [], False))):
        got, want, size = got.cpu().numpy()[there].astype(np.float64), want[there], size[there]
        g = want.reshape(*want.shape[:-1], -1, 64)
        # a step is at most range / top, the range reaches down by the bias's rounding (2^-7 of the lowest
        # value at most), both round up by 2^-7
        span = g.max(-1) - g.min(-1) + 2.0**-7 * np.abs(g.min(-1))
        step = np.repeat(span / (2**bits - 1) * (1 + 2.0**-7), 64, axis=-1).reshape(want.shape)
        assert np.all(np.abs(got - want) <= 0.5 * step * (1 + 2.0**-12) + 2 * TOL * np.maximum(size, size.max(-1, keepdims=True)))


def test_refusals():
    r = T.Rotary(64)
    x = torch.zeros((4, 2, 64), device="cuda")
    pt = ids(np.arange(4))
    cache, other = T.KvCache(1, 32, 2, 64), T.KvCache(1, 32, 2, 128)
    ok = dict(q=x, q_heads=2, positions=pt, q_out=x)
    for kw, word in ((dict(), "both NULL"), (dict(ok, q_heads=0), "q_heads"), (dict(ok, q_heads=8193), "q_heads"),
                     (dict(ok, q_out=None), "q_out is NULL"), (dict(ok, positions=None), "positions"),
                     (dict(ok, q=x.data_ptr() + 4, q_out=x.data_ptr() + 4), "aligned"),
                     (dict(k=x, kv_heads=2, positions=pt), "neither k_out nor a cache"),
                     (dict(k=x, kv_heads=2, positions=pt, k_out=x, v=x), "no cache"),
                     (dict(k=x, kv_heads=2, positions=pt, cache=cache, slots=pt), "needs k and v"),
                     (dict(k=x, v=x, kv_heads=2, positions=pt, cache=cache), "slots"),
                     (dict(k=x, v=x, kv_heads=2, positions=pt, cache=other, slots=pt), "another head_dim"),
                     (dict(k=x, v=x, kv_heads=1, positions=pt, cache=cache, slots=pt), "number of heads"),
                     (dict(ok, dtype=3), "dtype")):
        with pytest.raises(T.TurboError, match=word):
            r.apply(r.make_inputs(4, **kw))
    wide = torch.zeros((4, 3, 64), device="cuda")
    inp = r.make_inputs(4, q=wide[:, :2], q_heads=2, positions=pt, q_out=wide[:, :2])
    inp.q_out_stride = 0
    with pytest.raises(T.TurboError, match="another stride"):
        r.apply(inp)
    with pytest.raises(T.TurboError, match="tokens"):
        r.apply(r.make_inputs(-1, **ok))
    r.apply(r.make_inputs(0, **ok))


def test_replayed_in_a_graph():
    rng = np.random.default_rng(9)
    n, dim = 9, 256
    r = T.Rotary(dim)
    cache = T.KvCache(2, 32, 2, dim)
    row = torch.empty((n, 8, dim), device="cuda")
    pt, sl = ids(np.arange(n)), ids(np.arange(n))
    qo, kr, vr = (torch.empty((n, h, dim), device="cuda") for h in (4, 2, 2))
    inp = r.make_inputs(n, q=row[:, :4], k=row[:, 4:6], v=row[:, 6:], q_heads=4, kv_heads=2, positions=pt, q_out=qo, cache=cache,
                        slots=sl)
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        r.apply(inp, stream=st.cuda_stream)
        cache.read(sl, n, kr, vr, stream=st.cuda_stream)
    for i in range(3):
        x = heads_of(rng, n, 8, dim, "f32")
        pos = rng.integers(0, 10**6, n).astype(np.uint32)
        row.copy_(tensor(x, "f32")), pt.copy_(ids(pos)), sl.copy_(ids(rng.permutation(64)[:n]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        close(qo, *plain(x[:, :4], None, True, pos, freqs(10000.0, dim), False), "f32")
        same(vr, L.stored(x[:, 6:], 8).astype(np.float32))


def test_more_workgroups_than_a_grid_holds_are_refused():
    # 2^28 tokens, 1,024 heads of 512: 2^32 workgroups of 32 tokens and 2 heads for the values alone
    x = torch.zeros(64, device="cuda")
    cache = T.KvCache(1, 32, 1024, 512)
    with pytest.raises(T.TurboError, match="too large"):
        cache.write(x, x, ids(np.arange(1)), 1 << 28)
    r = T.Rotary(512)
    with pytest.raises(T.TurboError, match="too large"):
        r.apply(r.make_inputs(1 << 28, q=x, q_heads=8192, positions=ids(np.arange(1)), q_out=x))
