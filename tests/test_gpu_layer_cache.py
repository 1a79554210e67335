"""The quantised key/value cache: what is read back equals, bit for bit, the plain quantiser's values
(the format is defined by fp32 operations), over head sizes, widths, page sizes, types, strides and
orders of slots; other slots keep what they held; values that are not finite; caches past 4 GiB."""
import numpy as np
import pytest

import layer_util as L
import turbo_decode_tail as T

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def tensor(x, dtype):
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda()
    return t.bfloat16() if dtype == "bf16" else t


def code(dtype):
    return T.TURBO_HIDDEN_BF16 if dtype == "bf16" else T.TURBO_HIDDEN_F32


def ids(a):
    return torch.from_numpy(np.asarray(a, np.uint32).view(np.int32).copy()).cuda()


def data(rng, tokens, heads, dim, dtype):
    x = (rng.standard_normal((2, tokens, heads, dim)) + rng.standard_normal((2, 1, heads, dim))).astype(np.float32)
    return L.bf16(x) if dtype == "bf16" else x


def expect(x, bits, dtype):
    y = L.stored(x, bits).astype(np.float32)  # code * scale + bias is one rounding of an exact product and sum
    return L.bf16(y) if dtype == "bf16" else y


def same(got, want):
    got = got.float().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)])


ORDERS = {
    "run": lambda rng, n, cap: np.arange(5, 5 + n),                       # from inside a block on
    "scattered": lambda rng, n, cap: rng.permutation(cap)[:n],
    "backwards": lambda rng, n, cap: np.arange(cap - 1, cap - 1 - n, -1),
    "blocks": lambda rng, n, cap: (np.arange(n) // 32 * 32)[::-1] // 32 * 32 + np.arange(n) % 32 if n % 32 == 0 else np.arange(n),
}


@pytest.mark.parametrize("order", list(ORDERS))
@pytest.mark.parametrize("dim,heads,page,tokens", [(64, 1, 32, 1), (64, 9, 64, 70), (128, 3, 256, 64), (256, 8, 64, 33),
                                                   (512, 2, 128, 130)])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_reads_back_what_the_format_holds(dim, heads, page, tokens, bits, dtype, order):
    rng = np.random.default_rng(dim + tokens)
    pages = -(-(tokens + 40) // page) + 1
    cap = pages * page
    cache = T.KvCache(pages, page, heads, dim, bits=bits)
    first = data(rng, cap, heads, dim, dtype)
    every = ids(np.arange(cap))
    k, v = tensor(first[0], dtype), tensor(first[1], dtype)
    cache.write(k, v, every, cap, dtype=code(dtype))
    slots = ORDERS[order](rng, tokens, cap)
    second = data(rng, tokens, heads, dim, dtype)
    first[:, slots] = second
    k2, v2 = tensor(second[0], dtype), tensor(second[1], dtype)
    cache.write(k2, v2, ids(slots), tokens, dtype=code(dtype))
    for out in ("f32", "bf16"):
        ko, vo = (torch.empty((cap, heads, dim), device="cuda", dtype=torch.bfloat16 if out == "bf16" else torch.float32)
                  for _ in range(2))
        cache.read(every, cap, ko, vo, dtype=code(out))
        same(ko, expect(first[0], bits, out))
        same(vo, expect(first[1], bits, out))
    # one at a time, in the order of the slots
    ko = torch.empty((tokens, heads, dim), device="cuda")
    vo = torch.empty_like(ko)
    cache.read(ids(slots), tokens, ko, None)
    cache.read(ids(slots), tokens, None, vo)
    same(ko, expect(second[0], bits, "f32"))
    same(vo, expect(second[1], bits, "f32"))


@pytest.mark.parametrize("bits", [4, 8])
def test_slots_past_the_cache_are_skipped_and_read_as_nan(bits):
    rng = np.random.default_rng(3)
    cache = T.KvCache(2, 32, 2, 128, bits=bits)
    x = data(rng, 64, 2, 128, "f32")
    every = ids(np.arange(64))
    k, v = tensor(x[0], "f32"), tensor(x[1], "f32")
    cache.write(k, v, every, 64)
    slots = np.array([64, L.NO_SLOT, 7, 65, 2**31, 8], np.uint32)
    y = data(rng, 6, 2, 128, "f32")
    k2, v2, sl = tensor(y[0], "f32"), tensor(y[1], "f32"), ids(slots)
    cache.write(k2, v2, sl, 6)
    x[:, [7, 8]] = y[:, [2, 5]]
    ko, vo = torch.empty((64, 2, 128), device="cuda"), torch.empty((64, 2, 128), device="cuda")
    cache.read(every, 64, ko, vo)
    same(ko, expect(x[0], bits, "f32"))
    same(vo, expect(x[1], bits, "f32"))
    ko, vo = torch.zeros((6, 2, 128), device="cuda"), torch.zeros((6, 2, 128), device="cuda")
    cache.read(sl, 6, ko, vo)
    want = np.stack([expect(y[i], bits, "f32") for i in range(2)])
    want[:, [0, 1, 3, 4]] = np.nan
    same(ko, want[0])
    same(vo, want[1])


@pytest.mark.parametrize("bits", [4, 8])
def test_values_at_the_ends_of_the_type(bits):
    """Groups that are constant, zero, tiny, as wide as the type, or hold a value that is not finite."""
    x = np.zeros((1, 9, 1, 64), np.float32)
    rng = np.random.default_rng(4)
    x[0, 1] = -3.75
    x[0, 2] = rng.standard_normal(64) * 1e-40
    x[0, 3] = rng.uniform(-1e31, 1e31, 64)  # 2^103 is the first that is refused
    x[0, 3, 0, :2] = np.nextafter(np.float32(2.0**103), np.float32(0)), -np.nextafter(np.float32(2.0**103), np.float32(0))
    x[0, 4] = rng.standard_normal(64)
    x[0, 4, 0, 9] = np.nan
    x[0, 5] = rng.standard_normal(64)
    x[0, 5, 0, 63] = -np.inf
    x[0, 6] = 1000.0 + rng.uniform(0, 1e-3, 64)
    x[0, 7] = rng.standard_normal(64)
    x[0, 8, 0, 1] = 2.0**103
    cache = T.KvCache(1, 32, 1, 64, bits=bits)
    t, sl = tensor(x[0], "f32"), ids(np.arange(9))
    cache.write(t, t, sl, 9)
    ko, vo = torch.empty((9, 1, 64), device="cuda"), torch.empty((9, 1, 64), device="cuda")
    cache.read(sl, 9, ko, vo)
    want = L.stored(x[0], bits).astype(np.float32)
    assert np.isnan(want[[4, 5, 8]]).all() and np.isfinite(want[[0, 1, 2, 3, 6, 7]]).all()
    same(ko, want)
    same(vo, want)


def test_heads_as_slices_of_a_wider_row_and_a_wider_output():
    rng = np.random.default_rng(5)
    n, heads, dim = 45, 4, 128
    x = data(rng, n, heads, dim, "bf16")
    row = torch.zeros((n, 3 * heads, dim), device="cuda", dtype=torch.bfloat16)
    row[:, heads:2 * heads] = tensor(x[0], "bf16")
    row[:, 2 * heads:] = tensor(x[1], "bf16")
    cache = T.KvCache(2, 64, heads, dim)
    sl = ids(np.arange(3, 3 + n))
    cache.write(row[:, heads:2 * heads], row[:, 2 * heads:], sl, n, dtype=T.TURBO_HIDDEN_BF16)
    out = torch.full((n, 3 * heads, dim), 7.0, device="cuda")
    cache.read(sl, n, out[:, :heads], out[:, 2 * heads:])
    same(out[:, :heads], expect(x[0], 8, "f32"))
    same(out[:, 2 * heads:], expect(x[1], 8, "f32"))
    assert bool((out[:, heads:2 * heads] == 7.0).all())


def test_a_cache_past_four_gibibytes():
    heads, dim, page = 8, 512, 256
    pages = 2200  # 563,200 tokens of 8,704 bytes
    cache = T.KvCache(pages, page, heads, dim)
    assert pages * page * 2 * heads * (dim + dim // 16) > 4.5 * 2**30
    rng = np.random.default_rng(6)
    slots = np.concatenate([[0, 1, 2, 3, 250000, 493447], np.arange(pages * page - 40, pages * page)])
    x = data(rng, len(slots), heads, dim, "bf16")
    k, v, sl = tensor(x[0], "bf16"), tensor(x[1], "bf16"), ids(slots)
    cache.write(k, v, sl, len(slots), dtype=T.TURBO_HIDDEN_BF16)
    ko, vo = torch.empty(x.shape[1:], device="cuda"), torch.empty(x.shape[1:], device="cuda")
    cache.read(sl, len(slots), ko, vo)
    same(ko, expect(x[0], 8, "f32"))
    same(vo, expect(x[1], 8, "f32"))


def test_refusals():
    cache = T.KvCache(1, 32, 2, 64)
    x = torch.zeros((4, 2, 64), device="cuda")
    sl = ids(np.arange(4))
    for call, word in ((lambda: cache.write(x, x, sl, -1), "tokens"), (lambda: cache.write(x, x, sl, 2**28 + 1), "tokens"),
                       (lambda: cache.write(None, x, sl, 4), "k is NULL"), (lambda: cache.write(x, None, sl, 4), "v is NULL"),
                       (lambda: cache.write(x, x, None, 4), "slots"), (lambda: cache.write(x, x, sl, 4, dtype=2), "dtype"),
                       (lambda: cache.write(x.data_ptr() + 4, x, sl, 4), "aligned"),
                       (lambda: cache.read(sl, 4, None, None), "both NULL"), (lambda: cache.read(sl, 4, x, x), "same buffer")):
        with pytest.raises(T.TurboError, match=word):
            call()
    lib = T.load()
    for stride, word in ((100, "smaller"), (130, "multiple of 16 bytes"), (2**33, "above")):
        assert lib.turbo_kv_cache_write(cache.h, x.data_ptr(), stride, x.data_ptr(), 0, 0, sl.data_ptr(), 4, None) == 0
        assert word in T.last_error()
    with pytest.raises(ValueError, match="contiguous"):
        cache.write(x.transpose(0, 1).contiguous().transpose(0, 1), x, sl, 4)
    cache.write(None, None, None, 0)  # nothing to do


def test_on_another_stream_and_in_a_graph():
    """Write and read captured once and replayed with other inputs, with eager work between the replays."""
    rng = np.random.default_rng(7)
    n, heads, dim = 37, 3, 256
    cache = T.KvCache(3, 32, heads, dim, bits=4)
    k, v = torch.empty((n, heads, dim), device="cuda"), torch.empty((n, heads, dim), device="cuda")
    sl = ids(np.arange(n))
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        cache.write(k, v, sl, n, stream=st.cuda_stream)
        cache.read(sl, n, ko, vo, stream=st.cuda_stream)
    for i in range(4):
        x = data(rng, n, heads, dim, "f32")
        at = rng.permutation(96)[:n]
        k.copy_(tensor(x[0], "f32")), v.copy_(tensor(x[1], "f32")), sl.copy_(ids(at))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        same(ko, expect(x[0], 4, "f32"))
        same(vo, expect(x[1], 4, "f32"))
    with torch.cuda.stream(st):
        x = data(rng, n, heads, dim, "f32")
        k, v = tensor(x[0], "f32"), tensor(x[1], "f32")
        cache.write(k, v, sl, n, stream=st.cuda_stream)
        cache.read(sl, n, ko, vo, stream=st.cuda_stream)
    st.synchronize()
    same(ko, expect(x[0], 4, "f32"))
