"""Attention over the quantised cache against the formula in 64 bits on the values that the cache reads
back, over head sizes, ratios, widths, types, page sizes, prefixes, ragged lengths, several queries to a
sequence, windows and padded sequences. Slots that no token was written to hold NaN in every test.

Tolerance. With K = |code * scale| + |bias| of a key's value (the two enter as separate sums), a score
is off by at most scale * sum |q| K * (2^-22 + 80 * 2^-24): FP32 queries keep 22 bits, 64 products and the
groups add in FP32 (BF16 queries are exact, the same bound holds); the factor and the exponential add
(2 |s| + 2) 2^-23 to a weight's relative error. A weight is rounded to 2^-22 (FP32) or 2^-12 (BF16) of
itself for the product with the values, which adds at most 32 + keys / 32 roundings, and the join and
division 8 more. For BF16 queries a key or value is rounded to fp16: 2^-12 K, or half of fp16's smallest
step, which is 2^-24 of the largest K of its 32 tokens (4 bits: 2^-20; scale and bias as well, once more
each). So |off| <= (2 e + w + (40 + keys / 32) 2^-24) sum p (|code * scale| + |bias|), and BF16 rounds
the result by 2^-8 of it. Those are worst cases; the errors are independent, so the 2-norm must stay far
below: under 4e-6 (FP32: 8 roundings' worth of a 64-term sum at the scores' size here) and 2.5e-3 (BF16:
half a step is 2^-8 at most, 2^-9 / sqrt(3) * 1.4 on average over a binade)."""
import numpy as np
import pytest

import layer_util as L
import turbo_decode_tail as T
from test_gpu_layer_cache import code, ids, tensor

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


class Setup:
    """A cache whose unwritten slots are NaN, `batch` sequences with own[b] own tokens after a prefix, pages
    shuffled, and the values that the cache holds of every token, in order."""

    def __init__(self, rng, heads, dim, bits, page, prefix, own, spare=1, k_size=1.0, v_size=1.0, extra_pages=0):
        self.heads, self.dim, self.bits, self.page, self.prefix, self.own = heads, dim, bits, page, prefix, own
        need_p = -(-prefix // page)
        need = [-(-n // page) for n in own]
        self.width = max([1] + need) + spare
        pages = need_p + sum(need) + 1
        self.cache = T.KvCache(pages + extra_pages, page, heads, dim, bits=bits)
        order = rng.permutation(pages) + extra_pages
        bad = np.full((pages * page, heads, dim), np.nan, np.float32)
        every = np.arange(extra_pages * page, (extra_pages + pages) * page)
        t = tensor(bad, "f32")
        self.cache.write(t, t, ids(every), len(every))
        self.prefix_pages = order[:need_p].astype(np.uint32)
        self.pages = np.full((len(own), self.width), order[-1], np.uint32)  # ends point at the page of NaN
        at = need_p
        slots = [self.prefix_pages[np.arange(prefix) // page].astype(np.int64) * page + np.arange(prefix) % page]
        for b, n in enumerate(own):
            self.pages[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
            j = np.arange(n)
            slots.append(self.pages[b, j // page].astype(np.int64) * page + j % page)
        self.slots = np.concatenate(slots)
        n = len(self.slots)
        k = (rng.standard_normal((n, heads, dim)) * 0.7 + rng.standard_normal((heads, dim)) * 0.7) * k_size
        v = rng.standard_normal((n, heads, dim)) * v_size
        self.k, self.v = L.bf16(k.astype(np.float32)), L.bf16(v.astype(np.float32))
        self.write(np.arange(n))

    def write(self, which):
        kt, vt = tensor(self.k[which], "f32"), tensor(self.v[which], "f32")
        self.cache.write(kt, vt, ids(self.slots[which]), len(which))
        torch.cuda.synchronize()

    def tokens(self, b):
        first = self.prefix + sum(self.own[:b])
        return np.concatenate([np.arange(self.prefix), np.arange(first, first + self.own[b])])

    def stored(self, x):
        """(values, |code * scale| + |bias|)"""
        c, s, b = L.quantise(x, self.bits)
        a = c.astype(np.float64) * s[..., None]
        return (a + b[..., None]).reshape(x.shape), (np.abs(a) + np.abs(b)[..., None]).reshape(x.shape)


def inputs(s, q, out, q_heads, kv_len, *, dtype, q_len=1, window=0, scale=None, max_kv_len=None, batch=None, workspace=True):
    st = s.__dict__.setdefault("device", {})
    st["kv_len"], st["pages"] = ids(kv_len), ids(s.pages)
    st["prefix"] = ids(s.prefix_pages) if s.prefix else None
    inp = s.cache.make_attention_inputs(
        len(kv_len) if batch is None else batch, dtype=code(dtype), q=q, out=out, q_heads=q_heads, q_len=q_len, kv_len=st["kv_len"],
        max_kv_len=max(kv_len) if max_kv_len is None else max_kv_len, pages=st["pages"], prefix_len=s.prefix,
        prefix_pages=st["prefix"], window=window, scale=s.dim**-0.5 if scale is None else scale)
    if workspace:
        st["ws"] = torch.full((max(1, s.cache.attention_workspace(inp)),), 255, dtype=torch.uint8, device="cuda")  # NaN as floats
        inp.workspace, inp.workspace_bytes = st["ws"].data_ptr(), st["ws"].numel()
    return inp


def expect(s, q, b, q_len, kv_len, window, scale, dtype):
    """Sequence b's outputs and their bound. kv_len may end before the tokens that there are."""
    t = s.tokens(b)[:kv_len]
    (k, kk), (v, vv) = s.stored(s.k[t]), s.stored(s.v[t])
    q = q.astype(np.float64)
    g = q.shape[1] // s.heads
    out, bound = np.zeros_like(q), np.zeros_like(q)
    least = 2.0**-24 if s.bits == 8 else 2.0**-20
    for i in range(q_len):
        p = kv_len - q_len + i
        lo, hi = (max(0, p - window + 1) if window else 0), p + 1
        if hi <= lo:
            continue
        for h in range(q.shape[1]):
            sc = k[lo:hi, h // g] @ q[i, h] * scale
            w = np.exp(sc - sc.max())
            w /= w.sum()
            out[i, h] = w @ v[lo:hi, h // g]
            ka, va = kk[lo:hi, h // g], vv[lo:hi, h // g]
            e = scale * (ka @ np.abs(q[i, h])) * (2.0**-22 + 80 * 2.0**-24) + (2 * np.abs(sc) * 1.4427 + 2) * 2.0**-23
            rel = (2.0**-22 if dtype == "f32" else 2.0**-12) + (40 + (hi - lo) / 32) * 2.0**-24
            if dtype == "bf16":
                e = e + scale * (ka @ np.abs(q[i, h]) * 2.0**-11 + np.nanmax(ka) * np.abs(q[i, h]).sum() * least)
                rel += 2.0**-11
            bound[i, h] = (2 * e.max() + rel) * (w @ va) + (np.nanmax(va) * least if dtype == "bf16" else 0.0)
    if dtype == "bf16":
        bound += 2.0**-8 * (np.abs(out) + bound)
    return out, bound + 1e-37


def check(s, q, out, kv_len, q_len, window, dtype, scale=None, norm=True):
    scale = s.dim**-0.5 if scale is None else scale
    got = out.float().cpu().numpy().astype(np.float64)
    offs = wants = 0.0
    for b, n in enumerate(kv_len):
        rows = slice(b * q_len, (b + 1) * q_len)
        want, bound = expect(s, q[rows], b, q_len, n, window, scale, dtype)
        off = np.abs(got[rows] - want)
        assert np.all(off <= bound), (b, n, float((off / bound).max()))
        offs, wants = offs + float((off**2).sum()), wants + float((want**2).sum())
    if norm and wants:
        assert (offs / wants)**0.5 < (4e-6 if dtype == "f32" else 2.5e-3), (offs / wants)**0.5


def queries(rng, rows, heads, dim, dtype):
    q = (rng.standard_normal((rows, heads, dim)) * 1.5).astype(np.float32)
    return L.bf16(q) if dtype == "bf16" else q


def run(s, rng, q_heads, kv_len, *, dtype, q_len=1, window=0, **kw):
    q = queries(rng, len(kv_len) * q_len, q_heads, s.dim, dtype)
    qt = tensor(q, dtype)
    out = torch.full((qt.shape[0] + 2,) + qt.shape[1:], 5.0, device="cuda", dtype=qt.dtype)
    inp = inputs(s, qt, out, q_heads, kv_len, dtype=dtype, q_len=q_len, window=window, **kw)
    s.cache.attend(inp)
    torch.cuda.synchronize()
    assert bool((out[-2:] == 5.0).all())  # what lies behind the last sequence stays
    return q, out[:-2]


CASES = {  # prefix, own tokens, q_len, window
    "one_token": (0, [1], 1, 0),
    "one_sequence": (0, [777], 1, 0),
    "lengths": (0, [1, 31, 32, 33, 64, 100, 0, 257], 1, 0),
    "prefix_only": (300, [0, 0], 1, 0),
    "prefix": (1000, [1, 40, 0, 333, 65], 1, 0),
    "short_prefix": (7, [1, 2, 300], 1, 0),
    "drafts": (515, [5, 37, 90], 5, 0),
    "chunk": (70, [95], 90, 0),
    "window": (600, [3, 70, 410], 4, 100),
    "narrow": (64, [1, 129], 2, 1),
    "long": (3000, [1500, 2], 1, 0),
}


@pytest.mark.parametrize("case", list(CASES))
@pytest.mark.parametrize("dim,heads,group,page", [(64, 2, 3, 32), (128, 3, 8, 64), (256, 2, 2, 128), (512, 1, 5, 256), (256, 1, 16, 32)])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_against_the_formula(dim, heads, group, page, bits, dtype, case):
    prefix, own, q_len, window = CASES[case]
    rng = np.random.default_rng(dim + len(case))
    s = Setup(rng, heads, dim, bits, page, prefix, own)
    kv_len = [prefix + n if n or case in ("prefix_only", "prefix") else 0 for n in own]
    q, out = run(s, rng, heads * group, kv_len, dtype=dtype, q_len=q_len, window=window)
    check(s, q, out, kv_len, q_len, window, dtype)


MANY = {  # more than 32 rows over the same keys: prefix, own tokens, q_len, window
    "batch": (333, [1, 40, 0, 77, 5] * 8, 1, 0),
    "drafts": (100, [17, 60, 33] * 3, 17, 0),
    "chunk": (0, [333], 300, 0),
    "chunks": (64, [100, 0, 71], 71, 0),
    "window": (500, [3, 90, 300] * 5, 3, 90),
    "narrow": (40, [130], 130, 1),
    "early": (0, [40], 70, 0),
}


@pytest.mark.parametrize("case", list(MANY))
@pytest.mark.parametrize("dim,heads,group,page", [(64, 2, 3, 32), (128, 1, 8, 64), (256, 2, 2, 128), (512, 1, 5, 256)])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_rows_over_the_same_keys(dim, heads, group, page, bits, dtype, case):
    prefix, own, q_len, window = MANY[case]
    rng = np.random.default_rng(dim + len(case))
    s = Setup(rng, heads, dim, bits, page, prefix, own)
    kv_len = [prefix + n if n else 0 for n in own]
    q, out = run(s, rng, heads * group, kv_len, dtype=dtype, q_len=q_len, window=window)
    check(s, q, out, kv_len, q_len, window, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_queries_before_the_first_token_and_sequences_inside_the_prefix(dtype):
    """More queries than tokens: those at negative positions give zeros. A sequence that has not reached the
    prefix's end sees its part of it. max_kv_len below the lengths changes nothing but the split."""
    rng = np.random.default_rng(1)
    s = Setup(rng, 2, 128, 8, 32, 200, [30, 0, 0, 0])
    kv_len = [230, 150, 3, 0]
    for most in (None, 1):
        q, out = run(s, rng, 4, kv_len, dtype=dtype, q_len=6, max_kv_len=most)
        check(s, q, out, kv_len, 6, 0, dtype)
        assert bool((out[12:15] == 0).all()) and bool((out[18:] == 0).all()) and bool((out[15:18] != 0).any())


def test_queries_past_their_pages_and_pages_past_the_cache_give_nan():
    """... and reach no other row."""
    rng = np.random.default_rng(2)
    s = Setup(rng, 2, 64, 8, 32, 100, [20, 20, 20, 70], spare=0)  # three pages to a sequence
    s.pages[1, 0] = 10**6
    kv_len = [120, 120, 100 + 97, 170]
    q, out = run(s, rng, 4, kv_len, dtype="f32", q_len=2)
    good = torch.isfinite(out).all(dim=2).all(dim=1).cpu().numpy()
    nan = torch.isnan(out).all(dim=2).all(dim=1).cpu().numpy()
    assert good.tolist() == [True, True, False, False, False, False, True, True]
    # query 0 of sequence 2 is at the table's last place: it sees slots that hold NaN; query 1 is past it
    assert nan.tolist() == [False, False, True, True, True, True, False, False]
    for b in (0, 3):
        want, bound = expect(s, q[2 * b:2 * b + 2], b, 2, kv_len[b], 0, s.dim**-0.5, "f32")
        assert np.all(np.abs(out[2 * b:2 * b + 2].cpu().numpy() - want) <= bound)
    s.prefix_pages[1] = 2**32 - 1
    q, out = run(s, rng, 4, [120, 30, 0, 170], dtype="f32")
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all() and (out[2] == 0).all() and torch.isnan(out[3]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(dtype):
    rng = np.random.default_rng(3)
    s = Setup(rng, 2, 128, 8, 32, 64, [90, 90])
    s.v[64 + 50, 1, 70] = np.inf   # sequence 0's own token 50, head 1, second group
    s.k[64 + 90 + 10, 0, 3] = np.nan  # sequence 1's own token 10, head 0
    s.write(np.array([64 + 50, 64 + 90 + 10]))
    q = queries(rng, 80, 4, 128, dtype)
    q[79, 3, 5] = np.nan
    qt = tensor(q, dtype)
    out = torch.empty_like(qt)
    s.cache.attend(inputs(s, qt, out, 4, [64 + 60, 64 + 40], dtype=dtype, q_len=40))
    got = out.float().cpu().numpy()
    nan = np.isnan(got)
    want = np.zeros_like(nan)
    want[30:40, 2:, 64:] = True   # queries at own positions 50 .. 59 of sequence 0, heads 2 and 3, that group
    want[50:80, :2] = True        # queries at own positions 10 .. 39 of sequence 1, heads 0 and 1
    want[79, 3] = True
    assert np.array_equal(nan, want)
    for b, n in ((0, 124), (1, 104)):
        w, bound = expect(s, np.nan_to_num(q[b * 40:b * 40 + 40]), b, 40, n, 0, 128**-0.5, dtype)
        fine = ~want[b * 40:b * 40 + 40]
        assert np.all(np.abs(got[b * 40:b * 40 + 40][fine] - w[fine]) <= bound[fine])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_values_and_queries_of_any_size(bits, dtype):
    """Values whose size changes from token to token over 60 powers of ten, the largest last, first and in
    between; queries of 1e-30 and 1e30 against keys that bring the scores back."""
    rng = np.random.default_rng(4)
    s = Setup(rng, 1, 256, bits, 64, 96, [64, 100], k_size=1.0)
    for size in (10.0 ** np.linspace(-30, 30, 260), 10.0 ** np.linspace(30, -30, 260), 10.0 ** rng.uniform(-30, 30, 260), np.full(260, 1e-38)):
        s.v = (rng.standard_normal(s.v.shape) * size[:, None, None]).astype(np.float32)
        s.write(np.arange(260))
        q, out = run(s, rng, 2, [160, 196], dtype=dtype)
        check(s, q, out, [160, 196], 1, 0, dtype, norm=False)
    s = Setup(rng, 1, 256, bits, 64, 96, [64, 100], k_size=1e-30)
    q, out = run(s, rng, 2, [160, 196], dtype=dtype, scale=1e30 / 16)
    check(s, q, out, [160, 196], 1, 0, dtype, scale=1e30 / 16)
    for size in (1e-30, 1e30):
        s = Setup(rng, 1, 256, bits, 64, 96, [64, 100])
        q = queries(rng, 2, 2, 256, dtype) * np.float32(size)
        q = L.bf16(q) if dtype == "bf16" else q
        qt = tensor(q, dtype)
        out = torch.empty_like(qt)
        s.cache.attend(inputs(s, qt, out, 2, [160, 196], dtype=dtype, scale=1 / 16 / size))
        check(s, q, out, [160, 196], 1, 0, dtype, scale=1 / 16 / size)


@pytest.mark.parametrize("size", [1e-35, 1e-20, 1.0, 1e20, 1e36])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sizes_that_many_rows_share(size, dtype):
    """Keys and values of any size, also growing and shrinking from record to record (by 2^40 in all; inside a
    record a value of less than 2^-13 of the largest has fewer than 11 bits), 60 rows."""
    rng = np.random.default_rng(13)
    s = Setup(rng, 2, 128, 8, 64, 150, [100, 40, 1], k_size=size)
    for by in (np.zeros(291), np.linspace(-20, 20, 291), np.linspace(20, -20, 291)):
        s.v = (rng.standard_normal(s.v.shape) * (size if size < 1e30 else 1e30) * 2.0**by[:, None, None]).astype(np.float32)
        s.write(np.arange(291))
        q, out = run(s, rng, 20 * 2, [250, 190, 151], dtype=dtype, scale=128**-0.5 / size)
        if size > 2.0**103:  # the cache refuses such keys: they are NaN
            assert bool(torch.isnan(out).all())
            continue
        check(s, q, out, [250, 190, 151], 1, 0, dtype, scale=128**-0.5 / size, norm=not by.any())


def test_sharp_and_flat_weights():
    """scale 0 is the mean of the values; a large scale picks one token (or shares it between equal keys)."""
    rng = np.random.default_rng(5)
    s = Setup(rng, 1, 128, 8, 32, 40, [50])
    q, out = run(s, rng, 3, [90], dtype="f32", scale=0.0)
    want = s.stored(s.v[s.tokens(0)])[0].mean(axis=0)
    assert np.all(np.abs(out[0].cpu().numpy() - want) < 1e-5)
    s.k[:] = s.k[0]
    s.v[:] = s.v[7]
    s.write(np.arange(90))
    q, out = run(s, rng, 3, [90], dtype="f32", scale=50.0)
    assert np.all(np.abs(out[0].cpu().numpy() - s.stored(s.v[:1])[0][0]) < 1e-5)
    s.v = rng.standard_normal(s.v.shape).astype(np.float32)
    s.k[33] *= 3.0
    s.write(np.arange(90))
    q = s.stored(s.k[33:34])[0].repeat(3, axis=1).astype(np.float32)
    qt = tensor(q, "f32")
    out = torch.empty_like(qt)
    s.cache.attend(inputs(s, qt, out, 3, [90], dtype="f32", scale=10.0))
    assert np.all(np.abs(out[0].cpu().numpy() - s.stored(s.v[33:34])[0][0]) < 1e-5)


def test_a_sequence_without_a_table_and_an_empty_call():
    rng = np.random.default_rng(6)
    s = Setup(rng, 2, 64, 8, 32, 50, [0])
    q = tensor(queries(rng, 3, 4, 64, "f32"), "f32")
    out = torch.full_like(q, 5.0)
    lens, pre = ids([50, 20, 51]), ids(s.prefix_pages)
    inp = s.cache.make_attention_inputs(3, q=q, out=out, q_heads=4, kv_len=lens, max_kv_len=50, prefix_len=50, prefix_pages=pre, scale=0.125)
    ws = torch.empty(max(1, s.cache.attention_workspace(inp)), dtype=torch.uint8, device="cuda")
    inp.workspace, inp.workspace_bytes = ws.data_ptr(), ws.numel()
    s.cache.attend(inp)
    for b, n in enumerate((50, 20)):
        want, bound = expect(s, q[b:b + 1].cpu().numpy(), 0, 1, n, 0, 0.125, "f32")
        assert np.all(np.abs(out[b].cpu().numpy() - want[0]) <= bound[0])
    assert torch.isnan(out[2]).all()  # one token past the prefix and no page for it
    none = s.cache.make_attention_inputs(2, q=q, out=out, q_heads=4, kv_len=ids([0, 1]), max_kv_len=0, scale=1.0)
    s.cache.attend(none)
    assert (out[0] == 0).all() and torch.isnan(out[1]).all()
    none.batch = 0
    s.cache.attend(none)


def test_strided_queries_and_outputs():
    rng = np.random.default_rng(7)
    s = Setup(rng, 2, 128, 4, 64, 130, [70, 9, 200])
    kv_len = [200, 139, 330]
    q = queries(rng, 6, 4, 128, "bf16")
    wide = torch.zeros((6, 10, 128), device="cuda", dtype=torch.bfloat16)
    wide[:, 2:6] = tensor(q, "bf16")
    out = torch.full((6, 7, 128), 3.0, device="cuda", dtype=torch.bfloat16)
    s.cache.attend(inputs(s, wide[:, 2:6], out[:, 1:5], 4, kv_len, dtype="bf16", q_len=2))
    check(s, q, out[:, 1:5], kv_len, 2, 0, "bf16")
    assert bool((out[:, 0] == 3.0).all()) and bool((out[:, 5:] == 3.0).all())


def test_pages_past_four_gibibytes():
    """The pages of a long cache that lie more than 4 GiB from its start."""
    rng = np.random.default_rng(8)
    s = Setup(rng, 8, 512, 8, 256, 300, [200, 31], extra_pages=2100)  # 4.7e9 bytes before the first page used
    q, out = run(s, rng, 8, [500, 331], dtype="bf16")
    check(s, q, out, [500, 331], 1, 0, "bf16")


def test_the_same_call_gives_the_same_bits():
    rng = np.random.default_rng(9)
    s = Setup(rng, 4, 128, 8, 64, 3000, [5, 900, 333, 64] * 6)
    q = tensor(queries(rng, 24, 16, 128, "bf16"), "bf16")
    outs = [torch.empty_like(q) for _ in range(3)]
    for out in outs:
        s.cache.attend(inputs(s, q, out, 16, [3000 + n for n in s.own], dtype="bf16"))
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_two_graphs_with_a_workspace_each_on_two_streams():
    """Captured once, replayed side by side with other queries and lengths, eager work between the replays."""
    rng = np.random.default_rng(10)
    s = Setup(rng, 2, 128, 8, 32, 700, [500, 500, 500])
    graphs = []
    for i in range(2):
        st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        q = torch.zeros((3, 8, 128), device="cuda")
        out = torch.empty_like(q)
        inp = inputs(s, q, out, 8, [1200] * 3, dtype="f32")
        hold = dict(s.device)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=st):
            s.cache.attend(inp, stream=st.cuda_stream)
        graphs.append((st, graph, q, out, hold))
    for i in range(4):
        made = []
        for j, (st, graph, q, out, hold) in enumerate(graphs):
            x = queries(rng, 3, 8, 128, "f32")
            lens = [0 if i == 2 and j == 1 else 701 + 17 * i, 900 + 100 * j, 1200 - 300 * i]
            q.copy_(tensor(x, "f32")), hold["kv_len"].copy_(ids(lens))
            made.append((x, lens))
        torch.cuda.synchronize()
        for st, graph, *_ in graphs:
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for (x, lens), (st, graph, q, out, hold) in zip(made, graphs):
            check(s, x, out, lens, 1, 0, "f32")


def test_refusals():
    rng = np.random.default_rng(11)
    s = Setup(rng, 2, 64, 8, 32, 400, [40])
    q = torch.zeros((1, 4, 64), device="cuda")
    out = torch.zeros_like(q)

    def refuse(word, **kw):
        inp = inputs(s, q, out, 4, [440], dtype="f32")
        for k, v in kw.items():
            setattr(inp, k, v)
        with pytest.raises(T.TurboError, match=word):
            s.cache.attend(inp)

    refuse("batch", batch=-1), refuse("q_len", q_len=0), refuse("q_heads", q_heads=3), refuse("q_heads", q_heads=0)
    refuse("dtype", dtype=2), refuse("scale", scale=float("nan")), refuse("scale", scale=float("inf"))
    refuse("q is NULL", q=None), refuse("out is NULL", out=None), refuse("out is q", out=q.data_ptr())
    refuse("aligned", q=q.data_ptr() + 4), refuse("q_stride", q_stride=100), refuse("out_stride", out_stride=258)
    refuse("kv_len", kv_len=None), refuse("prefix_pages", prefix_pages=None), refuse("pages is NULL", pages=None)
    refuse("2\\^31", prefix_len=2**31), refuse("2\\^31", page_stride=2**26)
    refuse("too large", batch=2**20, q_len=2**20)
    refuse("workspace is NULL", workspace=None), refuse("workspace holds", workspace_bytes=16)
    inp = inputs(s, q, out, 4, [440], dtype="f32")
    inp.workspace += 4
    with pytest.raises(T.TurboError, match="workspace must be"):
        s.cache.attend(inp)


@pytest.mark.parametrize("bits", [4, 8])
def test_projections_to_attention_to_projection(bits):
    """The operators as a layer's decode step runs them: one grouped product gives q, k and v, one call norms,
    turns and stores them, one attends over a shared prefix, one more product projects back; several steps,
    each token attending to those before. Against the same steps in 64 bits with the cache's own rounding."""
    rng = np.random.default_rng(12)
    dim, hq, hk, hidden, prefix, steps = 64, 4, 2, 256, 45, 6

    def matrix(rows, cols):
        w = rng.integers(0, 256, (rows, cols // 2), dtype=np.uint8)
        sc = L.bf16(np.abs(rng.standard_normal((rows, cols // 64)) * 0.02).astype(np.float32) + np.float32(0.005))
        bi = L.bf16((-8 * sc).astype(np.float32))
        m = T.Int4Matrix(rows, cols)
        m.load_weights(w, L.bf16_bits(sc), L.bf16_bits(bi))
        codes = np.stack((w & 15, w >> 4), axis=-1).reshape(rows, -1, 64).astype(np.float64)
        return m, (codes * sc[..., None].astype(np.float64) + bi[..., None].astype(np.float64)).reshape(rows, cols)

    (mq, wq), (mk, wk), (mv, wv), (mo, wo) = (matrix(hq * dim, hidden), matrix(hk * dim, hidden), matrix(hk * dim, hidden),
                                              matrix(hidden, hq * dim))
    s = Setup(rng, hk, dim, bits, 32, prefix, [0])
    s.pages[:] = s.pages[0, 0]  # the page of NaN becomes the sequence's own
    rot = T.Rotary(dim, theta=1e4)
    inv = [1e4 ** (-2.0 * i / dim) for i in range(dim // 2)]
    x = torch.empty(hidden, device="cuda")
    q, k, v = (torch.empty((1, h, dim), device="cuda") for h in (hq, hk, hk))
    att, y = torch.empty_like(q), torch.empty(hidden, device="cuda")
    pos, slot = ids([0]), ids([0])
    inp_r = rot.make_inputs(1, q=q, k=k, v=v, q_heads=hq, kv_heads=hk, positions=pos, q_out=q, cache=s.cache, slots=slot)
    inp_a = inputs(s, q, att, hq, [0], dtype="f32", max_kv_len=prefix + steps)
    keys, values = list(s.stored(s.k)[0]), list(s.stored(s.v)[0])
    for i in range(steps):
        xs = rng.standard_normal(hidden).astype(np.float32)
        x.copy_(torch.from_numpy(xs)), pos.copy_(ids([prefix + i])), slot.copy_(ids([int(s.pages[0, 0]) * 32 + i]))
        s.device["kv_len"].copy_(ids([prefix + i + 1]))
        T.matvec_grouped([mq, mk, mv], [x, x, x], [q, k, v])
        rot.apply(inp_r)
        s.cache.attend(inp_a)
        T.matvec_grouped([mo], [att], [y])
        torch.cuda.synchronize()
        at = np.array([prefix + i])
        q64 = L.rotate(L.norm((wq @ xs).reshape(1, hq, dim), 1e-6), at, inv, False)
        k64 = L.rotate(L.norm((wk @ xs).reshape(1, hk, dim), 1e-6), at, inv, False)
        v64 = (wv @ xs).reshape(1, hk, dim)
        # the cache's own content of the new token: within a step of the exact one, then taken as it is
        kr, vr = torch.empty((1, hk, dim), device="cuda"), torch.empty((1, hk, dim), device="cuda")
        s.cache.read(slot, 1, kr, vr)
        for got, want in ((kr, k64), (vr, v64)):
            got = got.cpu().numpy().astype(np.float64)
            span = want.max(-1, keepdims=True) - want.min(-1, keepdims=True) + 2.0**-7 * np.abs(want).max(-1, keepdims=True)
            assert np.all(np.abs(got - want) <= 0.51 * span * (1 + 2.0**-7) / (2**bits - 1) + 1e-4 * np.abs(want).max())
        keys.append(kr.cpu().numpy()[0].astype(np.float64)), values.append(vr.cpu().numpy()[0].astype(np.float64))
        want = L.attention(q64, np.stack(keys), np.stack(values), prefix + i, 0, dim**-0.5)
        got = att.cpu().numpy()
        # q is off by the projection's rounding (2^-21 of a group's largest activation), which moves scores by 1e-5
        assert np.all(np.abs(got - want) <= 1e-4 * np.abs(want).max())
        assert np.all(np.abs(y.cpu().numpy() - wo @ want.reshape(-1)) <= 2e-4 * np.abs(wo @ want.reshape(-1)).max())
