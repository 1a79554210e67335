"""Attention of drafted trees over the quantised cache (turbo_tree_attention) against the formula in 64 bits, and a
speculative step from lengths to kept tokens."""
import math
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import layer_util as L
import step_util as S
import turbo_decode_tail as T

pytestmark = pytest.mark.gpu
F32, BF16 = T.TURBO_HIDDEN_F32, T.TURBO_HIDDEN_BF16
TYPES = {F32: torch.float32, BF16: torch.bfloat16}


class Case:
    """A batch of trees: before[b] tokens in front of sequence b's nodes (None: padded), the first `prefix` of them shared."""

    def __init__(self, before, nodes, hq, hk, d, *, bits=8, page=32, prefix=0, dtype=BF16, seed=0, masks=None, size=1.0):
        rng = random.Random(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.before, self.nodes, self.hq, self.hk, self.d, self.prefix, self.dtype = before, nodes, hq, hk, d, prefix, dtype
        b = len(before)
        own = [0 if n is None else max(0, n + nodes - prefix) for n in before]
        need_p, need = -(-prefix // page), [-(-n // page) for n in own]
        self.page, self.width = page, max(1, max(need))
        order = list(range(need_p + sum(need) + 1))
        rng.shuffle(order)
        self.bad_page = order.pop()  # in no table: its contents stay undefined
        prefix_pages = [order.pop() for _ in range(need_p)]
        tables = [[order.pop() for _ in range(n)] + [self.bad_page] * (self.width - n) for n in need]
        self.cache = T.KvCache(need_p + sum(need) + 1, page, hk, d, bits=bits)
        self.prefix_pages, self.tables = S.ids(prefix_pages or [0]), S.ids(tables, (b, self.width))
        rand = lambda n: torch.randn((n, hk, d), generator=g, device="cuda").bfloat16()  # noqa: E731
        shared = rand(prefix), rand(prefix)
        self.held, slots, keys, values = [], [], [shared[0]], [shared[1]]
        slots += [prefix_pages[i // page] * page + i % page for i in range(prefix)]
        for i in range(b):
            k, v = rand(own[i]), rand(own[i])
            keys.append(k)
            values.append(v)
            slots += [tables[i][j // page] * page + j % page for j in range(own[i])]
            self.held.append((torch.cat([shared[0], k]), torch.cat([shared[1], v])))
        self.slots = S.ids(slots or [0])
        if slots:
            self.cache.write(torch.cat(keys).contiguous(), torch.cat(values).contiguous(), self.slots, len(slots), dtype=BF16)
        self.bits = bits
        self.kv_len = S.ids([0 if n is None else n + nodes for n in before])
        self.masks = masks if masks is not None else [self.tree(rng) for _ in range(b)]
        self.q = (torch.randn((b * nodes, hq, d), generator=g, device="cuda") * size).to(TYPES[dtype])

    def tree(self, rng):
        out = []
        for t in range(self.nodes):
            p = -1 if t == 0 or rng.random() < 0.1 else rng.randint(max(0, t - 6), t - 1)
            out.append((out[p] if p >= 0 else 0) | 1 << t)
        return out

    def run(self, *, window=0, scale=None, masks=None, workspace=None, stream=None, sync=True, longest=None):
        b = len(self.before)
        self.scale = self.d**-0.5 if scale is None else scale
        self.out = torch.full(self.q.shape, 7.0, dtype=self.q.dtype, device="cuda")
        words = self.masks if masks is None else masks
        self.d_masks = torch.tensor([[m - 2**64 if m >= 2**63 else m for m in row] for row in words], dtype=torch.int64, device="cuda")
        longest = longest or max([n or 0 for n in self.before]) + self.nodes
        self.inp = self.cache.make_attention_inputs(b, dtype=self.dtype, q=self.q, out=self.out, q_heads=self.hq, q_len=self.nodes,
                                                    kv_len=self.kv_len, max_kv_len=longest, pages=self.tables,
                                                    prefix_len=self.prefix, prefix_pages=self.prefix_pages, window=window, scale=self.scale)
        self.workspace = torch.empty(max(1, self.cache.attention_workspace(self.inp)), dtype=torch.uint8, device="cuda")
        self.inp.workspace, self.inp.workspace_bytes = self.workspace.data_ptr(), self.workspace.numel()
        self.cache.attend_tree(self.inp, self.d_masks, stream)
        if sync:
            torch.cuda.synchronize()
        return self.out

    def stored(self, x):
        """What the cache holds, and the size of what enters the sums for it: a code counts from the middle one, so a
        small value may be the difference of the centre and a code times the scale, each of up to half its group's range."""
        x = x.float().cpu().numpy()
        half = np.repeat(L.quantise(x, self.bits)[1].astype(np.float64) * 2.0 ** (self.bits - 1), 64, axis=-1)
        held = L.stored(x, self.bits)
        return torch.from_numpy(held).cuda(), torch.from_numpy(np.abs(held) + 2 * half).cuda()

    def seen(self, i, window, masks=None):
        """[nodes][tokens] of sequence i."""
        n, t = self.before[i], self.nodes
        seen = torch.zeros((t, n + t), dtype=torch.bool)
        for j, m in enumerate((masks or self.masks)[i]):
            m &= 2**t - 1
            at = ([*range(n)] + [n + x for x in range(t) if m >> x & 1]) if m else []
            seen[j, at[-window:] if window else at] = True
        return seen.cuda()

    def check(self, window=0, masks=None, rounding=0.0):
        """rounding: of a key and a value, relative to it."""
        t = self.nodes
        for i, n in enumerate(self.before):
            out = self.out[i * t:(i + 1) * t]
            if n is None:
                assert bool((out == 0).all())
                continue
            (k, ks), (v, vs) = (self.stored(x[:n + t]) for x in self.held[i])
            want, mean, size = S.softmax_rows(self.q[i * t:(i + 1) * t], k, v, self.seen(i, window, masks), self.scale, ks, vs)
            # a score is off by roundings of 2^-22 (both parts of an FP32 query; a BF16 one is exact) and d + 64 of 2^-24 of
            # what enters it, and a weight by as much relative to itself; a weight times a scale keeps 22 bits, for BF16
            # 11 (2^-11 of each at most); sums of n tokens, n of 2^-24; the result is rounded once
            spread = 2 * (rounding + 2.0**-21 + (self.d + 64) * 2.0**-24) * abs(self.scale) * size[..., None]
            weight = spread + rounding + (n + t + 64) * 2.0**-24 + 2.0**-20 + (2.0**-11 if self.dtype == BF16 else 0)
            bound = 1.01 * mean * weight + want.abs() * (2.0**-8 if self.dtype == BF16 else 2.0**-23)
            far = (out.double() - want).abs()
            assert bool((far <= bound).all()), (i, (far / bound).max().item())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d,hq,hk", [(64, 4, 4), (128, 8, 1), (256, 4, 2), (256, 6, 2), (512, 8, 2)])
@pytest.mark.parametrize("nodes", [1, 2, 17, 33, 64])
def test_trees(d, hq, hk, nodes, bits, dtype):
    c = Case([0, 1, 31, None, 200, 77], nodes, hq, hk, d, bits=bits, dtype=dtype, seed=nodes)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [1, 2, 3, 9, 40, 100, 5000])
@pytest.mark.parametrize("prefix", [0, 50, 300])
def test_windows_and_prefixes(prefix, window, dtype):
    c = Case([prefix + n if n is not None else None for n in (0, 5, 64, None, 130)], 21, 8, 2, 128, prefix=prefix, dtype=dtype, seed=window)
    c.run(window=window)
    c.check(window)


@pytest.mark.parametrize("d", [64, 256])
def test_long_and_many(d):
    c = Case([2000 + 37 * i for i in range(9)], 40, 8, 2, d, page=64, prefix=2000, seed=3)
    c.run()
    c.check()


def test_a_chain_is_what_the_causal_attention_gives():
    """A run of drafts as a tree, and by turbo_prefix_attention: both within the bound of the same formula."""
    for dtype in (F32, BF16):
        c = Case([40, 7, 333], 16, 4, 2, 256, dtype=dtype, masks=[[2**(t + 1) - 1 for t in range(16)]] * 3)
        for window in (0, 5, 100):
            c.run(window=window)
            c.check(window)
            c.out.fill_(9.0)
            c.cache.attend(c.inp)
            torch.cuda.synchronize()
            c.check(window)


def test_masks_of_any_shape():
    """Nodes that see none of the others, themselves or later ones; all of them; bits past the nodes."""
    masks = [[1, 2**64 - 1, 1 << 9, (1 << 63) | 4, 2**10 - 1, 1 << 3, 0, 0b1010101010, 2**40, 1 << 9 | 1]] * 2
    for window in (0, 1, 4):
        c = Case([55, 0], 10, 2, 1, 128, masks=masks)
        c.run(window=window)
        c.check(window)
        assert bool((c.out[6] == 0).all()) and bool((c.out[8] == 0).all())


def test_sixty_four_nodes_and_the_top_bit():
    masks = [[1 << 63] * 32 + [2**64 - 1] * 32]
    c = Case([10], 64, 2, 2, 64, masks=masks, dtype=F32)
    c.run()
    c.check()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128, 256, 512])
def test_absent_nodes_may_lie_anywhere(d, bits):
    """Slots of nodes that nobody sees hold NaN, or were never written; neither has a part."""
    t = 12
    absent = {3, 4, 9, 11}
    keep = [0 if j in absent else sum(1 << x for x in range(j + 1) if x not in absent) for j in range(t)]
    for dtype in (F32, BF16):
        c = Case([45, 0, 90], t, 4, 2, d, bits=bits, dtype=dtype, masks=[keep] * 3)
        want = c.run().clone()
        c.check()
        nan = torch.full((1, 2, d), math.nan, dtype=torch.bfloat16, device="cuda")
        for i, n in enumerate(c.before):
            for j in absent:
                pos = n + j
                slot = S.words(c.tables)[i][pos // c.page] * c.page + pos % c.page
                c.cache.write(nan, nan, S.ids([slot]), 1, dtype=BF16)
        assert torch.equal(c.run(), want)


def test_a_sibling_of_nan():
    """A node whose values are NaN reaches its descendants and no other."""
    t = 6  # 0; 1 and 2 under 0; 3 under 1; 4 under 2; 5 under 3
    masks = [[1, 3, 5, 11, 21, 43]]
    for which in ("k", "v"):
        c = Case([70], t, 4, 2, 128, masks=masks)
        slot = S.words(c.tables)[0][71 // c.page] * c.page + 71 % c.page  # node 1
        k, v = (x[71:72].clone() for x in c.held[0])
        (k if which == "k" else v)[0, 0, 3] = math.nan
        c.cache.write(k.contiguous(), v.contiguous(), S.ids([slot]), 1, dtype=BF16)
        out = c.run()
        for node in (1, 3, 5):
            assert bool(out[node, :2, 0:64].isnan().all())
        out = out.clone()
        out[[1, 3, 5], :2] = 0
        assert bool(out.isfinite().all())


def test_the_workspace_holds_either_call():
    """What turbo_attention_workspace gives serves a tree and a run of the same sizes; a byte less than a call needs is refused."""
    c = Case([900, 1000], 8, 4, 1, 128, seed=5)
    for window in (0, 200):
        c.run(window=window)
        c.check(window)
        c.cache.attend(c.inp)
        if window == 0:  # the few records of a window are one part, which needs no scratch
            c.inp.workspace_bytes = 16
            with pytest.raises(T.TurboError, match="workspace holds"):
                c.cache.attend_tree(c.inp, c.d_masks)


def test_nodes_past_the_table_give_nan():
    c = Case([60, 20], 8, 2, 1, 64, page=32)
    c.tables = c.tables[:, :2].contiguous()  # room for 64 tokens: sequence 0 has 68
    c.masks = [[2**(t + 1) - 1 for t in range(8)]] * 2
    out = c.run()
    assert bool(out[4:8].isnan().all()) and bool(out[:4].isfinite().all()) and bool(out[8:].isfinite().all())


def test_graph_streams_and_two_workspaces():
    a, b = Case([300, 500], 24, 4, 2, 256, seed=1), Case([800], 24, 4, 2, 256, seed=2)
    want = [c.run().clone() for c in (a, b)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = torch.cuda.current_stream().cuda_stream
        for c in (a, b):
            c.cache.attend_tree(c.inp, c.d_masks, st)
    for _ in range(3):
        for c in (a, b):
            c.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a.out, want[0]) and torch.equal(b.out, want[1])
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for c, st in zip((a, b), side):
        c.out.zero_()
        st.wait_stream(torch.cuda.current_stream())
        c.cache.attend_tree(c.inp, c.d_masks, st.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(a.out, want[0]) and torch.equal(b.out, want[1])


# ---- trees of many rows, whose records are widened once for 128 of them --------------------------------

# A key and a value are rounded to fp16 there: half a step, 2^-11 of it; and, where it is small against the largest of its
# head, 2^-22 of that (4 bits: 2^-18), which is below 2^-14 of the size that Case.stored() gives, half a group's range.
ROUNDING = 2.0**-11 + 2.0**-14


class Many(Case):
    """Takes that form by the longest sequence that the call announces: its table has the columns, of no page."""

    def __init__(self, before, nodes, hq, hk, d, announced=40000, **rest):
        super().__init__(before, nodes, hq, hk, d, **rest)
        more = -(-announced // self.page) - self.width
        if more > 0:
            fill = torch.full((len(before), more), self.bad_page, dtype=self.tables.dtype, device="cuda")
            self.tables = torch.cat([self.tables, fill], dim=1).contiguous()
        self.announced = announced

    def run(self, **rest):
        return super().run(longest=self.announced, **rest)


MANY = [([0, 31, None, 500, 1999], 64, 32, 4), ([700, 33, 32, 1, 64], 40, 24, 4), ([300] * 9, 64, 16, 4), ([2500], 64, 128, 8)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("before,nodes,hq,hk", MANY)
def test_many_rows(before, nodes, hq, hk, d, bits):
    c = Many(before, nodes, hq, hk, d, bits=bits, seed=d)
    c.run()
    c.check(rounding=ROUNDING)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("prefix", [1, 32, 100, 999])
def test_many_rows_behind_a_prefix(prefix, d):
    """Some trees begin inside the shared tokens, one behind none of its own."""
    c = Many([prefix, prefix + 45, max(0, prefix - 70), None, prefix + 800], 64, 32, 4, d, prefix=prefix, seed=prefix)
    c.run()
    c.check(rounding=ROUNDING)


def test_many_rows_masks_that_leave_nothing():
    masks = [[0] * 64, [0 if t % 3 else 1 << t for t in range(64)], [2**64 - 1] * 64]
    c = Many([900, 100, 40], 64, 64, 4, 128, masks=masks)
    out = c.run().clone()
    c.check(rounding=ROUNDING)
    assert bool((out[:64] == 0).all()) and bool((out[65:67] == 0).all())
    assert torch.equal(c.run(), out)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_many_rows_large_values_without_weight(d, bits):
    """Values 2^60 times the others under keys that no row gives weight, between the others and before them all, cost the
    others nothing; nor do keys 2^20 times smaller. (The third sequence's last token is taken twice, 2^120: the cache holds
    2^103 and more as NaN, which all its rows see.)"""
    c = Many([600, 200, 64], 64, 32, 4, d, bits=bits, seed=1)
    c.q = c.q.abs() + 0.5
    for i, n in enumerate(c.before):
        k, v = c.held[i]
        for at in (0, 1, 63, n // 2, n - 1):
            k[at], v[at] = -100, v[at] * 2.0**60
        k[n // 3] *= 2.0**-20
        slots = S.ids([S.words(c.tables)[i][j // c.page] * c.page + j % c.page for j in range(n)])
        c.cache.write(k[:n].contiguous(), v[:n].contiguous(), slots, n, dtype=BF16)
    out = c.run()
    assert bool((out[:128].abs() < 100).all()) and bool(out[128:].isnan().all())
    c.before = c.before[:2]
    seen = c.seen

    def others(i, window, masks):  # those tokens have no weight: the bound is that of the others
        s, n = seen(i, window, masks), c.before[i]
        s[:, [0, 1, 63, n // 2, n - 1]] = False
        return s

    c.seen = others
    c.check(rounding=ROUNDING)


@pytest.mark.parametrize("scale", [-0.11, 0.0, 0.7])
def test_many_rows_scales(scale):
    c = Many([500, 90], 64, 64, 4, 128)
    c.run(scale=scale)
    c.check(rounding=ROUNDING)


@pytest.mark.parametrize("which", ["k", "v"])
def test_many_rows_nan(which):
    """NaN in a token before one tree: all its rows see it, the other sequences' none."""
    c = Many([400, 300], 64, 64, 4, 128)
    k, v = (x[77:78].clone() for x in c.held[0])
    (k if which == "k" else v)[0, 1, 3] = math.nan
    c.cache.write(k.contiguous(), v.contiguous(), S.ids([S.words(c.tables)[0][77 // c.page] * c.page + 77 % c.page]), 1, dtype=BF16)
    out = c.run()
    heads = slice(16, 32)  # of that key/value head
    assert bool(out[:64, heads, 0:64].isnan().all())
    out = out.clone()
    out[:64, heads] = 0
    assert bool(out.isfinite().all())


def test_many_rows_bad_pages_and_tables():
    c = Many([400, 300, 200], 64, 64, 4, 128)
    t = c.tables.clone()
    c.tables[0, 3] = -5  # no page of the cache
    out = c.run().clone()
    assert bool(out[:64].isnan().all()) and bool(out[64:].isfinite().all())
    c.tables = t
    c.kv_len = S.ids([c.announced + 500, 0, 264])  # past the table; padded
    out = c.run()
    assert bool(out[:64].isnan().all()) and bool((out[64:128] == 0).all()) and bool(out[128:].isfinite().all())


@pytest.mark.parametrize("d", [64, 256])
def test_many_rows_graphs_and_streams(d):
    a, b = Many([900, 30], 64, 64, 4, d, seed=1), Many([400, 1500], 64, 64, 4, d, seed=2)
    want = [c.run().clone() for c in (a, b)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = torch.cuda.current_stream().cuda_stream
        for c in (a, b):
            c.cache.attend_tree(c.inp, c.d_masks, st)
    for _ in range(3):
        for c in (a, b):
            c.out.zero_()
            c.workspace.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a.out, want[0]) and torch.equal(b.out, want[1])


# ---- a step from lengths to kept tokens --------------------------------------------------------------

def ids(n):
    return torch.zeros(n, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("bits", [4, 8])
def test_speculative_generation(bits):
    """Prompts of different lengths, then steps with drafted trees until each sequence has 24 tokens: what is kept must be
    what the same calls give one token at a time. The model: embeddings, one layer of rotation, cache and attention, and
    a head, all with the library's calls; the drafts are partly right."""
    rng = random.Random(bits)
    V, hq, hk, d, page, R, prompts, goal = 512, 4, 2, 64, 32, 9, [37, 5, 70], 24
    B, hidden = len(prompts), 256
    g = torch.Generator(device="cuda").manual_seed(4)
    emb = torch.randn((V, (hq + 2 * hk) * d), generator=g, device="cuda")
    head = torch.randn((hq * d, V), generator=g, device="cuda")
    text = [[rng.randrange(V) for _ in range(n)] for n in prompts]
    del hidden

    class Model:
        def __init__(self):
            self.cache, self.rotary = T.KvCache(40, page, hk, d, bits=bits), T.Rotary(d)
            self.pages, self.held = torch.zeros((B, 8), dtype=torch.int32, device="cuda"), ids(B)
            self.free, self.count, self.past = torch.arange(40, dtype=torch.int32, device="cuda"), S.ids([40]), ids(B)

        def plan(self, new, rows, n, parents=None):
            self.new = S.ids(new)
            self.out = dict(starts=ids(B + 1), kv_len=ids(B), positions=ids(n), slots=ids(n), totals=ids(4))
            if parents is not None:
                self.out["masks"] = torch.zeros((B, rows), dtype=torch.int64, device="cuda")
                self.parents = torch.tensor(parents, dtype=torch.int32, device="cuda")
            T.batch_plan(T.make_batch_plan(B, page_tokens=page, past_len=self.past, new_len=self.new, row_tokens=rows, max_tokens=n,
                                           parents=self.parents if parents is not None else None, pages=self.pages, held=self.held,
                                           free_pages=self.free, free_count=self.count, **self.out))
            assert S.words(self.out["totals"])[3] == 0

        def heads(self, tokens):
            """Projections, norms and rotation; keys and values into the cache."""
            x = emb[torch.tensor(tokens, device="cuda")].view(len(tokens), -1, d)
            self.q, self.k, self.v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
            q, k = torch.empty((len(tokens), hq, d), device="cuda"), torch.empty((len(tokens), hk, d), device="cuda")
            self.rotary.apply(self.rotary.make_inputs(len(tokens), q=self.q, k=self.k, v=self.v, q_heads=hq, kv_heads=hk,
                                                      positions=self.out["positions"], q_out=q, k_out=k, cache=self.cache,
                                                      slots=self.out["slots"]))
            return q, k

        def choose(self, out):
            return (out.reshape(out.shape[0], -1) @ head).argmax(dim=1).to(torch.int32)

        def prompt(self):
            n = sum(prompts)
            self.plan(prompts, 0, n)
            q, k = self.heads([t for p in text for t in p])
            out = torch.zeros_like(q)
            T.prompt_attention(T.make_prompt_inputs(B, n, q=q, k=k, v=self.v, out=out, q_heads=hq, kv_heads=hk, head_dim=d,
                                                    starts=self.out["starts"], scale=d**-0.5))
            self.past = self.out["kv_len"]
            last = [x - 1 for x in S.words(self.out["starts"])[1:]]
            return S.words(self.choose(out)[last])

        def attend(self, rows, q, masks):
            out = torch.empty_like(q)
            inp = self.cache.make_attention_inputs(B, q=q, out=out, q_heads=hq, q_len=rows, kv_len=self.out["kv_len"], max_kv_len=256,
                                                   pages=self.pages, scale=d**-0.5)
            ws = torch.empty(max(1, self.cache.attention_workspace(inp)), dtype=torch.uint8, device="cuda")
            inp.workspace, inp.workspace_bytes = ws.data_ptr(), ws.numel()
            if masks is None:
                self.cache.attend(inp)
            else:
                self.cache.attend_tree(inp, masks)
            torch.cuda.synchronize()
            return self.choose(out)

    # one token at a time
    plain = Model()
    token = plain.prompt()
    truth = [[t] for t in token]
    for _ in range(goal + R):
        plain.plan([1] * B, 1, B)
        q, _ = plain.heads(token)
        token = S.words(plain.attend(1, q, None))
        plain.past = plain.past + 1
        for b in range(B):
            truth[b].append(token[b])

    # trees
    tree = Model()
    token = tree.prompt()
    assert token == [t[0] for t in truth]
    made, steps = [[] for _ in range(B)], 0
    while min(map(len, made)) < goal:
        parents, drafts, new = [], [], []
        for b in range(B):
            n = rng.randint(1, R)
            par, tok = [-1], [token[b]]
            at, depth = 0, 1
            for i in range(1, n):  # the right continuation for a while, wrong siblings beside it
                right = len(made[b]) + depth < len(truth[b]) and rng.random() < 0.6
                par.append(at if right else rng.randrange(i))
                tok.append(truth[b][len(made[b]) + depth] if right else rng.randrange(V))
                if right:
                    at, depth = i, depth + 1
            parents.append(par + [-1] * (R - n))
            drafts.append(tok + [0] * (R - n))
            new.append(n)
        tree.plan(new, R, B * R, parents)
        q, _ = tree.heads([t for row in drafts for t in row])
        chosen = tree.attend(R, q, tree.out["masks"])
        res = {k: ids(B) for k in ("kept", "next", "length")} | {k: torch.zeros((B, R), dtype=torch.int32, device="cuda")
                                                                 for k in ("path", "source", "target")}
        T.tree_accept(T.make_tree_accept(B, R, parents=tree.parents, new_len=tree.new, tokens=(d_drafts := S.ids(drafts)), chosen=chosen,
                                         past_len=tree.past, slots=tree.out["slots"], **res))
        tree.cache.move(res["source"], res["target"])
        T.pages_release(B, page_tokens=page, keep_len=res["length"], pages=tree.pages, held=tree.held, free_pages=tree.free,
                        free_count=tree.count)
        torch.cuda.synchronize()
        for b, (n, path) in enumerate(zip(S.words(res["kept"]), S.words(res["path"]))):
            made[b] += [drafts[b][j] for j in path[:n]]
        tree.past, token = res["length"], S.words(res["next"])
        steps += 1
        assert sum(S.words(tree.held)) + S.words(tree.count)[0] == 40
    for b in range(B):
        n = min(len(made[b]), len(truth[b]))
        assert made[b][:n] == truth[b][:n]
    assert steps < goal  # some drafts were right
