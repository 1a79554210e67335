"""Page tables, slots, positions and masks from lengths, pages given back, a tree's confirmed path and moves inside the
cache, against plain Python."""
import random

import pytest

torch = pytest.importorskip("torch")
import step_util as S
import turbo_decode_tail as T

pytestmark = pytest.mark.gpu
NO = 0xFFFFFFFF


def empty(n, dtype=torch.int32):
    return torch.full((n,), 77, dtype=dtype, device="cuda") if isinstance(n, int) else torch.full(n, 77, dtype=dtype, device="cuda")


class Pool:
    """Sequences that hold the pages of their tokens, and the free pages."""

    def __init__(self, past, page, prefix, width, spare, seed=0):
        rng = random.Random(seed)
        self.past, self.page, self.prefix, self.width = list(past), page, prefix, width
        self.held = [-(-max(0, p - prefix) // page) for p in past]
        order = list(range(sum(self.held) + spare))
        rng.shuffle(order)
        self.tables = []
        for h in self.held:
            self.tables.append([order.pop() for _ in range(h)] + [NO - 1] * (width - h))
        self.free = order

    def device(self, capacity):
        self.d_pages = S.ids(self.tables, (len(self.past), self.width)) if self.past else empty((0, self.width))
        self.d_free = S.ids(self.free + [5] * (capacity - len(self.free)))
        self.d_count, self.d_held, self.d_past = S.ids([len(self.free)]), S.ids(self.held), S.ids(self.past)


def run_plan(pool, new, *, row_tokens=0, max_tokens=None, parents=None, in_place=True, capacity=None, stream=None):
    b = len(new)
    n = b * row_tokens if row_tokens else max_tokens
    pool.device(capacity or len(pool.free) + 8)
    out = {"starts": empty(b + 1), "kv_len": empty(b), "positions": empty(max(1, n)), "slots": empty(max(1, n)), "totals": empty(4)}
    if parents is not None:
        out["masks"] = empty((b, row_tokens), torch.int64)
        d_parents = torch.tensor(parents, dtype=torch.int32, device="cuda")
    more = {} if in_place else {"held_out": empty(max(1, b)), "free_count_out": empty(1)}
    inp = T.make_batch_plan(b, page_tokens=pool.page, prefix_len=pool.prefix, past_len=pool.d_past, new_len=(d_new := S.ids(new)),
                            row_tokens=row_tokens, max_tokens=n, parents=d_parents if parents is not None else None,
                            pages=pool.d_pages, held=pool.d_held, free_pages=pool.d_free, free_count=pool.d_count, **more, **out)
    T.batch_plan(inp, stream)
    torch.cuda.synchronize()
    held, count = (pool.d_held, pool.d_count) if in_place else (more["held_out"], more["free_count_out"])
    got = {k: S.words(x) for k, x in out.items() if k != "masks"}
    got["positions"], got["slots"] = got["positions"][:n], got["slots"][:n]
    got["masks"] = [[m & (2**64 - 1) for m in row] for row in out["masks"].cpu().tolist()] if parents is not None else None
    got["held"], got["count"] = S.words(held)[:b], S.words(count)[0]
    got["pages"] = S.words(pool.d_pages)
    del d_new
    return got


def compare(pool, new, **kw):
    tables = [list(t) for t in pool.tables]
    want = S.plan(pool.past, new, pool.held, tables, pool.free, pool.page, pool.prefix, pool.width, kw.get("row_tokens", 0),
                  kw.get("max_tokens"), kw.get("parents"))
    got = run_plan(pool, new, **kw)
    for k in ("starts", "kv_len", "positions", "slots", "masks", "totals", "held"):
        assert got[k] == want[k], k
    assert got["count"] == len(want["free"]) and got["pages"] == tables
    return want, tables


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("page,prefix", [(32, 0), (64, 100), (256, 1)])
@pytest.mark.parametrize("batch,longest", [(1, 1), (1, 9000), (3, 70), (70, 400), (300, 60)])
def test_packed(batch, longest, page, prefix, in_place):
    rng = random.Random(batch * 1000 + longest)
    past = [prefix + rng.choice([0, rng.randint(0, 500), page * rng.randint(0, 4)]) for _ in range(batch)]
    new = [rng.choice([0, 1, rng.randint(0, longest), longest]) for _ in range(batch)]
    need = sum(new) // page + 2 * batch
    pool = Pool(past, page, prefix, (600 + longest) // page + 2, need)
    compare(pool, new, max_tokens=sum(new) + 5, in_place=in_place)


@pytest.mark.parametrize("batch,longest", [(5, 20), (60, 700), (2100, 40)])
def test_lengths_in_the_place_of_the_past(batch, longest):
    """kv_len may be past_len itself: the lengths after the step, and the same slots, whatever runs first."""
    rng = random.Random(batch)
    past = [rng.randint(0, 300) for _ in range(batch)]
    new = [rng.randint(0, longest) for _ in range(batch)]
    pool = Pool(past, 32, 0, (300 + longest) // 32 + 2, sum(new) // 32 + 2 * batch)
    n, tables = sum(new), [list(t) for t in pool.tables]
    want = S.plan(pool.past, new, pool.held, tables, pool.free, 32, 0, pool.width, 0, n, None)
    pool.device(len(pool.free) + 1)
    slots, held, count = empty(n), empty(batch), empty(1)
    T.batch_plan(T.make_batch_plan(batch, page_tokens=32, past_len=pool.d_past, new_len=(d_new := S.ids(new)), max_tokens=n,
                                   pages=pool.d_pages, held=pool.d_held, free_pages=pool.d_free, free_count=pool.d_count,
                                   held_out=held, free_count_out=count, kv_len=pool.d_past, slots=slots))
    torch.cuda.synchronize()
    assert S.words(slots) == want["slots"] and S.words(pool.d_past) == want["kv_len"] and S.words(held) == want["held"]
    del d_new


@pytest.mark.parametrize("batch", [2047, 2048, 2049, 8192])
def test_the_largest_batches(batch):
    rng = random.Random(batch)
    past = [rng.randint(0, 90) for _ in range(batch)]
    new = [rng.choice([0, 1, 2, rng.randint(0, 70)]) for _ in range(batch)]
    pool = Pool(past, 32, 0, 6, 3 * batch)
    compare(pool, new, max_tokens=sum(new) + 3, in_place=bool(batch % 2))
    rows = [min(n, 4) for n in new]
    compare(pool, rows, row_tokens=4, parents=random_trees(rng, batch, 4, 0.05))


@pytest.mark.parametrize("batch,rows", [(1, 1), (5, 1), (40, 7), (9, 64), (600, 3), (2, 5000)])
def test_rows(batch, rows):
    rng = random.Random(batch)
    past = [rng.randint(0, 300) for _ in range(batch)]
    new = [rng.choice([0, rows, rng.randint(0, rows), rows + 3]) for _ in range(batch)]
    pool = Pool(past, 64, 0, (300 + rows) // 64 + 2, 3 * batch + batch * rows // 64)
    compare(pool, new, row_tokens=rows)


@pytest.mark.parametrize("spare", [0, 1, 5])
def test_a_pool_that_runs_out_and_is_filled_again(spare):
    pool = Pool([10, 64, 0, 200, 63], 64, 0, 6, spare)
    new = [100, 1, 130, 0, 2]
    want, tables = compare(pool, new, max_tokens=300)
    assert want["totals"][3] > 0 and want["totals"][2] == spare
    pool.tables, pool.held = tables, want["held"]
    pool.free = [1000 + i for i in range(20)]
    want, _ = compare(pool, new, max_tokens=300)  # the same step again: what is missing is taken now
    assert want["totals"][3] == 0


def test_a_table_that_is_too_short():
    pool = Pool([0, 100], 32, 0, 4, 50)
    want, _ = compare(pool, [500, 60], max_tokens=560)
    assert want["totals"][3] == 16 - 4 + 1


def test_tokens_past_the_arrays_and_of_the_prefix():
    pool = Pool([0, 30], 32, 40, 4, 20)  # both begin inside the shared prefix
    want, _ = compare(pool, [60, 20], max_tokens=70)
    assert want["totals"][:2] == [80, 10] and want["slots"][:40] == [NO] * 40


def test_nothing_to_do():
    pool = Pool([3, 64], 64, 0, 2, 4)
    compare(pool, [0, 0], max_tokens=0)
    compare(pool, [0, 0], max_tokens=6)
    got = run_plan(Pool([], 64, 0, 2, 3), [], max_tokens=4)
    assert got["starts"] == [0] and got["slots"] == [NO] * 4 and got["positions"] == [0] * 4 and got["totals"] == [0] * 4


def random_trees(rng, batch, rows, bad=0.0):
    out = []
    for _ in range(batch):
        t = [-1 if i == 0 or rng.random() < 0.1 else rng.randint(max(0, i - 5), i - 1) for i in range(rows)]
        out.append([rng.choice([-2, i, i + 1, 10**9, -2**31]) if rng.random() < bad else p for i, p in enumerate(t)])
    return out


@pytest.mark.parametrize("bad", [0.0, 0.1])
@pytest.mark.parametrize("batch,rows", [(1, 1), (1, 64), (3, 2), (33, 40), (130, 63)])
def test_trees(batch, rows, bad):
    rng = random.Random(rows)
    past = [50 + rng.randint(0, 300) for _ in range(batch)]
    new = [rng.choice([0, rows, rng.randint(0, rows)]) for _ in range(batch)]
    pool = Pool(past, 32, 50, 14, 4 * batch)
    compare(pool, new, row_tokens=rows, parents=random_trees(rng, batch, rows, bad))
    chain = [[i - 1 for i in range(rows)]] * batch
    compare(pool, new, row_tokens=rows, parents=chain)


def test_results_that_are_not_wanted():
    pool = Pool([10, 20], 32, 0, 3, 9)
    pool.device(20)
    T.batch_plan(T.make_batch_plan(2, page_tokens=32, past_len=pool.d_past, new_len=S.ids([40, 50]), max_tokens=90, pages=pool.d_pages,
                                   held=pool.d_held, free_pages=pool.d_free, free_count=pool.d_count))
    torch.cuda.synchronize()
    assert S.words(pool.d_held) == [2, 3] and S.words(pool.d_count) == [6]


@pytest.mark.parametrize("batch", [1, 7, 700])
def test_release(batch):
    rng = random.Random(batch)
    past = [20 + rng.randint(0, 400) for _ in range(batch)]
    pool = Pool(past, 32, 20, 16, 11)
    keep = [rng.choice([0, p, rng.randint(0, p + 50), 20, 21]) for p in past]
    free, held = list(pool.free), []
    for i in range(batch):
        n = min(pool.held[i], -(-max(0, keep[i] - 20) // 32))
        free += pool.tables[i][n:pool.held[i]]
        held.append(n)
    capacity = len(pool.free) + sum(pool.held)
    pool.device(capacity)
    T.pages_release(batch, page_tokens=32, keep_len=S.ids(keep), pages=pool.d_pages, held=pool.d_held, free_pages=pool.d_free,
                    free_count=pool.d_count, prefix_len=20)
    torch.cuda.synchronize()
    assert S.words(pool.d_held) == held and S.words(pool.d_count) == [len(free)] and S.words(pool.d_free)[:len(free)] == free
    assert S.words(pool.d_pages) == pool.tables


def test_plan_and_release_in_a_graph():
    """Steps of one captured plan: lengths change between the replays, the pool lives on."""
    rng = random.Random(5)
    pool = Pool([0] * 6, 32, 0, 40, 150)
    pool.device(150)
    new, slots, totals = empty(6), empty(300), empty(4)
    inp = T.make_batch_plan(6, page_tokens=32, past_len=pool.d_past, new_len=new, max_tokens=300, pages=pool.d_pages, held=pool.d_held,
                            free_pages=pool.d_free, free_count=pool.d_count, slots=slots, totals=totals)
    new.zero_()
    T.batch_plan(inp)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        T.batch_plan(inp, torch.cuda.current_stream().cuda_stream)
    free, held, tables, past = list(pool.free), [0] * 6, pool.tables, [0] * 6
    for _ in range(8):
        add = [rng.randint(0, 49) for _ in range(6)]
        new.copy_(S.ids(add))
        pool.d_past.copy_(S.ids(past))
        graph.replay()
        torch.cuda.synchronize()
        want = S.plan(past, add, held, tables, free, 32, 0, 40, 0, 300)
        assert S.words(slots) == want["slots"] and S.words(totals) == want["totals"] and S.words(pool.d_held) == want["held"]
        free, held = want["free"], want["held"]
        past = [p + a for p, a in zip(past, add)]
    T.pages_release(6, page_tokens=32, keep_len=S.ids([0] * 6), pages=pool.d_pages, held=pool.d_held, free_pages=pool.d_free,
                    free_count=pool.d_count)
    torch.cuda.synchronize()
    assert sorted(S.words(pool.d_free)) == sorted(pool.free) and S.words(pool.d_count) == [150]


# ---- the confirmed path ------------------------------------------------------------------------------

@pytest.mark.parametrize("bad", [0.0, 0.1])
@pytest.mark.parametrize("batch,rows", [(1, 1), (1, 64), (5, 3), (257, 40)])
def test_accept(batch, rows, bad):
    rng = random.Random(batch + rows)
    parents = random_trees(rng, batch, rows, bad)
    tokens = [[rng.randint(0, 3) for _ in range(rows)] for _ in range(batch)]  # siblings with the same token among them
    chosen = [[rng.choice([0, 1, 2, 3, NO]) for _ in range(rows)] for _ in range(batch)]
    new = [rng.choice([0, rows, rng.randint(0, rows), rows + 9]) for _ in range(batch)]
    past = [rng.randint(0, 1000) for _ in range(batch)]
    slots = [[rng.randint(0, 10**6) for _ in range(rows)] for _ in range(batch)]
    out = {k: empty(batch) for k in ("kept", "next", "length")} | {k: empty((batch, rows)) for k in ("path", "source", "target")}
    keep = dict(parents=torch.tensor(parents, dtype=torch.int32, device="cuda"), new_len=S.ids(new), tokens=S.ids(tokens),
                chosen=S.ids(chosen), past_len=S.ids(past), slots=S.ids(slots))
    T.tree_accept(T.make_tree_accept(batch, rows, **keep, **out))
    torch.cuda.synchronize()
    got = {k: S.words(x) for k, x in out.items()}
    for b in range(batch):
        path, after = S.accept(parents[b], tokens[b], chosen[b], min(new[b], rows))
        rest = [NO] * (rows - len(path))
        assert (got["kept"][b], got["next"][b], got["length"][b]) == (len(path), after, past[b] + len(path))
        assert got["path"][b] == path + rest
        assert got["source"][b] == [slots[b][i] for i in path] + rest
        assert got["target"][b] == slots[b][:len(path)] + rest


def test_accept_without_the_optional_results():
    one = S.ids([[4]])
    kept, after = empty(1), empty(1)
    T.tree_accept(T.make_tree_accept(1, 1, parents=torch.tensor([[-1]], dtype=torch.int32, device="cuda"), new_len=S.ids([1]),
                                     tokens=one, chosen=S.ids([[9]]), kept=kept, next=after))
    torch.cuda.synchronize()
    assert (S.words(kept), S.words(after)) == ([1], [9])


# ---- moves -------------------------------------------------------------------------------------------

def contents(cache, n, heads, d):
    """What every slot reads back, as bits (a stored value is code * scale + bias: FP32 holds nearly all of it)."""
    k, v = (torch.empty((n, heads, d), dtype=torch.float32, device="cuda") for _ in range(2))
    cache.read(torch.arange(n, dtype=torch.int32, device="cuda"), n, k, v)
    torch.cuda.synchronize()
    return torch.stack([k, v]).view(torch.int32)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d,heads,page", [(64, 1, 32), (64, 3, 256), (128, 8, 64), (256, 2, 128), (512, 3, 32)])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 17), (5, 64)])
def test_move(d, heads, page, bits, rows, width):
    rng = random.Random(d + rows)
    n = 1024
    cache = T.KvCache(n // page, page, heads, d, bits=bits)
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn((n, heads, d), generator=g, device="cuda") * 3 for _ in range(2))
    cache.write(k, v, torch.arange(n, dtype=torch.int32, device="cuda"), n)
    want = contents(cache, n, heads, d)
    before = want.clone()
    source, target = [], []
    places = rng.sample(range(n), rows * width)
    for r in range(rows):  # a row moves among its own places: it writes slots that it reads
        mine = places[r * width:(r + 1) * width]
        to = rng.sample(mine, width)
        src = [rng.choice(mine) for _ in range(width)]
        for i in range(width):
            x = rng.random()
            if x < 0.1:
                src[i] = rng.choice([NO, n, n + 7])
            elif x < 0.2:
                to[i] = rng.choice([NO, n])
            if src[i] < n and to[i] < n:
                want[:, to[i]] = before[:, src[i]]
        source.append(src)
        target.append(to)
    cache.move(S.ids(source), S.ids(target))
    assert torch.equal(contents(cache, n, heads, d), want)
    cache.close()


def test_move_in_a_graph_and_of_groups_of_nan():
    cache = T.KvCache(2, 32, 1, 64)
    k = torch.randn((64, 1, 64), device="cuda")
    v = k + 1
    k[5, 0, 3], v[9, 0, 0] = float("nan"), float("inf")
    every = torch.arange(64, dtype=torch.int32, device="cuda")
    source, target = S.ids([[5, 9]]), S.ids([[40, 41]])
    cache.move(source, target)  # of undefined contents: only the first launch before the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.move(source, target, torch.cuda.current_stream().cuda_stream)
    for shift in (0, 1, 2):
        cache.write(k, v, every, 64)
        want = contents(cache, 64, 1, 64)
        target.copy_(S.ids([[40 + shift, 50 + shift]]))
        want[:, 40 + shift], want[:, 50 + shift] = want[:, 5].clone(), want[:, 9].clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(contents(cache, 64, 1, 64), want)
    cache.close()
