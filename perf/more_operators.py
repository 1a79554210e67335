"""A serving step from request lengths to kept tokens, as cases that can be timed and compared.

A case is a dict of plain values. `prepare` makes what the caller holds before the call, `run` makes
one pass in plain torch operations or, with `own` set, through the entry points of turbo_decode_tail,
`exact` gives the same outputs from the definitions in 64 bits.

Kinds
  plan    a batch's page tables, slots, positions, offsets (and the masks of drafted trees) from the
          lengths of its sequences
  prompt  causal attention over whole prompts, packed one after another, keys and values as the
          projections leave them
  tree    attention of a tree of drafted tokens over the quantised cache: a node sees the tokens before
          the tree and its own ancestors
  keep    what follows the tree's step: its keys and values are in the cache (written here), the path
          that the model's choices confirm is found, its tokens move to the places after the sequence,
          and the tree's slots are read back

Heads of 256 (16 queries, 8 key/value heads) are those of the benchmark's 4,096 x 2,816 projection;
the other head sizes and ratios are generic.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

GROUP = 64
VOCAB = 262144


# ---- the cases ---------------------------------------------------------------------------------

def _plan(**kw):
    c = {"kind": "plan", "batch": 32, "past_hi": 4000, "new_lo": 1, "new_hi": 1, "prefix": 0, "page": 64, "row_tokens": 0,
         "tree": False, "spare": 0}
    c.update(kw)
    return c


def _prompt(**kw):
    c = {"kind": "prompt", "batch": 1, "lo": 1, "hi": 1, "q_heads": 16, "kv_heads": 8, "head_dim": 256, "window": 0,
         "dtype": "bf16", "packed": False, "spare": 0}
    c.update(kw)
    return c


def _tree(**kw):
    c = {"kind": "tree", "batch": 1, "nodes": 8, "q_heads": 16, "kv_heads": 8, "head_dim": 256, "bits": 8, "page": 64,
         "prefix": 0, "own_lo": 1, "own_hi": 1, "window": 0, "dtype": "bf16", "padded": 0, "reach": 8}
    c.update(kw)
    return c


def _keep(**kw):
    c = {"kind": "keep", "batch": 1, "nodes": 8, "kv_heads": 8, "head_dim": 256, "bits": 8, "page": 64, "dtype": "bf16",
         "past_hi": 4000, "reach": 8}
    c.update(kw)
    return c


def listed():
    return [
        # a batch of prompts that comes in at once: every page is new, tens of thousands of slots
        _plan(name="plan_prompts_24", batch=24, past_hi=0, new_lo=11, new_hi=2700, spare=100),
        # a decode step with drafted trees: few new pages, the masks and the depths of the nodes
        _plan(name="plan_trees_48x40", batch=48, past_hi=9000, new_lo=0, new_hi=40, row_tokens=40, tree=True, prefix=1000),
        # one short question: launch and one round trip
        _prompt(name="prompt_1x37", lo=37, hi=37),
        # a batch of ragged prompts as FP32 projections leave them
        _prompt(name="prompt_ragged_13_f32", batch=13, lo=5, hi=1900, dtype="f32"),
        # documents in a local layer: the window leaves most keys out; heads are slices of one projection
        _prompt(name="prompt_window_3", batch=3, lo=4100, hi=6001, window=1024, packed=True, spare=61),
        # a global layer: wide heads, eight queries to a key/value head
        _prompt(name="prompt_wide_4", batch=4, lo=700, hi=3500, q_heads=16, kv_heads=2, head_dim=512),
        # one long document with heads of 128: the largest
        _prompt(name="prompt_long_16384", lo=16384, hi=16384, q_heads=32, kv_heads=8, head_dim=128),
        # interactive decoding with a tree of 24 drafts, 32-bit activations
        _tree(name="tree_1x24_f32", nodes=24, own_lo=2000, own_hi=2000, dtype="f32"),
        # a local layer over a 4-bit cache, small trees, a padded batch
        _tree(name="tree_window_7x17", batch=7, nodes=17, q_heads=32, kv_heads=4, head_dim=128, bits=4, page=32, prefix=1111,
              own_lo=40, own_hi=1700, window=1024, padded=1),
        # a server's batch of trees behind a system prompt
        _tree(name="tree_shared_24x64", batch=24, nodes=64, prefix=8192, own_lo=1, own_hi=2000),
        # the end of an interactive step
        _keep(name="keep_1x16", nodes=16),
        # the end of a server's step
        _keep(name="keep_64x48", batch=64, nodes=48, bits=4, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choices(["plan", "prompt", "tree", "keep"], [15, 40, 30, 15])[0]
    dim = rng.choice([64, 128, 128, 256, 256, 512])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 8])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    page = rng.choice([32, 64, 128, 256])
    if kind == "plan":
        shape = rng.choice(["prompts", "decode", "trees"])
        common = dict(batch=_log(rng, 1, 512), page=page, prefix=rng.choice([0, 0, _log(rng, 1, 8192)]))
        if shape == "prompts":
            hi = _log(rng, 1, 8192)
            return _plan(**common, past_hi=rng.choice([0, _log(rng, 16, 4096)]), new_lo=rng.randint(0, hi), new_hi=hi,
                         spare=rng.choice([0, 0, 200]))
        if shape == "decode":
            rows = _log(rng, 1, 16)
            return _plan(**common, past_hi=_log(rng, 16, 32768), new_lo=rng.choice([0, rows]), new_hi=rows, row_tokens=rows)
        rows = rng.randint(2, 64)
        return _plan(**common, past_hi=_log(rng, 16, 32768), new_lo=rng.randint(0, rows), new_hi=rows, row_tokens=rows, tree=True)
    if kind == "prompt":
        hi = _log(rng, 1, 16384)
        return _prompt(batch=_log(rng, 1, 32), lo=rng.choice([hi, rng.randint(0, hi)]), hi=hi, q_heads=heads, kv_heads=kv,
                       head_dim=dim, window=rng.choice([0, 0, _log(rng, 1, 4096)]), dtype=dtype, packed=rng.random() < 0.3,
                       spare=rng.choice([0, 0, 33]))
    if kind == "tree":
        batch, own_hi = _log(rng, 1, 64), _log(rng, 1, 4000)
        return _tree(batch=batch, nodes=rng.randint(2, 64), q_heads=heads, kv_heads=kv, head_dim=dim, bits=rng.choice([4, 8, 8]),
                     page=page, prefix=rng.choice([0, _log(rng, 1, 32768)]), own_lo=rng.randint(0, own_hi), own_hi=own_hi,
                     window=rng.choice([0, 0, _log(rng, 2, 8192)]), dtype=dtype, padded=min(batch - 1, rng.choice([0, 0, 1, 3])),
                     reach=rng.choice([1, 4, 16]))
    return _keep(batch=_log(rng, 1, 96), nodes=rng.randint(2, 64), kv_heads=kv, head_dim=dim, bits=rng.choice([4, 8]), page=page,
                 dtype=dtype, past_hi=_log(rng, 16, 32768), reach=rng.choice([1, 4, 16]))


def draw(rng):
    """One more case of the same ranges: batches up to 512, prompts up to 16,384 tokens, trees up to 64
    nodes, prefixes up to 32,768 tokens, every head size, ratio and width; at most the largest listed
    case's work."""
    most = max(_price(c) for c in listed())
    while True:
        c = _draw(rng)
        if _price(c) <= most:
            return c


def _price(c):
    """Seconds the plain form would take, roughly: the larger of its work at plain rates and, for an
    attention, the score tables that it makes."""
    w = work(c)
    s = max(w["bytes"] / 1e11, w["flops"] / 2e13)
    if c["kind"] == "prompt":
        n = _lengths(c, 0, c["lo"], c["hi"])
        s = max(s, 1e-3 * len(n), sum(x * x for x in n) * c["q_heads"] * 24 / 1e12)
    if c["kind"] == "tree":
        keys = c["prefix"] + c["batch"] * (c["own_hi"] + c["nodes"])
        rows = c["batch"] * c["nodes"] * c["q_heads"]
        s = max(s, (keys * c["kv_heads"] * c["head_dim"] * 32 + rows * (c["prefix"] + c["own_hi"]) * 24) / 1e12)
    return s


# ---- inputs, from the seed alone -----------------------------------------------------------------

def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + what) & 0x7FFFFFFFFFFFFFFF)
    return g


def _host_gen(seed, what):
    g = torch.Generator()
    g.manual_seed((int(seed) * 1000033 + what) & 0x7FFFFFFFFFFFFFFF)
    return g


def _randn(shape, g):
    return torch.randn(shape, generator=g, device="cuda")


def _cast(x, dtype):
    return x.bfloat16().contiguous() if dtype == "bf16" else x.contiguous()


def _code(dtype):
    return T().TURBO_HIDDEN_BF16 if dtype == "bf16" else T().TURBO_HIDDEN_F32


_binding = None


def T():
    """The framework's binding; only the passes through the framework's own calls need it."""
    global _binding
    if _binding is None:
        pkg = str(Path(__file__).resolve().parents[1] / "turbo-winfare_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import turbo_decode_tail
        _binding = turbo_decode_tail
    return _binding


def _lengths(c, seed, lo, hi):
    """One length for each sequence, spread evenly over the range (so that the work does not depend on the
    seed), in a random order."""
    n = c["batch"]
    spread = [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]
    order = torch.randperm(n, generator=_host_gen(seed, 1)).tolist()
    return [spread[i] for i in order]


def _u32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _trees(c, seed, batch, nodes):
    """[batch][nodes] parents: node 0 hangs on the sequence, every other one on one of the `reach` nodes
    before it (1: a chain)."""
    g = _host_gen(seed, 2)
    back = torch.randint(1, c.get("reach", 8) + 1, (batch, nodes), generator=g)
    return (torch.arange(nodes) - back).clamp_min(0).index_fill_(1, torch.tensor([0]), -1).to(torch.int32).cuda()


def _keys_values(tokens, c, g):
    """Keys with a few strong channels, as trained keys have them, and values without."""
    shape = (tokens, c["kv_heads"], c["head_dim"])
    k = _randn(shape, g) * 0.7 + _randn(shape[1:], g) * 0.7
    return k, _randn(shape, g)


class State:
    """What the program holds."""

    def __init__(self, case):
        self.case = case


def prepare(case, seed):
    c, st = case, State(case)
    {"plan": _prepare_plan, "prompt": _prepare_prompt, "tree": _prepare_tree, "keep": _prepare_keep}[c["kind"]](c, seed, st)
    if own:
        _prepare_own(c, st)
    elif c["kind"] in ("tree", "keep"):
        st.store = _plain_store(st.pages * c["page"], c)
        if c["kind"] == "tree":
            _plain_write(st.store, st.all_slots.long(), *st.all_kv, c["bits"])
            st.slot_table = _slot_table(st, c)
    if c["kind"] == "tree":
        del st.all_kv, st.all_slots
    torch.cuda.synchronize()
    return st


def _prepare_plan(c, seed, st):
    """Sequences in the middle of their lives: each holds the pages of its tokens, the other pages are in a
    pool in any order."""
    g = _gen(seed, 3)
    b, page, p = c["batch"], c["page"], c["prefix"]
    past = torch.randint(0, c["past_hi"] + 1, (b,), generator=g, device="cuda") + p
    new = torch.tensor(_lengths(c, seed, c["new_lo"], c["new_hi"]), device="cuda")
    held = -(-(past - p) // page)
    need = -(-(past - p + new) // page)
    st.width = -(-(c["past_hi"] + c["new_hi"]) // page) + 1
    total, take = int(held.sum().item()), int((need - held).sum().item())
    order = torch.randperm(total + take + 20, generator=g, device="cuda").to(torch.int32)
    st.pages = torch.zeros((b, st.width), dtype=torch.int32, device="cuda")
    st.pages[torch.arange(st.width, device="cuda")[None] < held[:, None]] = order[:total]
    st.free_pages = order[total:].contiguous()
    st.free_count = _u32([take + 20])
    st.past, st.new, st.held = past.int(), new.int(), held.int()
    st.parents = _trees(c, seed, b, c["row_tokens"]) if c["tree"] else None
    st.tokens = b * c["row_tokens"] if c["row_tokens"] else int(new.sum().item()) + c["spare"]


def _prepare_prompt(c, seed, st):
    g = _gen(seed, 4)
    st.lengths = _lengths(c, seed, c["lo"], c["hi"])
    st.tokens = n = sum(st.lengths) + c["spare"]  # rows behind the last sequence belong to nobody
    hq, hk, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    starts = [0]
    for x in st.lengths:
        starts.append(starts[-1] + x)
    st.starts = _u32(starts)
    k, v = _keys_values(n, c, g)
    parts = [_randn((n, hq, d), g) * 1.5, k, v]
    if c["packed"]:  # one projection's output, the heads are slices of it
        rows = _cast(torch.cat(parts, dim=1), c["dtype"])
        st.q, st.k, st.v = rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:]
    else:
        st.q, st.k, st.v = (_cast(x, c["dtype"]) for x in parts)
    st.out = torch.zeros((n, hq, d), dtype=st.q.dtype, device="cuda")


def _prepare_tree(c, seed, st):
    """Queries, a cache's contents, the page tables and the nodes' masks: pages of the prefix and of every
    sequence in shuffled order, the tables' unused ends filled with page 0. Padded sequences hold nothing
    and their nodes see nothing."""
    g = _gen(seed, 5)
    b, t, page, d, p = c["batch"], c["nodes"], c["page"], c["head_dim"], c["prefix"]
    past = _lengths(c, seed, c["own_lo"], c["own_hi"])
    there = torch.ones(b, dtype=torch.bool)
    there[torch.randperm(b, generator=_host_gen(seed, 6))[:c["padded"]]] = False
    st.there = there.tolist()
    st.own_len = [n + t if here else 0 for n, here in zip(past, st.there)]
    st.kv_len = _u32([p + n if n else 0 for n in st.own_len])
    st.masks = _masks(_trees(c, seed, b, t)) * there.cuda()[:, None]
    st.q = _cast(_randn((b * t, c["q_heads"], d), g) * 1.5, c["dtype"])
    need_p = -(-p // page)
    need = [-(-n // page) for n in st.own_len]
    st.pages = max(1, need_p + sum(need))
    order = torch.randperm(st.pages, generator=g, device="cuda").to(torch.int32)
    st.prefix_pages = order[:need_p].contiguous()
    width = max(1, max(need))
    takes = torch.arange(width, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    st.own_pages = torch.zeros((b, width), dtype=torch.int32, device="cuda")
    st.own_pages[takes] = order[need_p:need_p + sum(need)]
    at = torch.arange(width * page, device="cuda")[None].expand(b, -1)
    written = at < torch.tensor(st.own_len, device="cuda")[:, None]
    slots = st.own_pages.long().repeat_interleave(page, dim=1) * page + at % page
    at = torch.arange(p, device="cuda")
    st.all_slots = torch.cat([st.prefix_pages.long()[at // page] * page + at % page, slots[written]]).to(torch.int32)
    st.all_kv = [x.bfloat16() for x in _keys_values(st.all_slots.numel(), c, g)]


def _prepare_keep(c, seed, st):
    """The step's keys and values and where they go, the trees, the drafted tokens and the model's choice
    after each node: most choices are the token of one of the node's children, as a good draft's are."""
    g = _gen(seed, 7)
    b, t, page = c["batch"], c["nodes"], c["page"]
    st.parents = _trees(c, seed, b, t)
    st.tokens = torch.randint(0, VOCAB, (b, t), generator=g, device="cuda", dtype=torch.int32)
    child = torch.full((b, t + 1), -1, device="cuda")
    child.scatter_reduce_(1, torch.where(st.parents < 0, t, st.parents).long(), torch.arange(t, device="cuda").expand(b, t),
                          "amax")
    child = child[:, :t]
    follow = (child >= 0) & (torch.rand((b, t), generator=g, device="cuda") < 0.85)
    st.chosen = torch.where(follow, st.tokens.gather(1, child.clamp_min(0)),
                            torch.randint(0, VOCAB, (b, t), generator=g, device="cuda", dtype=torch.int32))
    st.past = torch.randint(0, c["past_hi"] + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    st.new = torch.full((b,), t, dtype=torch.int32, device="cuda")
    first = st.past.long() % page  # where the tree begins on its first page
    width = -(-(page - 1 + t) // page)
    st.pages = b * width
    order = torch.randperm(st.pages, generator=g, device="cuda").view(b, width)
    at = first[:, None] + torch.arange(t, device="cuda")
    st.slots = (order.gather(1, at // page) * page + at % page).to(torch.int32)
    st.k, st.v = (_cast(x, c["dtype"]) for x in _keys_values(b * t, c, g))


def _prepare_own(c, st):
    """Handles, output buffers and argument blocks that a program sets up once."""
    t, kind = T(), c["kind"]
    new = lambda shape, dtype=torch.int32: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    if kind == "plan":
        b = c["batch"]
        st.out = {"starts": new(b + 1), "kv_len": new(b), "positions": new(st.tokens), "slots": new(st.tokens), "held": new(b),
                  "free_count": new(1), "totals": new(4)}
        if c["tree"]:
            st.out["masks"] = new((b, c["row_tokens"]), torch.int64)
        st.inp = t.make_batch_plan(b, page_tokens=c["page"], prefix_len=c["prefix"], past_len=st.past, new_len=st.new,
                                   row_tokens=c["row_tokens"], max_tokens=st.tokens, parents=st.parents, pages=st.pages,
                                   held=st.held, free_pages=st.free_pages, free_count=st.free_count, held_out=st.out["held"],
                                   free_count_out=st.out["free_count"], starts=st.out["starts"], kv_len=st.out["kv_len"],
                                   positions=st.out["positions"], slots=st.out["slots"], masks=st.out.get("masks"),
                                   totals=st.out["totals"])
    elif kind == "prompt":
        st.inp = t.make_prompt_inputs(c["batch"], st.tokens, dtype=_code(c["dtype"]), q=st.q, k=st.k, v=st.v, out=st.out,
                                      q_heads=c["q_heads"], kv_heads=c["kv_heads"], head_dim=c["head_dim"], starts=st.starts,
                                      window=c["window"], scale=c["head_dim"] ** -0.5)
    elif kind == "tree":
        st.cache = t.KvCache(st.pages, c["page"], c["kv_heads"], c["head_dim"], bits=c["bits"])
        st.cache.write(st.all_kv[0], st.all_kv[1], st.all_slots, st.all_slots.numel(), dtype=t.TURBO_HIDDEN_BF16)
        st.out = torch.empty(st.q.shape, dtype=st.q.dtype, device="cuda")
        st.inp = st.cache.make_attention_inputs(c["batch"], dtype=_code(c["dtype"]), q=st.q, out=st.out, q_heads=c["q_heads"],
                                                q_len=c["nodes"], kv_len=st.kv_len,
                                                max_kv_len=c["prefix"] + c["own_hi"] + c["nodes"], pages=st.own_pages,
                                                prefix_len=c["prefix"], prefix_pages=st.prefix_pages, window=c["window"],
                                                scale=c["head_dim"] ** -0.5)
        st.workspace = torch.empty(max(1, st.cache.attention_workspace(st.inp)), dtype=torch.uint8, device="cuda")
        st.inp.workspace, st.inp.workspace_bytes = st.workspace.data_ptr(), st.workspace.numel()
    else:
        b, n = c["batch"], c["nodes"]
        st.cache = t.KvCache(st.pages, c["page"], c["kv_heads"], c["head_dim"], bits=c["bits"])
        st.out = {"kept": new(b), "next": new(b), "length": new(b), "path": new((b, n)), "from": new((b, n)), "to": new((b, n)),
                  "k": new(st.k.shape, torch.bfloat16), "v": new(st.v.shape, torch.bfloat16)}
        st.inp = t.make_tree_accept(b, n, parents=st.parents, new_len=st.new, tokens=st.tokens, chosen=st.chosen,
                                    past_len=st.past, slots=st.slots, kept=st.out["kept"], next=st.out["next"],
                                    length=st.out["length"], path=st.out["path"], source=st.out["from"], target=st.out["to"])


# ---- one pass --------------------------------------------------------------------------------------

def run(st):
    c, kind = st.case, st.case["kind"]
    if own:
        if kind == "plan":
            T().batch_plan(st.inp)
            return {**st.out, "pages": st.pages}
        if kind == "prompt":
            T().prompt_attention(st.inp)
            return st.out
        if kind == "tree":
            st.cache.attend_tree(st.inp, st.masks)
            return st.out
        n = c["batch"] * c["nodes"]
        st.cache.write(st.k, st.v, st.slots, n, dtype=_code(c["dtype"]))
        T().tree_accept(st.inp)
        st.cache.move(st.out["from"], st.out["to"])
        st.cache.read(st.slots, n, st.out["k"], st.out["v"], dtype=T().TURBO_HIDDEN_BF16)
        return st.out
    return {"plan": _plain_plan, "prompt": _plain_prompt, "tree": _plain_tree, "keep": _plain_keep}[kind](st)


def _ancestors(parents):
    """[batch][node][node]: whether the second is the first or one of its ancestors. With A the table of
    parents, (1 + A)^n counts the walks of up to n steps."""
    b, t = parents.shape
    step = torch.zeros((b, t, t + 1), dtype=torch.float64, device="cuda")
    step.scatter_(2, torch.where(parents < 0, t, parents).long()[..., None], 1.0)
    return torch.linalg.matrix_power(step[..., :t] + torch.eye(t, dtype=torch.float64, device="cuda"), t) > 0.5


def _masks(parents):
    """Bit j of a node's mask: it sees node j."""
    bits = torch.ones((), dtype=torch.int64, device="cuda") << torch.arange(parents.shape[1], device="cuda")
    return (_ancestors(parents) * bits).sum(dim=-1)


def _plain_plan(st):
    c = st.case
    b, page, p, rows, n = c["batch"], c["page"], c["prefix"], c["row_tokens"], st.tokens
    past, new, held = st.past.long(), st.new.long(), st.held.long()
    need = -(-(past - p + new) // page)
    take = (need - held).clamp_min(0)
    upto = torch.cumsum(take, 0)
    at = torch.arange(st.width, device="cuda")
    number = upto[:, None] - take[:, None] + at[None] - held[:, None]  # of a taken page, in the order of taking
    taken = (at[None] >= held[:, None]) & (at[None] < need[:, None])
    fresh = st.free_pages[(st.free_count.long() - 1 - number).clamp(0, st.free_pages.numel() - 1)]
    st.pages.copy_(torch.where(taken, fresh, st.pages))
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    i = torch.arange(n, device="cuda")
    if rows:
        starts, seq, t = torch.arange(b + 1, device="cuda") * rows, i // rows, i % rows
        there = t < new[seq]
        kv_len = torch.where(new > 0, past + rows, zero)
    else:
        starts = torch.cat([zero, torch.cumsum(new, 0)])
        seq = (torch.searchsorted(starts, i, right=True) - 1).clamp_max(b - 1)
        t, there, kv_len = i - starts[seq], i < starts[-1], past + new
    index = past[seq] + t - p
    slots = torch.where(there, st.pages[seq, (index // page).clamp_max(st.width - 1)].long() * page + index % page, -1)
    depth = t
    out = {"starts": starts.int(), "kv_len": kv_len.int(), "held": torch.maximum(held, need).int(),
           "free_count": st.free_count - upto[-1:].int(), "slots": slots.int(), "pages": st.pages,
           "totals": torch.cat([new.sum().view(1), zero, upto[-1:], zero]).int()}
    if c["tree"]:
        out["masks"] = torch.where(there.view(b, rows), _masks(st.parents), 0)
        seen = _ancestors(st.parents) & there.view(b, rows)[..., None]
        depth = (seen.sum(dim=-1) - 1).clamp_min(0).view(-1)
    out["positions"] = torch.where(there, past[seq] + depth, 0).int()
    return out


def _plain_prompt(st):
    """Sequence by sequence, 1,024 queries at a time over the keys that one of them sees."""
    c = st.case
    hk, d, w = c["kv_heads"], c["head_dim"], c["window"]
    g = c["q_heads"] // hk
    first = 0
    for n in st.lengths:
        k, v = (x[first:first + n].float().transpose(0, 1).contiguous() for x in (st.k, st.v))  # [hk, n, d]
        kt = k.transpose(1, 2).contiguous()
        for lo in range(0, n, 1024):
            hi = min(n, lo + 1024)
            begin = max(0, lo - w + 1) if w else 0
            q = st.q[first + lo:first + hi].float().view(hi - lo, hk, g, d).permute(1, 2, 0, 3).reshape(hk, -1, d) * d ** -0.5
            s = torch.matmul(q, kt[:, :, begin:hi].contiguous()).view(hk, g, hi - lo, hi - begin)
            i, j = torch.arange(lo, hi, device="cuda")[:, None], torch.arange(begin, hi, device="cuda")[None]
            s.masked_fill_((j > i) | (j <= i - w) if w else j > i, -math.inf)
            e = s.sub_(s.amax(dim=-1, keepdim=True)).exp_()
            out = torch.matmul((e / e.sum(dim=-1, keepdim=True)).view(hk, -1, hi - begin), v[:, begin:hi].contiguous())
            st.out[first + lo:first + hi] = out.view(hk, g, hi - lo, d).permute(2, 0, 1, 3).reshape(hi - lo, -1, d)
        first += n
    return st.out


def _plain_keep(st):
    c = st.case
    b, t = c["batch"], c["nodes"]
    slots = st.slots.long()
    _plain_write(st.store, slots.view(-1), st.k, st.v, c["bits"])
    above = torch.where(st.parents < 0, 0, st.parents).long()
    agrees = (st.parents >= 0) & (st.tokens == st.chosen.gather(1, above))
    # of siblings with the same token the first counts
    same = (st.parents[:, :, None] == st.parents[:, None]) & agrees[:, None] & agrees[:, :, None]
    agrees &= ~torch.tril(same, diagonal=-1).any(dim=-1)
    agrees[:, 0] = True
    kept = (agrees[:, None] | ~_ancestors(st.parents)).all(dim=-1)
    count = kept.sum(dim=-1)
    path = torch.argsort(~kept, dim=-1, stable=True)  # a node comes after its ancestors
    held = torch.arange(t, device="cuda") < count[:, None]
    last = path.gather(1, (count - 1)[:, None])
    source, target = slots.gather(1, path)[held], slots[held]
    for part in st.store:
        for x in part:
            x[target] = x[source]
    k, v = _plain_read(st.store, slots.view(-1))
    none = lambda x: torch.where(held, x, -1).int()  # noqa: E731
    return {"kept": count.int(), "next": st.chosen.gather(1, last)[:, 0], "length": st.past + count.int(), "path": none(path),
            "from": none(slots.gather(1, path)), "to": none(slots), "k": k.bfloat16(), "v": v.bfloat16()}


def _plain_store(slots, c):
    """A cache in plain layout: codes, scales and biases of the keys and of the values."""
    hk, d = c["kv_heads"], c["head_dim"]
    codes = lambda: torch.zeros((slots, hk, d), dtype=torch.uint8, device="cuda")  # noqa: E731
    pair = lambda: torch.zeros((slots, hk, d // GROUP), dtype=torch.bfloat16, device="cuda")  # noqa: E731
    return [(codes(), pair(), pair()) for _ in range(2)]


def _outward(x, up):
    """x rounded to BF16 upwards or downwards, as fp32: the low half is cut off, which rounds towards
    zero, and one unit is added where that went the wrong way."""
    bits = x.contiguous().view(torch.int32)
    cut = bits & -65536
    wrong = (cut != bits) & ((bits >= 0) if up else (bits < 0))
    return (cut + wrong.int() * 65536).view(torch.float32)


def _plain_quantise(x, bits):
    """Codes, scale and bias of every group of 64 values; the quotients in 64 bits, as 16-bit values fall on a
    border between two codes or two scales often."""
    top = 2 ** bits - 1
    x = x.float().unflatten(-1, (-1, GROUP))
    bias = _outward(x.amin(dim=-1, keepdim=True), False)
    scale = _outward(((x.amax(dim=-1, keepdim=True) - bias).double() / top).float(), True).clamp_min(2.0 ** -126)
    codes = ((x.double() - bias) / scale).round().clamp(0, top)
    return codes.flatten(-2).to(torch.uint8), scale.squeeze(-1).bfloat16(), bias.squeeze(-1).bfloat16()


def _plain_write(store, slots, k, v, bits):
    for (codes, scale, bias), x in zip(store, (k, v)):
        a, b, c = _plain_quantise(x, bits)
        codes[slots], scale[slots], bias[slots] = a, b, c


def _plain_read(store, slots):
    """The values that the codes at these slots stand for, in fp32."""
    return [torch.addcmul(bias[slots].float().unsqueeze(-1), codes[slots].float().unflatten(-1, (-1, GROUP)),
                          scale[slots].float().unsqueeze(-1)).flatten(-2) for codes, scale, bias in store]


def _slot_table(st, c):
    """The slots of the prefix's tokens and of every sequence's own tokens, as a plain program keeps them."""
    page, at = c["page"], torch.arange(c["prefix"], device="cuda")
    prefix = st.prefix_pages.long()[at // page] * page + at % page
    at = torch.arange(max(1, max(st.own_len)), device="cuda")
    return prefix, st.own_pages.long()[:, at // page] * page + at % page


def _plain_tree(st):
    """Scores against the prefix as one product per key/value head over the rows of the whole batch,
    against the sequences' own keys as one per sequence and head; one softmax over both."""
    c = st.case
    b, t, hk, d, p, w = c["batch"], c["nodes"], c["kv_heads"], c["head_dim"], c["prefix"], c["window"]
    m = t * (c["q_heads"] // hk)
    pre, mine = st.slot_table
    n = mine.shape[1]
    kp, vp = (x.transpose(0, 1).contiguous() for x in _plain_read(st.store, pre))          # [hk, p, d]
    ko, vo = (x.transpose(1, 2).contiguous() for x in _plain_read(st.store, mine))         # [b, hk, n, d]
    q = st.q.float().reshape(b, t, hk, m // t, d).permute(2, 0, 1, 3, 4).reshape(hk, b, m, d) * d ** -0.5
    sp = torch.matmul(q.reshape(hk, b * m, d), kp.transpose(1, 2).contiguous()).reshape(hk, b, m, p)
    so = torch.matmul(q.transpose(0, 1).contiguous(), ko.transpose(2, 3).contiguous()).transpose(0, 1)
    s = torch.cat((sp, so), dim=-1)
    del sp, so
    at = torch.arange(p + n, device="cuda")
    before = st.kv_len.long() - t                                                           # tokens before the tree
    node = at[None] - before[:, None]                                                       # [b, keys]
    seen_node = ((st.masks[..., None] >> node.clamp(0, 63)[:, None]) & 1).bool() & ((node >= 0) & (node < t))[:, None]
    seen = (node < 0)[:, None] | seen_node                                                  # [b, t, keys]
    if w:  # the last w of the tokens that a node sees
        seen &= seen.flip(-1).cumsum(dim=-1).flip(-1) <= w
    seen &= (st.masks != 0)[..., None]
    seen = seen.repeat_interleave(m // t, dim=1)
    s = s.masked_fill_(~seen, -math.inf)
    e = (s - s.amax(dim=-1, keepdim=True).clamp_min(-3e38)).exp_()
    total = e.sum(dim=-1, keepdim=True)
    out = torch.matmul(e[..., :p].reshape(hk, b * m, p), vp).reshape(hk, b, m, d)
    out = out + torch.matmul(e[..., p:].transpose(0, 1).contiguous(), vo).transpose(0, 1)
    out = torch.where(total > 0, out / total, torch.zeros((), device="cuda"))
    return out.reshape(hk, b, t, m // t, d).permute(1, 2, 0, 3, 4).reshape(b * t, c["q_heads"], d).to(st.q.dtype)


# ---- what a pass cannot do without -------------------------------------------------------------------

def _stored(tokens, c):
    """Bytes of `tokens` tokens' keys and values in the cache."""
    return 2 * tokens * c["kv_heads"] * (c["head_dim"] * c["bits"] // 8 + 4 * c["head_dim"] // GROUP)


def work(case):
    c, kind = case, case["kind"]
    size = 2 if c.get("dtype") == "bf16" else 4
    if kind == "plan":
        b = c["batch"]
        new = sum(_lengths(c, 0, c["new_lo"], c["new_hi"]))
        n = b * c["row_tokens"] or new + c["spare"]
        # lengths and pages in, offsets and lengths out; a position and a slot (a parent and a mask) for each
        # token; the pages of the new tokens, out of the pool and into the tables
        return {"bytes": 24 * b + n * (20 if c["tree"] else 8) + 8 * (new // c["page"]), "flops": 2 * n}
    d = c["head_dim"]
    if kind == "prompt":
        w, pairs = c["window"], 0
        lengths = _lengths(c, 0, c["lo"], c["hi"])
        for n in lengths:
            m = min(n, w or n)
            pairs += m * (m + 1) // 2 + (n - m) * m
        return {"bytes": sum(lengths) * 2 * (c["q_heads"] + c["kv_heads"]) * d * size, "flops": 4 * d * c["q_heads"] * pairs}
    b, t = c["batch"], c["nodes"]
    if kind == "tree":
        w, p, keys, first = c["window"], c["prefix"], 0, 0
        depth = _depths(c, t)
        pairs = 0
        for n in _lengths(c, 0, c["own_lo"], c["own_hi"])[:b - c["padded"]]:
            pairs += sum(min(p + n + x, w or p + n + x) for x in depth)
            begin = max(0, p + n + 1 - w) if w else 0
            keys += n + t - min(n, max(0, begin - p))
            first = max(first, p - begin)
        return {"bytes": 2 * b * t * c["q_heads"] * d * size + _stored(first + keys, c), "flops": 4 * d * c["q_heads"] * pairs}
    n = b * t
    kv = n * c["kv_heads"] * d
    moved = b * min(t, 6)  # a path confirms a handful of nodes
    return {"bytes": 2 * kv * size + 2 * _stored(n, c) + 2 * _stored(moved, c) + 2 * kv * 2 + 32 * n, "flops": 12 * kv}


def _depths(c, t):
    """About how many tokens of the tree its nodes see, themselves included."""
    step = (c["reach"] + 1) / 2
    return [1 + int(x / step) for x in range(t)]


# ---- the same outputs from the definitions, in 64 bits -------------------------------------------------

def exact(case, seed):
    c, st = case, State(case)
    if c["kind"] == "plan":
        return None  # whole numbers
    if c["kind"] == "prompt":
        _prepare_prompt(c, seed, st)
        return _exact_prompt(c, st)
    if c["kind"] == "tree":
        _prepare_tree(c, seed, st)
        return _exact_tree(c, st)
    _prepare_keep(c, seed, st)
    k, v = (_exact_stored(x.double(), c["bits"]).unflatten(0, (c["batch"], c["nodes"])) for x in (st.k, st.v))
    for i, (parents, tokens, chosen) in enumerate(zip(st.parents.tolist(), st.tokens.tolist(), st.chosen.tolist())):
        path, at = [0], 0
        while at is not None:
            at = next((j for j in range(c["nodes"]) if parents[j] == at and tokens[j] == chosen[at]), None)
            path += [] if at is None else [at]
        for x in (k, v):
            x[i, :len(path)] = x[i, path].clone()
    return {"kept": None, "next": None, "length": None, "path": None, "from": None, "to": None, "k": k.flatten(0, 1),
            "v": v.flatten(0, 1)}


def _exact_prompt(c, st):
    hk, d, w = c["kv_heads"], c["head_dim"], c["window"]
    g = c["q_heads"] // hk
    out = torch.zeros(st.out.shape, dtype=torch.float64, device="cuda")
    first = 0
    for n in st.lengths:
        at = torch.arange(n, device="cuda")
        for h in range(hk):
            k, v = st.k[first:first + n, h].double(), st.v[first:first + n, h].double().contiguous()
            kt = k.t().contiguous() / math.sqrt(d)
            for head in range(h * g, (h + 1) * g):
                for lo in range(0, n, 4096):
                    rows = at[lo:lo + 4096]
                    hi = lo + rows.numel()
                    s = st.q[first + lo:first + hi, head].double() @ kt[:, :hi].contiguous()
                    hidden = at[None, :hi] > rows[:, None]
                    if w:
                        hidden |= at[None, :hi] <= rows[:, None] - w
                    out[first + lo:first + hi, head] = s.masked_fill_(hidden, -math.inf).softmax(dim=-1) @ v[:hi]
        first += n
    return out


def _next_bf16(x, up):
    """The nearest BF16 number that is not below (above) x, from the round-to-nearest one and its neighbour."""
    r = x.bfloat16()
    wrong = r.double() < x if up else r.double() > x
    return torch.where(wrong, torch.nextafter(r, torch.full_like(r, math.inf if up else -math.inf)), r).double()


def _exact_stored(x, bits):
    """What a cache of this width holds of x."""
    shape = x.shape
    x = x.reshape(*shape[:-1], shape[-1] // GROUP, GROUP)
    bias = _next_bf16(x.min(dim=-1).values, False)
    scale = _next_bf16((x.max(dim=-1).values - bias) / (2 ** bits - 1), True).clamp(min=2.0 ** -126)
    q = torch.round((x - bias[..., None]) / scale[..., None]).clamp(0, 2 ** bits - 1)
    return (q * scale[..., None] + bias[..., None]).reshape(shape)


def _exact_tree(c, st):
    """Sequence by sequence over the tokens in order, which is how they were laid out before the pages
    were shuffled: the prefix first, then each sequence's own, its tree last."""
    p, t, hk, d, w = c["prefix"], c["nodes"], c["kv_heads"], c["head_dim"], c["window"]
    g = c["q_heads"] // hk
    held = [_exact_stored(x.double(), c["bits"]) for x in st.all_kv]
    out = torch.zeros(c["batch"] * t, c["q_heads"], d, dtype=torch.float64, device="cuda")
    lo = p
    for i, n in enumerate(st.own_len):
        if n == 0:
            continue
        k, v = (torch.cat((x[:p], x[lo:lo + n])) for x in held)
        lo += n
        before = p + n - t
        seen = torch.ones((t, p + n), dtype=torch.bool, device="cuda")
        for node, mask in enumerate(st.masks[i].tolist()):
            seen[node, before:] = torch.tensor([bool(mask >> j & 1) for j in range(t)], device="cuda")
            if w:
                at = seen[node].nonzero()[:, 0]
                seen[node, at[:max(0, at.numel() - w)]] = False
        for h in range(hk):
            q = st.q[i * t:(i + 1) * t, h * g:(h + 1) * g].double().reshape(t * g, d)
            s = (q @ k[:, h].t().contiguous() / math.sqrt(d)).reshape(t, g, p + n)
            e = s.masked_fill(~seen[:, None], -math.inf).softmax(dim=-1).reshape(t * g, p + n)
            out[i * t:(i + 1) * t, h * g:(h + 1) * g] = (e @ v[:, h].contiguous()).reshape(t, g, d)
    return out
