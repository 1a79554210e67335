"""The attention side of a layer loop over int4 projections, as cases that can be timed and compared.

A case is a dict of plain values. `prepare` makes what the caller holds before the call, `run` makes
one pass in plain torch operations or, with `own` set, through the entry points of turbo_decode_tail,
`exact` gives the same outputs from the definitions in 64 bits.

Kinds
  rotary     norms of the query and key heads and the position rotation in one pass
  cache      keys and values quantised into a paged cache (affine, groups of 64 values, BF16 scale
             and bias, 4 or 8 bits), then the same tokens read back
  append     both at once: norms and rotation, the keys and values quantised into the cache as they
             are made, then read back
  attention  a batch of sequences over the cache; all of them share a prefix that is stored once

Heads of 256 (16 queries, 8 key/value heads) are those of the benchmark's 4,096 x 2,816 projection;
the other head sizes and ratios are generic.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-6
GROUP = 64


# ---- the cases ---------------------------------------------------------------------------------

def _rotary(**kw):
    c = {"kind": "rotary", "tokens": 1, "q_heads": 16, "kv_heads": 8, "head_dim": 256, "rotary_dim": 256,
         "layout": "halves", "theta": 10000.0, "dtype": "bf16", "far": 4096, "consecutive": False, "packed": False}
    c.update(kw)
    return c


def _cache(**kw):
    c = {"kind": "cache", "tokens": 64, "kv_heads": 8, "head_dim": 256, "bits": 8, "page": 64, "dtype": "bf16",
         "consecutive": False}
    c.update(kw)
    return c


def _append(**kw):
    c = _rotary(packed=True, bits=8, page=64)
    c.update(kind="append", **kw)
    return c


def _attention(**kw):
    c = {"kind": "attention", "batch": 1, "q_len": 1, "q_heads": 16, "kv_heads": 8, "head_dim": 256, "bits": 8,
         "page": 64, "prefix": 0, "own_lo": 1, "own_hi": 1, "window": 0, "dtype": "bf16", "padded": 0}
    c.update(kw)
    return c


def listed():
    return [
        # one decoded token between its projections and its attention: launch and one round trip
        _rotary(name="rotary_decode_1", dtype="f32"),
        # a prompt of 2,048 tokens
        _rotary(name="rotary_prompt_2048", tokens=2048, consecutive=True),
        # a ragged batch far into long contexts: half of each head rotates, neighbours as pairs, the
        # heads are slices of one projection's output
        _rotary(name="rotary_far_777", tokens=777, q_heads=20, kv_heads=4, head_dim=128, rotary_dim=64, layout="pairs",
                theta=1e6, dtype="f32", far=4000000, packed=True),
        # a decode step's keys and values, each to its own sequence's page
        _cache(name="cache_decode_64", tokens=64, bits=4),
        # a prompt written from the middle of a page on
        _cache(name="cache_prompt_4001", tokens=4001, consecutive=True),
        # a decode step of 32 sequences, straight from the projections to the cache
        _append(name="append_decode_32", tokens=32),
        # a chunk of a prompt, the same way
        _append(name="append_chunk_1500", tokens=1500, consecutive=True, rotary_dim=128),
        # interactive decoding of one sequence, 32-bit activations
        _attention(name="attend_1x2000", own_lo=2000, own_hi=2000, dtype="f32"),
        # eight drafted tokens checked at once for each of seven sequences, local layer, 4-bit cache
        _attention(name="attend_drafts_7x8", batch=7, q_len=8, q_heads=32, kv_heads=4, head_dim=128, bits=4, page=32,
                   prefix=1111, own_lo=40, own_hi=1700, window=1024),
        # a global layer: wide heads, eight queries to a key/value head, padded batch
        _attention(name="attend_wide_16", batch=16, kv_heads=2, head_dim=512, page=128, prefix=6000, own_lo=9, own_hi=900,
                   padded=2),
        # a chunk of 512 prompt tokens after a shared prefix
        _attention(name="attend_chunk_512", q_len=512, prefix=4096, own_lo=700, own_hi=700),
        # a server's batch behind one long system prompt: the largest
        _attention(name="attend_shared_64", batch=64, prefix=32768, own_lo=1, own_hi=2000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choices(["rotary", "cache", "append", "attention"], [20, 20, 15, 45])[0]
    dim = rng.choice([64, 128, 128, 256, 256, 512])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 8])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    page = rng.choice([32, 64, 128, 256])
    if kind in ("rotary", "append"):
        c = dict(tokens=_log(rng, 1, 4096), q_heads=heads, kv_heads=kv, head_dim=dim,
                 rotary_dim=rng.choice([dim, dim, dim // 2, 32]), layout=rng.choice(["halves", "pairs"]),
                 theta=rng.choice([1e4, 5e5, 1e6]), dtype=dtype, far=_log(rng, 4096, 4000000),
                 consecutive=rng.random() < 0.5)
        if kind == "rotary":
            return _rotary(**c, packed=rng.random() < 0.5)
        if not c["consecutive"]:
            c["tokens"] = _log(rng, 1, 256)
        return _append(**c, page=page)
    if kind == "cache":  # one run of a prompt, or a decode step's tokens
        together = rng.random() < 0.5
        return _cache(tokens=_log(rng, 1, 8192 if together else 256), kv_heads=kv, head_dim=dim, bits=rng.choice([4, 8]),
                      page=page, dtype=dtype, consecutive=together)
    shape = rng.choices(["decode", "drafts", "chunk"], [60, 20, 20])[0]
    q_len = {"decode": 1, "drafts": rng.randint(2, 16), "chunk": _log(rng, 17, 700)}[shape]
    batch = _log(rng, 1, 2 if shape == "chunk" else 128)
    prefix = rng.choice([0, _log(rng, 1, 32768), _log(rng, 256, 32768)])
    hi = q_len + _log(rng, 1, 4000)
    lo = rng.choice([q_len, hi, rng.randint(q_len, hi)])
    return _attention(batch=batch, q_len=q_len, q_heads=heads, kv_heads=kv, head_dim=dim, bits=rng.choice([4, 8, 8]),
                      page=page, prefix=prefix, own_lo=lo, own_hi=hi, window=rng.choice([0, 0, 0, _log(rng, 64, 8192)]),
                      dtype=dtype, padded=min(batch - 1, rng.choice([0, 0, 1, 3])))


def draw(rng):
    """One more case of the same ranges: 1 to thousands of tokens, batches up to 128, prefixes up to
    32,768 tokens, every head size, ratio, width and layout; at most the largest listed case's work."""
    most = _price(listed()[-1])
    while True:
        c = _draw(rng)
        if _price(c) <= most:
            return c


def _price(c):
    """Seconds the plain form would take, roughly: the larger of its work at plain rates, and for an
    attention the dequantised copies and score tables that it makes."""
    w = work(c)
    s = max(w["bytes"] / 1e11, w["flops"] / 2e13)
    if c["kind"] == "attention":
        keys = c["prefix"] + c["batch"] * c["own_hi"]
        rows = c["batch"] * c["q_len"] * c["q_heads"]
        s = max(s, (keys * c["kv_heads"] * c["head_dim"] * 32 + rows * (c["prefix"] + c["own_hi"]) * 24) / 1e12)
    return s


# ---- inputs, from the seed alone -----------------------------------------------------------------

def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + what) & 0x7FFFFFFFFFFFFFFF)
    return g


def _randn(shape, g):
    return torch.randn(shape, generator=g, device="cuda")


def _cast(x, dtype):
    return x.bfloat16().contiguous() if dtype == "bf16" else x.contiguous()


def _code(dtype):
    return T().TURBO_HIDDEN_BF16 if dtype == "bf16" else T().TURBO_HIDDEN_F32


def T():
    """The framework's binding; only the passes through the framework's own calls need it."""
    pkg = str(Path(__file__).resolve().parents[1] / "turbo-winfare_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import turbo_decode_tail
    return turbo_decode_tail


def _keys_values(tokens, c, g):
    """Keys with a few strong channels, as trained keys have them, and values without."""
    shape = (tokens, c["kv_heads"], c["head_dim"])
    k = _randn(shape, g) * 0.7 + _randn(shape[1:], g) * 0.7
    return k, _randn(shape, g)


def _freqs(c):
    """theta^(-2i / R) in 64 bits."""
    i = torch.arange(c["rotary_dim"] // 2, device="cuda", dtype=torch.float64)
    return c["theta"] ** (-2.0 * i / c["rotary_dim"])


def _positions(c, g):
    n = c["tokens"]
    if c["consecutive"]:
        start = int(torch.randint(0, c["far"], (1,), generator=g, device="cuda").item())
        return torch.arange(start, start + n, device="cuda", dtype=torch.int32)
    return torch.randint(0, c["far"], (n,), generator=g, device="cuda", dtype=torch.int32)


def _slots(c, g):
    """The places of `tokens` tokens in a cache, and the number of its pages: one run through pages in
    shuffled order that begins inside its first page, or every token in a sequence of its own."""
    n, page = c["tokens"], c["page"]
    if c["consecutive"]:
        pages = (n + page - 1) // page + 2
        order = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(n, device="cuda") + int(torch.randint(0, page, (1,), generator=g, device="cuda").item())
        return (order[at // page] * page + at % page).to(torch.int32), pages
    order = torch.randperm(2 * n, generator=g, device="cuda")[:n]
    at = torch.randint(0, page, (n,), generator=g, device="cuda")
    return (order * page + at).to(torch.int32), 2 * n


def _own_lengths(c, seed):
    """Own tokens of each sequence, the queries' included: spread evenly over the range (so that the
    work does not depend on the seed), in a random order; padded sequences have none and see nothing."""
    n = c["batch"] - c["padded"]
    own = [c["own_hi"] - (c["own_hi"] - c["own_lo"]) * i // max(1, n - 1) for i in range(n)]
    order = torch.randperm(c["batch"], generator=torch.Generator().manual_seed(seed)).tolist()
    spread = own + [None] * c["padded"]
    return [spread[i] for i in order]


class State:
    """What the program holds."""

    def __init__(self, case):
        self.case = case


def prepare(case, seed):
    c, st = case, State(case)
    kind = c["kind"]
    if kind in ("rotary", "append"):
        n, hq, hk, d = c["tokens"], c["q_heads"], c["kv_heads"], c["head_dim"]
        g = _gen(seed, 1)
        parts = [_randn((n, hq, d), g) * 2.0, _randn((n, hk, d), g) * 2.0, _randn((n, hk, d), g)]
        if c["packed"]:  # one projection's output, the heads are slices of it
            rows = _cast(torch.cat(parts, dim=1), c["dtype"])
            st.q, st.k, st.v = rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:]
        else:
            st.q, st.k, st.v = (_cast(p, c["dtype"]) for p in parts)
        st.q_norm, st.k_norm = ((1.0 + 0.2 * _randn((d,), g)).bfloat16() for _ in range(2))
        st.positions = _positions(c, g)
        st.freqs = _freqs(c)
    if kind in ("cache", "append"):
        n, hk, d = c["tokens"], c["kv_heads"], c["head_dim"]
        g = _gen(seed, 2)
        st.slots, st.pages = _slots(c, g)
        if kind == "cache":
            st.k, st.v = (_cast(x, c["dtype"]) for x in _keys_values(n, c, g))
    if kind == "attention":
        _prepare_attention(c, seed, st)
    if own:
        _prepare_own(c, st)
    elif kind in ("cache", "append"):
        st.store = _plain_store(st.pages * c["page"], c)
    elif kind == "attention":
        st.store = _plain_store(st.pages * c["page"], c)
        _plain_write(st.store, st.all_slots.long(), *st.all_kv, c["bits"])
        st.slot_table = _slot_table(st, c)
    if kind == "attention":
        del st.all_kv, st.all_slots
    torch.cuda.synchronize()
    return st


def _prepare_attention(c, seed, st):
    """Queries, a cache's contents and the page tables: pages of the prefix and of every sequence in
    shuffled order, the tables' unused ends filled with page 0."""
    g = _gen(seed, 3)
    b, page, d = c["batch"], c["page"], c["head_dim"]
    st.own_len = _own_lengths(c, seed)
    st.kv_len = torch.tensor([0 if n is None else c["prefix"] + n for n in st.own_len], dtype=torch.int32, device="cuda")
    st.q = _cast(_randn((b * c["q_len"], c["q_heads"], d), g) * 1.5, c["dtype"])
    need_p = -(-c["prefix"] // page)
    need = [-(-(n or 0) // page) for n in st.own_len]
    st.pages = max(1, need_p + sum(need))
    order = torch.randperm(st.pages, generator=g, device="cuda").to(torch.int32)
    st.prefix_pages = order[:need_p].contiguous()
    width = max(1, max(need))
    takes = torch.arange(width, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    st.own_pages = torch.zeros((b, width), dtype=torch.int32, device="cuda")
    st.own_pages[takes] = order[need_p:need_p + sum(need)]
    at = torch.arange(width * page, device="cuda")[None].expand(b, -1)
    written = at < torch.tensor([n or 0 for n in st.own_len], device="cuda")[:, None]
    slots = st.own_pages.long().repeat_interleave(page, dim=1) * page + at % page
    at = torch.arange(c["prefix"], device="cuda")
    st.all_slots = torch.cat([st.prefix_pages.long()[at // page] * page + at % page, slots[written]]).to(torch.int32)
    st.all_kv = [x.bfloat16() for x in _keys_values(st.all_slots.numel(), c, g)]


def _prepare_own(c, st):
    """Handles, output buffers and argument blocks that a program sets up once."""
    t, kind, code = T(), c["kind"], _code(c["dtype"])
    if kind in ("rotary", "append"):
        st.rotary = t.Rotary(c["head_dim"], rotary_dim=c["rotary_dim"], theta=c["theta"], eps=EPS,
                             layout=t.TURBO_ROPE_PAIRS if c["layout"] == "pairs" else t.TURBO_ROPE_HALVES,
                             q_norm=st.q_norm, k_norm=st.k_norm)
        st.q_out = torch.empty(st.q.shape, dtype=st.q.dtype, device="cuda")
    if kind in ("cache", "append", "attention"):
        st.cache = t.KvCache(st.pages, c["page"], c["kv_heads"], c["head_dim"], bits=c["bits"])
    if kind in ("cache", "append"):
        st.k_out, st.v_out = (torch.empty(st.k.shape, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    if kind == "rotary":
        st.k_out = torch.empty(st.k.shape, dtype=st.k.dtype, device="cuda")
        st.inp = st.rotary.make_inputs(c["tokens"], dtype=code, q=st.q, k=st.k, q_heads=c["q_heads"], kv_heads=c["kv_heads"],
                                       positions=st.positions, q_out=st.q_out, k_out=st.k_out)
    elif kind == "append":
        st.inp = st.rotary.make_inputs(c["tokens"], dtype=code, q=st.q, k=st.k, v=st.v, q_heads=c["q_heads"],
                                       kv_heads=c["kv_heads"], positions=st.positions, q_out=st.q_out, cache=st.cache,
                                       slots=st.slots)
    elif kind == "attention":
        st.cache.write(st.all_kv[0], st.all_kv[1], st.all_slots, st.all_slots.numel(), dtype=t.TURBO_HIDDEN_BF16)
        st.out = torch.empty(st.q.shape, dtype=st.q.dtype, device="cuda")
        st.inp = st.cache.make_attention_inputs(c["batch"], dtype=code, q=st.q, out=st.out, q_heads=c["q_heads"],
                                                q_len=c["q_len"], kv_len=st.kv_len, max_kv_len=c["prefix"] + c["own_hi"],
                                                pages=st.own_pages, prefix_len=c["prefix"], prefix_pages=st.prefix_pages,
                                                window=c["window"], scale=c["head_dim"] ** -0.5)
        st.workspace = torch.empty(max(1, st.cache.attention_workspace(st.inp)), dtype=torch.uint8, device="cuda")
        st.inp.workspace, st.inp.workspace_bytes = st.workspace.data_ptr(), st.workspace.numel()


# ---- one pass --------------------------------------------------------------------------------------

def run(st):
    c, kind = st.case, st.case["kind"]
    if own:
        code = T().TURBO_HIDDEN_BF16
        if kind == "rotary":
            st.rotary.apply(st.inp)
            return {"q": st.q_out, "k": st.k_out}
        if kind == "cache":
            st.cache.write(st.k, st.v, st.slots, c["tokens"], dtype=_code(c["dtype"]))
            st.cache.read(st.slots, c["tokens"], st.k_out, st.v_out, dtype=code)
            return {"k": st.k_out, "v": st.v_out}
        if kind == "append":
            st.rotary.apply(st.inp)
            st.cache.read(st.slots, c["tokens"], st.k_out, st.v_out, dtype=code)
            return {"q": st.q_out, "k": st.k_out, "v": st.v_out}
        st.cache.attend(st.inp)
        return st.out
    if kind == "attention":
        return _plain_attention(st).to(st.q.dtype)
    if kind == "cache":
        slots = st.slots.long()
        _plain_write(st.store, slots, st.k, st.v, c["bits"])
        k, v = _plain_read(st.store, slots)
        return {"k": k.bfloat16(), "v": v.bfloat16()}
    angle = st.positions.double()[:, None] * st.freqs[None]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _plain_rotate(_plain_norm(st.q, st.q_norm), cos, sin, c)
    k = _plain_rotate(_plain_norm(st.k, st.k_norm), cos, sin, c)
    if kind == "rotary":
        return {"q": q.to(st.q.dtype), "k": k.to(st.k.dtype)}
    slots = st.slots.long()
    _plain_write(st.store, slots, k, st.v, c["bits"])
    k, v = _plain_read(st.store, slots)
    return {"q": q.to(st.q.dtype), "k": k.bfloat16(), "v": v.bfloat16()}


def _plain_norm(x, w):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * w.float()


def _plain_rotate(x, cos, sin, c):
    r = c["rotary_dim"]
    if c["layout"] == "pairs":
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., r:]), dim=-1)


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
    """Codes, scale and bias of every group of 64 values. The quotients are taken in 64 bits: 16-bit values
    fall on a border between two codes or two scales often, and a division by way of a 32-bit reciprocal
    would decide those by its rounding."""
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
    page = c["page"]
    at = torch.arange(c["prefix"], device="cuda")
    prefix = st.prefix_pages.long()[at // page] * page + at % page
    at = torch.arange(c["own_hi"], device="cuda")
    return prefix, st.own_pages.long()[:, at // page] * page + at % page


def _plain_attention(st):
    """Scores against the prefix as one product per key/value head over the rows of the whole batch,
    against the sequences' own keys as one per sequence and head; one softmax over both."""
    c = st.case
    b, t, hk, d, p = c["batch"], c["q_len"], c["kv_heads"], c["head_dim"], c["prefix"]
    m = t * (c["q_heads"] // hk)
    pre, mine = st.slot_table
    kp, vp = (x.transpose(0, 1).contiguous() for x in _plain_read(st.store, pre))          # [hk, p, d]
    ko, vo = (x.transpose(1, 2).contiguous() for x in _plain_read(st.store, mine))         # [b, hk, n, d]
    q = st.q.float().reshape(b, t, hk, m // t, d).permute(2, 0, 1, 3, 4).reshape(hk, b, m, d) * d ** -0.5
    sp = torch.matmul(q.reshape(hk, b * m, d), kp.transpose(1, 2).contiguous()).reshape(hk, b, m, p)
    so = torch.matmul(q.transpose(0, 1).contiguous(), ko.transpose(2, 3).contiguous()).transpose(0, 1)
    s = torch.cat((sp, so), dim=-1)
    del sp, so
    at = torch.arange(p + c["own_hi"], device="cuda")
    last = st.kv_len[:, None] - t + torch.arange(t, device="cuda")                          # [b, t]
    seen = at <= last[..., None]
    if c["window"]:
        seen &= at > last[..., None] - c["window"]
    seen = seen.repeat_interleave(m // t, dim=1)                                            # [b, m, keys]
    s = s.masked_fill_(~seen, -math.inf)
    e = (s - s.amax(dim=-1, keepdim=True).clamp_min(-3e38)).exp_()
    total = e.sum(dim=-1, keepdim=True)
    out = torch.matmul(e[..., :p].reshape(hk, b * m, p), vp).reshape(hk, b, m, d)
    out = out + torch.matmul(e[..., p:].transpose(0, 1).contiguous(), vo).transpose(0, 1)
    out = torch.where(total > 0, out / total, torch.zeros((), device="cuda"))
    return out.reshape(hk, b, t, m // t, d).permute(1, 2, 0, 3, 4).reshape(b * t, c["q_heads"], d)


# ---- what a pass cannot do without -------------------------------------------------------------------

def _stored(tokens, c):
    """Bytes of `tokens` tokens' keys and values in the cache."""
    return 2 * tokens * c["kv_heads"] * (c["head_dim"] * c["bits"] // 8 + 4 * c["head_dim"] // GROUP)


def work(case):
    c, kind = case, case["kind"]
    size = 2 if c["dtype"] == "bf16" else 4
    d = c["head_dim"]
    if kind == "attention":
        rows = c["batch"] * c["q_len"]
        keys = pairs = first = 0
        for n in _own_lengths(c, 0):
            if n is None:
                continue
            for last in range(c["prefix"] + n - c["q_len"], c["prefix"] + n):
                pairs += min(last + 1, c["window"] or last + 1)
            begin = max(0, c["prefix"] + n - c["q_len"] + 1 - c["window"]) if c["window"] else 0
            keys += n - max(0, begin - c["prefix"])
            first = max(first, c["prefix"] - begin)
        return {"bytes": 2 * rows * c["q_heads"] * d * size + _stored(first + keys, c), "flops": 4 * d * c["q_heads"] * pairs}
    n = c["tokens"]
    q, kv = n * c["q_heads"] * d if "q_heads" in c else 0, n * c["kv_heads"] * d
    if kind == "rotary":
        return {"bytes": 2 * (q + kv) * size + 4 * n, "flops": 10 * (q + kv)}
    back = 2 * kv * 2 + 2 * _stored(n, c) + 4 * n  # written, read, handed out
    if kind == "cache":
        return {"bytes": 2 * kv * size + back, "flops": 12 * kv}
    return {"bytes": (2 * q + 2 * kv) * size + back, "flops": 10 * (q + kv) + 12 * kv}


# ---- the same outputs from the definitions, in 64 bits -------------------------------------------------

def exact(case, seed):
    global own
    c = case
    was, own = own, False
    try:
        if c["kind"] == "attention":
            st = State(c)
            _prepare_attention(c, seed, st)
            return _exact_attention(c, st)
        st = prepare(c, seed)
    finally:
        own = was
    out = {}
    if c["kind"] != "cache":
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           st.positions.double()[:, None] * st.freqs)[:, None]
        rotated = [_exact_rotate(x, w, turn, c) for x, w in ((st.q, st.q_norm), (st.k, st.k_norm))]
        out["q"] = rotated[0]
        if c["kind"] == "rotary":
            return {**out, "k": rotated[1]}
    k = st.k.double() if c["kind"] == "cache" else rotated[1]
    return {**out, "k": _exact_stored(k, c["bits"]), "v": _exact_stored(st.v.double(), c["bits"])}


def _exact_rotate(x, w, turn, c):
    x = x.double()
    x = x / (x.pow(2).sum(-1, keepdim=True) / c["head_dim"] + EPS).sqrt() * w.double()
    r = c["rotary_dim"]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if c["layout"] == "pairs" else (x[..., :r // 2], x[..., r // 2:r])
    z = torch.complex(a.contiguous(), b.contiguous()) * turn
    y = x.clone()
    if c["layout"] == "pairs":
        y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
    else:
        y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
    return y


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


def _exact_attention(c, st):
    """Sequence by sequence over the tokens in order, which is how they were laid out before the pages
    were shuffled: the prefix first, then each sequence's own."""
    p, t, hk, d = c["prefix"], c["q_len"], c["kv_heads"], c["head_dim"]
    g = c["q_heads"] // hk
    stored = [_plain_quantise(x, c["bits"]) for x in st.all_kv]  # the codes are this operator's inputs

    def values(which, lo, hi):
        codes, scale, bias = (x[lo:hi] for x in stored[which])
        x = codes.double().reshape(hi - lo, hk, d // GROUP, GROUP) * scale.double()[..., None] + bias.double()[..., None]
        return x.reshape(hi - lo, hk, d)

    shared = [values(i, 0, p) for i in range(2)]
    out = torch.zeros(c["batch"] * t, c["q_heads"], d, dtype=torch.float64, device="cuda")
    lo = p
    for i, n in enumerate(st.own_len):
        if n is None:
            continue
        k, v = (torch.cat((shared[j], values(j, lo, lo + n))) for j in range(2))
        lo += n
        at, last = torch.arange(p + n, device="cuda"), p + n - t + torch.arange(t, device="cuda")
        hidden = at[None] > last[:, None]
        if c["window"]:
            hidden |= at[None] <= last[:, None] - c["window"]
        for h in range(hk):
            q = st.q[i * t:(i + 1) * t, h * g:(h + 1) * g].double().reshape(t * g, d)
            s = (q @ k[:, h].t().contiguous() / math.sqrt(d)).reshape(t, g, p + n)
            w = s.masked_fill(hidden[:, None], -math.inf).softmax(dim=-1).reshape(t * g, p + n)
            out[i * t:(i + 1) * t, h * g:(h + 1) * g] = (w @ v[:, h].contiguous()).reshape(t, g, d)
    return out
