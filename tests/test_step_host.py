"""The calls around a serving step without a GPU: struct layouts, refusals that come before a device is touched, the
binding's view of the arrays, and where a workgroup's LDS and tile numbers end."""
import ctypes as C

import pytest

import turbo_decode_tail as T

torch = pytest.importorskip("torch")
F32, BF16 = T.TURBO_HIDDEN_F32, T.TURBO_HIDDEN_BF16


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_struct_sizes():
    lib = T.load()
    for which, st in ((10, T.TurboBatchPlan), (11, T.TurboPagesRelease), (12, T.TurboTreeAccept), (13, T.TurboPromptInputs)):
        assert lib.turbo_abi_struct_size(which) == C.sizeof(st), st.__name__


def refused(call, inp, word):
    assert call(C.byref(inp), None) == 0
    assert word in T.last_error(), T.last_error()


KEEP = {k: i32(256) for k in ("a", "b", "c", "d", "e", "f", "g")}  # arrays that outlive the structs below


def plan(**kw):
    a = dict(page_tokens=64, past_len=KEEP["a"], new_len=KEEP["b"], max_tokens=20, pages=KEEP["c"].view(4, 64), held=KEEP["d"],
             free_pages=KEEP["e"], free_count=KEEP["f"], slots=KEEP["g"])
    a.update(kw)
    return T.make_batch_plan(4, **a)


@pytest.mark.parametrize("field,value,word", [
    ("batch", -1, "batch"), ("batch", 8193, "batch"), ("page_tokens", 48, "page_tokens"), ("page_tokens", 512, "page_tokens"),
    ("max_tokens", 2**28 + 1, "max_tokens"), ("past_len", None, "past_len"), ("new_len", None, "new_len"), ("held", None, "held"),
    ("held_out", None, "held_out"), ("pages", None, "pages"), ("free_pages", None, "free_pages"), ("free_count", None, "free_count"),
    ("free_count_out", None, "free_count_out"), ("row_tokens", 7, "batch * row_tokens"), ("page_stride", 2**31, "page_stride"),
    ("prefix_len", 2**31 - 255, "prefix_len"), ("past_len", 6, "aligned"), ("slots", 6, "aligned"), ("masks", 8, "parents")])
def test_plan_refuses(field, value, word):
    inp = plan()
    setattr(inp, field, value)
    refused(T.load().turbo_batch_plan, inp, word)


@pytest.mark.parametrize("result,taken", [("slots", "past_len"), ("kv_len", "new_len"), ("held_out", "past_len"), ("starts", "pages"),
                                          ("free_count_out", "held"), ("totals", "free_count"), ("kv_len", "slots"), ("positions", "slots")])
def test_plan_refuses_results_in_the_place_of_others(result, taken):
    inp = plan()
    setattr(inp, result, getattr(inp, taken))
    refused(T.load().turbo_batch_plan, inp, "of the plan")


@pytest.mark.parametrize("rows,word", [(0, "row_tokens"), (65, "row_tokens")])
def test_plan_refuses_trees_that_masks_do_not_hold(rows, word):
    inp = plan()
    inp.parents, inp.row_tokens, inp.max_tokens = KEEP["a"].data_ptr(), rows, 4 * rows or 20
    refused(T.load().turbo_batch_plan, inp, word)
    inp.row_tokens, inp.max_tokens, inp.masks = 5, 20, 12
    refused(T.load().turbo_batch_plan, inp, "8-byte")


@pytest.mark.parametrize("field,value,word", [("batch", 8193, "batch"), ("page_tokens", 33, "page_tokens"), ("keep_len", None, "keep_len"),
                                              ("pages", None, "pages"), ("held", None, "held"), ("free_pages", None, "free_pages"),
                                              ("free_count", None, "free_count"), ("held", 2, "aligned")])
def test_release_refuses(field, value, word):
    inp = T.TurboPagesRelease(4, 64, 0, KEEP["a"].data_ptr(), KEEP["b"].data_ptr(), 8, KEEP["c"].data_ptr(), KEEP["d"].data_ptr(),
                              KEEP["e"].data_ptr(), 9, 0)
    setattr(inp, field, value)
    refused(T.load().turbo_pages_release, inp, word)


@pytest.mark.parametrize("field,value,word", [
    ("batch", -1, "batch"), ("batch", 2**20 + 1, "batch"), ("row_tokens", 0, "row_tokens"), ("row_tokens", 65, "row_tokens"),
    ("parents", None, "parents"), ("new_len", None, "new_len"), ("tokens", None, "tokens"), ("chosen", None, "chosen"),
    ("kept", None, "kept"), ("next", None, "next"), ("length", 4, "past_len"), ("source", 4, "together"), ("target", 4, "together"),
    ("path", 5, "aligned")])
def test_accept_refuses(field, value, word):
    p = KEEP["a"].data_ptr()
    inp = T.TurboTreeAccept(2, 4, p, p, p, p, None, None, p, p, None, None, None, None, 0)
    setattr(inp, field, value)
    refused(T.load().turbo_tree_accept, inp, word)


def test_accept_refuses_moves_without_slots():
    p = KEEP["a"].data_ptr()
    refused(T.load().turbo_tree_accept, T.TurboTreeAccept(2, 4, p, p, p, p, None, None, p, p, None, None, p, p, 0), "slots")


def prompt(dtype=BF16, hq=4, hk=2, d=64):
    x = torch.zeros((9, hq + 2 * hk, d), dtype=torch.bfloat16 if dtype == BF16 else torch.float32)
    out = torch.zeros((9, hq, d), dtype=x.dtype)
    inp = T.make_prompt_inputs(2, 9, dtype=dtype, q=x[:, :hq], k=x[:, hq:hq + hk], v=x[:, hq + hk:], out=out, q_heads=hq, kv_heads=hk,
                               head_dim=d, starts=KEEP["a"], scale=0.1)
    return inp, (x, out)


@pytest.mark.parametrize("field,value,word", [
    ("batch", -1, "batch"), ("batch", 2**20 + 1, "batch"), ("tokens", -1, "tokens"), ("tokens", 2**28 + 1, "tokens"),
    ("q_heads", 0, "q_heads"), ("q_heads", 5, "q_heads"), ("q_heads", 8194, "q_heads"), ("kv_heads", 0, "kv_heads"),
    ("kv_heads", 1025, "kv_heads"), ("head_dim", 96, "head_dim"), ("dtype", 2, "dtype"), ("q", None, "q is"), ("k", None, "k is"),
    ("v", None, "v is"), ("out", None, "out is"), ("q_stride", 100, "q_stride"), ("k_stride", 127, "k_stride"),
    ("v_stride", 516, "v_stride"), ("out_stride", 2**24 + 8, "2^24"), ("starts", None, "starts"), ("starts", 7, "aligned"),
    ("scale", float("nan"), "scale"), ("scale", float("inf"), "scale"), ("scale", 3e38, "scale")])
def test_prompt_refuses(field, value, word):
    inp, keep = prompt()
    setattr(inp, field, value)
    refused(T.load().turbo_prompt_attention, inp, word)


def test_prompt_refuses_what_would_overlap_or_not_fit():
    lib = T.load()
    for name in ("q", "k", "v"):
        inp, keep = prompt()
        inp.out = getattr(inp, name)
        refused(lib.turbo_prompt_attention, inp, "out is")
    inp, keep = prompt()
    inp.v += 8
    refused(lib.turbo_prompt_attention, inp, "16-byte")
    inp, keep = prompt()
    inp.tokens, inp.q_heads, inp.kv_heads = 2**28, 64, 1
    refused(lib.turbo_prompt_attention, inp, "too large")


def test_tree_and_move_refuse():
    lib = T.load()
    assert lib.turbo_tree_attention(None, None, None, None) == 0 and "handle" in T.last_error()
    assert lib.turbo_kv_cache_move(None, None, None, 1, 1, None) == 0 and "handle" in T.last_error()
    for name in ("turbo_batch_plan", "turbo_pages_release", "turbo_tree_accept", "turbo_prompt_attention"):
        assert getattr(lib, name)(None, None) == 0 and "NULL" in T.last_error()


class Library:
    def __getattr__(self, name):
        return lambda *args: pytest.fail(f"{name} was called")


def test_binding_refuses_arrays_of_another_kind():
    c = object.__new__(T.KvCache)
    c.lib, c.h = Library(), None
    with pytest.raises(ValueError, match="32-bit"):
        c.move(torch.zeros((2, 3), dtype=torch.int64), torch.zeros((2, 3), dtype=torch.int64))
    for a, b in ((i32(2, 3), i32(3, 2)), (i32(6), i32(6))):
        with pytest.raises(ValueError, match="width"):
            c.move(a, b)
    with pytest.raises(ValueError, match="32-bit"):
        c.move(i32(2, 6)[:, :3], i32(2, 3))
    q = torch.zeros((6, 2, 64))
    inp = T.KvCache.make_attention_inputs(2, q=q, out=torch.zeros_like(q), q_heads=2, q_len=3, kv_len=i32(2), max_kv_len=9, scale=1.0)
    for bad in (i32(2, 3), torch.zeros((2, 3)).double(), torch.zeros((2, 2), dtype=torch.int64), torch.zeros((2, 6), dtype=torch.int64)[:, ::2]):
        with pytest.raises(ValueError, match="64-bit"):
            c.attend_tree(inp, bad)
    with pytest.raises(ValueError, match="past_len"):
        plan(past_len=i32(3))
    with pytest.raises(ValueError, match="slots"):
        plan(slots=i32(19))
    with pytest.raises(ValueError, match="page_stride"):
        plan(pages=i32(3, 64))
    with pytest.raises(ValueError, match="32-bit"):
        plan(new_len=torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="starts"):
        T.make_prompt_inputs(2, 6, q=q, k=q, v=q, out=q, q_heads=2, kv_heads=2, head_dim=64, starts=i32(2), scale=1.0)
    with pytest.raises(ValueError, match="element size"):
        T.make_prompt_inputs(1, 6, dtype=BF16, q=q, k=q, v=q, out=q, q_heads=2, kv_heads=2, head_dim=64, starts=i32(2), scale=1.0)
    with pytest.raises(ValueError, match="fewer"):
        T.make_prompt_inputs(1, 7, q=q, k=q, v=q, out=q, q_heads=2, kv_heads=2, head_dim=64, starts=i32(2), scale=1.0)
    with pytest.raises(ValueError, match="fewer"):
        T.make_prompt_inputs(1, 6, q=q, k=q, v=q, out=q, q_heads=4, kv_heads=2, head_dim=64, starts=i32(2), scale=1.0)
    with pytest.raises(ValueError, match="tokens"):
        T.make_tree_accept(2, 4, parents=i32(8), new_len=i32(2), tokens=i32(7), chosen=i32(8), kept=i32(2), next=i32(2))
