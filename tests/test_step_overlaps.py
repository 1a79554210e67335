"""Arrays of the calls around a serving step that lie on each other, refused before a device is touched: a call reads some of them
while it writes others."""
import ctypes as C

import pytest

import turbo_decode_tail as T

torch = pytest.importorskip("torch")
WORDS = torch.zeros(4096, dtype=torch.int32)


def at(word):
    return WORDS.data_ptr() + 4 * word


def plan():
    """Four sequences with tables of 8 pages, 20 tokens in rows of 5, everything apart."""
    return T.TurboBatchPlan(4, 64, 0, at(0), at(4), 5, 20, at(8), at(32), 8, at(64), at(70), at(170), 100, at(180), at(190), at(200), at(210),
                            at(220), at(240), at(260), at(300), 99)


def release():
    return T.TurboPagesRelease(4, 64, 0, at(0), at(8), 8, at(40), at(50), at(160), 100, 99)


def accept():
    """Two trees of 4 nodes."""
    return T.TurboTreeAccept(2, 4, at(0), at(8), at(10), at(18), at(26), at(28), at(40), at(42), at(44), at(50), at(58), at(66), 99)


def answer(call, inp):
    assert call(C.byref(inp), None) == 0
    return T.last_error()


@pytest.mark.parametrize("make,call", [(plan, "turbo_batch_plan"), (release, "turbo_pages_release"), (accept, "turbo_tree_accept")])
def test_what_lies_apart_goes_on_to_the_device(make, call):
    assert "device" in answer(getattr(T.load(), call), make()).lower()


@pytest.mark.parametrize("field,word,of", [
    ("kv_len", 1, "of the plan"),           # past_len, but one further
    ("kv_len", 3, "of the plan"), ("held_out", 65, "of the plan"), ("held_out", 61, "of the plan"), ("starts", 60, "of the plan"),
    ("positions", 51, "of the plan"), ("slots", 225, "of the plan"), ("masks", 28, "of the plan"), ("masks", 266, "of the plan"),
    ("totals", 169, "of the plan"), ("free_count_out", 169, "of the plan"), ("free_count_out", 183, "of the plan"), ("starts", 179, "of the plan"),
    ("pages", 39, "of the plan"), ("pages", 60, "of the plan"), ("pages", 1, "of the plan")])
def test_plan(field, word, of):
    inp = plan()
    setattr(inp, field, at(word))
    assert of in answer(T.load().turbo_batch_plan, inp)


@pytest.mark.parametrize("fields", [{"held_out": 64}, {"free_count_out": 170}, {"kv_len": 0}, {"held_out": 64, "free_count_out": 170, "kv_len": 0},
                                    {"starts": None, "kv_len": None, "positions": None, "slots": None, "masks": None, "totals": None}])
def test_plan_in_place(fields):
    inp = plan()
    for k, v in fields.items():
        setattr(inp, k, None if v is None else at(v))
    assert "device" in answer(T.load().turbo_batch_plan, inp).lower()


@pytest.mark.parametrize("field,word", [("held", 3), ("held", 39), ("held", 0), ("free_pages", 20), ("free_pages", 41), ("free_count", 2),
                                        ("free_count", 149), ("pages", 42), ("keep_len", 160)])
def test_release(field, word):
    inp = release()
    setattr(inp, field, at(word))
    assert "of the release" in answer(T.load().turbo_pages_release, inp)


@pytest.mark.parametrize("field,word", [("kept", 9), ("kept", 10), ("next", 41), ("length", 27), ("path", 1), ("path", 59), ("source", 65),
                                        ("target", 35), ("next", 0)])
def test_accept(field, word):
    inp = accept()
    setattr(inp, field, at(word))
    assert "of the tree" in answer(T.load().turbo_tree_accept, inp)


@pytest.mark.parametrize("fields", [{"length": 26}, {"kept": 8}, {"path": 10}, {"target": 28, "length": 26}, {"path": None, "length": None}])
def test_accept_in_place(fields):
    inp = accept()
    for k, v in fields.items():
        setattr(inp, k, None if v is None else at(v))
    assert "device" in answer(T.load().turbo_tree_accept, inp).lower()
