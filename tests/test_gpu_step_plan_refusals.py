"""Refusals of the calls around a serving step that need a cache."""
import pytest

torch = pytest.importorskip("torch")
import turbo_decode_tail as T

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["source", "target"])
def test_moves_refuse_slots_that_are_not_words(name):
    cache = T.KvCache(2, 32, 1, 64)
    slots = torch.zeros(64, dtype=torch.int32, device="cuda")
    args = {"source": slots.data_ptr(), "target": slots.data_ptr() + 128}
    for off, word in ((1, "aligned"), (2, "aligned"), (None, "NULL")):
        bad = dict(args)
        bad[name] = None if off is None else args[name] + off
        assert cache.lib.turbo_kv_cache_move(cache.h, bad["source"], bad["target"], 2, 4, None) == 0
        assert f"{name} " in T.last_error() and word in T.last_error()
    cache.close()
