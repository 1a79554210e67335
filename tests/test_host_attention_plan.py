"""How attention calls are split, from the library's own host code compiled here (csrc/dt_plan.h), for a card of 256
compute units: the partial results that the join reads are those that the kernels of the form that was chosen write."""
import itertools
import random
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
FIELDS = ("prefix_tile_rows", "own_tile_rows", "prefix_tiles", "prefix_splits", "own_tiles", "own_splits", "wide_tiles",
          "wide_splits", "wide_items", "prefix_items", "items", "rows", "parts", "stats_bytes", "bytes")
PROGRAM = """
#include <cstdio>
#include "dt_plan.h"
int main() {
    unsigned long long v[11];
    auto next = [&] {
        for (unsigned long long& x : v)
            if (std::scanf("%%llu", &x) != 1) return false;
        return true;
    };
    while (next()) {
        const tdt::AttnPlan p = tdt::plan_attention(v[0], v[1], v[2], v[3], v[4], v[5] == 0u, v[6], v[7], v[8], 256u, v[9] != 0u, v[10]);
        const unsigned long long out[] = {%s};
        for (unsigned long long x : out) std::printf("%%llu ", x);
        std::puts("");
    }
}
""" % ", ".join("p." + f for f in FIELDS)
F32, BF16 = 0, 1


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    """Plans of shapes (batch, q_len, q_heads, kv_heads, head_dim, dtype, prefix, own tokens, window, tree) and, where it is
    given, the partial results that a tree may leave, in bytes."""
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++20", "-O2", f"-I{ROOT / 'turbo-winfare_amd' / 'csrc'}", str(d / "plan.cpp"),
                    "-o", str(d / "plan")], check=True)

    def run(shapes):
        text = "\n".join(" ".join(str(int(x)) for x in (*s, 2**64 - 1)[:11]) for s in shapes)
        out = subprocess.run([str(d / "plan")], input=text, check=True, capture_output=True, text=True).stdout.splitlines()
        assert len(out) == len(shapes)
        return [dict(zip(FIELDS, map(int, line.split()))) for line in out]

    return run


def parts_written(shape, p):
    """Numbers of the partial results of a row that the kernels write, by the workgroups that a call has."""
    batch, q_len, q_heads, kv_heads = shape[:4]
    rows = q_len * (q_heads // kv_heads)
    assert p["own_tiles"] * p["own_tile_rows"] >= rows
    if p["wide_splits"]:  # 128 rows of a sequence, then its other records in one part
        assert p["wide_tiles"] * 128 >= rows and p["wide_items"] == batch * kv_heads * p["wide_tiles"] * p["wide_splits"]
        assert p["items"] == p["wide_items"] + batch * kv_heads * p["own_tiles"]
        return list(range(p["wide_splits"])) + [p["wide_splits"]]
    assert p["wide_tiles"] == p["wide_items"] == 0
    if p["prefix_splits"]:
        assert p["prefix_tiles"] * p["prefix_tile_rows"] >= batch * rows
    assert p["prefix_items"] == kv_heads * p["prefix_tiles"] * p["prefix_splits"]
    assert p["items"] == p["prefix_items"] + batch * kv_heads * p["own_tiles"] * p["own_splits"]
    return list(range(p["prefix_splits"])) + [p["prefix_splits"] + s for s in range(p["own_splits"])]


def hold(plans, shapes):
    got = plans(shapes)
    for shape, p in zip(shapes, got):
        assert parts_written(shape, p) == list(range(p["parts"])), (shape, p)
        assert p["rows"] == shape[0] * shape[1] * shape[2]
        values = p["rows"] * p["parts"] if p["parts"] > 1 else 0
        assert p["stats_bytes"] >= 8 * values and p["bytes"] == p["stats_bytes"] + 4 * values * shape[4], (shape, p)
    return got


# Trees whose tiles of 32 rows take the prefix with their own tokens, while tiles of 16 rows take it apart.
TWO_KINDS = [(18, 10, 64, 32, 64, 1536, 40), (34, 21, 16, 16, 64, 1600, 21), (49, 7, 96, 32, 64, 256, 7), (57, 21, 9, 9, 64, 1000, 600),
             (66, 21, 8, 8, 64, 336, 600)]


def test_trees_that_one_tile_takes_apart_and_another_does_not(plans):
    hold(plans, [(b, t, hq, hk, d, BF16, prefix, own, 0, True) for b, t, hq, hk, d, prefix, own in TWO_KINDS])


def test_every_part_is_written_by_somebody(plans):
    heads = [(4, 4), (8, 1), (16, 8), (9, 9), (64, 32), (24, 8)]
    shapes = [(b, t, hq, hk, d, dtype, prefix, own, window, tree)
              for b, t, (hq, hk), d, dtype, prefix, own, window, tree in itertools.product(
                  (1, 2, 18, 57), (1, 7, 17, 21, 64), heads, (64, 256, 512), (F32, BF16), (0, 100, 1536), (0, 40, 2000), (0, 300),
                  (False, True))]
    hold(plans, shapes)


def test_every_part_of_random_trees_is_written_by_somebody(plans):
    rng = random.Random(1)
    shapes = []
    for _ in range(150000):
        hk = rng.choice([1, 2, 3, 4, 8, 9, 16, 32])
        shapes.append((rng.randint(1, 80), rng.randint(1, 64), hk * rng.choice([1, 1, 2, 3, 4, 8]), hk, rng.choice([64, 128, 256]), BF16,
                       rng.randint(0, 3000), rng.randint(0, 1500), 0, True))
    got = hold(plans, shapes)
    assert sum(p["wide_splits"] > 0 for p in got) > 1000 and sum(p["prefix_splits"] > 0 for p in got) > 1000


def test_a_tree_takes_the_scratch_that_there_is(plans):
    """In as many bytes as the tree's best plan needs that plan; in fewer another that fits them and is whole; a run's bytes are
    always enough."""
    rng = random.Random(2)
    shapes = [(b, t, hq, hk, d, BF16, prefix, own, 0, True) for b, t, hq, hk, d, prefix, own in TWO_KINDS]
    shapes += [(256, 64, 16, 8, 256, BF16, 0, 2000, 0, True), (64, 64, 16, 8, 256, BF16, 0, 2000, 0, True)]
    for _ in range(20000):
        hk = rng.choice([1, 2, 4, 8, 16])
        shapes.append((rng.randint(1, 80), rng.randint(1, 64), hk * rng.choice([1, 2, 4]), hk, rng.choice([64, 128, 256, 512]),
                       rng.choice([F32, BF16]), rng.choice([0, rng.randint(0, 3000)]), rng.randint(0, 3000), rng.choice([0, 0, 700]), True))
    best = hold(plans, shapes)
    assert plans([(*s, p["bytes"]) for s, p in zip(shapes, best)]) == best
    runs = hold(plans, [(*s[:9], False) for s in shapes])
    for limit in ([p["bytes"] for p in runs], [0] * len(best), [rng.randint(0, p["bytes"]) for p in best]):
        for p, most in zip(hold(plans, [(*s, n) for s, n in zip(shapes, limit)]), limit):
            assert p["bytes"] <= most
    grown = [(s, r["bytes"], p["bytes"]) for s, r, p in zip(shapes, runs, best) if p["bytes"] > r["bytes"]]
    assert grown and runs[5]["bytes"] == 0  # 256 sequences of 64 rows are one part each as a run


def test_the_tests_of_many_rows_take_that_form(plans):
    """The cases of test_gpu_tree_attention.py (Many) and test_gpu_tree_many_rows.py that are there for the workgroups of 128 rows."""
    pytest.importorskip("torch")
    from test_gpu_tree_attention import MANY

    dims, announced = (64, 128, 256), 40000
    shapes = [(len(before), nodes, hq, hk, d, 0) for before, nodes, hq, hk in MANY for d in dims]
    shapes += [(5, 64, 32, 4, d, prefix) for d in dims for prefix in (1, 32, 100, 999)]
    shapes += [(3, 64, 32, 4, d, 0) for d in dims] + [(2, 64, 64, 4, d, 0) for d in dims] + [(3, 64, 64, 4, 128, 0)]
    for shape, p in zip(shapes, hold(plans, [(*s[:5], BF16, s[5], announced - s[5], 0, True) for s in shapes])):
        assert p["wide_splits"] > 0, shape
