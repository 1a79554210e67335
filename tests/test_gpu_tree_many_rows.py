"""Attention of drafted trees of many rows (turbo_tree_attention's workgroups of 128 rows): what their splits, their units and
their scratch must hold, against the formula in 64 bits."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
import step_util as S
import turbo_decode_tail as T
from test_gpu_tree_attention import ROUNDING, Case, Many

pytestmark = pytest.mark.gpu


def again_over(c, byte):
    """The same call over a workspace of this byte in every place."""
    c.workspace.fill_(byte)
    c.out.fill_(7.0)
    c.cache.attend_tree(c.inp, c.d_masks)
    torch.cuda.synchronize()
    return c.out


# shapes of test_host_attention_plan.py whose tiles of 32 and of 16 rows take the prefix in different ways
@pytest.mark.parametrize("batch,nodes,hq,hk,prefix,own", [(18, 10, 64, 32, 1536, 40), (34, 21, 16, 16, 1600, 21), (49, 7, 96, 32, 256, 7),
                                                         (57, 21, 9, 9, 1000, 600), (66, 21, 8, 8, 336, 600)])
def test_the_join_reads_what_the_call_wrote(batch, nodes, hq, hk, prefix, own):
    """Whatever the scratch held before: NaN (255), zeros, or numbers."""
    c = Case([prefix + own - nodes - (i % 5 if own > nodes + 5 else 0) for i in range(batch)], nodes, hq, hk, 64, prefix=prefix, seed=batch)
    want = c.run(longest=prefix + own).clone()
    c.check(rounding=ROUNDING)
    for byte in (255, 0, 64):
        assert torch.equal(again_over(c, byte), want), byte


@pytest.mark.parametrize("power", [20, 28, 34, 60])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_large_values_that_lose_their_weight(d, bits, power):
    """Every third record holds nothing but large values under keys that lead while no others are met, and have 2^-100 of the
    weight of those: what they leave is below 2^-40 of the result, and the others' bits must be as without them."""
    c = Many([640, 200, 1999], 64, 32, 4, d, bits=bits, seed=power)
    c.q = c.q.abs() + 0.5
    large = [torch.arange(n, device="cuda") // 32 % 3 == 0 for n in c.before]
    large[1][:] = False
    for i, n in enumerate(c.before):
        k, v = (x[:n] for x in c.held[i])
        v.copy_(v.abs() + 0.5)
        k[large[i]] = -70.0 / (1.3 * d**0.5)
        v[large[i]] *= 2.0**power
        slots = S.ids([S.words(c.tables)[i][j // c.page] * c.page + j % c.page for j in range(n)])
        c.cache.write(k.contiguous(), v.contiguous(), slots, n, dtype=T.TURBO_HIDDEN_BF16)
    out = c.run().double()
    small = 2.0**-18 if bits == 4 else 2.0**-22  # of a head's largest
    for i, n in enumerate(c.before):
        k, v = (c.stored(x)[0].double() for x in c.held[i])
        seen = c.seen(i, 0)
        seen[:, :n] &= ~large[i]
        for h in range(c.hq):
            kk, vv = k[:, h // 8], v[:, h // 8]
            q = c.q[i * 64:(i + 1) * 64, h].double()
            s = (q @ kk.T.contiguous() * c.scale).masked_fill_(~seen, -torch.inf)
            w = s.softmax(dim=1)
            want = w @ vv
            # Of a key and a value 2^-11 and `small` of the head's largest; a weight is off by as much, relative to itself, as
            # twice a score, and by 2^-11 when it is rounded. A weighted value that is small keeps 2^-20 of the row's largest.
            wrong = (q.abs() @ (2.0**-11 * kk.abs() + small * kk.abs().amax(dim=1, keepdim=True)).T.contiguous() * c.scale).masked_fill_(~seen, 0.0)
            weight = 2 * wrong.amax(dim=1, keepdim=True) + 2.0**-11 + 2.0**-16
            top = vv.masked_fill(~seen.any(dim=0)[:, None], 0.0).abs().amax(dim=1)
            rest = (w * top).amax(dim=1, keepdim=True) * 2.0**-20 * (n + 64) + small * (w @ top)[:, None]
            bound = 1.01 * ((w @ vv.abs()) * (weight + 2.0**-11) + rest) + want.abs() * 2.0**-8
            far = (out[i * 64:(i + 1) * 64, h] - want).abs()
            assert bool((far <= bound).all()), (i, h, (far / bound).max().item())


def sizes(c):
    """What the two calls of the C interface give for the case's last call."""
    n = C.c_size_t()
    out = []
    for call in (c.cache.lib.turbo_attention_workspace, c.cache.lib.turbo_tree_workspace):
        assert call(c.cache.h, C.byref(c.inp), C.byref(n)) == 1
        out.append(n.value)
    return out


def test_a_run_needs_what_it_needed_before_there_were_trees():
    """256 sequences of 64 rows, one part each: no scratch, where a tree would have use for 540 MB."""
    cache = T.KvCache(1, 64, 8, 256)
    inp = cache.make_attention_inputs(256, dtype=T.TURBO_HIDDEN_BF16, q=None, out=None, q_heads=16, q_len=64, kv_len=None,
                                      max_kv_len=2000, pages=torch.zeros((256, 32), dtype=torch.int32, device="cuda"), scale=1.0)
    n = C.c_size_t()
    assert cache.lib.turbo_attention_workspace(cache.h, C.byref(inp), C.byref(n)) == 1 and n.value == 0
    assert cache.lib.turbo_tree_workspace(cache.h, C.byref(inp), C.byref(n)) == 1 and n.value > 2**29
    assert cache.attention_workspace(inp, tree=False) == 0 and cache.attention_workspace(inp) == cache.attention_workspace(inp, tree=True) == n.value
    inp.q_len = 65
    assert cache.lib.turbo_tree_workspace(cache.h, C.byref(inp), C.byref(n)) == 0 and "q_len" in T.last_error()
    assert cache.attention_workspace(inp) == cache.attention_workspace(inp, tree=False)
    cache.close()


def test_a_run_that_no_tree_could_be():
    """As a tree these sizes are more workgroups than a grid holds; that does not refuse the run's scratch."""
    cache = T.KvCache(1, 32, 32, 64)
    inp = cache.make_attention_inputs(218774, dtype=T.TURBO_HIDDEN_BF16, q=None, out=None, q_heads=64, q_len=19, kv_len=None,
                                      max_kv_len=100000, pages=torch.zeros((1, 3125), dtype=torch.int32, device="cuda"), scale=1.0)
    with pytest.raises(T.TurboError, match="too large"):
        cache.attention_workspace(inp, tree=True)
    assert cache.attention_workspace(inp) == cache.attention_workspace(inp, tree=False)
    cache.close()


@pytest.mark.parametrize("shape", [([900, 1000], 8, 4, 1, 128, 0), ([300] * 9, 64, 16, 4, 64, 0), ([1600] * 34, 21, 16, 16, 64, 1600),
                                   ([2500, 700], 64, 128, 8, 256, 0)], ids=str)
@pytest.mark.parametrize("dtype", [T.TURBO_HIDDEN_F32, T.TURBO_HIDDEN_BF16])
def test_a_tree_in_the_scratch_of_a_run(shape, dtype):
    """Any size from the smaller of both on, and a byte less is refused."""
    before, nodes, hq, hk, d, prefix = shape
    c = Case(before, nodes, hq, hk, d, prefix=prefix, dtype=dtype, seed=9)
    c.run()
    c.check(rounding=ROUNDING)
    run, tree = sizes(c)
    for n in sorted({run, tree, (run + tree) // 2, min(run, tree)}):
        c.workspace = torch.empty(n + 64, dtype=torch.uint8, device="cuda")
        c.inp.workspace, c.inp.workspace_bytes = c.workspace.data_ptr(), n
        again_over(c, 255)
        c.check(rounding=ROUNDING)
        assert bool((c.workspace[n:] == 255).all())
    if min(run, tree) > 0:
        c.inp.workspace_bytes = min(run, tree) - 1
        with pytest.raises(T.TurboError, match="workspace holds"):
            c.cache.attend_tree(c.inp, c.d_masks)
        c.inp.workspace, c.inp.workspace_bytes = None, tree
        with pytest.raises(T.TurboError, match="workspace is NULL"):
            c.cache.attend_tree(c.inp, c.d_masks)
