"""Attention of drafted trees of many rows (turbo_tree_attention's workgroups of 128 rows): what their splits, their units and
their scratch must hold, against the formula in 64 bits."""
import pytest

torch = pytest.importorskip("torch")
import turbo_decode_tail as T
from test_gpu_tree_attention import ROUNDING, Case

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
