"""Attention for drafted tokens at its edges: blocks of few rows beside numbers that are none, positions that are none of the
entry's.  Tolerances: those of ``test_drafts_gpu.Case.check``."""
import math

import pytest
import torch

from test_drafts_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd, ps", [(128, 16), (64, 16), (128, 128)])
@pytest.mark.parametrize("tokens", [1, 5, 13, 20])                 # 4, 20, 52, 80 of 128 rows: one to three warps in four have none
@pytest.mark.parametrize("window", [0, 30])
def test_blocks_of_few_rows_beside_numbers_that_are_none(hd, ps, tokens, window):
    """The warps of a block that have no rows clear its values with the others: places that nobody sees, behind the last key,
    in front of the window, on both halves of a tile, hold NaN and infinities, and none of them arrives, however often."""
    for ctx in (0, 3, 61, 70, 300):
        c = Case([tokens, tokens], [ctx, ctx + 128], 8, 2, hd, ps, torch.bfloat16, window=window, seed=ctx + tokens)
        for e in range(2):
            dead = (~c.visible(e).any(0)).nonzero().flatten().tolist()
            for n, j in enumerate(dead + list(range(c.kv[e], len(c.tables[e]) * ps))):
                for t in (c.k, c.v):
                    t[c.tables[e][j // ps], :, j % ps] = (math.nan, math.inf, -math.inf)[n % 3]
        for t in (c.k, c.v):
            t[torch.tensor(c.unused, device=t.device)] = math.nan
        first = c.run().clone()
        c.check()
        for _ in range(20):
            c.out.fill_(7.0)
            c.run()
            assert torch.equal(c.out, first)
