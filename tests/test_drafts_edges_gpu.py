"""Attention for drafted tokens at its edges: blocks of few rows beside numbers that are none, positions that are none of the
entry's.  Tolerances: those of ``test_drafts_gpu.Case.check``."""
import math
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from safetyraise_lmengine_b200.errors import ShapeError
from safetyraise_lmengine_b200.kernels import ops
from test_drafts_gpu import DEV, Case, ints

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


def test_pools_of_one_byte_numbers():
    """Copied and moved at even addresses, refused at odd ones."""
    flat = torch.randint(0, 256, (2 * 4 * 3 * 4 * 6 + 2,), dtype=torch.uint8, device=DEV)
    for at in (0, 2):
        pool = flat[at:at + 576].view(2, 4, 3, 4, 6)
        want = pool.clone()
        want[:, 3] = want[:, 1]
        ops.copy_pages(pool, [1], [3])
        assert torch.equal(pool, want)
        want[:, 2, :, 1] = want[:, 2, :, 3]
        ops.keep_drafts(pool, ints([[2]]), ints([0, 4]), ints([4]), ints([[0, 3]]), ints([2]))
        assert torch.equal(pool, want)
    was, pool = flat.clone(), flat[1:577].view(2, 4, 3, 4, 6)
    with pytest.raises(ShapeError, match="odd address"):
        ops.copy_pages(pool, [1], [3])
    with pytest.raises(ShapeError, match="odd address"):
        ops.keep_drafts(pool, ints([[2]]), ints([0, 4]), ints([4]), ints([[0, 3]]), ints([2]))
    assert torch.equal(flat, was)


@pytest.mark.parametrize("dt, hd, ps", [(torch.bfloat16, 128, 16), (torch.bfloat16, 64, 8), (torch.bfloat16, 80, 16), (torch.float32, 64, 16)])
@pytest.mark.parametrize("tokens", [3, 40])
def test_positions_that_are_none_of_the_entry_s(dt, hd, ps, tokens):
    """Under a window a position in front of the entry's first token, or behind its last key, raises the error word and counts as
    the nearest that is the entry's, wherever tiles begin and end."""
    dev = torch.device(DEV)
    for ctx, window in ((900, 200), (516, 37), (20, 300)):
        c = Case([tokens, 5], [ctx, 300], 8, 2, hd, ps, dt, window=window, seed=ctx)
        ops.gemm_error_flag(dev)
        c.run()
        c.check()
        assert ops.gemm_error_flag(dev) == 0
        right = c.positions.clone()
        for wrong, nearest in ((ctx + tokens, ctx + tokens - 1), (ctx + tokens + 150, ctx + tokens - 1), (2 ** 31 - 1, ctx + tokens - 1),
                               (ctx - 1, ctx), (ctx - 70, ctx), (-2 ** 31, ctx)):
            at = tokens // 2
            c.positions[at] = nearest
            want = c.run().clone()
            assert ops.gemm_error_flag(dev) == 0
            c.positions[at] = wrong
            c.run()
            assert ops.gemm_error_flag(dev) != 0, wrong
            assert torch.equal(c.out, want), wrong
            c.positions.copy_(right)


@pytest.mark.parametrize("dt, hd, ps", [(torch.bfloat16, 128, 16), (torch.bfloat16, 64, 8), (torch.bfloat16, 80, 16), (torch.float32, 64, 16)])
@pytest.mark.parametrize("tokens, ctx", [(20, 600), (5, 200), (20, 5000)])
def test_values_that_are_no_numbers_add_up(dt, hd, ps, tokens, ctx):
    """Of a committed key that every row sees, and of a drafted one that some see: NaN stays NaN beside an infinity, and infinities of
    both signs make NaN."""
    c = Case([tokens], [ctx], 8, 2, hd, ps, dt, seed=3)

    def put(j, d, value):
        c.v[c.tables[0][j // ps], :, j % ps, d] = value

    node = 3
    sees = torch.from_numpy(c.seen[0][:, node]).to(DEV)
    assert sees.any() and not sees.all()
    early = 10
    put(early, 3, math.nan), put(early, 7, -math.inf), put(early, 9, math.inf)
    for d in (3, 5, 7, 9):
        put(ctx + node, d, math.inf)
    out = c.run().view(tokens, 8, hd).float()
    assert out[..., 3].isnan().all()
    assert (out[sees][..., 5] == math.inf).all() and out[~sees][..., 5].isfinite().all()
    assert out[sees][..., 7].isnan().all() and (out[~sees][..., 7] == -math.inf).all()
    assert (out[..., 9] == math.inf).all()
    assert out[..., 0].isfinite().all()


@pytest.mark.parametrize("dt, sizes", [(torch.bfloat16, (144, 256, 160, 240)), (torch.float32, (132, 256, 140, 255))])
@pytest.mark.parametrize("tokens", [4, 8, 40])
def test_calls_of_several_threads(dt, sizes, tokens):
    """Heads of unlike sizes that one kernel takes, from several host threads at once, each on a stream of its own: a call's
    shared memory is not another's to take away."""
    cases = [Case([tokens, 3], [100, 40], 4, 2, hd, 20, dt, seed=hd) for hd in sizes]
    ops.gemm_error_flag(torch.device(DEV))

    def serve(c):
        torch.cuda.set_device(DEV)
        outs = []
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                outs.append(c.run().clone())
        torch.cuda.synchronize()
        return all(torch.equal(o, outs[0]) for o in outs)

    torch.cuda.synchronize()
    with ThreadPoolExecutor(len(cases)) as pool:
        assert all(pool.map(serve, cases))
    for c in cases:
        c.check()
    assert ops.gemm_error_flag(torch.device(DEV)) == 0


@pytest.mark.parametrize("dt, hd, ps", [(torch.bfloat16, 128, 16), (torch.bfloat16, 64, 8), (torch.bfloat16, 128, 128), (torch.bfloat16, 80, 16),
                                        (torch.float32, 64, 16)])
@pytest.mark.parametrize("ctx, window", [(700, 50), (515, 130), (1030, 3)])
def test_pages_that_a_window_has_passed(dt, hd, ps, ctx, window):
    """Given back, -1 in the table: not missed, with whatever page 0 holds by now; the first page that the window still needs is."""
    dev = torch.device(DEV)
    c = Case([20, 3], [ctx, 40], 8, 2, hd, ps, dt, window=window, seed=ctx)
    want = c.run().clone()
    c.check()
    needed = max(0, ctx - window + 1) // ps
    assert needed > 0
    for t in (c.k, c.v):                                           # page 0 is another request's: numbers that would show
        if 0 not in c.tables[0][needed:].tolist() + c.tables[1].tolist():
            t[0] = math.nan
    ops.gemm_error_flag(dev)
    c.table[0, :needed] = -1
    c.out.fill_(7.0)
    c.run()
    assert ops.gemm_error_flag(dev) == 0
    assert torch.equal(c.out, want)
    c.table[0, needed] = -1
    c.run()
    assert ops.gemm_error_flag(dev) != 0
