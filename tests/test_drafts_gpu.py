"""Attention for drafted tokens, and what stands around it, against their formulas in 64 bits.

Tolerance of the attention, from the arithmetic.  With u = 2^-24: a score is scale * sum of hd products, off by at most
(hd + 2) u times scale * sum |q_d k_d|, and its exponential's argument by another 4 u |score| and 2^-21 (the exponential's own
error); a weight is off by twice that (its own and the sum's), relatively, and by half a step of bfloat16 (2^-8) where the
tensor cores read it so; sums over n keys add n u.  The result is rounded to its type at the end.
"""
import math

import numpy as np
import pytest
import torch

from safetyraise_lmengine_b200.errors import ShapeError, Unavailable
from safetyraise_lmengine_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U}


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def tree(q, r, chain=False):
    if chain:
        return np.arange(-1, q - 1)
    p = np.array([-1] + [int(r.randint(max(0, i - 5), i)) for i in range(1, q)])
    p[0] = -1
    return p


def ancestors(parents):
    """[q, q] truth values, and depths."""
    q = len(parents)
    seen, depth = np.zeros((q, q), dtype=bool), np.zeros(q, dtype=int)
    for i in range(q):
        k = i
        while k >= 0:
            seen[i, k] = True
            k = parents[k]
        depth[i] = seen[i].sum() - 1
    return seen, depth


def packed(seen, words):
    out = np.zeros((seen.shape[0], words), dtype=np.uint32)
    for i, k in zip(*np.nonzero(seen)):
        out[i, k // 32] |= np.uint32(1 << (k % 32))
    return out.view(np.int32)


class Case:
    """A batch on pages in no order; ``masks``: what each entry's tokens see of one another (a tree's lines, or given)."""

    def __init__(self, lens, ctx, nq, nkv, hd, ps, dt, window=0, masks=None, seed=0, spare=0, words=None):
        g, r = torch.Generator(device=DEV).manual_seed(seed), np.random.RandomState(seed)
        self.lens, self.ctx, self.nq, self.nkv, self.hd, self.ps, self.window = lens, ctx, nq, nkv, hd, ps, window
        self.kv = [c + q for c, q in zip(ctx, lens)]
        need = [-(-k // ps) for k in self.kv]
        pages = sum(need) + 2
        order = r.permutation(pages)
        table = np.zeros((len(lens), max(need) + 1), dtype=np.int32)
        self.tables, at = [], 0
        for e, k in enumerate(need):
            table[e, :k] = order[at:at + k]
            self.tables.append(torch.tensor(order[at:at + k], device=DEV))
            at += k
        self.unused = order[at:]
        self.T = sum(lens) + spare
        self.words = words or -(-max(lens) // 32)
        rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dt)
        self.q, self.k, self.v = rnd(self.T, nq * hd), rnd(pages, nkv, ps, hd), rnd(pages, nkv, ps, hd)
        self.cu = np.concatenate([[0], np.cumsum(lens)])
        self.seen, pos = [], []
        for e, q in enumerate(lens):
            if masks is None:
                seen, depth = ancestors(tree(q, r, chain=e % 3 == 2))
                if window:
                    seen &= depth[:, None] - depth[None, :] < window
            else:
                seen, depth = masks[e], np.arange(q)
            self.seen.append(seen)
            pos += [ctx[e] + int(d) for d in depth]
        mask = np.zeros((self.T, self.words), dtype=np.int32)
        if sum(lens):
            mask[:sum(lens)] = np.concatenate([packed(s, self.words) for s in self.seen])
        self.mask, self.table, self.cu_q, self.kv_lens = ints(mask), ints(table), ints(self.cu), ints(self.kv)
        self.positions = ints(pos + [0] * spare)
        self.scale = 1.0 / math.sqrt(hd)
        self.out = torch.full_like(self.q, 7.0)

    def run(self, **kw):
        a = dict(positions=self.positions if self.window else None, window=self.window)
        a.update(kw)
        ops.tree_attention(self.q, self.k, self.v, self.out, self.table, self.cu_q, self.kv_lens, self.mask, self.nq, self.nkv, self.hd,
                           self.ps, self.scale, max(self.lens), **a)
        return self.out

    def visible(self, e):
        c, q = self.ctx[e], self.lens[e]
        vis = torch.zeros((q, self.kv[e]), dtype=torch.bool, device=DEV)
        j = torch.arange(c, device=DEV)
        p = self.positions[int(self.cu[e]):int(self.cu[e + 1]), None]
        vis[:, :c] = (p - j < self.window) if self.window else True
        vis[:, c:] = torch.from_numpy(self.seen[e]).to(DEV)
        return vis

    def check(self, p_half=None):
        """Every entry against the formula; returns the largest share of the tolerance that was used."""
        dt, worst = self.q.dtype, 0.0
        p_half = p_half if p_half is not None else (HALF[dt] if dt == torch.bfloat16 else 0.0)
        for e, q in enumerate(self.lens):
            lo, hi = int(self.cu[e]), int(self.cu[e + 1])
            vis = self.visible(e)
            for h in range(self.nq):
                kh = h // (self.nq // self.nkv)
                k = self.k[self.tables[e], kh].reshape(-1, self.hd)[:self.kv[e]].double()
                v = self.v[self.tables[e], kh].reshape(-1, self.hd)[:self.kv[e]].double()
                x = self.q[lo:hi, h * self.hd:(h + 1) * self.hd].double()
                seen_any = vis.any(0)
                k, v = torch.where(seen_any[:, None], k, 0.0), torch.where(seen_any[:, None], v, 0.0)
                s = (x @ k.T) * self.scale
                size = ((x.abs() @ k.abs().T) * self.scale).masked_fill(~vis, 0.0)
                w = torch.softmax(s.masked_fill(~vis, -math.inf), 1)
                w = torch.where(vis.any(1)[:, None], w, 0.0)
                want = w @ v
                n = vis.sum(1, keepdim=True)
                ds = (self.hd + 6) * U * size.amax(1, keepdim=True) + 2.0 ** -21
                tol = HALF[dt] * want.abs() + (p_half + 2 * ds + (n + 16) * U) * (w @ v.abs()) * (1 + HALF[dt])
                got = self.out[lo:hi, h * self.hd:(h + 1) * self.hd].double()
                assert torch.isfinite(got).all(), (e, h)
                assert (got[~vis.any(1)] == 0).all(), "a row that sees nothing"
                over = (got - want).abs() - tol
                assert (over <= 0).all(), (e, h, float(over.max()), float((got - want).abs().max()))
                worst = max(worst, float(((got - want).abs() / tol.clamp(min=1e-300)).max()))
        return worst


SIZES = [
    # lens, ctx, nq, nkv, hd, ps
    ([1], [0], 1, 1, 16, 4),                                        # one token behind nothing
    ([5], [600], 32, 8, 128, 16),                                   # a chain behind a short context
    ([24], [1000], 32, 8, 128, 16),
    ([33, 1, 64, 17], [500, 0, 129, 63], 8, 2, 128, 16),            # ragged; contexts that end on and inside tiles and pages
    ([64, 40], [1500, 700], 40, 8, 128, 64),
    ([7, 12, 3], [100, 31, 33], 6, 2, 64, 8),
    ([20, 9], [257, 1000], 16, 4, 64, 20),                          # pages of an odd size
    ([6, 40], [300, 5], 5, 5, 80, 16),
    ([11], [77], 8, 1, 256, 32),
    ([30, 2], [90, 400], 3, 1, 48, 7),
    ([70, 100], [40, 3000], 4, 2, 128, 128),                        # pages of a tile
    ([130], [200], 2, 1, 128, 16),                                  # masks of several words
]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens, ctx, nq, nkv, hd, ps", SIZES)
@pytest.mark.parametrize("window", [0, 37])
def test_trees(lens, ctx, nq, nkv, hd, ps, dt, window):
    c = Case(lens, ctx, nq, nkv, hd, ps, dt, window=window, seed=hd + ps)
    c.run()
    c.check()


@pytest.mark.parametrize("dt, lens, ctx, nq, nkv, hd, ps", [
    (torch.bfloat16, [64, 50], [9000, 12000], 64, 8, 128, 16),     # blocks of rows side by side over more keys than L2 holds
    (torch.bfloat16, [64, 33, 50], [12000, 9000, 1], 16, 8, 256, 32),
    (torch.bfloat16, [64, 5, 64], [9000, 4000, 9000], 40, 8, 128, 64),     # ... and entries of too unlike numbers of them
    (torch.float32, [20, 20], [5000, 4500], 32, 8, 128, 16)])
def test_long_contexts(dt, lens, ctx, nq, nkv, hd, ps):
    c = Case(lens, ctx, nq, nkv, hd, ps, dt, seed=6)
    c.run()
    c.check()


@pytest.mark.parametrize("dt, hd", [(torch.float32, 18), (torch.float32, 5), (torch.bfloat16, 36)])
def test_heads_of_odd_sizes(dt, hd):
    c = Case([9, 14], [50, 120], 4, 2, hd, 16, dt, seed=hd)
    c.run()
    c.check()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd, ps", [(128, 16), (64, 20), (80, 16)])
def test_any_mask(dt, hd, ps):
    """Masks that are no trees': rows that see nothing at all, nothing but later tokens, everything; entries without a context."""
    r = np.random.RandomState(3)
    lens, ctx = [40, 8, 3, 33], [0, 0, 200, 0]
    masks = [r.rand(q, q) < 0.3 for q in lens]
    masks[0][5], masks[0][17] = False, True
    masks[1][:] = False                                          # nobody in it sees anything
    masks[3][0] = False
    masks[3][0, 32] = True                                       # one key of the second word alone
    c = Case(lens, ctx, 8, 2, hd, ps, dt, masks=masks, seed=2, words=3)
    c.run()
    c.check()
    assert (c.out[40:48] == 0).all()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd, ps", [(128, 16), (64, 20), (128, 64), (80, 16)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_seen_never_arrives(dt, hd, ps, bad):
    """Numbers that are none in every place that no row sees, and in drafted tokens' keys and values that only their descendants
    see: the other rows are the formula's."""
    c = Case([20, 40], [333, 50], 8, 2, hd, ps, dt, window=60, seed=4)
    for e in range(2):
        vis = c.visible(e)
        dead = (~vis.any(0)).nonzero().flatten().tolist()
        places = dead + list(range(c.kv[e], len(c.tables[e]) * ps))          # behind the last key too
        for j in places:
            c.k[c.tables[e][j // ps], :, j % ps] = bad
            c.v[c.tables[e][j // ps], :, j % ps] = bad
    c.k[torch.tensor(c.unused, device=DEV)] = bad
    c.v[torch.tensor(c.unused, device=DEV)] = bad
    clean = c.run().clone()
    c.check()
    # a drafted token of each entry: the rows that do not see it stay bit for bit what they were
    for what in ("v", "k"):
        for e, node in ((0, 3), (1, 7)):
            j = c.ctx[e] + node
            getattr(c, what)[c.tables[e][j // ps], :, j % ps] = bad
        c.out.fill_(7.0)
        c.run()
        for e, node in ((0, 3), (1, 7)):
            sees = torch.from_numpy(c.seen[e][:, node]).to(DEV)
            rows, was = (t[int(c.cu[e]):int(c.cu[e + 1])] for t in (c.out, clean))
            assert sees.any() and not sees.all()
            assert torch.equal(rows[~sees], was[~sees])
            if what == "v" or not math.isinf(bad):
                assert not torch.isfinite(rows[sees].float()).all(dim=1).any()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_far_apart_scores_and_the_lowest_values(dt):
    """Scores of +-10^4 (a softmax with one key left), and keys of the type's lowest value behind the mask."""
    c = Case([12, 5], [700, 64], 8, 4, 128, 16, dt, seed=9)
    c.q *= 100.0
    c.v[torch.tensor(c.unused, device=DEV)] = torch.finfo(dt).min
    c.run()
    rows = 0
    for e in range(2):
        vis = c.visible(e)
        lo, hi = int(c.cu[e]), int(c.cu[e + 1])
        for h in range(8):
            k = c.k[c.tables[e], h // 2].reshape(-1, 128)[:c.kv[e]].double()
            v = c.v[c.tables[e], h // 2].reshape(-1, 128)[:c.kv[e]].double()
            x = c.q[lo:hi, h * 128:(h + 1) * 128].double()
            s = (x @ k.T * c.scale).masked_fill(~vis, -math.inf)
            top = s.topk(2, dim=1)
            sure = top.values[:, 0] - top.values[:, 1] > 40        # what else there is weighs less than e^-40
            got = c.out[lo:hi, h * 128:(h + 1) * 128].double()[sure]
            want = v[top.indices[:, 0]][sure]
            assert ((got - want).abs() <= v.abs().max() * (HALF[dt] + 2 ** -20)).all()
            rows += int(sure.sum())
    assert rows > 0


def test_rows_behind_the_last_entry_and_entries_without_tokens():
    for dt in (torch.float32, torch.bfloat16):
        c = Case([9, 20], [100, 30], 8, 2, 128, 16, dt, spare=7, seed=1)
        c.run()
        c.check()
        assert (c.out[29:] == 7.0).all()
        # a third entry of no tokens between them
        c.cu_q, c.kv_lens = ints([0, 9, 9, 29]), ints([c.kv[0], 0, c.kv[1]])
        was = c.out.clone()
        c.table = torch.stack([c.table[0], c.table[0] * 0, c.table[1]])
        c.out.fill_(7.0)
        ops.tree_attention(c.q, c.k, c.v, c.out, c.table, c.cu_q, c.kv_lens, c.mask, 8, 2, 128, 16, c.scale, 20)
        assert torch.equal(c.out, was)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_many_entries(dt):
    """More entries than a warp counts at a time, of every length."""
    r = np.random.RandomState(8)
    lens = [int(x) for x in r.randint(1, 20, size=70)]
    ctx = [int(x) for x in r.randint(0, 400, size=70)]
    c = Case(lens, ctx, 4, 2, 64, 16, dt, seed=5)
    c.run()
    c.check()


def test_a_chain_is_causal_attention():
    """Chains of drafted tokens are what the engine's causal attention computes for them."""
    lens, ctx = [5, 17], [300, 41]
    masks = [np.tril(np.ones((q, q), dtype=bool)) for q in lens]
    c = Case(lens, ctx, 8, 2, 128, 16, torch.float32, masks=masks)
    c.run()
    want = torch.empty_like(c.out)
    eot = ints([0] * 5 + [1] * 17)
    ops.paged_attention_simt(c.q, c.k, c.v, want, c.table, eot, c.positions, 8, 2, 128, 16, c.scale)
    assert (c.out - want).abs().max() <= 2 ** -18 * c.v.abs().max()


def test_graphs_streams_and_repeats():
    """Recorded and replayed with other lengths, on two streams at once, and twice over: bit for bit the eager results."""
    cases = [Case([24, 30], [900, 300], 32, 8, 128, 16, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [c.run().clone() for c in cases]
    again = [c.run().clone() for c in cases]
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                c.out.zero_()
                c.run()
    torch.cuda.synchronize()
    assert all(torch.equal(c.out, w) for c, w in zip(cases, want))
    graphs = []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.run()
        graphs.append(g)
    for c in cases:
        c.out.zero_()
    for g in graphs:
        g.replay()
    assert all(torch.equal(c.out, w) for c, w in zip(cases, want))
    # shorter contexts under the same graph
    c = cases[0]
    short = Case([24, 30], [900, 300], 32, 8, 128, 16, torch.bfloat16, seed=1)
    c.kv_lens.copy_(ints([400, 31]))
    short.kv_lens.copy_(ints([400, 31]))
    short.run()
    graphs[0].replay()
    assert torch.equal(c.out, short.out) and not torch.equal(c.out, want[0])


def test_bad_pages_and_lengths_raise_the_error_word():
    ops.gemm_error_flag(torch.device(DEV))
    for dt in (torch.float32, torch.bfloat16):
        c = Case([9, 20], [100, 30], 8, 2, 128, 16, dt, seed=1)
        good = c.run().clone()
        assert ops.gemm_error_flag(torch.device(DEV)) == 0
        for number in (-1, 10 ** 6, c.k.shape[0]):
            c.table[0, 1] = number
            c.run()
            assert ops.gemm_error_flag(torch.device(DEV)) != 0
            assert torch.equal(c.out[9:], good[9:])
        c.table[0, 1] = int(c.tables[0][1])
        for kv in (8, 10 ** 6):                                    # fewer keys than tokens; more than the table has pages
            c.kv_lens[0] = kv
            c.out.fill_(7.0)
            c.run()
            assert ops.gemm_error_flag(torch.device(DEV)) != 0
            assert (c.out[:9] == 7.0).all() and torch.equal(c.out[9:], good[9:])
        c.kv_lens[0] = c.kv[0]
        c.out.fill_(7.0)                                           # more tokens than the call said
        ops.tree_attention(c.q, c.k, c.v, c.out, c.table, c.cu_q, c.kv_lens, c.mask, 8, 2, 128, 16, c.scale, 9)
        assert ops.gemm_error_flag(torch.device(DEV)) != 0
        assert torch.equal(c.out[:9], good[:9]) and (c.out[9:] == 7.0).all()


def test_lengths_whose_sums_pass_32_bits_raise_the_error_word():
    """Differences and sums of such lengths come out as numbers that would do."""
    low, high = -2 ** 31, 2 ** 31 - 1
    ops.gemm_error_flag(torch.device(DEV))
    for dt, hd in ((torch.float32, 64), (torch.bfloat16, 128), (torch.bfloat16, 32)):
        c = Case([9, 20], [100, 30], 8, 2, hd, 16, dt, seed=1)
        good = c.run().clone()
        for kv in (low, low + 3, low + 8):                         # less 9 tokens: 2^31 - 9 and so on
            c.kv_lens[0] = kv
            c.out.fill_(7.0)
            c.run()
            assert ops.gemm_error_flag(torch.device(DEV)) != 0
            assert (c.out[:9] == 7.0).all() and torch.equal(c.out[9:], good[9:])
        c.kv_lens[0] = c.kv[0]
        c.cu_q.copy_(ints([high - 3, low + 5, low + 14]))          # entry 0: 9 tokens from 2^31 - 4 on; entry 1: below none
        c.out.fill_(7.0)
        c.run()
        assert ops.gemm_error_flag(torch.device(DEV)) != 0 and (c.out == 7.0).all()
    parents, cu = ints([-1, 0, 1, 2, 3]), ints([0, 5])
    for lens, kv in (([0, 5], low), ([0, 5], low + 4), ([high - 1, low + 3], 100)):
        positions, mask = ints([7] * 5), ints([[7]] * 5)
        ops.draft_tree(parents, ints(lens), ints([kv]), positions, mask)
        assert ops.gemm_error_flag(torch.device(DEV)) != 0
        assert (positions == 7).all() and (mask == 7).all()
    path, count, following = ints([[7] * 5]), ints([7]), ints([7])
    ops.accept_drafts(parents, parents, parents, ints([high - 1, low + 3]), path, count, following)
    assert ops.gemm_error_flag(torch.device(DEV)) != 0
    assert (path == -1).all() and int(count) == 0 and int(following) == -1
    for lens, kv in (([0, 5], low), ([0, 5], low + 4), ([0, -5], 100), ([0, 5], 4)):
        pool = torch.randn(2, 4, 1, 4, 8, device=DEV)
        was = pool.clone()
        ops.keep_drafts(pool, ints([[1, 2]]), ints(lens), ints([kv]), ints([[0, 2, 4]]), ints([3]))
        assert ops.gemm_error_flag(torch.device(DEV)) != 0 and torch.equal(pool, was)


@pytest.mark.parametrize("lens, chain, window", [([1], False, 0), ([7, 1, 32, 33], False, 0), ([200, 64, 90], False, 5), ([130, 31], True, 0),
                                                 ([130], True, 1), ([40, 256], True, 33)])
def test_draft_tree(lens, chain, window):
    r = np.random.RandomState(len(lens))
    trees = [tree(q, r, chain) for q in lens]
    trees[0][len(trees[0]) // 2] = -1                              # a second root
    kv = [q + int(r.randint(0, 500)) for q in lens]
    T, words = sum(lens), -(-max(lens) // 32) + 1
    positions, mask = ints(np.full(T + 2, -7)), ints(np.full((T + 2, words), -7))
    ops.draft_tree(ints(np.concatenate(trees + [[0, 0]])), ints(np.concatenate([[0], np.cumsum(lens)])), ints(kv), positions, mask, window)
    at = 0
    for q, k, p in zip(lens, kv, trees):
        seen, depth = ancestors(p)
        if window:
            seen &= depth[:, None] - depth[None, :] < window
        assert positions[at:at + q].tolist() == (k - q + depth).tolist()
        assert (mask[at:at + q].cpu().numpy() == packed(seen, words)).all()
        at += q
    assert (mask[T:] == -7).all() and (positions[T:] == -7).all()  # rows of no entry
    assert ops.gemm_error_flag(torch.device(DEV)) == 0


def test_draft_tree_with_wrong_parents():
    ops.gemm_error_flag(torch.device(DEV))
    for wrong in (3, 4, 100, -2):
        positions, mask = ints(np.zeros(5)), ints(np.zeros((5, 1)))
        ops.draft_tree(ints([-1, 0, 0, wrong, 2]), ints([0, 5]), ints([9]), positions, mask)
        assert ops.gemm_error_flag(torch.device(DEV)) != 0
        assert mask.flatten().tolist() == [1, 3, 5, 8, 21] and positions.tolist() == [4, 5, 5, 4, 6]
    positions, mask = ints(np.full(40, -7)), ints(np.full((40, 1), -7))
    ops.draft_tree(ints(np.arange(-1, 39)), ints([0, 40]), ints([50]), positions, mask)      # 32 bits for 40 tokens
    assert ops.gemm_error_flag(torch.device(DEV)) != 0 and (mask == -7).all() and (positions == -7).all()


def walk(tokens, parents, targets, room):
    path = [0]
    while len(path) < room:
        child = [k for k in range(len(tokens)) if parents[k] == path[-1] and tokens[k] == targets[path[-1]] and k > path[-1]]
        if not child:
            break
        path.append(child[0])
    return path, targets[path[-1]]


@pytest.mark.parametrize("lens, room", [([1], 3), ([5, 1, 40, 33], 8), ([100, 64], 3), ([70], 1), ([64, 300], 64)])
def test_accept_drafts(lens, room):
    """Small vocabularies: siblings of the same token, targets that several children have."""
    r = np.random.RandomState(room)
    for vocab in (2, 5):
        trees, tok = [tree(q, r, chain=room == 64) for q in lens], [r.randint(0, vocab, size=q) for q in lens]
        want = [r.randint(0, vocab, size=q) for q in lens]
        n = len(lens)
        path, count, nxt = ints(np.full((n, room), -7)), ints(np.full(n, -7)), ints(np.full(n, -7))
        ops.accept_drafts(ints(np.concatenate(tok)), ints(np.concatenate(trees)), ints(np.concatenate(want)),
                          ints(np.concatenate([[0], np.cumsum(lens)])), path, count, nxt)
        for e in range(n):
            line, token = walk(tok[e].tolist(), trees[e].tolist(), want[e].tolist(), room)
            assert path[e].tolist() == line + [-1] * (room - len(line))
            assert count[e].item() == len(line) and nxt[e].item() == token


def test_accept_drafts_of_an_entry_without_tokens():
    path, count, nxt = ints(np.full((3, 4), -7)), ints([-7] * 3), ints([-7] * 3)
    ops.accept_drafts(ints([4, 5]), ints([-1, -1]), ints([9, 8]), ints([0, 1, 1, 2]), path, count, nxt)
    assert path.tolist() == [[0, -1, -1, -1], [-1] * 4, [0, -1, -1, -1]]
    assert count.tolist() == [1, 0, 1] and nxt.tolist() == [9, -1, 8]


@pytest.mark.parametrize("dt, nkv, ps, hd", [(torch.bfloat16, 8, 16, 128), (torch.float32, 2, 5, 20), (torch.bfloat16, 3, 4, 1), (torch.float32, 1, 8, 3),
                                             (torch.bfloat16, 2, 32, 36)])
@pytest.mark.parametrize("room", [1, 6, 150])
def test_keep_drafts(dt, nkv, ps, hd, room):
    """Paths whose moves read where earlier ones write, whole chains (nothing moves), long paths; every other place stays."""
    r = np.random.RandomState(room)
    g = torch.Generator(device=DEV).manual_seed(room)
    lens, ctx, layers = [200, 9, 1, 160], [33, 0, 7, 100], 3
    need = [-(-(c + q) // ps) for c, q in zip(ctx, lens)]
    order = r.permutation(sum(need) + 2)
    table, at = np.zeros((4, max(need)), dtype=np.int32), 0
    for e, k in enumerate(need):
        table[e, :k] = order[at:at + k]
        at += k
    pool = torch.randn(layers, 2, sum(need) + 2, nkv, ps, hd, generator=g, device=DEV).to(dt)
    paths = []
    for q in lens:
        a = min(room, int(r.randint(1, q + 1)))
        paths.append([0] + sorted((1 + r.choice(q - 1, size=a - 1, replace=False)).tolist()))
    paths[3] = list(range(min(room, 160)))
    if room > 1:
        paths[1] = [0, 2, 3, 4, 5, 8][:room]                       # each place is read behind where the one before is written
    path = np.full((4, room), -1)
    for e, p in enumerate(paths):
        path[e, :len(p)] = p
    want = pool.clone()
    for e, p in enumerate(paths):
        for i, k in enumerate(p):
            a, b = ctx[e] + k, ctx[e] + i
            want[:, :, table[e, b // ps], :, b % ps] = pool[:, :, table[e, a // ps], :, a % ps]
    ops.keep_drafts(pool, ints(table), ints(np.concatenate([[0], np.cumsum(lens)])), ints([c + q for c, q in zip(ctx, lens)]), ints(path),
                    ints([len(p) for p in paths]))
    assert torch.equal(pool, want)
    assert ops.gemm_error_flag(torch.device(DEV)) == 0


def test_keep_drafts_stops_at_a_wrong_step():
    ops.gemm_error_flag(torch.device(DEV))
    for path, table, moved in (([0, 3, 2, 5], [1, 2], 2), ([0, 2, 9, 5], [1, 2], 2), ([1, 0, -1, 5], [1, 2], 1), ([0, 2, 6, 7], [1, 5], 2),
                               ([0, 2, 3, 7], [-1, 2], 0)):
        pool = torch.randn(2, 4, 1, 4, 8, device=DEV)
        was = pool.clone()
        ops.keep_drafts(pool, ints([table]), ints([0, 8]), ints([8]), ints([path]), ints([4]))
        assert ops.gemm_error_flag(torch.device(DEV)) != 0
        for i in range(moved):
            was[:, table[0], 0, i] = was[:, table[path[i] // 4], 0, path[i] % 4].clone()
        assert torch.equal(pool, was)


@pytest.mark.parametrize("shape, dt", [((3, 2, 40, 8, 16, 128), torch.bfloat16), ((40, 1, 1, 1), torch.bfloat16), ((2, 40, 3, 5, 7), torch.float32),
                                       ((2, 40, 1, 3, 3), torch.bfloat16), ((1, 2, 1200, 1, 2, 8), torch.float32)])
def test_copy_pages(shape, dt):
    r = np.random.RandomState(len(shape))
    pool = torch.randn(*shape, device=DEV).to(dt)
    pages = shape[-4]
    for n in sorted({0, 1, 5, pages // 2}):
        order = r.permutation(pages)
        dst, src = order[:n], r.choice(order[n:], size=n)          # pages that go to several places among them
        want = pool.clone().view(-1, pages, *shape[-3:])
        want[:, torch.tensor(dst, device=DEV)] = want[:, torch.tensor(src, device=DEV)]
        ops.copy_pages(pool, src.tolist() if n % 2 else src, dst.tolist())
        assert torch.equal(pool, want.view(shape))


def test_pages_far_into_a_pool():
    """Offsets that pass 32 bits: elements behind the first 2^31 of a pool, copied, moved and attended to."""
    pages = 530000                                                 # x 16 x 256 elements > 2^31
    pool = torch.empty(pages, 1, 16, 256, dtype=torch.bfloat16, device=DEV)
    assert pool.numel() > 2 ** 31
    far = pages - 3
    pool[:4] = torch.randn(4, 1, 16, 256, device=DEV)
    ops.copy_pages(pool, [0, 1, 2], [far, far + 1, far + 2])
    assert torch.equal(pool[far:far + 3], pool[:3])
    near = Case([9], [30], 2, 1, 256, 16, torch.bfloat16)
    near.k = near.v = pool[:4]
    near.table, near.tables = ints([[0, 1, 2]]), [torch.tensor([0, 1, 2], device=DEV)]
    want = near.run().clone()
    near.check()
    near.k = near.v = pool
    near.table = ints([[far, far + 1, far + 2]])
    near.run()
    assert torch.equal(near.out, want)
    ops.keep_drafts(pool, near.table, near.cu_q, near.kv_lens, ints([[0, 4, 5]]), ints([3]))
    assert torch.equal(pool[far + 1, 0, 15], pool[2, 0, 2]) and torch.equal(pool[far + 2, 0, 0], pool[2, 0, 3])


@pytest.mark.parametrize("dt, hd, keys", [(torch.float32, 16, 200_000_001), (torch.bfloat16, 16, 330_000_001), (torch.bfloat16, 64, 1 << 30)])
def test_as_many_keys_as_an_entry_may_have(dt, hd, keys):
    """One page over and over: parts times tiles pass 32 bits.  Scores are zero, so a weight is 1, sums of up to 2^24 of them
    are exact in float32, and what comes out is the page's value."""
    page = 512
    k, v = torch.randn(1, 1, page, hd, device=DEV).to(dt), torch.full((1, 1, page, hd), 0.75, device=DEV, dtype=dt)
    q, out = torch.zeros(1, hd, device=DEV, dtype=dt), torch.full((1, hd), 7.0, device=DEV, dtype=dt)
    table = torch.zeros(1, -(-keys // page), dtype=torch.int32, device=DEV)
    ops.gemm_error_flag(torch.device(DEV))
    ops.tree_attention(q, k, v, out, table, ints([0, 1]), ints([keys]), ints([[1]]), 1, 1, hd, page, 1.0, 1)
    assert ops.gemm_error_flag(torch.device(DEV)) == 0
    # what is added of the parts, at most 1,200 of them, is off by 2^-24 each
    assert (out.double() - 0.75).abs().max() <= 0.75 * (1200 * 2 * U + HALF[dt])


def test_a_table_of_more_keys_than_an_entry_may_have_is_refused():
    k = torch.zeros(1, 1, 1024, 16, device=DEV)
    q = torch.zeros(1, 16, device=DEV)
    with pytest.raises(Exception, match="more work than a call takes"):
        ops.tree_attention(q, k, k, q.clone(), ints(np.zeros((1, (1 << 20) + 1))), ints([0, 1]), ints([5]), ints([[1]]), 1, 1, 16, 1024, 1.0, 1)


def test_a_verification_as_it_is_used():
    """Mask, attention, the walk and the move, in a row and in a graph: the kept rows are the accepted tokens', and attention
    over them is that of the same tokens decoded one behind another."""
    r = np.random.RandomState(0)
    lens, ctx = [13, 30], [200, 77]
    trees = [tree(q, r) for q in lens]
    c = Case(lens, ctx, 8, 2, 128, 16, torch.float32, seed=3)
    parents = ints(np.concatenate(trees))
    tok = r.permutation(1000)[:43]
    want = 1000 + np.arange(43)
    line = [12]                                                    # of entry 0: the last token and what it descends from
    while line[0] > 0:
        line.insert(0, int(trees[0][line[0]]))
    want[line[:-1]] = tok[line[1:]]
    tokens, targets = ints(tok), ints(want)
    path, count, nxt = ints(np.zeros((2, 14))), ints([0, 0]), ints([0, 0])
    pool = torch.stack([c.k, c.v])
    start = pool.clone()

    def step():
        ops.draft_tree(parents, c.cu_q, c.kv_lens, c.positions, c.mask)
        ops.tree_attention(c.q, pool[0], pool[1], c.out, c.table, c.cu_q, c.kv_lens, c.mask, 8, 2, 128, 16, c.scale, 30)
        ops.accept_drafts(tokens, parents, targets, c.cu_q, path, count, nxt)
        ops.keep_drafts(pool, c.table, c.cu_q, c.kv_lens, path, count)

    step()
    out, kept = c.out.clone(), pool.clone()
    assert path[0, :len(line)].tolist() == line and count.tolist() == [len(line), 1] and nxt.tolist() == [1012, 1013]
    # the accepted tokens as a chain over the kept rows
    chain = Case([len(line)], [200], 8, 2, 128, 16, torch.float32, masks=[np.tril(np.ones((len(line),) * 2, dtype=bool))])
    chain.q, chain.k, chain.v = c.q[torch.tensor(line, device=DEV)].contiguous(), pool[0], pool[1]
    chain.table, chain.out = c.table[:1].contiguous(), torch.empty(len(line), 8 * 128, device=DEV)
    chain.run()
    assert (chain.out - out[torch.tensor(line, device=DEV)]).abs().max() <= 2 ** -18 * c.v.abs().max()
    pool.copy_(start)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    pool.copy_(start)
    c.out.zero_(), path.zero_(), c.mask.zero_()
    g.replay()
    assert torch.equal(c.out, out) and torch.equal(pool, kept) and path[0, :len(line)].tolist() == line


def test_refusals():
    c = Case([9, 20], [100, 30], 8, 2, 128, 16, torch.bfloat16)
    call = lambda **kw: ops.tree_attention(*[kw.get(n, d) for n, d in (
        ("q", c.q), ("k", c.k), ("v", c.v), ("out", c.out), ("table", c.table), ("cu", c.cu_q), ("kv", c.kv_lens), ("mask", c.mask),
        ("nq", 8), ("nkv", 2), ("hd", 128), ("ps", 16), ("scale", c.scale), ("most", 20))], positions=kw.get("pos"), window=kw.get("window", 0))
    call()
    for kw in ({"q": c.q.float()}, {"out": c.out.float()}, {"v": c.v.float()}, {"k": c.k.half(), "v": c.v.half(), "q": c.q.half(), "out": c.out.half()},
               {"q": c.q[:, :512]}, {"q": c.q.t().contiguous().t()}, {"k": c.k[:, :, ::2]}, {"nq": 7}, {"hd": 64}, {"ps": 8}, {"nkv": 4},
               {"cu": c.cu_q.long()}, {"cu": c.cu_q[:2]}, {"kv": c.kv_lens[:1]}, {"mask": c.mask[:5]}, {"mask": c.mask.long()}, {"table": c.table[:1]},
               {"most": 33}, {"most": 0}, {"window": 5}, {"window": -1}, {"pos": c.positions[:3]}, {"v": c.v[:3]}):
        with pytest.raises(ShapeError):
            call(**kw)
    with pytest.raises((ShapeError, Unavailable)):
        call(q=c.q.cpu())
    with pytest.raises(ShapeError):                                # 9 heads over 2 KV heads
        ops.tree_attention(torch.zeros(3, 9 * 128, device=DEV), torch.zeros(2, 2, 16, 128, device=DEV), torch.zeros(2, 2, 16, 128, device=DEV),
                           torch.zeros(3, 9 * 128, device=DEV), ints([[0]]), ints([0, 3]), ints([3]), ints(np.zeros((3, 1))), 9, 2, 128, 16, 1.0, 3)
    big = torch.zeros(2, 1, 16, 512, device=DEV)
    with pytest.raises(ShapeError):                                # heads of 512
        ops.tree_attention(torch.zeros(3, 512, device=DEV), big, big, torch.zeros(3, 512, device=DEV), ints([[0]]), ints([0, 3]), ints([3]),
                           ints(np.zeros((3, 1))), 1, 1, 512, 16, 1.0, 3)
    with pytest.raises(ShapeError):
        ops.draft_tree(ints([-1, 0]).long(), ints([0, 2]), ints([5]), ints([0, 0]), ints([[0], [0]]))
    with pytest.raises(ShapeError):
        ops.draft_tree(ints([-1, 0]), ints([0, 2]), ints([5]), ints([0, 0]), ints([[0], [0]]), window=-1)
    with pytest.raises(ShapeError):
        ops.draft_tree(ints([-1, 0]), ints([0, 2]), ints([5]), ints([0, 0]), ints(np.zeros((2, 0))))
    with pytest.raises(ShapeError):
        ops.accept_drafts(ints([1, 2]), ints([-1, 0]), ints([1, 2]), ints([0, 2]), ints(np.zeros((1, 0))), ints([0]), ints([0]))
    with pytest.raises(ShapeError):
        ops.accept_drafts(ints([1, 2]), ints([-1]), ints([1, 2]), ints([0, 2]), ints([[0]]), ints([0]), ints([0]))
    pool = torch.zeros(2, 6, 1, 4, 8, device=DEV)
    for src, dst in (([0], [6]), ([-1], [0]), ([2 ** 64], [1]), (np.array([7]), [1]), ([0], np.array([-1])), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([3], [3]), ([0], [1, 2]), ([0.5], [1]), ([[0]], [[1]]),
                     (ints([0]), [1])):
        with pytest.raises(ShapeError):
            ops.copy_pages(pool, src, dst)
    with pytest.raises(ShapeError):
        ops.copy_pages(pool.transpose(0, 1), [0], [1])
    with pytest.raises(ShapeError):
        ops.copy_pages(pool[0, 0], [0], [1])
    with pytest.raises(Unavailable):
        ops.copy_pages(pool.cpu(), [0], [1])
    with pytest.raises(ShapeError):
        ops.keep_drafts(pool, ints([[0]]), ints([0, 1]), ints([1]), ints([[0]]), ints([1, 1]))
    assert not pool.any()
