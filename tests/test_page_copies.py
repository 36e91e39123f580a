"""Copies of pages that cannot be made (no GPU: pools on the host, the copying kernel's part played there)."""
import contextlib
import random

import numpy as np
import pytest
import torch

from safetyraise_lmengine_b200.cache.manager import FIXED_STATE, PAGED_ALL, PAGED_WINDOW, CacheGroupSpec, CacheManager
from safetyraise_lmengine_b200.kernels import ops

GROUPS = [CacheGroupSpec("all", PAGED_ALL, (0, 1), kv_heads=2, head_dim=16),
          CacheGroupSpec("split", PAGED_ALL, (2,), kv_heads=1, head_dim=8, v_head_dim=4),
          CacheGroupSpec("win", PAGED_WINDOW, (3,), kv_heads=1, head_dim=16, window=100)]
STATE = CacheGroupSpec("st", FIXED_STATE, (4,), state_shape=(4,))


class Device:
    """Copies on the host; from the call ``fails_at`` on there is no memory."""

    def __init__(self, monkeypatch):
        self.calls, self.fails_at = 0, None
        monkeypatch.setattr(torch.cuda, "device", lambda _: contextlib.nullcontext())
        monkeypatch.setattr(ops, "copy_pages", self.copy_pages, raising=False)

    def copy_pages(self, pool, src, dst):
        self.calls += 1
        if self.fails_at is not None and self.calls > self.fails_at:
            raise MemoryError("no memory")
        at = pool.dim() - 4
        pool.index_copy_(at, torch.tensor(dst).long(), pool.index_select(at, torch.tensor(src).long()))


def manager(groups, pages=16):
    m = CacheManager(groups, page_size=4, num_pages=pages, max_requests=4, dtype=torch.float32, device=torch.device("cpu"))
    for pools in (m.kv_pools, m.k_pools, m.v_pools):
        for p in pools.values():
            p.copy_(torch.rand_like(p))
    return m


def filled(m, n):
    s = m.open_request()
    assert m.reserve(s, n)
    m.commit(s, n)
    return s


def read(m, slot):
    """What the request's tokens hold, in every pool."""
    n, out = m.length(slot), []
    for g in m.paged_groups:
        table = torch.tensor(m.table(g.name, slot)).long()
        for pools in (m.kv_pools, m.k_pools, m.v_pools):
            if g.name in pools:
                p = pools[g.name]
                rows = p.index_select(p.dim() - 4, table).transpose(-4, -3).flatten(-3, -2)
                out.append(rows[..., :n, :].clone())
    return out


def standing(m, slots):
    return ([m.free_pages(g.name) for g in m.paged_groups], [[m.table(g.name, s) for g in m.paged_groups] for s in slots],
            [m.length(s) for s in slots], m.audit())


CALLS = {"fork": lambda m, a, b: m.fork(a, 10), "truncate": lambda m, a, b: m.truncate(b, 10), "compact": lambda m, a, b: m.compact()}


@pytest.mark.parametrize("what", CALLS)
@pytest.mark.parametrize("fails_at", [0, 1, 2, 3])
def test_a_copy_that_cannot_be_made_changes_nothing(monkeypatch, what, fails_at):
    dev, m = Device(monkeypatch), manager(GROUPS)
    low = filled(m, 12)
    a = filled(m, 16)
    b = m.fork(a)                                                  # shares a's four pages
    m.close_request(low)
    before, held = standing(m, (a, b)), [read(m, s) for s in (a, b)]
    dev.calls, dev.fails_at = 0, fails_at
    with pytest.raises(MemoryError):
        CALLS[what](m, a, b)
    assert standing(m, (a, b)) == before and before[-1] == 0
    for s, was in zip((a, b), held):
        assert all(torch.equal(x, y) for x, y in zip(read(m, s), was))
    dev.fails_at = None
    made = CALLS[what](m, a, b)                                    # goes through once there is memory
    assert m.audit() == 0
    for s, was in [(a, held[0]), (b, held[1])] + ([(made, held[0])] if what == "fork" else []):
        n = m.length(s)
        assert all(torch.equal(x, y[..., :n, :]) for x, y in zip(read(m, s), was))
    for s in [a, b] + ([made] if what == "fork" else []):
        m.close_request(s)
    assert [m.free_pages(g.name) for g in m.paged_groups] == [16] * 3


def test_a_state_that_cannot_be_copied_leaves_no_fork(monkeypatch):
    Device(monkeypatch)
    m = manager([GROUPS[0], STATE])
    a = filled(m, 10)
    before = standing(m, (a,))

    class Full:
        def __getitem__(self, _):
            raise MemoryError("no memory")

    with monkeypatch.context() as p:
        p.setitem(m.state_pools, "st", Full())
        with pytest.raises(MemoryError):
            m.fork(a)
    assert standing(m, (a,)) == before
    assert len([m.open_request() for _ in range(3)]) == 3          # every other slot is free


def test_what_is_planned_is_what_is_done():
    """The copies that a call would make, and those that it makes."""
    import ctypes as C
    rng, lib = random.Random(5), None
    m = CacheManager([GROUPS[0], GROUPS[2]], page_size=4, num_pages=30, max_requests=6)
    lib, slots, seen = m._lib, [], set()

    def ask(fn, *args):
        rows, n = np.zeros((64, 3), dtype=np.int32), C.c_int()
        r = fn(m._h, *args, rows.ctypes.data, 64, C.byref(n))
        return r, rows[:n.value].tolist()

    for _ in range(500):
        what = rng.choice(["open", "fork", "cut", "cut", "close", "compact"])
        if what == "open" and len(slots) < 6:
            s = m.open_request()
            if m.reserve(s, 4 * rng.randint(1, 5)):
                m.commit(s, m._lib.srlm_cache_reserved(m._h, s))
            slots.append(s)
        elif what == "close" and slots:
            m.close_request(slots.pop(rng.randrange(len(slots))))
        elif what in ("fork", "cut") and slots:
            s = rng.choice(slots)
            args = (s, rng.randint(0, m.length(s)))
            call = "fork" if what == "fork" else "unshare"
            before = standing(m, slots)
            plan = ask(lib.srlm_cache_plan, m._PAGE_CALLS[call], *args)
            assert standing(m, slots) == before
            assert ask(getattr(lib, "srlm_cache_" + call), *args) == plan
            seen.add((call, len(plan[1])))
            if call == "fork" and plan[0] >= 0:
                slots.append(plan[0])
        elif what == "compact":
            before = standing(m, slots)
            plan = ask(lib.srlm_cache_plan, 2, 0, 0)
            assert standing(m, slots) == before
            assert ask(lib.srlm_cache_compact) == plan
            seen.add((what, bool(plan[1])))
        assert m.audit() == 0
    assert {("fork", 0), ("fork", 2), ("unshare", 0), ("unshare", 2), ("compact", True)} <= seen
