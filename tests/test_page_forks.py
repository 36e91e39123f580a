"""Pages in several requests' tables (no GPU): who holds what after forks, truncations and compactions, and that no page that
two requests hold is ever written again."""
import random

import numpy as np
import pytest

from safetyraise_lmengine_b200.cache.manager import FIXED_STATE, PAGED_ALL, PAGED_WINDOW, CacheGroupSpec, CacheManager
from safetyraise_lmengine_b200.errors import ResourceExhausted

ALL = CacheGroupSpec("all", PAGED_ALL, (0, 1), kv_heads=2, head_dim=16)
WIN = CacheGroupSpec("win", PAGED_WINDOW, (2,), kv_heads=1, head_dim=16, window=10)
STATE = CacheGroupSpec("st", FIXED_STATE, (3,), state_shape=(4,))


def filled(m, n):
    s = m.open_request()
    assert m.reserve(s, n)
    m.commit(s, n)
    return s


def test_a_fork_shares_full_pages_and_copies_the_last():
    m = CacheManager([ALL], page_size=4, num_pages=8, max_requests=4)
    a = filled(m, 10)                                              # pages 0, 1 and half of 2
    b = m.fork(a)
    assert m.length(b) == 10 and m.table("all", b)[:2] == [0, 1] and m.table("all", b)[2] == 3
    assert m.free_pages("all") == 4 and m.audit() == 0
    c = m.fork(a, 8)                                               # at a page's border: nothing to copy
    assert m.table("all", c) == [0, 1] and m.length(c) == 8 and m.free_pages("all") == 4
    d = m.fork(c, 0)
    assert m.table("all", d) == [] and m.length(d) == 0
    for s in (a, b, c):                                            # each writes on pages of its own
        assert m.reserve(s, 12)
    own = [m.table("all", s)[2] for s in (a, b, c)]
    assert len(set(own)) == 3 and m.audit() == 0
    m.close_request(a)
    assert m.free_pages("all") == 4 and m.audit() == 0             # its own page; 0 and 1 stand in two more tables
    m.close_request(b)
    m.close_request(c)
    m.close_request(d)
    assert m.free_pages("all") == 8 and m.audit() == 0


def test_truncation_into_a_shared_page_gives_a_copy():
    m = CacheManager([ALL], page_size=4, num_pages=4, max_requests=3)
    a = filled(m, 8)
    b = m.fork(a)
    m.truncate(b, 6)                                               # inside page 1, which a holds too
    assert m.table("all", b) == [0, 2] and m.table("all", a) == [0, 1] and m.length(b) == 6 and m.audit() == 0
    m.truncate(b, 5)                                               # its own by now
    assert m.table("all", b) == [0, 2] and m.audit() == 0
    m.truncate(b, 4)
    assert m.table("all", b) == [0] and m.free_pages("all") == 2
    assert m.reserve(b, 12)
    with pytest.raises(ResourceExhausted):                         # no page left for the copy: nothing changes
        m.truncate(a, 2)
    assert m.table("all", a) == [0, 1] and m.length(a) == 8 and m.audit() == 0
    m.close_request(b)
    m.truncate(a, 2)                                               # nobody else's now
    assert m.table("all", a) == [0] and m.free_pages("all") == 3 and m.audit() == 0


def test_windows():
    m = CacheManager([ALL, WIN], page_size=4, num_pages=16, max_requests=3)
    a = filled(m, 30)
    passed = m.table("win", a)
    assert passed[:5] == [-1] * 5 and min(passed[5:]) >= 0         # a query at 30 sees keys from 21 on
    b = m.fork(a)
    assert m.table("win", b)[:5] == [-1] * 5 and m.table("win", b)[5:7] == passed[5:7] and m.audit() == 0
    with pytest.raises(ValueError):                                # the window needs pages that are gone
        m.fork(a, 20)
    c = m.fork(a, 29)                                              # a query there sees keys from 20 on: page 5
    assert m.audit() == 0 and m.table("win", c)[5:7] == passed[5:7]
    assert m.reserve(b, 50)
    m.commit(b, 50)                                                # passes the pages that it shares: a keeps them
    assert m.table("win", a) == passed and m.table("win", b)[:10] == [-1] * 10 and m.audit() == 0
    for s in (a, b, c):
        m.close_request(s)
    assert m.free_pages("win") == 16 and m.free_pages("all") == 16 and m.audit() == 0


def test_refusals_change_nothing():
    m = CacheManager([ALL, STATE], page_size=4, num_pages=3, max_requests=2)
    a = filled(m, 9)
    before = (m.table("all", a), m.free_pages("all"))
    with pytest.raises(ResourceExhausted):                         # no page for the copy of the third
        m.fork(a)
    with pytest.raises(ValueError):                                # the fixed-size state stands at 9 tokens
        m.fork(a, 8)
    n = CacheManager([ALL], page_size=4, num_pages=3, max_requests=2)
    s = filled(n, 9)
    for length in (10, -1):
        with pytest.raises(ValueError):
            n.fork(s, length)
    with pytest.raises(ValueError):
        n.fork(1)                                                  # not open
    with pytest.raises(ValueError):
        n.fork(7)
    n.fork(s, 8)
    with pytest.raises(ResourceExhausted):                         # no slot
        n.fork(s, 8)
    assert (m.table("all", a), m.free_pages("all")) == before and m.audit() == 0 and n.audit() == 0


def test_the_generation_of_a_forked_slot_grows():
    m = CacheManager([ALL], page_size=4, num_pages=8, max_requests=2)
    a = filled(m, 5)
    b = m.open_request()
    g = m.generation(b)
    m.close_request(b)
    assert m.fork(a) == b and m.generation(b) == g + 1


def test_compaction_moves_pages_to_the_lowest_numbers():
    m = CacheManager([ALL, WIN], page_size=4, num_pages=20, max_requests=4)
    a, b = filled(m, 16), filled(m, 15)
    c = m.fork(b)
    m.close_request(a)                                             # pages 0 .. 3 are free
    held = [m.table("all", s) for s in (b, c)]
    assert held[0][:3] == held[1][:3] and min(held[0]) == 4
    moved = m.compact()
    assert moved > 0 and m.audit() == 0
    now = [m.table("all", s) for s in (b, c)]
    assert sorted(set(sum(now, []))) == list(range(5)) and now[0][:3] == now[1][:3]
    assert m.compact() == 0                                        # nothing left to move
    assert m.reserve(c, 20) and m.table("all", c)[-1] == 5         # the lowest free page is next
    for s in (b, c):
        m.close_request(s)
    assert m.free_pages("all") == m.free_pages("win") == 20 and m.audit() == 0 and m.compact() == 0


@pytest.mark.parametrize("seed", range(6))
def test_drawn_at_random(seed):
    """Opens, forks, steps, steps taken back, truncations, compactions; beside it what each request's cells hold, written the way a
    device would: a cell that two requests hold must never be written by one of them."""
    rng = random.Random(seed)
    ps, pages = rng.choice([1, 3, 4]), 40
    m = CacheManager([ALL], page_size=ps, num_pages=pages, max_requests=6)
    pool, told = np.full((pages, ps), -1), {}
    count = 0

    # the copies that a call makes on the device: recorded as they are made
    real = m._with_copies

    def with_copies(what, room, *args):
        import ctypes as C
        copies, n = np.empty((max(room, 1), 3), dtype=np.int32), C.c_int()
        r = getattr(m._lib, "srlm_cache_" + what)(m._h, *args, copies.ctypes.data, max(room, 1), C.byref(n))
        src, dst = copies[:max(n.value, 0), 1], copies[:max(n.value, 0), 2]
        assert len(set(dst.tolist())) == len(dst) and not set(src.tolist()) & set(dst.tolist())
        if r >= 0:
            pool[dst] = pool[src]
        return r

    m._with_copies = with_copies
    assert real is not None
    for _ in range(400):
        what = rng.choice(["open", "fork", "step", "step", "step", "back", "cut", "close", "compact"])
        slots = list(told)
        if what == "open" and len(told) < 6:
            told[m.open_request()] = []
        elif what == "fork" and slots and len(told) < 6:
            s = rng.choice(slots)
            n = rng.randint(0, len(told[s]))
            try:
                told[m.fork(s, n)] = told[s][:n]
            except ResourceExhausted:
                pass
        elif what in ("step", "back") and slots:
            s = rng.choice(slots)
            have, n = len(told[s]), rng.randint(1, 9)
            if m.reserve(s, have + n):
                table = m.table("all", s)
                new = list(range(count, count + n))
                count += n
                for i, v in enumerate(new):
                    pool[table[(have + i) // ps], (have + i) % ps] = v
                if what == "step":
                    m.commit(s, have + n)
                    told[s] = told[s] + new
                else:
                    m.truncate(s, have)
        elif what == "cut" and slots:
            s = rng.choice(slots)
            n = rng.randint(0, len(told[s]))
            try:
                m.truncate(s, n)
                told[s] = told[s][:n]
            except ResourceExhausted:
                pass
        elif what == "close" and slots:
            s = rng.choice(slots)
            m.close_request(s)
            del told[s]
        elif what == "compact":
            m.compact()
        assert m.audit() == 0
        for s, cells in told.items():
            table = m.table("all", s)
            assert m.length(s) == len(cells)
            assert [int(pool[table[i // ps], i % ps]) for i in range(len(cells))] == cells
    for s in list(told):
        m.close_request(s)
    assert m.free_pages("all") == pages and m.audit() == 0
