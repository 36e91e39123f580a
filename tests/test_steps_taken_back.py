"""Steps that are taken back while forks hold their pages (no GPU: accounting alone)."""
import contextlib
import types

import pytest
import torch

from safetyraise_lmengine_b200.cache.manager import PAGED_ALL, CacheGroupSpec, CacheManager
from safetyraise_lmengine_b200.engine.step import Engine, StepEntry
from safetyraise_lmengine_b200.errors import ResourceExhausted

ALL = CacheGroupSpec("all", PAGED_ALL, (0,), kv_heads=1, head_dim=8)


@pytest.fixture
def served(monkeypatch):
    monkeypatch.setattr(torch.cuda, "device", lambda _: contextlib.nullcontext())

    def make(pages):
        eng = Engine.__new__(Engine)
        eng.cache = CacheManager([ALL], page_size=4, num_pages=pages, max_requests=4)
        eng.mctx = types.SimpleNamespace(device=None)
        return eng
    return make


def filled(m, n):
    s = m.open_request()
    assert m.reserve(s, n)
    m.commit(s, n)
    return s


def ran(m, *steps):
    """Steps as ``Engine.run`` leaves them: (slot, tokens) each, committed."""
    starts = [m.length(s) for s, _ in steps]
    for (s, n), start in zip(steps, starts):
        assert m.reserve(s, start + n)
        m.commit(s, start + n)
    return types.SimpleNamespace(entries=[StepEntry(s, [1] * n) for s, n in steps], starts=starts, state_snapshot=None)


def test_a_step_whose_pages_a_fork_shares_is_taken_back_with_the_pages_that_its_others_return(served):
    eng = served(5)
    m = eng.cache
    a, b = filled(m, 6), filled(m, 4)
    prep = ran(m, (a, 2), (b, 4))                                  # a's second page is full, b has a second one
    f = m.fork(a, 8)
    c = filled(m, 4)                                               # the last free page
    assert m.free_pages("all") == 0
    eng.revoke(prep)                                               # a's copy goes into what b gives back
    assert [m.length(s) for s in (a, b, f, c)] == [6, 4, 8, 4] and m.audit() == 0
    assert m.table("all", a)[0] == m.table("all", f)[0] and m.table("all", a)[1] != m.table("all", f)[1]


def test_what_cannot_be_taken_back_is_said_behind_the_rest(served):
    eng = served(6)
    m = eng.cache
    a, b = filled(m, 6), filled(m, 5)
    prep = ran(m, (a, 2), (b, 2))
    f = m.fork(a, 8)
    c = filled(m, 8)
    assert m.free_pages("all") == 0
    with pytest.raises(ResourceExhausted, match=f"slot {a}|slots.*{a}"):
        eng.revoke(prep)
    assert m.length(b) == 5 and m.length(a) == 8 and m.audit() == 0
    m.close_request(c)
    m.truncate(a, 6)
    assert m.length(a) == 6 and m.length(f) == 8 and m.audit() == 0
