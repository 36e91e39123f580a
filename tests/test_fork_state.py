"""The fixed-size state of forked requests, between the cache manager and the engine that runs them (no GPU)."""
import pytest
import torch

from safetyraise_lmengine_b200.cache.manager import FIXED_STATE, PAGED_ALL, CacheGroupSpec, CacheManager
from safetyraise_lmengine_b200.engine.step import Engine, StepEntry

ALL = CacheGroupSpec("all", PAGED_ALL, (0,), kv_heads=1, head_dim=8)
STATE = CacheGroupSpec("st", FIXED_STATE, (1,), state_shape=(4,))


def served():
    """(engine, manager) with pools on the host; only what greets a step's slots is there of the engine."""
    m = CacheManager([ALL, STATE], page_size=4, num_pages=8, max_requests=4, dtype=torch.float32, device=torch.device("cpu"))
    eng = Engine.__new__(Engine)
    eng.cache, eng._slot_generation = m, [0] * m.max_requests
    return eng, m


def greet(eng, *slots):
    eng._greet_new_occupants([StepEntry(s, [1]) for s in slots], [eng.cache.generation(s) for s in slots])


def begun(eng, m, state):
    """A request of four tokens whose state is ``state``."""
    s = m.open_request()
    greet(eng, s)
    assert m.reserve(s, 4)
    m.commit(s, 4)
    m.state_pools["st"][:, s] = state
    return s


def test_the_state_of_a_fork_outlives_its_first_step():
    eng, m = served()
    a = begun(eng, m, 5.0)
    b = m.fork(a)
    c = m.fork(b)                                                  # of one that has not run a step of its own yet
    greet(eng, a, b, c)
    for s in (a, b, c):
        assert (m.state_pools["st"][:, s] == 5.0).all()


def test_a_slot_that_was_a_fork_starts_its_next_request_from_zero():
    eng, m = served()
    a = begun(eng, m, 5.0)
    b = m.fork(a)
    m.close_request(b)
    assert m.open_request() == b
    greet(eng, a, b)
    assert (m.state_pools["st"][:, a] == 5.0).all() and not m.state_pools["st"][:, b].any()


@pytest.mark.parametrize("ran", [False, True])
def test_a_fork_of_a_request_without_tokens_starts_from_zero(ran):
    """What the slot's state holds by then is the request's before it."""
    eng, m = served()
    a = begun(eng, m, 5.0)
    m.close_request(a)
    assert m.open_request() == a
    if ran:
        greet(eng, a)
    b = m.fork(a)
    greet(eng, b)
    assert not m.state_pools["st"][:, b].any()
