"""Forks and drafted tokens through the engine, at their edges."""
import numpy as np
import pytest
from helpers import TOL, random_tokens

pytestmark = pytest.mark.gpu


def test_a_fork_made_by_the_cache_takes_the_fixed_size_state_along(tmp_path_factory):
    """CacheManager.fork beside Engine.fork_request, and a fork of a fork: each goes on from the request's state."""
    from safetyraise_lmengine_b200 import StepEntry
    import test_nekedra_gpu as nekedra
    folder, cfg, _ = nekedra.folder_of("delta", tmp_path_factory)
    eng, alone = nekedra.build(folder, "float32"), nekedra.build(folder, "float32")
    rng = np.random.default_rng(6)
    seq = random_tokens(rng, 19, cfg["vocab"])
    news = [random_tokens(rng, n, cfg["vocab"]) for n in (6, 4, 1, 3)]
    a = eng.open_request()
    eng.step([StepEntry(a, seq)])
    b = eng.cache.fork(a)
    slots = [a, b, eng.fork_request(b), eng.cache.fork(b)]
    got = eng.step([StepEntry(s, new, [len(new) - 1]) for s, new in zip(slots, news)]).cpu().numpy()
    for row, new in zip(got, news):
        s = alone.open_request()
        alone.step([StepEntry(s, seq)])
        ref = alone.step([StepEntry(s, new, [len(new) - 1])]).cpu().numpy()[0]
        assert np.abs(row - ref).max() <= TOL["float32"] * np.abs(ref).max()
        alone.close_request(s)
