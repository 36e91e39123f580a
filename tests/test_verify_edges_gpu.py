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


def test_a_wide_tree_at_the_end_of_the_context(folder_a):
    """Its lines fit, its tokens side by side do not; page and table have places for them all, and what is kept is the context's
    last tokens."""
    from safetyraise_lmengine_b200 import Engine, StepEntry
    from safetyraise_lmengine_b200.errors import ShapeError
    import plain_qwen3
    cfg, w = plain_qwen3.read_model_folder(folder_a)
    eng = Engine.from_folder(folder_a, dtype="float32", page_size=4, num_pages=24, max_requests=2, max_batch_tokens=64, max_context=32)
    prompt = random_tokens(np.random.default_rng(8), 28, cfg["vocab_size"])
    truth = plain_qwen3.greedy_generate(cfg, w, prompt, 5)
    s = eng.open_request()
    assert int(eng.step([StepEntry(s, prompt, [27])]).argmax()) == truth[0]
    wrong = [(t + 1) % cfg["vocab_size"] for t in truth]
    # the line of four behind wrong siblings at every place
    tokens, parents = [truth[0]] + [wrong[1]] * 6 + [truth[1], wrong[2], truth[2], wrong[3], truth[3]], [-1] + [0] * 7 + [7, 7, 9, 9]
    with pytest.raises(ShapeError):
        eng.verify([StepEntry(s, tokens + [1], parents=parents + [11])])
    v, = eng.verify([StepEntry(s, tokens, parents=parents)])
    assert v.path == [0, 7, 9, 11] and v.next_token == truth[4]
    assert eng.cache.length(s) == 32 and eng.cache.audit() == 0
    assert eng.cache.free_pages() == 16
