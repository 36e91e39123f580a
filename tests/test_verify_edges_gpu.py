"""Forks and drafted tokens through the engine, at their edges."""
import numpy as np
import pytest
from helpers import TOL, plain_logits, random_tokens

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


HEADS = {128: dict(num_attention_heads=8, num_key_value_heads=2, head_dim=128), 64: dict(num_attention_heads=6, num_key_value_heads=3, head_dim=64)}


def folder_of_heads(hd, tmp_path_factory):
    """A tiny model whose heads and pages the tensor-memory form of the drafted tokens' attention takes."""
    from conftest import TINY_B
    from safetyraise_lmengine_b200.weights.random_init import write_model_folder
    config = dict(TINY_B, **HEADS[hd])
    return config, write_model_folder(config, 20 + hd, str(tmp_path_factory.mktemp(f"heads{hd}") / "model"))


@pytest.mark.parametrize("hd, ps", [(128, 16), (64, 8), (128, 128)])
def test_trees_over_heads_of_the_served_models(hd, ps, tmp_path_factory):
    """bfloat16 heads of 128 and 64: the logits of every token of a tree are those of its line, and the walk takes the model's own
    tokens wherever they are ahead of the next best by more than both logits may be off."""
    from safetyraise_lmengine_b200 import Engine, StepEntry
    import plain_qwen3
    config, folder = folder_of_heads(hd, tmp_path_factory)
    cfg, w = plain_qwen3.read_model_folder(folder)
    vocab, rng = config["vocab_size"], np.random.default_rng(hd + ps)
    eng = Engine.from_folder(folder, dtype="bfloat16", page_size=ps, num_pages=64, max_requests=4, max_batch_tokens=256)
    slots, seqs, kept = [], [], []
    for n in (140, 21, 3):
        slots.append(eng.open_request())
        seqs.append(random_tokens(rng, n, vocab))
        eng.step([StepEntry(slots[-1], seqs[-1])])
    for turn in range(3):
        entries, trees = [], []
        for s, seq in zip(slots, seqs):
            first = int(rng.integers(0, vocab))
            truth = plain_qwen3.greedy_generate(cfg, w, seq + [first], 6)
            tokens, parents, line = [first], [-1], [0]
            for t in truth[:5]:
                at = line[-1]
                tokens += [(t + 1) % vocab, t, (t + 2) % vocab]
                parents += [at] * 3
                line.append(len(tokens) - 2)
            entries.append(StepEntry(s, tokens, (), None, parents))
            trees.append((tokens, parents, line))
        prep = eng.prepare([StepEntry(e.slot, e.tokens, range(len(e.tokens)), None, e.parents) for e in entries], drafts=True)
        logits = eng.launch(prep).cpu().numpy().copy()
        eng.revoke(prep)
        found, at = eng.verify(entries), 0
        for r, (v, (tokens, parents, line)) in enumerate(zip(found, trees)):
            sure, targets = True, []
            for i in range(len(tokens)):
                up, k = [], i
                while k >= 0:
                    up.insert(0, tokens[k])
                    k = parents[k]
                ref = plain_logits(folder, seqs[r] + up)[-1]
                assert np.abs(logits[at + i] - ref).max() <= TOL["bfloat16"] * np.abs(ref).max(), (r, i)
                if i in line and sure:
                    top = np.sort(ref)[-2:]
                    sure = bool(top[1] - top[0] > 2 * TOL["bfloat16"] * np.abs(ref).max())
                    if sure:
                        targets.append(i)
            at += len(tokens)
            n = min(len(targets) + 1, len(line))                   # the places behind sure choices
            assert v.path[:n] == line[:n]
            kept.append(len(v.path))
            seqs[r] = seqs[r] + [tokens[k] for k in v.path]
            assert eng.cache.length(slots[r]) == len(seqs[r])
    assert max(kept) >= 3 and eng.cache.audit() == 0
    # and what stands in the cache by now is the kept tokens'
    for s, seq in zip(slots, seqs):
        got = eng.step([StepEntry(s, [5], [0])]).cpu().numpy()[0]
        ref = plain_logits(folder, seq + [5])[-1]
        assert np.abs(got - ref).max() <= TOL["bfloat16"] * np.abs(ref).max()
