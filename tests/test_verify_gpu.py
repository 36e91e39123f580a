"""Drafted tokens, forks and compactions through the engine: the tokens and logits of requests that were served one token at a
time."""
import numpy as np
import pytest
import torch
from conftest import TINY
from helpers import TOL, plain_logits, random_tokens

import plain_qwen3

pytestmark = pytest.mark.gpu


def build(folder, dtype="float32", **kw):
    from safetyraise_lmengine_b200 import Engine
    kw.setdefault("num_pages", 64)
    kw.setdefault("page_size", 4)
    return Engine.from_folder(folder, dtype=dtype, max_requests=6, max_batch_tokens=256, **kw)


def drafted(rng, first, truth, vocab, size):
    """A tree of ``size`` tokens behind ``first``: some lines follow the truth for a while, siblings and the rest are wrong."""
    tokens, parents, good = [first], [-1], {0: 0}                 # good: place -> how many true tokens lead to it
    while len(tokens) < size:
        p = int(rng.integers(max(0, len(tokens) - 6), len(tokens)))
        right = p in good and good[p] < len(truth) and rng.random() < 0.6
        t = truth[good[p]] if right else int(rng.integers(0, vocab))
        if p in good and good[p] < len(truth) and t == truth[good[p]] \
                and not any(parents[k] == p and tokens[k] == t for k in range(len(tokens))):
            good[len(tokens)] = good[p] + 1
        tokens.append(t)
        parents.append(p)
    return tokens, parents


def best_line(tokens, parents, truth):
    line = [0]
    while len(line) - 1 < len(truth):
        child = [k for k in range(line[-1] + 1, len(tokens)) if parents[k] == line[-1] and tokens[k] == truth[len(line) - 1]]
        if not child:
            break
        line.append(child[0])
    return line


def test_drafts_give_the_tokens_of_greedy_decoding(tiny_folder):
    """Trees of every size, several requests at once, a plain step among them: the greedy continuation, token for token, and
    logits afterwards that are those of the whole sequence."""
    from safetyraise_lmengine_b200 import StepEntry
    name, folder = tiny_folder
    vocab = TINY[name][0]["vocab_size"]
    cfg, w = plain_qwen3.read_model_folder(folder)
    rng = np.random.default_rng(3)
    eng = build(folder)
    want, slots, done = {}, {}, {}
    for r, n in enumerate((5, 17, 1)):
        prompt = random_tokens(rng, n, vocab)
        want[r] = (prompt, plain_qwen3.greedy_generate(cfg, w, prompt, 24))
        slots[r] = eng.open_request()
        logits = eng.step([StepEntry(slots[r], prompt, [n - 1])])
        done[r] = [int(logits.argmax())]
    kept = []
    for turn in range(6):
        entries, lines = [], []
        for r in slots:
            truth = want[r][1]
            assert done[r] == truth[:len(done[r])]
            size = (1, 2, 7, 12, 33, 5)[(turn + r) % 6]
            ahead = truth[len(done[r]):]
            if turn == 4 and r == 0:                              # a chain, its parents left out
                tokens, parents = [done[r][-1]] + ahead[:3], None
                lines.append(best_line(tokens, [-1, 0, 1, 2], ahead))
            else:
                tokens, parents = drafted(rng, done[r][-1], ahead, vocab, size)
                lines.append(best_line(tokens, parents, ahead))
            entries.append(StepEntry(slots[r], tokens, (), eng.generation(slots[r]), parents))
        found = eng.verify(entries)
        for r, e, v, line in zip(slots, entries, found, lines):
            assert v.path == line
            done[r] += [e.tokens[k] for k in v.path[1:]] + [v.next_token]
            kept.append(len(v.path))
            assert eng.cache.length(slots[r]) == len(want[r][0]) + len(done[r]) - 1
        assert eng.cache.audit() == 0
    assert max(kept) >= 3 and min(kept) == 1
    for r in slots:
        seq = want[r][0] + done[r]
        assert done[r][:24] == want[r][1][:len(done[r])]
        logits = eng.step([StepEntry(slots[r], done[r][-1:], [0])]).cpu().numpy()
        ref = plain_logits(folder, seq)[-1:]
        assert np.abs(logits - ref).max() <= TOL["float32"] * np.abs(ref).max()
    for s in slots.values():
        eng.close_request(s)
    assert eng.cache.free_pages() == 64 and eng.cache.audit() == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logits_of_a_tree_are_those_of_its_lines(folder_b, dtype):
    """Every token of a tree, against the whole sequence that its line makes, in both types; heads of 32."""
    from safetyraise_lmengine_b200 import StepEntry
    rng = np.random.default_rng(0)
    vocab = TINY["B"][0]["vocab_size"]
    eng = build(folder_b, dtype)
    prompt = random_tokens(rng, 21, vocab)
    s = eng.open_request()
    eng.step([StepEntry(s, prompt)])
    tokens = random_tokens(rng, 11, vocab)
    parents = [-1, 0, 0, 1, 1, 2, 5, 6, 3, 8, 0]
    prep = eng.prepare([StepEntry(s, tokens, range(11), None, parents)], drafts=True)
    logits = eng.launch(prep).cpu().numpy()
    eng.revoke(prep)
    for i in range(11):
        line, k = [], i
        while k >= 0:
            line.insert(0, tokens[k])
            k = parents[k]
        ref = plain_logits(folder_b, prompt + line)[-1]
        assert np.abs(logits[i] - ref).max() <= TOL[dtype] * np.abs(ref).max(), i
    assert eng.cache.length(s) == 21 and eng.cache.audit() == 0


def test_drafts_under_a_window():
    """Attention over a window of 10 keys: trees deeper than the window, pages given back under them."""
    from safetyraise_lmengine_b200 import Engine, StepEntry, spec_from_config
    from safetyraise_lmengine_b200.parts.model import tensor_decls
    from safetyraise_lmengine_b200.weights.random_init import RandomWeights
    import test_toy_parts_gpu as toy
    toy.define_window_toy()
    src = RandomWeights(tensor_decls(spec_from_config(toy.WINDOW_CONFIG)), seed=11)
    w = {n: src.get(n) for n in src.names()}
    rng = np.random.default_rng(5)
    seq = [int(t) for t in rng.integers(0, 70, size=9)]
    eng = Engine.from_source(toy.WINDOW_CONFIG, src, dtype="float32", page_size=4, num_pages=16, max_requests=2, max_batch_tokens=128)
    for pool in eng.cache.kv_pools.values():
        pool.fill_(float("nan"))
    s = eng.open_request()
    first = int(eng.step([StepEntry(s, seq, [8])]).argmax())
    truth, t = [], seq + [first]
    for _ in range(45):
        t = t + [int(np.argmax(toy.plain_window_logits(w, t)[-1]))]
    truth = t[len(seq):]
    done = [first]
    while len(done) < 40:
        ahead = truth[len(done):]
        n = min(14, len(ahead))
        # a line of 14, and wrong siblings at every place of it
        tokens, parents = [done[-1]], [-1]
        for k in range(n):
            p = len(tokens) - 2 if k else 0
            tokens += [ahead[k], (ahead[k] + 1) % 70]
            parents += [p, p]
        v, = eng.verify([StepEntry(s, tokens, (), None, parents)])
        assert v.path == best_line(tokens, parents, ahead) and len(v.path) == n + 1
        done += [tokens[k] for k in v.path[1:]] + [v.next_token]
        assert done == truth[:len(done)] and eng.cache.audit() == 0
    eng.close_request(s)
    assert eng.cache.free_pages() == 16


def test_verify_refuses_and_fails_like_a_step(folder_a):
    from safetyraise_lmengine_b200 import StepEntry
    from safetyraise_lmengine_b200.errors import ResourceExhausted, ShapeError, StepFailed
    eng = build(folder_a, num_pages=6)
    s = eng.open_request()
    eng.step([StepEntry(s, [1, 2, 3, 4, 5])])
    before = (eng.cache.length(s), eng.cache.free_pages())
    for tokens, kw in (([1, 2], {"parents": [-1]}), ([1, 2], {"parents": [0, 0]}), ([1, 2], {"parents": [-1, 1]}), ([1, 2], {"parents": [-1, -1]}),
                       ([1, 2], {"want": [0]}), ([1, -1], {}), ([1, 10 ** 6], {}), ([], {}), ([1], {"generation": 77})):
        with pytest.raises(ShapeError):
            eng.verify([StepEntry(s, tokens, **kw)])
    with pytest.raises(ShapeError):
        eng.step([StepEntry(s, [1, 2], [0], parents=[-1, 0])])
    with pytest.raises(ResourceExhausted):
        eng.verify([StepEntry(s, list(range(30)))])
    eng.status[1] = 5                                             # the host stands in for a kernel that raises it
    with pytest.raises(StepFailed):
        eng.verify([StepEntry(s, [6, 7, 8], parents=[-1, 0, 0])])
    assert (eng.cache.length(s), eng.cache.free_pages()) == before and eng.cache.audit() == 0 and eng.read_faults() == [0] * 8
    got = eng.step([StepEntry(s, [6], [0])]).cpu().numpy()
    ref = plain_logits(folder_a, [1, 2, 3, 4, 5, 6])[-1:]
    assert np.abs(got - ref).max() <= TOL["float32"] * np.abs(ref).max()


@pytest.mark.parametrize("name", ["argmax", "accept_drafts", "keep_drafts"])
def test_an_error_on_the_host_behind_the_forward_keeps_nothing(folder_a, monkeypatch, name):
    from safetyraise_lmengine_b200 import StepEntry
    from safetyraise_lmengine_b200.kernels import ops
    eng = build(folder_a, num_pages=6)
    s = eng.open_request()
    eng.step([StepEntry(s, [1, 2, 3, 4, 5])])
    before = (eng.cache.length(s), eng.cache.free_pages())

    def fails(*_, **__):
        raise MemoryError("no memory")
    with monkeypatch.context() as m:
        m.setattr(ops, name, fails, raising=False)
        with pytest.raises(MemoryError):
            eng.verify([StepEntry(s, [6, 7, 8, 9, 10, 11, 12, 13], parents=[-1, 0, 0, 1, 1, 2, 2, 3])])
    assert (eng.cache.length(s), eng.cache.free_pages()) == before and eng.cache.audit() == 0
    got = eng.step([StepEntry(s, [6], [0])]).cpu().numpy()
    ref = plain_logits(folder_a, [1, 2, 3, 4, 5, 6])[-1:]
    assert np.abs(got - ref).max() <= TOL["float32"] * np.abs(ref).max()


def test_other_mixers_refuse_drafts(tmp_path_factory):
    from safetyraise_lmengine_b200 import StepEntry
    from safetyraise_lmengine_b200.errors import Unsupported
    import test_nekedra_gpu as nekedra
    for name in ("delta", "attention", "latent"):
        folder, cfg, _ = nekedra.folder_of(name, tmp_path_factory)
        eng = nekedra.build(folder, "float32")
        s = eng.open_request()
        with pytest.raises(Unsupported):
            eng.verify([StepEntry(s, [1, 2, 3])])
        assert eng.cache.length(s) == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_forked_requests_go_their_own_ways(folder_b, dtype):
    """Forks inside a page, at a page's border and behind one another; the branches are the sequences they stand for, the
    pages in front are held once; compaction in between moves what is held and changes nothing."""
    from safetyraise_lmengine_b200 import StepEntry
    rng = np.random.default_rng(1)
    vocab = TINY["B"][0]["vocab_size"]
    eng = build(folder_b, dtype)
    gone = eng.open_request()
    eng.step([StepEntry(gone, random_tokens(rng, 30, vocab))])    # low pages that are free later
    seqs = {}
    s = eng.open_request()
    seqs[s] = random_tokens(rng, 22, vocab)
    eng.step([StepEntry(s, seqs[s])])
    free = eng.cache.free_pages()
    for length in (None, 20, 3):
        f = eng.fork_request(s, length)
        seqs[f] = seqs[s][:22 if length is None else length]
    assert free - eng.cache.free_pages() == 2                      # the last page of two of them; the third ends at a border
    g = eng.fork_request(f)
    seqs[g] = list(seqs[f])
    eng.close_request(gone)
    assert eng.cache.compact() > 0 and eng.cache.audit() == 0
    for turn in range(5):
        entries = []
        for slot in seqs:
            new = random_tokens(rng, 1 + (turn + slot) % 3, vocab)
            entries.append(StepEntry(slot, new, range(len(new))))
        logits = eng.step(entries).cpu().numpy()
        at = 0
        for e in entries:
            seqs[e.slot] = seqs[e.slot] + list(e.tokens)
            ref = plain_logits(folder_b, seqs[e.slot])[-len(e.tokens):]
            assert np.abs(logits[at:at + len(e.tokens)] - ref).max() <= TOL[dtype] * np.abs(ref).max()
            at += len(e.tokens)
        if turn == 2:
            dead = next(iter(seqs))
            eng.close_request(dead)                                # the one that the others came from
            del seqs[dead]
            eng.cache.compact()
    for slot in seqs:
        eng.close_request(slot)
    assert eng.cache.free_pages() == 64 and eng.cache.audit() == 0


def test_a_request_truncated_into_a_shared_page(folder_b):
    """Goes on with other tokens; the one that it shares the page with still reads its own."""
    from safetyraise_lmengine_b200 import StepEntry
    rng = np.random.default_rng(2)
    vocab = TINY["B"][0]["vocab_size"]
    eng = build(folder_b)
    seq, other = random_tokens(rng, 16, vocab), random_tokens(rng, 9, vocab)
    a = eng.open_request()
    eng.step([StepEntry(a, seq)])
    b = eng.fork_request(a)
    eng.cache.truncate(a, 14)
    for slot, tokens in ((a, seq[:14] + other), (b, seq + other)):
        new = tokens[eng.cache.length(slot):]
        got = eng.step([StepEntry(slot, new, [len(new) - 1])]).cpu().numpy()
        ref = plain_logits(folder_b, tokens)[-1:]
        assert np.abs(got - ref).max() <= TOL["float32"] * np.abs(ref).max()


def test_a_fork_takes_the_fixed_size_state_along(tmp_path_factory):
    """A mixer with a state of its own: the fork's state is the request's, and both go on from it."""
    from safetyraise_lmengine_b200 import StepEntry
    from safetyraise_lmengine_b200.errors import ShapeError
    import test_nekedra_gpu as nekedra
    folder, cfg, _ = nekedra.folder_of("delta", tmp_path_factory)
    eng = nekedra.build(folder, "float32")
    rng = np.random.default_rng(4)
    seq, one, two = (random_tokens(rng, n, cfg["vocab"]) for n in (19, 6, 4))
    a = eng.open_request()
    with pytest.raises(ShapeError):                                # nothing of this request has run: the slot's state is not its own yet
        eng.fork_request(a)
    eng.step([StepEntry(a, seq)])
    b = eng.fork_request(a)
    with pytest.raises(ValueError):
        eng.fork_request(a, 7)
    got = eng.step([StepEntry(a, one, [5]), StepEntry(b, two, [3])]).cpu().numpy()
    alone = nekedra.build(folder, "float32")
    for row, new in zip(got, (one, two)):
        s = alone.open_request()
        alone.step([StepEntry(s, seq)])
        ref = alone.step([StepEntry(s, new, [len(new) - 1])]).cpu().numpy()[0]
        assert np.abs(row - ref).max() <= TOL["float32"] * np.abs(ref).max()
