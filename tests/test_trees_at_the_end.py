"""Trees of drafted tokens near the end of a context (no GPU: the checks alone)."""
import types

import pytest

from safetyraise_lmengine_b200.cache.manager import PAGED_ALL, CacheGroupSpec, CacheManager
from safetyraise_lmengine_b200.engine.step import Engine, StepEntry
from safetyraise_lmengine_b200.errors import ShapeError


def test_a_tree_counts_by_its_longest_line():
    eng = Engine.__new__(Engine)
    eng.cache = CacheManager([CacheGroupSpec("all", PAGED_ALL, (0,), kv_heads=1, head_dim=8)], page_size=4, num_pages=16, max_requests=2)
    eng.spec, eng.mctx, eng.max_context = types.SimpleNamespace(vocab_size=50), types.SimpleNamespace(max_batch_tokens=64), 32
    s = eng.cache.open_request()
    assert eng.cache.reserve(s, 28)
    eng.cache.commit(s, 28)
    wide = [-1] + [0] * 9 + [3, 10]                                # twelve tokens, lines of up to four
    eng._validate([StepEntry(s, [1] * 12, parents=wide)])
    for parents in (wide + [11], None, list(range(-1, 11))):       # a line of five; a chain of twelve
        with pytest.raises(ShapeError, match="context"):
            eng._validate([StepEntry(s, [1] * 12 + [1] * (parents is not None and len(parents) > 12), parents=parents)])
    eng._validate([StepEntry(s, [1] * 4)])
