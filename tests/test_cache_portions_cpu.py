"""Which prompts may be continued from a cache, and how: what is refused is refused before the sequence has grown."""
import pytest
import torch

from pisceslx_b200 import YvConfig
from pisceslx_b200.models import build_model, generation
from pisceslx_b200.models.cache import YvCacheConfig, YvPagedKVCache
from pisceslx_b200.ops import cache as C
from pisceslx_b200.serve.engine import YvEngineConfig, YvInferenceEngine

TOKENS = torch.randint(0, 300, (80,), generator=torch.Generator().manual_seed(5)).tolist()


def _model(**kw):
    cfg = YvConfig.tiny_text_moe(vocab_size=300)
    cfg.n_layer = 2
    for k, v in kw.items():
        setattr(cfg, k, v)
    return build_model(cfg, "cpu", torch.float32, seed=1).eval()


@pytest.fixture(scope="module")
def model():
    return _model()


def _cache(model, **kw):
    cfg = model.cfg
    return YvPagedKVCache(cfg.n_layer, cfg.n_kv_head, cfg.head_dim, YvCacheConfig(block_size=16, num_blocks=16, dtype=torch.float32, **kw), torch.device("cpu"))


def _run(model, cache, tokens):
    return generation._prefill(model, torch.tensor([tokens]), cache, [1])


def test_tables_that_are_cut_are_not_continued(model):
    """A sliding window's tables hold a sequence's last pages only: a later portion would read others' tokens at other positions."""
    cache = _cache(model, sliding_window=32)
    assert not cache.continues and _cache(model).continues
    cache.add_sequence(1)
    _run(model, cache, TOKENS[:70])
    before = (cache.lengths[1], list(cache.tables[1]), cache.alloc.available())
    with pytest.raises(ValueError, match="continue"):
        _run(model, cache, TOKENS[70:76])
    assert before == (cache.lengths[1], list(cache.tables[1]), cache.alloc.available())


def test_8_bit_pages_are_not_read_through_cut_tables():
    with pytest.raises(ValueError, match="sliding_window"):
        YvPagedKVCache(1, 1, 64, YvCacheConfig(num_blocks=2, dtype=torch.float8_e4m3fn, sliding_window=64), torch.device("cpu"))


def test_pages_that_no_kernel_reads_are_refused_before_slots_are_taken(model, monkeypatch):
    cache = _cache(model)
    cache.add_sequence(1)
    _run(model, cache, TOKENS[:20])
    monkeypatch.setattr(YvPagedKVCache, "continues", property(lambda self: False))
    with pytest.raises(ValueError, match="continue"):
        _run(model, cache, TOKENS[20:50])
    assert cache.lengths[1] == 20 and len(cache.tables[1]) == 2
    fresh = _cache(model)
    fresh.add_sequence(1)
    assert _run(model, fresh, TOKENS[:50]).shape == (1, 300)                     # prompts from their start need no pages
    engine = YvInferenceEngine(model, cfg=YvEngineConfig(num_blocks=16, block_size=16, prefill_portion=8, eos_token_id=-1))
    engine.cache.add_sequence(1)
    assert engine.run_tokens(1, TOKENS[:50], [49]).shape == (1, 300)             # as a whole


def test_experts_with_a_capacity_see_prompts_as_a_whole():
    """Which assignments a full expert drops depends on all tokens of the call."""
    dropping = _model(moe_drop_tokens=True, moe_capacity_factor=0.5, moe_min_capacity=1)
    assert any(blk.is_moe for blk in dropping.model.layers) and not dropping.supports_portions
    kw = dict(num_blocks=16, block_size=16, eos_token_id=-1)
    logits = []
    for portion in (0, 9):
        engine = YvInferenceEngine(dropping, cfg=YvEngineConfig(prefill_portion=portion, **kw))
        engine.cache.add_sequence(1)
        logits.append(engine.run_tokens(1, TOKENS, [79]))
    assert torch.equal(*logits)
    engine.cache.add_sequence(2)
    engine.run_tokens(2, TOKENS[:40], [])
    with pytest.raises(ValueError, match="continue"):
        engine.run_tokens(2, TOKENS[40:50], [9])
    assert engine.cache.lengths[2] == 40


def test_routes_that_are_kept_from_call_to_call_are_not_those_of_another_portion():
    model = _model(moe_gate_type="research", extra={"path_moe_stage_size": 2})
    assert model.model.layers[-1].mlp.router.path_stage_size == 2 and not model.supports_portions
    assert _model(moe_gate_type="research").supports_portions


def test_more_new_tokens_than_announced_are_refused():
    q, page = torch.randn(5, 2, 64), torch.randn(1, 16, 1, 64)
    args = (q, page, page, torch.zeros(2, 1, dtype=torch.int32), torch.tensor([9, 7], dtype=torch.int32), torch.tensor([0, 3, 5], dtype=torch.int32))
    want = C.cache_attention(*args, 3)
    assert torch.equal(C.cache_attention(*args), want) and torch.equal(C.cache_attention(*args, max_q=5), want)
    with pytest.raises(ValueError, match="new tokens"):
        C.cache_attention(*args, max_q=2)


def test_a_saved_cache_of_another_form_leaves_the_cache_as_it_was(model):
    def filled(**kw):
        cache = _cache(model, **kw)
        cache.add_sequence(1)
        _run(model, cache, TOKENS[:40])
        return cache
    plain, small = filled(), YvPagedKVCache(2, model.cfg.n_kv_head, model.cfg.head_dim, YvCacheConfig(
        block_size=16, num_blocks=16, dtype=torch.float8_e4m3fn), torch.device("cpu"))
    small.add_sequence(7)
    _run_in(model, small, 7, TOKENS[:20])
    one_layer = {k: v[:1] if k in ("k", "v") else v for k, v in plain.state().items()}
    other_pages = {k: [t[:, :8] for t in v] if k in ("k", "v") else v for k, v in plain.state().items()}
    for cache, states in ((plain, (small.state(), one_layer, other_pages)), (small, (plain.state(), other_pages))):
        before = cache.state()
        free, refs = list(cache.alloc.free), dict(cache.alloc.refs)
        before = {k: [t.clone() for t in v] if isinstance(v, list) else v for k, v in before.items()}
        for state in states:
            with pytest.raises(ValueError):
                cache.load_state(state)
        after = cache.state()
        assert (after["tables"], after["lengths"], cache.alloc.free, cache.alloc.refs) == (before["tables"], before["lengths"], free, refs)
        for name in ("k", "v", "k_scale", "v_scale"):
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before[name], after[name]))
    copy = _cache(model)
    copy.load_state(plain.state())
    assert torch.equal(copy.k[1], plain.k[1]) and copy.lengths == {1: 40}


def _run_in(model, cache, seq, tokens):
    return generation._prefill(model, torch.tensor([tokens]), cache, [seq])
