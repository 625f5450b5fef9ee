"""Serving over 8-bit pages, over a window with first tokens, and in portions: the engine's paths on the CPU."""
import pytest
import torch

from pisceslx_b200 import YvConfig
from pisceslx_b200.models import build_model
from pisceslx_b200.models.cache import RELEASED, YvCacheConfig, YvPagedKVCache, YvPagedLayeredCache, cache_for_model
from pisceslx_b200.serve.engine import YvEngineConfig, YvInferenceEngine

F8 = torch.float8_e4m3fn


def _model(layers=2):
    cfg = YvConfig.tiny_text_moe(vocab_size=300)
    cfg.n_layer = layers
    return build_model(cfg, "cpu", torch.float32, seed=1).eval()


@pytest.fixture(scope="module")
def model():
    return _model()


def _engine(model, **kw):
    return YvInferenceEngine(model, cfg=YvEngineConfig(**{**dict(max_num_seqs=4, num_blocks=64, block_size=16, eos_token_id=-1), **kw}))


def _logits(engine, tokens, cuts):
    """Logits of every token of a sequence that is run in the given portions."""
    engine.cache.add_sequence(1)
    out = []
    for lo, hi in zip(cuts, cuts[1:]):
        out.append(engine.run_tokens(1, tokens[lo:hi], list(range(hi - lo))))
    return torch.cat(out)


TOKENS = torch.randint(0, 300, (90,), generator=torch.Generator().manual_seed(2)).tolist()


def test_a_prompt_in_portions_gives_the_logits_of_the_whole(model):
    assert model.supports_portions
    whole = _logits(_engine(model), TOKENS, [0, 90])
    parts = _logits(_engine(model), TOKENS, [0, 33, 34, 35, 64, 90])
    assert torch.allclose(whole, parts, atol=2e-4, rtol=2e-4)              # sums of up to 90 and 256 products in 32 bits, other orders
    engine = _engine(model, prefill_portion=7)
    assert torch.allclose(_logits(engine, TOKENS, [0, 90]), whole, atol=2e-4, rtol=2e-4)


@pytest.mark.parametrize("window,first", [(20, 0), (20, 4), (5, 20), (200, 3)])
def test_a_window_does_not_depend_on_the_cuts_and_gives_pages_back(model, window, first):
    kw = dict(attention_window=window, first_tokens=first)
    whole = _logits(_engine(model, **kw), TOKENS, [0, 90])
    engine = _engine(model, **kw)
    parts = _logits(engine, TOKENS, [0, 33, 34, 35, 64, 89, 90])
    assert torch.allclose(whole, parts, atol=2e-4, rtol=2e-4)
    full = _logits(_engine(model), TOKENS, [0, 90])
    same = min(window, 90)
    assert torch.allclose(whole[:same], full[:same], atol=2e-4, rtol=2e-4)
    assert (window >= 90) == torch.allclose(whole, full, atol=2e-4, rtol=2e-4)
    table = engine.cache.tables[1]
    assert all(b != RELEASED for b in table[:-(-first // 16)])
    assert (RELEASED in table) == (window < 64)
    engine.cache.free_sequence(1)
    assert engine.cache.alloc.available() == 64


def test_a_window_masks_as_the_definition_says():
    """One layer: the hidden keys have no other way to reach a token."""
    model = _model(1)
    got = _logits(_engine(model, attention_window=8, first_tokens=2), TOKENS[:40], [0, 40])
    for i in (5, 20, 39):
        # the same token with the same positions, its hidden predecessors replaced: nothing changes
        other = [t if j < 2 or j > i - 8 else 299 - t for j, t in enumerate(TOKENS[:i + 1])]
        mine = _logits(_engine(model, attention_window=8, first_tokens=2), other, [0, i + 1])[-1]
        assert torch.allclose(mine, got[i], atol=1e-5)
    assert not torch.allclose(_logits(_engine(model), TOKENS[:40], [0, 40])[-1], got[-1], atol=1e-3)


def test_8_bit_pages_hold_a_little_over_half_and_answer_alike(model):
    exact, small = _engine(model), _engine(model, kv_cache_dtype="fp8_e4m3")
    assert small.cache.bytes() < 0.27 * exact.cache.bytes()                # codes for fp32 here
    a = _logits(exact, TOKENS, [0, 60, 89, 90])
    b = _logits(small, TOKENS, [0, 60, 89, 90])
    assert torch.allclose(a[:60], b[:60], atol=2e-4, rtol=2e-4)            # the first portion meets its keys as they were computed
    assert 0 < float((a[60:] - b[60:]).norm() / a[60:].norm()) < 0.1
    for idx in range(2):
        for x, y in zip(exact.cache.read(1, idx, 0, 60), small.cache.read(1, idx, 0, 60)):
            rows = x.double().view(60, -1, small.cache.d)
            off = (rows - y.double().view_as(rows)).abs()
            # half a step of a code
            assert bool((off <= torch.maximum(2.0 ** -4 * rows.abs(), 2.0 ** -10 / 224 * rows.abs().amax(-1, keepdim=True)) * (1 + 1e-6)).all())
    r = [small.add_request(TOKENS[:n], max_new_tokens=6) for n in (3, 40)]
    small.cache.free_sequence(1)
    small.run_until_done()
    assert all(len(x.output_ids) == 6 for x in r)


def test_a_saved_8_bit_cache_is_restored(model):
    engine = _engine(model, kv_cache_dtype="fp8_e4m3")
    _logits(engine, TOKENS, [0, 30])
    other = _engine(model, kv_cache_dtype="fp8_e4m3")
    other.cache.load_state(engine.cache.state())
    a, b = (e.run_tokens(1, TOKENS[30:37], [6]) for e in (engine, other))
    assert torch.equal(a, b)
    with pytest.raises(ValueError):
        _engine(model).cache.load_state(engine.cache.state())


def test_refusals(model):
    dev = torch.device("cpu")
    for kw in (dict(attention_window=0), dict(first_tokens=4), dict(attention_window=8, first_tokens=-1), dict(attention_window=8, sliding_window=8)):
        with pytest.raises(ValueError):
            YvPagedKVCache(1, 1, 64, YvCacheConfig(num_blocks=2, **kw), dev)
    for kw in (dict(dtype=F8), dict(attention_window=8)):
        with pytest.raises(ValueError):
            YvPagedLayeredCache([{"row": 64}], YvCacheConfig(num_blocks=2, **kw), dev)
    with pytest.raises(ValueError):
        _engine(model, kv_cache_dtype="int4")
    assert cache_for_model(model.cfg, dev, 2, dtype=F8).scales(0)[0].shape == (2, model.cfg.n_kv_head, model.cfg.kv_cache_block_size)


def test_pages_that_the_gpu_cannot_read_are_not_continued():
    """The kernels take heads of 64 or 128 numbers and pages of a multiple of 16 tokens: a prompt over other pages runs as a whole."""
    def at(d, block, dtype=torch.bfloat16):
        cache = YvPagedKVCache(1, 1, d, YvCacheConfig(num_blocks=2, block_size=block, dtype=dtype), torch.device("cpu"))
        here = cache.continues
        cache.device = torch.device("cuda")
        return here, cache.continues
    assert at(64, 16) == at(128, 64) == at(64, 48, F8) == (True, True)
    assert at(32, 16) == at(64, 8) == at(64, 16, torch.float32) == (True, False)
    cache = YvPagedLayeredCache([{"row": 24}], YvCacheConfig(num_blocks=2, block_size=8), torch.device("cpu"))
    cache.device = torch.device("cuda")
    assert cache.continues


def test_a_window_is_refused_where_prompts_are_padded(model, monkeypatch):
    with pytest.raises(ValueError, match="tensor parallelism"):
        cache_for_model(model.cfg, torch.device("cpu"), 2, tp_size=2, attention_window=8)
    from pisceslx_b200.models import generation
    engine = _engine(model, attention_window=8)
    engine.cache.add_sequence(1)
    monkeypatch.setattr(generation, "_tp_size", lambda m: 2)
    with pytest.raises(ValueError, match="pads"):
        generation._prefill(model, torch.zeros(1, 3, dtype=torch.long), engine.cache, [1])


def test_the_command_line_reaches_the_engine(monkeypatch):
    import sys
    import manage
    from pisceslx_b200.serve import server
    seen = {}
    monkeypatch.setitem(sys.modules, "uvicorn", type(sys)("uvicorn"))
    sys.modules["uvicorn"].run = lambda app, **kw: seen.update(kw)

    class Engine:
        def __init__(self, model, cfg):
            seen["cfg"] = cfg

    monkeypatch.setattr(server, "YvInferenceEngine", Engine)
    monkeypatch.setattr(server, "PiscesLxInferService", lambda *a: type("S", (), {"build_app": lambda self: None})())
    monkeypatch.setattr("pisceslx_b200.engine.loader.load_model_for_inference", lambda *a: None)
    args = manage.build_parser().parse_args(["serve", "--kv_cache_dtype", "fp8_e4m3", "--attention_window", "4096", "--first_tokens", "4", "--prefill_portion", "512"])
    server.PiscesLxBackendServer(args).run()
    cfg = seen["cfg"]
    assert (cfg.kv_cache_dtype, cfg.attention_window, cfg.first_tokens, cfg.prefill_portion) == ("fp8_e4m3", 4096, 4, 512)
