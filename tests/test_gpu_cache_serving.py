"""Serving over 8-bit pages, over a window with first tokens, and in portions: the engine's paths on the GPU."""
import pytest
import torch

from pisceslx_b200 import YvConfig
from pisceslx_b200.models import build_model
from pisceslx_b200.ops import check_status
from pisceslx_b200.serve.engine import YvEngineConfig, YvInferenceEngine

pytestmark = pytest.mark.gpu
TOKENS = torch.randint(0, 2048, (300,), generator=torch.Generator().manual_seed(2)).tolist()
FORMS = [dict(), dict(kv_cache_dtype="fp8_e4m3"), dict(attention_window=70, first_tokens=4), dict(kv_cache_dtype="fp8_e4m3", attention_window=70, first_tokens=4)]


@pytest.fixture(scope="module")
def model():
    cfg = YvConfig.tiny_text_moe(vocab_size=2048)
    cfg.n_layer = 3
    return build_model(cfg, "cuda", torch.bfloat16, seed=3).eval()


def _engine(model, **kw):
    return YvInferenceEngine(model, cfg=YvEngineConfig(**{**dict(max_num_seqs=8, num_blocks=64, block_size=64, eos_token_id=-1), **kw}))


def _logits(engine, tokens, cuts):
    engine.cache.add_sequence(1)
    out = torch.cat([engine.run_tokens(1, tokens[lo:hi], list(range(hi - lo))).clone() for lo, hi in zip(cuts, cuts[1:])])
    check_status()
    return out


def _near(a, b, share):
    assert float((a - b).norm() / b.norm()) < share, float((a - b).norm() / b.norm())


@pytest.mark.parametrize("form", FORMS)
def test_portions_of_any_size_agree(model, form):
    """Long portions, a few tokens, single ones through the captured step: kernels of three kinds over the same pages.  bf16 rounds
    each of some ten intermediate results of a layer to 2^-8, differently where sums run in another order; with 8 bits the first
    portion of a prompt without a window meets unrounded keys and values as well (2^-4)."""
    whole = _logits(_engine(model, **form), TOKENS, [0, 300])
    cuts = [0, 130, 200, 205, 206, 221, 299, 300]
    parts = _logits(_engine(model, **form), TOKENS, cuts)
    _near(parts, whole, 0.06 if "kv_cache_dtype" in form else 0.03)
    portion = _logits(_engine(model, prefill_portion=100, **form), TOKENS, [0, 300])
    _near(portion, whole, 0.06 if "kv_cache_dtype" in form else 0.03)


@pytest.mark.parametrize("form", FORMS[1:])
def test_captured_steps_equal_eager_ones(model, form):
    outs = []
    for graphs in (True, False):
        engine = _engine(model, use_cuda_graphs=graphs, graph_max_seq_len=512, **form)
        reqs = [engine.add_request(TOKENS[i:i + n], max_new_tokens=k) for i, (n, k) in enumerate([(60, 12), (5, 3), (190, 7), (130, 20), (2, 2)])]
        engine.run_until_done()
        check_status()
        outs.append([r.output_ids for r in reqs])
        stats = engine.get_stats()["decode_graphs"]
        assert (stats["disabled_reason"] is None and stats["graph_replays"] > 0) == graphs
        assert engine.cache.alloc.available() == 64 - (1 if graphs else 0)
    assert outs[0] == outs[1]


def test_two_engines_with_caches_of_their_own_take_turns(model):
    """Captured steps of two engines, replayed in turn, do not share scratch."""
    forms = [FORMS[1], FORMS[3]]
    alone = []
    for f in forms:
        e = _engine(model, graph_max_seq_len=512, **f)
        r = e.add_request(TOKENS[:150], max_new_tokens=12)
        e.run_until_done()
        alone.append(r.output_ids)
    engines = [_engine(model, graph_max_seq_len=512, **f) for f in forms]
    reqs = [e.add_request(TOKENS[:150], max_new_tokens=12) for e in engines]
    while any(not r.finished for r in reqs):
        for e, r in zip(engines, reqs):
            if not r.finished:
                e.step()
    check_status()
    assert [r.output_ids for r in reqs] == alone


def test_a_prefix_is_read_back(model):
    exact, small = _engine(model), _engine(model, kv_cache_dtype="fp8_e4m3")
    for e in (exact, small):
        _logits(e, TOKENS, [0, 200])
    hk, d = small.cache.hk, small.cache.d
    for x, y in zip(exact.cache.read(1, 0), small.cache.read(1, 0)):
        assert x.shape == y.shape == (200, hk * d)
        x, y = x.double().view(200, hk, d), y.double().view(200, hk, d)
        assert bool(((x - y).abs() <= torch.maximum(2.0 ** -4 * x.abs(), 2.0 ** -10 / 224 * x.abs().amax(-1, keepdim=True))).all())
