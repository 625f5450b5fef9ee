"""Admission of requests whose window gives pages back: what counts is what a sequence holds at once."""
import pytest
import torch

from pisceslx_b200 import YvConfig
from pisceslx_b200.models import build_model
from pisceslx_b200.models.cache import RELEASED
from pisceslx_b200.serve.engine import YvEngineConfig, YvInferenceEngine

TOKENS = torch.randint(0, 300, (400,), generator=torch.Generator().manual_seed(5)).tolist()


@pytest.fixture(scope="module")
def model():
    cfg = YvConfig.tiny_text_moe(vocab_size=300)
    cfg.n_layer = 1
    return build_model(cfg, "cpu", torch.float32, seed=1).eval()


def _engine(model, **kw):
    return YvInferenceEngine(model, cfg=YvEngineConfig(**{**dict(max_num_seqs=4, block_size=16, eos_token_id=-1), **kw}))


def _most(engine):
    """Runs to the end; the most pages that were held at once, and by one sequence."""
    total = engine.cache.alloc.available()
    seen, one = [0], [0]
    alloc = engine.cache.alloc.alloc

    def counted():
        block = alloc()
        seen[0] = max(seen[0], total - engine.cache.alloc.available())
        held = max((sum(b != RELEASED for b in t) for t in engine.cache.tables.values()), default=0)
        one[0] = max(one[0], held + 1)
        return block

    engine.cache.alloc.alloc = counted
    engine.run_until_done()
    assert engine.cache.alloc.available() == total
    return seen[0], one[0]


def test_a_stream_longer_than_the_pool_runs_in_its_window(model):
    engine = _engine(model, num_blocks=10, attention_window=40, first_tokens=3, prefill_portion=20)
    reqs = [engine.add_request(TOKENS[:n], max_new_tokens=m) for n, m in ((300, 20), (5, 260), (400, 1))]
    _most(engine)
    assert [len(r.output_ids) for r in reqs] == [20, 260, 1] and all(r.finish_reason == "length" for r in reqs)
    # the same answers as with room for all
    wide = _engine(model, num_blocks=80, attention_window=40, first_tokens=3, prefill_portion=20)
    again = [wide.add_request(TOKENS[:n], max_new_tokens=m) for n, m in ((300, 20), (5, 260), (400, 1))]
    wide.run_until_done()
    assert [r.output_ids for r in reqs] == [r.output_ids for r in again]


@pytest.mark.parametrize("window", [1, 16, 17, 40, 1000])
@pytest.mark.parametrize("first", [0, 1, 33])
@pytest.mark.parametrize("portion", [0, 7, 16, 50])
def test_no_sequence_holds_more_than_was_reserved(model, window, first, portion):
    for n, m in ((120, 4), (3, 50)):
        engine = _engine(model, num_blocks=40, attention_window=window, first_tokens=first, prefill_portion=portion)
        req = engine.add_request(TOKENS[:n], max_new_tokens=m)
        need = engine._worst_case_blocks(req)
        _, held = _most(engine)
        assert len(req.output_ids) == m and held <= need <= -(-(n + m) // 16)


def test_a_prompt_that_runs_as_a_whole_needs_all_its_pages(model):
    engine = _engine(model, num_blocks=10, attention_window=40)
    long, short = engine.add_request(TOKENS[:300], max_new_tokens=2), engine.add_request(TOKENS[:60], max_new_tokens=200)
    engine.run_until_done()
    assert long.finish_reason.startswith("error") and len(short.output_ids) == 200


def test_several_streams_share_a_small_pool(model):
    engine = _engine(model, num_blocks=16, attention_window=30, first_tokens=2, prefill_portion=16)
    reqs = [engine.add_request(TOKENS[i:i + 90 + i], max_new_tokens=80) for i in range(6)]
    most, _ = _most(engine)
    assert all(len(r.output_ids) == 80 for r in reqs) and engine.stats["preemptions"] == 0 and most <= 16


def test_without_a_window_nothing_changes(model):
    engine = _engine(model, num_blocks=10)
    req = engine.add_request(TOKENS[:100], max_new_tokens=30)
    assert engine._worst_case_blocks(req) == 9
    long = engine.add_request(TOKENS[:300], max_new_tokens=2)
    engine.run_until_done()
    assert len(req.output_ids) == 30 and long.finish_reason.startswith("error")
