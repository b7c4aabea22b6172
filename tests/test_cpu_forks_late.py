"""Samples that are added when their prompt has been computed already."""
import pytest
import torch

from omni_npu_b200 import SamplingParams
from omni_npu_b200.config import ModelConfig
from omni_npu_b200.engine.llm import LLM


def _llm(**kw):
    cfg = ModelConfig(hidden_size=64, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=16, intermediate_size=128, vocab_size=97,
                      rope_theta=10000.0, max_position_embeddings=512, dtype=torch.float32)
    args = dict(model=cfg, device="cpu", max_num_seqs=8, max_num_batched_tokens=64, max_model_len=128, num_gpu_blocks=64,
                block_size=4, seed=1)
    args.update(kw)
    return LLM(**args)


def _sp(i=0, **kw):
    return SamplingParams(**{**dict(max_tokens=9, temperature=1.0, seed=3 + i, ignore_eos=True), **kw})


@pytest.mark.parametrize("tokens", [1, 4, 5, 11, 30])
@pytest.mark.parametrize("steps", [1, 2, 5])
@pytest.mark.parametrize("kw", [dict(), dict(enable_prefix_caching=True), dict(enable_mixed_batches=True),
                                dict(scheduling_policy="priority"), dict(additional_config={"async_scheduling": False})])
def test_a_late_sample_shares_the_prompt(tokens, steps, kw):
    p = torch.randint(1, 97, (tokens,), generator=torch.Generator().manual_seed(tokens)).tolist()
    alone = _llm()
    want = [alone.generate([p], _sp(i))[0].output_token_ids for i in range(3)]
    e = _llm(**kw).engine
    free, outs = e.scheduler.pool.num_free, {}

    def step():
        for o in e.step():
            outs[o.request_id] = o.output_token_ids
    a = e.add_request(p, _sp(0))
    for _ in range(steps):
        step()
    b = e.add_request(p, _sp(1), fork_of=a)
    step()
    c = e.add_request(p, _sp(2), fork_of=a)
    while e.has_unfinished_requests():
        step()
    assert [outs[r] for r in (a, b, c)] == want
    assert e.scheduler.fork_stats["requests"] == 2 and e.scheduler.fork_stats["shared_tokens"] == 2 * (tokens - 1)
    assert e.scheduler.pool.num_free == free and not e.scheduler.pool._ref and not e.scheduler.held


def test_a_sample_of_a_finished_or_evicted_request():
    p = list(range(1, 12))
    e = _llm().engine
    want = [_llm().generate([p], _sp(i))[0].output_token_ids for i in range(3)]
    a = e.add_request(p, _sp(0))
    outs = {}
    for _ in range(3):
        for o in e.step():
            outs[o.request_id] = o.output_token_ids
    for o in e._settle():
        outs[o.request_id] = o.output_token_ids
    first = e.scheduler.requests[a]
    e.scheduler.preempt_for_recompute(first)                  # its blocks are gone: the sample waits for the prompt once more
    e.worker.model_runner.input_batch.remove_request(a)
    b = e.add_request(p, _sp(1), fork_of=a)
    assert list(e.scheduler.held) == [b]
    while e.has_unfinished_requests():
        for o in e.step():
            outs[o.request_id] = o.output_token_ids
    c = e.add_request(p, _sp(2), fork_of=a)                   # nobody holds it any more
    assert not e.scheduler.held and e.scheduler.requests[c].block_ids == []
    while e.has_unfinished_requests():
        for o in e.step():
            outs[o.request_id] = o.output_token_ids
    assert [outs[r] for r in (a, b, c)] == want
    assert e.scheduler.pool.num_free == 64 and not e.scheduler.pool._ref
