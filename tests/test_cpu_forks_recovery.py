"""Samples of one prompt when blocks that they share are lost in a failed step."""
import pytest
import torch

from omni_npu_b200 import SamplingParams
from omni_npu_b200.config import ModelConfig
from omni_npu_b200.engine.llm import LLM


def _llm(**kw):
    cfg = ModelConfig(hidden_size=64, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=16, intermediate_size=128, vocab_size=97,
                      rope_theta=10000.0, max_position_embeddings=512, dtype=torch.float32)
    args = dict(model=cfg, device="cpu", max_num_seqs=8, max_num_batched_tokens=64, max_model_len=128, num_gpu_blocks=64,
                block_size=4, seed=1, additional_config={"async_scheduling": False})
    args.update(kw)
    return LLM(**args)


P = [11, 12, 13, 14, 15, 16, 17, 18, 19, 20, 21]             # two whole blocks and two rows before the last token


def _wipe(llm, block):
    for t in llm.engine.worker.model_runner.page_cache.tensors:
        t[block] = 9.0


def _run(llm):
    outs = {}
    while llm.engine.has_unfinished_requests():
        for o in llm.engine.step():
            outs[o.request_id] = o
    return outs


def _sp(i=0):
    return SamplingParams(max_tokens=6, temperature=1.0, seed=3 + i, ignore_eos=True)


@pytest.mark.parametrize("which", [1, 2])                     # a block that is shared, and the one whose rows are copied
@pytest.mark.parametrize("caching", [False, True])
def test_a_waiting_sample_computes_a_lost_prompt_again(which, caching):
    want = {i: _llm().generate([P], _sp(i))[0].output_token_ids for i in range(3)}
    llm = _llm(max_num_seqs=1, enable_prefix_caching=caching)
    e = llm.engine
    a = e.add_request(P, _sp(0))
    b = e.add_request(P, _sp(1), fork_of=a)
    c = e.add_request(P, _sp(2), fork_of=a)
    e.step()                                                  # the prompt: the samples wait for a place with its blocks
    sched = e.scheduler
    first, waiting = sched.requests[a], [sched.requests[r] for r in (b, c)]
    assert all(r.block_ids == first.block_ids[:2] and r.fork_source for r in waiting)
    lost = first.block_ids[which]
    out = sched.schedule()
    _wipe(llm, lost)
    done = e._after_recovered_step(out, {"opt": "abort", "bad_blocks": [lost]})
    assert [o.request_id for o in done] == [a] and all(not r.block_ids and r.fork_source is None for r in waiting)
    outs = _run(llm)
    assert outs[b].output_token_ids == want[1] and outs[c].output_token_ids == want[2]
    assert sched.pool.num_free == 64 and not sched.pool._ref


def test_a_running_sample_outside_the_step_is_aborted():
    llm = _llm(max_num_seqs=4)
    e = llm.engine
    a = e.add_request(P, _sp(0))
    b = e.add_request(P, _sp(1), fork_of=a)
    e.step()
    e.step()                                                  # b runs with a's blocks
    other = e.add_request([5, 6, 7], _sp(2))
    sched = e.scheduler
    out = sched.schedule()
    assert [s.request.request_id for s in out.seqs] == [other]
    lost = sched.requests[a].block_ids[0]
    assert lost == sched.requests[b].block_ids[0]
    done = e._after_recovered_step(out, {"opt": "abort", "bad_blocks": [lost]})
    assert sorted(o.request_id for o in done) == sorted([a, b])
    assert _run(llm)[other].output_token_ids == _llm().generate([[5, 6, 7]], _sp(2))[0].output_token_ids
    assert sched.pool.num_free == 64 and not sched.pool._ref


def test_a_recomputed_step_leaves_shared_blocks_alone():
    want = [_llm().generate([P], _sp(i))[0].output_token_ids for i in range(2)]
    llm = _llm(max_num_seqs=1)
    e = llm.engine
    a = e.add_request(P, _sp(0))
    b = e.add_request(P, _sp(1), fork_of=a)
    e.step()
    out = e.scheduler.schedule()
    assert e._after_recovered_step(out, {"opt": "recompute", "bad_blocks": []}) == []
    assert e.scheduler.requests[b].fork_source is not None
    outs = _run(llm)
    assert [outs[a].output_token_ids, outs[b].output_token_ids] == want
    assert e.scheduler.pool.num_free == 64 and not e.scheduler.pool._ref
