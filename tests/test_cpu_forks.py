"""Several samples of one prompt: the prompt is computed once, its blocks are shared, the partly filled one is copied."""
import pytest
import torch

from omni_npu_b200 import SamplingParams
from omni_npu_b200.config import CacheConfig, ModelConfig, SchedulerConfig
from omni_npu_b200.engine.block_manager import BlockPool
from omni_npu_b200.engine.llm import LLM
from omni_npu_b200.engine.request import Request
from omni_npu_b200.engine.scheduler import Scheduler


def _llm(**kw):
    cfg = ModelConfig(hidden_size=64, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=16, intermediate_size=128, vocab_size=97,
                      rope_theta=10000.0, max_position_embeddings=512, dtype=torch.float32)
    args = dict(model=cfg, device="cpu", max_num_seqs=8, max_num_batched_tokens=64, max_model_len=128, num_gpu_blocks=64,
                block_size=4, seed=1)
    args.update(kw)
    return LLM(**args)


def prompt(n, seed=0):
    return torch.randint(1, 97, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def separate(llm, p, sp, n):
    """The same samples as requests of their own, one after another."""
    return [llm.generate([p], SamplingParams(**{**sp, "seed": sp["seed"] + i}))[0].output_token_ids for i in range(n)]


@pytest.mark.parametrize("tokens", [1, 2, 4, 5, 9, 30, 70])
@pytest.mark.parametrize("kw", [dict(), dict(enable_prefix_caching=True), dict(enable_mixed_batches=True),
                                dict(additional_config={"async_scheduling": False})])
def test_samples_equal_separate_requests(tokens, kw):
    p, sp = prompt(tokens, tokens), dict(max_tokens=6, temperature=1.0, seed=5, ignore_eos=True)
    want = separate(_llm(), p, sp, 5)
    llm = _llm(**kw)
    free = llm.engine.scheduler.pool.num_free
    outs = llm.generate([p, prompt(7)], [SamplingParams(**sp, n=5), SamplingParams(max_tokens=3, ignore_eos=True)])
    assert [outs[0].output_token_ids, *[o.output_token_ids for o in outs[0].others]] == want
    assert not outs[1].others and len(outs) == 2
    sched = llm.engine.scheduler
    assert sched.fork_stats["requests"] == 4 and sched.fork_stats["shared_tokens"] == 4 * (tokens - 1)
    assert sched.pool.num_free == free and not sched.pool._ref and not sched.held and not sched.requests


@pytest.mark.parametrize("blocks", [9, 11, 14])
def test_a_full_cache_evicts_and_recomputes(blocks):
    p, sp = prompt(14, 3), dict(max_tokens=9, temperature=1.0, seed=2, ignore_eos=True)
    want = separate(_llm(), p, sp, 6)
    llm = _llm(num_gpu_blocks=blocks)
    o = llm.generate([p], [SamplingParams(**sp, n=6)])[0]
    assert [o.output_token_ids, *[x.output_token_ids for x in o.others]] == want
    assert llm.engine.scheduler.pool.num_free == blocks and not llm.engine.scheduler.pool._ref


def test_one_token_samples():
    """A parent that ends with the step that computed its prompt."""
    p, sp = prompt(10, 3), dict(max_tokens=1, temperature=1.0, seed=2, ignore_eos=True)
    want = separate(_llm(), p, sp, 4)
    llm = _llm()
    o = llm.generate([p], [SamplingParams(**sp, n=4)])[0]
    assert [o.output_token_ids, *[x.output_token_ids for x in o.others]] == want
    assert llm.engine.scheduler.pool.num_free == 64


def test_cache_without_page_copies_shares_whole_blocks():
    p, sp = prompt(10, 3), dict(max_tokens=4, temperature=1.0, seed=2, ignore_eos=True)
    want = separate(_llm(), p, sp, 3)
    llm = _llm()
    llm.engine.scheduler.copies_pages = False
    o = llm.generate([p], [SamplingParams(**sp, n=3)])[0]
    assert [o.output_token_ids, *[x.output_token_ids for x in o.others]] == want
    assert llm.engine.scheduler.fork_stats["shared_tokens"] == 2 * 8


def _scheduler(num_blocks=32, **kw):
    s = Scheduler(SchedulerConfig(max_num_seqs=4, max_num_batched_tokens=8, max_model_len=64, **kw), CacheConfig(block_size=4),
                  num_blocks=num_blocks)
    s.copies_pages = True
    return s


def _req(rid, toks, **kw):
    return Request(rid, toks, SamplingParams(**{**dict(max_tokens=3, ignore_eos=True), **kw}))


def test_blocks_and_copies_of_a_step():
    s = _scheduler()
    p = list(range(1, 12))                                    # 11 tokens: two whole blocks and two rows before the last token
    a, b, c, late = _req("a", p), _req("b", p), _req("c", p), _req("late", [9, 9])
    s.add_request(a)
    s.add_fork(b, "a")
    s.add_fork(c, "a")
    s.add_request(late)
    out = s.schedule()                                        # the first chunk: its samples wait
    assert [q.request for q in out.seqs] == [a] and set(s.held) == {"b", "c"} and s.num_unfinished == 4
    s.update_from_output(out, [0])
    out = s.schedule()                                        # the rest, and the request behind it
    assert [q.request for q in out.seqs] == [a, late] and not out.block_copies
    s.update_from_output(out, [7, 8])
    assert not s.held and b.block_ids == a.block_ids[:2] and b.num_computed_tokens == 10
    out = s.schedule()                                        # both samples compute the last token
    new = {q.request: q for q in out.seqs}
    assert set(new) == {b, c} and all(q.start == 10 and q.num_new_tokens == 1 and q.samples for q in new.values())
    assert sorted(out.block_copies) == sorted([(a.block_ids[2], b.block_ids[2], 2), (a.block_ids[2], c.block_ids[2], 2)])
    assert len({a.block_ids[2], b.block_ids[2], c.block_ids[2]}) == 3
    s.update_from_output(out, [1, 2])
    while s.has_unfinished():
        out = s.schedule()
        s.update_from_output(out, [3] * len(out.seqs))
    assert s.pool.num_free == 32 and not s.pool._ref


def test_a_source_is_not_given_out_before_it_was_copied():
    s = _scheduler(num_blocks=6)
    p = list(range(1, 7))
    a, b = _req("a", p, max_tokens=1), _req("b", p)
    s.add_request(a)
    s.add_fork(b, "a")
    out = s.schedule()
    tail = a.block_ids[1]
    s.update_from_output(out, [7])                            # the parent is done
    assert a.is_finished
    out = s.schedule()
    assert out.block_copies == [(tail, b.block_ids[1], 1)] and b.block_ids[1] != tail and tail not in s.pool._free
    s.update_from_output(out, [8])
    assert tail in s.pool._free


def test_aborts():
    p = list(range(1, 12))
    # of the parent before its prompt is done: a sample takes its place
    s = _scheduler()
    a, b, c = _req("a", p), _req("b", p), _req("c", p)
    s.add_request(a)
    s.add_fork(b, "a")
    s.add_fork(c, "a")
    s.update_from_output(s.schedule(), [0])
    s.abort_request("a")
    assert list(s.waiting) == [b] and set(s.held) == {"c"} and b.forks == [c]
    while s.has_unfinished():
        out = s.schedule()
        s.update_from_output(out, [3] * len(out.seqs))
    assert b.output_token_ids == c.output_token_ids == [3, 3, 3] and s.fork_stats["requests"] == 1
    assert s.pool.num_free == 32 and not s.pool._ref
    # of a sample that is held, and of one that has its blocks but does not run yet
    s = _scheduler()
    a, b, c = _req("a", p), _req("b", p), _req("c", p)
    s.add_request(a)
    s.add_fork(b, "a")
    s.add_fork(c, "a")
    s.abort_request("b")
    assert a.forks == [c] and set(s.held) == {"c"}
    for _ in range(2):
        s.update_from_output(s.schedule(), [0])
    assert list(s.waiting) == [c] and c.fork_source is not None
    s.abort_request("c")
    s.abort_request("a")
    assert s.pool.num_free == 32 and not s.pool._ref and not s.has_unfinished()


def test_requests_that_cannot_share_are_ordinary():
    p = list(range(1, 12))
    s = _scheduler()
    a = _req("a", p)
    s.add_request(a)
    s.add_fork(_req("other", p[:-1]), "a")
    s.add_fork(_req("unknown", p), "nobody")
    s.add_fork(_req("rows", p, prompt_logprobs=0), "a")
    assert not s.held and len(s.waiting) == 4
    b = _req("b", p)
    b.adapter = "x"
    s.add_fork(b, "a")
    assert not s.held and len(s.waiting) == 5


def test_shared_blocks_return_with_their_last_user():
    pool = BlockPool(8, 4)
    a = pool.allocate(3)
    pool.share(a[:2])
    pool.share(a[:1])
    pool.free(a)
    assert pool.num_free == 6
    pool.free(a[:2])
    assert pool.num_free == 7
    pool.free(a[:1])
    assert pool.num_free == 8 and not pool._ref and sorted(pool._free) == list(range(8))


def test_n_is_checked():
    with pytest.raises(ValueError):
        _llm().generate([[1, 2]], SamplingParams(n=0))
