"""Several samples of one prompt asked of a server."""
import threading

import pytest
import torch

from omni_npu_b200 import SamplingParams
from omni_npu_b200.config import ModelConfig
from omni_npu_b200.engine.llm import LLM

pytest.importorskip("fastapi")
from starlette.testclient import TestClient  # noqa: E402

from omni_npu_b200.serving.api_server import EngineLoop, build_app  # noqa: E402


def _llm(**kw):
    cfg = ModelConfig(hidden_size=64, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=16, intermediate_size=128, vocab_size=97,
                      rope_theta=10000.0, max_position_embeddings=4096, dtype=torch.float32)
    args = dict(model=cfg, device="cpu", max_num_seqs=16, max_num_batched_tokens=64, max_model_len=2048, num_gpu_blocks=1024,
                block_size=4, seed=1)
    args.update(kw)
    return LLM(**args)


class Noticing:
    """A lock that lets the engine's thread in whenever it is given back."""

    def __init__(self, engine):
        self.lock, self.engine = threading.Lock(), engine

    def __enter__(self):
        self.lock.acquire()

    def __exit__(self, *exc):
        for _ in range(3):
            if self.engine.has_unfinished_requests():
                self.engine.step()
        self.lock.release()


def test_no_step_runs_between_the_samples_of_a_request():
    llm = _llm()
    loop = EngineLoop(llm)
    loop.shutdown()                                           # (this test steps)
    loop.lock = Noticing(llm.engine)
    p = list(range(1, 12))
    sps = [SamplingParams(max_tokens=2, temperature=1.0, seed=i, ignore_eos=True) for i in range(8)]
    rids = loop.submit_samples(p, sps)
    assert len(set(rids)) == 8 and set(loop.waiters) == set(rids)
    assert llm.engine.scheduler.fork_stats["requests"] == 7


def test_all_samples_are_added_or_none():
    llm = _llm()
    loop = EngineLoop(llm)
    loop.shutdown()
    good, calls = SamplingParams(max_tokens=2), []

    def add(*a, inner=llm.engine.add_request, **kw):
        calls.append(kw["request_id"])
        if len(calls) == 3:
            raise ValueError("no")
        return inner(*a, **kw)
    llm.engine.add_request = add
    with pytest.raises(ValueError):
        loop.submit_samples([1, 2, 3], [good] * 4)
    assert not loop.waiters and not llm.engine.has_unfinished_requests() and loop.counters["requests"] == 0
    assert llm.engine.scheduler.pool.num_free == 1024


def test_a_busy_server_shares_the_prompt():
    llm = _llm()
    app = build_app(llm, model_name="base")
    loop = app.state.engine_loop
    body = {"prompt": list(range(1, 40)), "max_tokens": 1, "temperature": 1.0, "seed": 4, "ignore_eos": True}
    with TestClient(app) as client:
        alone = [client.post("/v1/completions", json={**body, "seed": 4 + i}).json()["choices"][0]["token_ids"] for i in range(8)]
        for round_ in range(1, 4):
            rid = loop.submit([3, 4, 5], SamplingParams(max_tokens=1500, ignore_eos=True))
            got = client.post("/v1/completions", json={**body, "n": 8}).json()["choices"]
            assert [c["token_ids"] for c in got] == alone
            assert llm.engine.scheduler.fork_stats["requests"] == 7 * round_
            loop.abort(rid)
    loop.shutdown()
