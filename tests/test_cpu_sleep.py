"""What sleep mode discards and what has to outlive it."""
import json
from contextlib import contextmanager

import pytest
import torch

from omni_npu_b200 import SamplingParams, ops
from omni_npu_b200.config import ModelConfig
from omni_npu_b200.engine.llm import LLM
from omni_npu_b200.worker import mem_pool


class FakePool:
    """Records which tag is active, and what was asked of it."""

    def __init__(self):
        self.tag, self.calls, self._sleeping = None, [], False

    @contextmanager
    def use_memory_pool(self, tag=None):
        old, self.tag = self.tag, tag
        try:
            yield
        finally:
            self.tag = old

    def sleep(self, offload_tags=None):
        self.calls.append(("sleep", tuple(offload_tags)))
        self._sleeping = True
        return 1

    def wake_up(self, tags=None):
        self.calls.append(("wake", tags))
        self._sleeping = tags is not None
        return 1


@pytest.fixture
def pool(monkeypatch):
    fake = FakePool()
    monkeypatch.setattr(mem_pool.B200MemAllocator, "get_instance", staticmethod(lambda: fake))
    monkeypatch.setattr(mem_pool.B200MemAllocator, "instance", fake)
    return fake


def _llm(**kw):
    cfg = ModelConfig(hidden_size=64, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=16, intermediate_size=96, vocab_size=97,
                      rope_theta=10000.0, max_position_embeddings=512, dtype=torch.float32)
    args = dict(model=cfg, device="cpu", max_num_seqs=8, max_num_batched_tokens=64, max_model_len=128, num_gpu_blocks=64,
                block_size=4, seed=3)
    args.update(kw)
    return LLM(**args)


def test_the_addresses_of_page_copies_lie_outside_the_pool_that_is_discarded(pool, monkeypatch):
    """A table of raw pointers in discarded memory would be read as pointers after the wake-up."""
    worker = _llm().engine.worker
    made = []

    class Recording(ops.CacheBlocks):
        def __init__(self, tensors):
            made.append(("addresses", pool.tag))
            super().__init__(tensors)

    def init(num_blocks, inner=worker.model_runner._init_kv_cache_tensors):
        made.append(("cache", pool.tag))
        inner(num_blocks)
    monkeypatch.setattr(ops, "CacheBlocks", Recording)
    monkeypatch.setattr(worker.model_runner, "_init_kv_cache_tensors", init)
    monkeypatch.setattr(worker, "device", torch.device("cuda"))
    worker.config.enable_sleep_mode = True
    worker.initialize_from_config(16)
    assert made == [("cache", "kv_cache"), ("addresses", None)]
    assert worker.model_runner.page_cache.num_blocks == 16


def adapter(rank=4):
    g = torch.Generator().manual_seed(rank)
    tensors = {}
    for layer in range(2):
        name = f"base_model.model.model.layers.{layer}.self_attn.q_proj.lora_"
        tensors[name + "A.weight"] = torch.randn(rank, 64, generator=g)
        tensors[name + "B.weight"] = torch.randn(64, rank, generator=g)
    return {"r": rank, "lora_alpha": 2 * rank}, tensors


def test_adapters_outlive_the_first_level_and_not_the_second(pool):
    llm = _llm(enable_lora=True, max_loras=2)
    m = llm.engine.adapters()
    config, tensors = adapter()
    m.load_tensors("a", config, tensors.items())
    sp = SamplingParams(max_tokens=5, ignore_eos=True)
    want = llm.generate([[5, 6, 7]], sp, adapter="a")[0].output_token_ids
    llm.sleep(1)
    llm.wake_up()
    assert llm.generate([[5, 6, 7]], sp, adapter="a")[0].output_token_ids == want
    llm.sleep(2)
    for s in m.stacks.values():                                 # what the device may hold after the wake-up
        s.a.fill_(7), s.b.fill_(7), s.ranks.fill_(1 << 20)
    llm.wake_up()
    assert not m.slots and not m.keys
    with pytest.raises(ValueError):
        llm.generate([[5, 6, 7]], sp, adapter="a")
    assert m.load_tensors("a", config, tensors.items()) == 0
    # also where the adapter has no factors
    assert all(not s.ranks[1].any() and (s.ranks[0, :-1] <= 16).all() for s in m.stacks.values())
    assert llm.generate([[5, 6, 7]], sp, adapter="a")[0].output_token_ids == want


def test_adapters_are_not_written_while_their_memory_is_away(pool, tmp_path):
    from safetensors.torch import save_file
    config, tensors = adapter()
    (tmp_path / "adapter_config.json").write_text(json.dumps(config))
    save_file(tensors, str(tmp_path / "adapter_model.safetensors"))
    llm = _llm(enable_lora=True, max_loras=2, enable_sleep_mode=True)
    llm.load_adapter("a", str(tmp_path))
    llm.sleep(1)
    for _ in range(2):
        with pytest.raises(ValueError, match="awake"):
            llm.load_adapter("b", str(tmp_path))
        with pytest.raises(ValueError, match="awake"):
            llm.unload_adapter("a")
        llm.wake_up(["kv_cache"])                               # the factors are still away
    assert list(llm.engine.adapters().slots) == ["a"]
    llm.wake_up()
    assert llm.load_adapter("b", str(tmp_path)) == 1
    llm.unload_adapter("a")
    # an engine whose memory never lies in the pool
    other = _llm(enable_lora=True, max_loras=1)
    llm.sleep(1)
    assert other.load_adapter("a", str(tmp_path)) == 0


def test_the_server_sleeps_when_no_adapter_is_being_loaded(pool):
    pytest.importorskip("fastapi")
    from starlette.testclient import TestClient
    from omni_npu_b200.serving.api_server import build_app
    llm = _llm(enable_lora=True, max_loras=1, enable_sleep_mode=True)
    app = build_app(llm, model_name="base")
    lock, held = app.state.engine_loop.lock, []
    for name in ("sleep", "wake_up"):
        def call(*a, inner=getattr(llm, name)):
            held.append(lock.locked())
            return inner(*a)
        setattr(llm, name, call)
    with TestClient(app) as client:
        assert client.post("/sleep").status_code == 200
        assert client.post("/v1/load_lora_adapter", json={"lora_name": "a", "lora_path": "/nowhere"}).status_code == 400
        assert client.post("/wake_up").status_code == 200
    app.state.engine_loop.shutdown()
    assert held == [True, True]


def test_cached_prefixes_are_forgotten_with_the_cache(pool):
    p = list(range(5, 25))
    sp = SamplingParams(max_tokens=5, ignore_eos=True)
    want = _llm().generate([p], sp)[0].output_token_ids
    llm = _llm(enable_prefix_caching=True)
    assert llm.generate([p], sp)[0].output_token_ids == want
    for t in llm.engine.worker.model_runner.page_cache.tensors:
        t.fill_(7.0)                                            # what the device may hold after the wake-up
    llm.sleep(1)
    llm.wake_up()
    stats = llm.engine.scheduler.prefix_stats
    assert llm.generate([p], sp)[0].output_token_ids == want and stats["hit_tokens"] == 0
    assert llm.generate([p], sp)[0].output_token_ids == want and stats["hit_tokens"] == 16
    assert llm.engine.scheduler.pool.num_free == 64
