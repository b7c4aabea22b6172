"""Adapters that a server loads while it answers."""
import json

import pytest
import torch

from omni_npu_b200 import SamplingParams
from omni_npu_b200.config import ModelConfig
from omni_npu_b200.engine.llm import LLM
from omni_npu_b200.ops.lora import LoraStack

pytest.importorskip("fastapi")
from starlette.testclient import TestClient  # noqa: E402

from omni_npu_b200.serving.api_server import build_app  # noqa: E402


def _llm(**kw):
    cfg = ModelConfig(hidden_size=64, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=16, intermediate_size=96, vocab_size=97,
                      rope_theta=10000.0, max_position_embeddings=512, dtype=torch.float32)
    args = dict(model=cfg, device="cpu", max_num_seqs=8, max_num_batched_tokens=64, max_model_len=128, num_gpu_blocks=64,
                block_size=4, seed=3, enable_lora=True, max_loras=2)
    args.update(kw)
    return LLM(**args)


def tensors(rank=4):
    g = torch.Generator().manual_seed(rank)
    return {f"base_model.model.model.layers.{i}.self_attn.q_proj.lora_{w}.weight": torch.randn(*s, generator=g)
            for i in range(2) for w, s in (("A", (rank, 64)), ("B", (64, rank)))}


def save(path, config=None, factors=None):
    from safetensors.torch import save_file
    path.mkdir()
    (path / "adapter_config.json").write_text(config if isinstance(config, str) else json.dumps(config or {"r": 4, "lora_alpha": 8}))
    save_file(factors or tensors(), str(path / "adapter_model.safetensors"))
    return str(path)


@pytest.fixture
def server():
    llm = _llm()
    app = build_app(llm, model_name="base")
    with TestClient(app, raise_server_exceptions=False) as client:
        yield llm, app.state.engine_loop, client
    app.state.engine_loop.shutdown()


def test_files_are_read_beside_the_steps(server, tmp_path, monkeypatch):
    llm, loop, client = server
    seen = []
    from omni_npu_b200.models import utils

    def reading(path, inner=utils.iter_safetensors):
        seen.append(("read", loop.lock.locked()))
        return inner(path)

    def load(self, *a, inner=LoraStack.load):
        seen.append(("packed", loop.lock.locked()))
        inner(self, *a)
    monkeypatch.setattr(utils, "iter_safetensors", reading)
    monkeypatch.setattr(LoraStack, "load", load)
    path = save(tmp_path / "a")
    assert client.post("/v1/load_lora_adapter", json={"lora_name": "a", "lora_path": path}).status_code == 200
    assert seen == [("read", False)] + [("packed", True)] * 2
    assert [m["id"] for m in client.get("/v1/models").json()["data"]] == ["base", "a"]
    # a name or a slot that was taken meanwhile
    b, c = (llm.engine.read_adapter(n, path) for n in "bc")
    llm.engine.install_adapter(b)
    with pytest.raises(ValueError):
        llm.engine.install_adapter(b)
    with pytest.raises(ValueError):
        llm.engine.install_adapter(c)
    assert llm.engine.adapters().slots == {"a": 0, "b": 1}


def test_models_are_listed_while_one_is_loaded(server, tmp_path):
    llm, loop, client = server
    path = save(tmp_path / "a")
    adapters = llm.engine.adapters()

    class Slots(dict):
        """Another thread's load, as soon as the first name has been listed."""
        def __iter__(self):
            for i, name in enumerate(super().__iter__()):
                yield name
                if i == 0 and not loop.lock.locked():
                    self["b"] = 1
    adapters.slots = Slots()
    assert client.post("/v1/load_lora_adapter", json={"lora_name": "a", "lora_path": path}).status_code == 200
    got = client.get("/v1/models")
    assert got.status_code == 200 and [m["id"] for m in got.json()["data"]] == ["base", "a"]


@pytest.mark.parametrize("config", ["[1]", "{", json.dumps({"r": None}), json.dumps({"r": 4, "lora_alpha": None}),
                                    json.dumps({"lora_alpha": 4}), json.dumps({"r": [4]}), json.dumps({"r": 4, "lora_alpha": float("nan")})])
def test_a_configuration_that_is_none_is_the_callers_mistake(server, tmp_path, config):
    llm, loop, client = server
    got = client.post("/v1/load_lora_adapter", json={"lora_name": "a", "lora_path": save(tmp_path / "a", config)})
    assert got.status_code == 400 and not llm.engine.adapters().slots


@pytest.mark.parametrize("keep", [0, 4, 100, -10])
def test_a_damaged_file_is_the_callers_mistake(server, tmp_path, keep):
    llm, loop, client = server
    path = save(tmp_path / "a")
    file = tmp_path / "a" / "adapter_model.safetensors"
    file.write_bytes(file.read_bytes()[:keep])
    got = client.post("/v1/load_lora_adapter", json={"lora_name": "a", "lora_path": path})
    assert got.status_code == 400 and not llm.engine.adapters().slots


def test_factors_of_another_rank_than_the_configurations():
    """They would be scaled by a rank that is not theirs."""
    m = _llm().engine.adapters()
    with pytest.raises(ValueError, match="rank should be 8"):
        m.load_tensors("a", {"r": 8, "lora_alpha": 16}, tensors(4).items())
    with pytest.raises(ValueError, match="rank should be 4"):
        m.load_tensors("a", {"r": 4}, {k: v[0] for k, v in tensors(4).items()}.items())
    assert not m.slots and m.load_tensors("a", {"r": 4}, tensors(4).items()) == 0


def test_a_server_without_routes_for_adapters(tmp_path):
    from omni_npu_b200.serving.api_server import make_parser
    llm = _llm()
    path = save(tmp_path / "a")
    llm.load_adapter("a", path)
    app = build_app(llm, model_name="base", adapter_routes=False)
    with TestClient(app) as client:
        assert client.post("/v1/load_lora_adapter", json={"lora_name": "b", "lora_path": path}).status_code == 404
        assert client.post("/v1/unload_lora_adapter", json={"lora_name": "a"}).status_code == 404
        assert [m["id"] for m in client.get("/v1/models").json()["data"]] == ["base", "a"]
        body = {"prompt": [5, 6, 7, 8], "max_tokens": 3, "ignore_eos": True, "model": "a"}
        assert client.post("/v1/completions", json=body).json()["model"] == "a"
    app.state.engine_loop.shutdown()
    args = make_parser().parse_args(["--model", "m"])
    assert not args.no_lora_routes and make_parser().parse_args(["--model", "m", "--no-lora-routes"]).no_lora_routes


def test_the_served_models_name_stays_the_served_models(server, tmp_path):
    llm, loop, client = server
    path = save(tmp_path / "a", factors={k: 3 * v for k, v in tensors().items()})
    body = {"prompt": [5, 6, 7, 8], "max_tokens": 6, "ignore_eos": True, "model": "base"}
    want = client.post("/v1/completions", json=body).json()["choices"][0]["token_ids"]
    assert client.post("/v1/load_lora_adapter", json={"lora_name": "base", "lora_path": path}).status_code == 400
    llm.load_adapter("base", path)                            # (not over HTTP)
    with loop.lock:                                           # (the server's thread steps the engine otherwise)
        other = llm.generate([[5, 6, 7, 8]], SamplingParams(max_tokens=6, ignore_eos=True), adapter="base")[0].output_token_ids
    assert other != want
    assert client.post("/v1/completions", json=body).json()["choices"][0]["token_ids"] == want
