"""Low-rank adapters through the engine: requests with and without them in one batch, against models whose weights hold the
adapter."""
import json

import pytest
import torch

from omni_npu_b200 import SamplingParams
from omni_npu_b200.config import ModelConfig
from omni_npu_b200.engine.llm import LLM

H, HEADS, KV, D, I, V = 64, 4, 2, 16, 96, 97


def _cfg(**kw):
    return ModelConfig(hidden_size=H, num_layers=2, num_heads=HEADS, num_kv_heads=KV, head_dim=D, intermediate_size=I,
                       vocab_size=V, rope_theta=10000.0, max_position_embeddings=512, dtype=torch.float32, **kw)


def _llm(**kw):
    args = dict(model=_cfg(), device="cpu", max_num_seqs=8, max_num_batched_tokens=64, max_model_len=128, num_gpu_blocks=64,
                block_size=4, seed=3)
    args.update(kw)
    return LLM(**args)


SHAPES = {"q_proj": (HEADS * D, H), "k_proj": (KV * D, H), "v_proj": (KV * D, H), "o_proj": (H, HEADS * D),
          "gate_proj": (I, H), "up_proj": (I, H), "down_proj": (H, I)}


def adapter(seed, rank, targets=tuple(SHAPES), layers=2, alpha=None, gain=0.3):
    g = torch.Generator().manual_seed(seed)
    tensors = {}
    for layer in range(layers):
        for t in targets:
            out, inp = SHAPES[t]
            name = f"base_model.model.model.layers.{layer}.{'mlp' if t in ('gate_proj', 'up_proj', 'down_proj') else 'self_attn'}.{t}"
            tensors[name + ".lora_A.weight"] = torch.randn(rank, inp, generator=g) * gain
            tensors[name + ".lora_B.weight"] = torch.randn(out, rank, generator=g) * gain
    return {"peft_type": "LORA", "r": rank, "lora_alpha": alpha or 2 * rank, "bias": "none", "target_modules": list(targets)}, tensors


def save(path, config, tensors):
    from safetensors.torch import save_file
    path.mkdir()
    (path / "adapter_config.json").write_text(json.dumps(config))
    save_file(tensors, str(path / "adapter_model.safetensors"))
    return str(path)


def merge(llm, config, tensors):
    """Add the adapter to the weights."""
    scale = config["lora_alpha"] / (config["r"] ** 0.5 if config.get("use_rslora") else config["r"])
    model = llm.engine.worker.get_model()
    for name, a in tensors.items():
        if ".lora_A." not in name:
            continue
        delta = scale * tensors[name.replace("lora_A", "lora_B")].double() @ a.double()
        parts = name.removeprefix("base_model.model.").split(".")
        layer = model.model.layers[int(parts[2])]
        proj = parts[4]
        if proj in ("q_proj", "k_proj", "v_proj"):
            mod, at = layer.self_attn.qkv_proj, {"q_proj": 0, "k_proj": HEADS * D, "v_proj": (HEADS + KV) * D}[proj]
            mod.weight.data[at: at + delta.shape[0]] += delta.float()
        elif proj in ("gate_proj", "up_proj"):
            mod = layer.mlp.gate_up_proj
            mod.weight.data[mod._rows_of(int(proj == "up_proj"))] += delta.float()
        else:
            mod = layer.self_attn.o_proj if proj == "o_proj" else layer.mlp.down_proj
            mod.weight.data += delta.float()


def prompts(n, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(1, V, (3 + 5 * i % 17,), generator=g).tolist() for i in range(n)]


SP = SamplingParams(max_tokens=7, ignore_eos=True)


def test_a_mixed_batch_answers_like_the_merged_models(tmp_path):
    specs = {"a": adapter(1, 4), "b": adapter(2, 16, targets=("q_proj", "v_proj", "down_proj")),
             "c": dict(zip((0, 1), adapter(5, 3, targets=("gate_proj", "o_proj"))))}
    specs["c"] = ({**specs["c"][0], "use_rslora": True}, specs["c"][1])
    ps = prompts(8)
    names = ["a", None, "b", "a", "c", "b", None, "c"]
    llm = _llm(enable_lora=True, max_loras=3)
    for name, (config, tensors) in specs.items():
        llm.load_adapter(name, save(tmp_path / name, config, tensors))
    got = [o.output_token_ids for o in llm.generate(ps, SP, adapter=names)]
    want = {}
    for name in (None, *specs):
        other = _llm()
        if name:
            merge(other, *specs[name])
        want[name] = [o.output_token_ids for o in other.generate(ps, SP)]
    assert got == [want[name][i] for i, name in enumerate(names)]
    assert want["a"] != want[None] and want["b"] != want[None] and want["c"] != want[None]
    # the same requests one after another, and none of them with an adapter
    for i in (0, 2, 4):
        assert llm.generate([ps[i]], SP, adapter=names[i])[0].output_token_ids == got[i]
    assert [o.output_token_ids for o in llm.generate(ps, SP)] == want[None]


def test_chunked_prompts_preemption_and_mixed_steps_keep_the_adapters():
    config, tensors = adapter(1, 4)
    ps = prompts(6, seed=4)
    names = ["a", None, "a", "a", None, "a"]
    want = None
    for kw in (dict(), dict(max_num_batched_tokens=9), dict(num_gpu_blocks=12), dict(enable_mixed_batches=True),
               dict(additional_config={"async_scheduling": False}),
               dict(speculative_config={"method": "ngram", "num_speculative_tokens": 2})):
        llm = _llm(enable_lora=True, max_loras=2, **kw)
        llm.engine.adapters().load_tensors("a", config, tensors.items())
        got = [o.output_token_ids for o in llm.generate(ps, SP, adapter=names)]
        want = want or got
        assert got == want, kw


def test_cached_prefixes_belong_to_an_adapter():
    (ca, ta), (cb, tb) = adapter(1, 4), adapter(2, 4)
    p = prompts(1, seed=7)[0] * 6
    plain = _llm(enable_lora=True, max_loras=2)
    cached = _llm(enable_lora=True, max_loras=2, enable_prefix_caching=True)
    for llm in (plain, cached):
        llm.engine.adapters().load_tensors("a", ca, ta.items())
        llm.engine.adapters().load_tensors("b", cb, tb.items())
    for name in ("a", "b", None, "a", "b"):
        assert cached.generate([p], SP, adapter=name)[0].output_token_ids == plain.generate([p], SP, adapter=name)[0].output_token_ids
    hits = cached.engine.scheduler.prefix_stats["hit_tokens"]
    assert hits == 2 * ((len(p) - 1) // 4 * 4)                # the second "a" and the second "b"
    # another adapter under a name used before does not find the earlier one's blocks
    for llm in (plain, cached):
        llm.unload_adapter("a")
        llm.engine.adapters().load_tensors("a", cb, tb.items())
    assert cached.generate([p], SP, adapter="a")[0].output_token_ids == plain.generate([p], SP, adapter="a")[0].output_token_ids
    assert cached.engine.scheduler.prefix_stats["hit_tokens"] == hits


def test_slots_are_given_out_and_taken_back():
    llm = _llm(enable_lora=True, max_loras=2)
    m = llm.engine.adapters()
    c, t = adapter(1, 4)
    assert (m.load_tensors("a", c, t.items()), m.load_tensors("b", c, t.items())) == (0, 1)
    with pytest.raises(ValueError):
        m.load_tensors("c", c, t.items())
    with pytest.raises(ValueError):
        m.load_tensors("a", c, t.items())
    rid = llm.engine.add_request([1, 2, 3], SP, adapter="a")
    with pytest.raises(ValueError):
        llm.unload_adapter("a")
    while llm.engine.has_unfinished_requests():
        llm.engine.step()
    assert rid not in llm.engine.scheduler.requests
    llm.unload_adapter("a")
    assert m.load_tensors("c", c, t.items()) == 0
    # what an earlier adapter of the slot left elsewhere is gone
    llm.unload_adapter("c")
    only_q = adapter(9, 2, targets=("q_proj",), layers=1)
    m.load_tensors("q", only_q[0], only_q[1].items())
    other = _llm()
    merge(other, *only_q)
    p = prompts(1, seed=2)
    assert llm.generate(p, SP, adapter="q")[0].output_token_ids == other.generate(p, SP)[0].output_token_ids


def test_refusals(tmp_path):
    off = _llm()
    with pytest.raises(ValueError):
        off.load_adapter("a", str(tmp_path))
    with pytest.raises(ValueError):
        off.generate([[1]], SP, adapter="a")
    llm = _llm(enable_lora=True, max_loras=2, max_lora_rank=8)
    m = llm.engine.adapters()
    c, t = adapter(1, 4)
    with pytest.raises(ValueError):
        llm.generate([[1], [2]], SP, adapter=["a", None])
    with pytest.raises(ValueError):
        llm.generate([[1], [2]], SP, adapter=[None])
    name = next(iter(t))
    for config, tensors in (({**c, "use_dora": True}, t), ({**c, "bias": "all"}, t), ({**c, "modules_to_save": ["lm_head"]}, t),
                            ({**c, "rank_pattern": {"q_proj": 2}}, t), ({**c, "r": 0}, t), (adapter(1, 9)[0], adapter(1, 9)[1]),
                            (c, {}), (c, {"base_model.model.lm_head.lora_A.weight": torch.zeros(4, H)}),
                            (c, {k: v for k, v in t.items() if k != name}), (c, {**t, name: torch.zeros(4, H + 8)}),
                            (c, {**t, "base_model.model.model.norm.weight": torch.zeros(H)})):
        with pytest.raises(ValueError):
            m.load_tensors("x", config, tensors.items())
    assert not m.slots and all(not r.any() for r in (s.ranks[:, :-1] for s in m.stacks.values()))
    with pytest.raises(ValueError):
        llm.unload_adapter("x")
    for kw in (dict(tensor_parallel_size=2), dict(pipeline_parallel_size=2), dict(kv_transfer_config={"kv_connector": "P2PKVConnector"}),
               dict(speculative_config={"method": "mtp", "num_speculative_tokens": 1})):
        with pytest.raises(ValueError):
            _llm(enable_lora=True, **kw)
    mc = ModelConfig(architecture="DeepseekV2ForCausalLM", model_type="deepseek_v2", hidden_size=64, num_layers=1, num_heads=2,
                     num_kv_heads=2, head_dim=16, intermediate_size=64, vocab_size=64, dtype=torch.float32, use_mla=True,
                     kv_lora_rank=512, qk_nope_head_dim=16, qk_rope_head_dim=64, v_head_dim=16)
    with pytest.raises(ValueError):
        LLM(model=mc, device="cpu", enable_lora=True, num_gpu_blocks=16)


def test_the_server_takes_an_adapter_as_model(tmp_path):
    pytest.importorskip("fastapi")
    from starlette.testclient import TestClient
    from omni_npu_b200.serving.api_server import build_app
    llm = _llm(enable_lora=True, max_loras=1)
    path = save(tmp_path / "a", *adapter(1, 4))
    app = build_app(llm, model_name="base")
    with TestClient(app) as client:
        body = {"prompt": [5, 6, 7, 8], "max_tokens": 6, "ignore_eos": True}
        base = client.post("/v1/completions", json=body).json()["choices"][0]["token_ids"]
        assert client.post("/v1/load_lora_adapter", json={"lora_name": "a", "lora_path": path}).status_code == 200
        assert client.post("/v1/load_lora_adapter", json={"lora_name": "b", "lora_path": path}).status_code == 400
        assert client.post("/v1/load_lora_adapter", json={"lora_name": "c", "lora_path": str(tmp_path / "none")}).status_code == 400
        assert [m["id"] for m in client.get("/v1/models").json()["data"]] == ["base", "a"]
        with_a = client.post("/v1/completions", json={**body, "model": "a"}).json()["choices"][0]["token_ids"]
        assert with_a != base
        assert client.post("/v1/completions", json={**body, "model": "a"}).json()["model"] == "a"
        assert client.post("/v1/completions", json={**body, "model": "base"}).json()["choices"][0]["token_ids"] == base
        three = client.post("/v1/completions", json={**body, "model": "a", "n": 3}).json()["choices"]
        assert [c["token_ids"] for c in three] == [with_a] * 3
        assert llm.engine.scheduler.fork_stats["requests"] == 2
        assert client.post("/v1/unload_lora_adapter", json={"lora_name": "a"}).status_code == 200
        assert client.post("/v1/unload_lora_adapter", json={"lora_name": "a"}).status_code == 400
    app.state.engine_loop.shutdown()
