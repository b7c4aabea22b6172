"""Adapters and shared prompts through the engine on a GPU."""
import pytest
import torch

from omni_npu_b200 import SamplingParams, ops
from omni_npu_b200.attention.metadata import AttentionMetadata, set_forward_context
from omni_npu_b200.config import ModelConfig
from omni_npu_b200.engine.llm import LLM
from lora_cases import check_silu, check_sum, exact

pytestmark = pytest.mark.gpu
H, HEADS, KV, D, I, V = 512, 4, 2, 128, 1408, 2048


def _llm(**kw):
    cfg = ModelConfig(hidden_size=H, num_layers=2, num_heads=HEADS, num_kv_heads=KV, head_dim=D, intermediate_size=I, vocab_size=V,
                      max_position_embeddings=2048)
    args = dict(model=cfg, device="cuda", max_num_seqs=16, max_num_batched_tokens=1024, max_model_len=512, num_gpu_blocks=512, seed=3)
    args.update(kw)
    return LLM(**args)


SHAPES = {"self_attn.q_proj": (HEADS * D, H), "self_attn.k_proj": (KV * D, H), "self_attn.v_proj": (KV * D, H),
          "self_attn.o_proj": (H, HEADS * D), "mlp.gate_proj": (I, H), "mlp.up_proj": (I, H), "mlp.down_proj": (H, I)}


def adapter(seed, rank, targets=tuple(SHAPES)):
    g = torch.Generator().manual_seed(seed)
    tensors = {}
    for layer in range(2):
        for t in targets:
            out, inp = SHAPES[t]
            tensors[f"base_model.model.model.layers.{layer}.{t}.lora_A.weight"] = torch.randn(rank, inp, generator=g) / inp ** 0.5
            tensors[f"base_model.model.model.layers.{layer}.{t}.lora_B.weight"] = torch.randn(out, rank, generator=g) / 8
    return {"peft_type": "LORA", "r": rank, "lora_alpha": 2 * rank}, tensors


def _load(llm, names=("a", "b", "c")):
    specs = {"a": adapter(1, 16), "b": adapter(2, 5, ("self_attn.q_proj", "mlp.up_proj")), "c": adapter(3, 32)}
    for n in names:
        llm.engine.adapters().load_tensors(n, specs[n][0], specs[n][1].items())
    return specs


def prompts(n, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(1, V, (5 + 37 * i % 200,), generator=g).tolist() for i in range(n)]


@pytest.mark.parametrize("tokens", [1, 13, 300])
def test_projections_match_64_bits(tokens):
    llm = _llm(enable_lora=True, max_loras=3, max_lora_rank=32)
    specs = _load(llm)
    model = llm.engine.worker.get_model()
    slots = (torch.arange(tokens, device="cuda") % 4 - 1).int()
    md = AttentionMetadata(True, 1, tokens, tokens, tokens, 0, slots, slots, slots.view(1, -1), slots, slots)
    md.extra["lora"] = llm.engine.adapters().plan(slots)

    def factors(layer, parts):
        out = []
        for n in ("a", "b", "c"):
            t = specs[n][1]
            get = [[t.get(f"base_model.model.model.layers.{layer}.{p}.lora_{w}.weight") for p in parts] for w in "AB"]
            out.append((*([None if x is None else x.bfloat16().cuda() for x in f] for f in get), 2.0))
        return out
    layer = model.model.layers[1]
    with torch.inference_mode(), set_forward_context(md, [], llm.config):
        x = torch.randn(tokens, H, device="cuda").bfloat16()
        for mod, parts in ((layer.self_attn.qkv_proj, ["self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj"]),
                           (layer.self_attn.o_proj, ["self_attn.o_proj"])):
            base = ops.gemm(x, mod.weight)
            z, bound = exact(x, base, factors(1, parts), slots, [SHAPES[p][0] for p in parts])
            got = mod(x)
            check_sum(torch.cat(got, dim=1) if isinstance(got, tuple) else got, z, bound)
        mod = layer.mlp.gate_up_proj
        z, bound = exact(x, ops.gemm(x, mod.weight), factors(1, ["mlp.gate_proj", "mlp.up_proj"]), slots, [I, I], interleaved=True)
        h = mod(x, fuse_swiglu=True)
        check_silu(h, z, bound)
        mod = layer.mlp.down_proj
        z, bound = exact(h, ops.gemm(h, mod.weight), factors(1, ["mlp.down_proj"]), slots, [H])
        check_sum(mod(h), z, bound)


def test_engine_with_graphs_without_and_with_asynchronous_steps():
    ps = prompts(12)
    names = ["a", None, "b", "c", "a", None, "c", "b", "a", "a", None, "c"]
    sp = SamplingParams(max_tokens=12, ignore_eos=True)
    got = []
    for kw in (dict(), dict(enforce_eager=True), dict(additional_config={"async_scheduling": False})):
        llm = _llm(enable_lora=True, max_loras=3, max_lora_rank=32, **kw)
        _load(llm)
        got.append([o.output_token_ids for o in llm.generate(ps, sp, adapter=names)])
        plain = [o.output_token_ids for o in llm.generate(ps, sp)]
        del llm
    assert got[0] == got[1] == got[2]
    # steps without an adapter run the kernels of an engine without them
    assert plain == [o.output_token_ids for o in _llm().generate(ps, sp)]
    assert sum(g != p for g, p, n in zip(got[0], plain, names) if n) >= 8


@pytest.mark.parametrize("tokens", [1, 16, 17, 200])
def test_samples_share_and_copy_the_prompts_pages(tokens):
    llm = _llm(enable_lora=True, max_loras=3, max_lora_rank=32)
    _load(llm)
    eng, p = llm.engine, prompts(1, seed=tokens)[0] * 40
    p = p[:tokens]
    sp = SamplingParams(max_tokens=20, ignore_eos=True)
    first = eng.add_request(p, sp, adapter="a")
    rids = [eng.add_request(p, sp, adapter="a", fork_of=first) for _ in range(3)]
    reqs = [eng.scheduler.requests[r] for r in (first, *rids)]
    done = {}
    while any(len(r.output_token_ids) < 3 for r in reqs):
        for o in eng.step():
            done[o.request_id] = o
    torch.cuda.synchronize()
    full, rows = divmod(tokens - 1, 16)
    for r in reqs[1:]:
        assert r.block_ids[:full] == reqs[0].block_ids[:full] and r.block_ids[full] != reqs[0].block_ids[full]
        for cache in eng.worker.model_runner.kv_caches:
            for t in cache:
                assert torch.equal(t[r.block_ids[full]][:, :rows], t[reqs[0].block_ids[full]][:, :rows])
    while eng.has_unfinished_requests():
        for o in eng.step():
            done[o.request_id] = o
    outs = [done[r].output_token_ids for r in (first, *rids)]
    assert all(len(o) == 20 for o in outs) and outs[1] == outs[2] == outs[3]
    assert eng.scheduler.pool.num_free == 512 and eng.scheduler.fork_stats["requests"] == 3


def test_many_samples_of_several_prompts_with_adapters():
    llm = _llm(enable_lora=True, max_loras=3, max_lora_rank=32, enable_prefix_caching=True)
    _load(llm)
    ps = prompts(4, seed=9)
    sp = [SamplingParams(max_tokens=9, temperature=0.8, seed=i, n=1 + 2 * i, ignore_eos=True) for i in range(4)]
    a = llm.generate(ps, sp, adapter=["a", None, "b", "c"])
    b = llm.generate(ps, sp, adapter=["a", None, "b", "c"])
    for x, y, s in zip(a, b, sp):
        assert len(x.others) == s.n - 1 and all(len(o.output_token_ids) == 9 for o in (x, *x.others))
        assert len({tuple(o.output_token_ids) for o in (x, *x.others)}) > s.n // 2
        assert len(y.others) == s.n - 1
    assert llm.engine.scheduler.fork_stats["requests"] == 2 * (2 + 4 + 6)
