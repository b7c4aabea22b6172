"""The engine after its memory was given back and mapped again."""
import pytest
import torch

from omni_npu_b200 import SamplingParams
from omni_npu_b200.config import ModelConfig
from omni_npu_b200.engine.llm import LLM

pytestmark = pytest.mark.gpu
H, HEADS, KV, D, I, V = 512, 4, 2, 128, 1408, 2048


def _llm(**kw):
    cfg = ModelConfig(hidden_size=H, num_layers=2, num_heads=HEADS, num_kv_heads=KV, head_dim=D, intermediate_size=I, vocab_size=V,
                      max_position_embeddings=2048)
    args = dict(model=cfg, device="cuda", max_num_seqs=8, max_num_batched_tokens=256, max_model_len=512, num_gpu_blocks=256, seed=3,
                enable_sleep_mode=True)
    args.update(kw)
    return LLM(**args)


def prompt(n):
    return torch.randint(1, V, (n,), generator=torch.Generator().manual_seed(n)).tolist()


def test_samples_of_one_prompt_after_a_wake_up():
    llm = _llm()
    from omni_npu_b200.worker.mem_pool import B200MemAllocator
    sp = SamplingParams(max_tokens=8, temperature=1.0, seed=7, ignore_eos=True, n=3)

    def samples():
        before = llm.engine.scheduler.fork_stats["shared_tokens"]
        o = llm.generate([prompt(45)], sp)[0]
        assert llm.engine.scheduler.fork_stats["shared_tokens"] == before + 2 * 44      # two whole blocks and 12 rows of a copy
        return [o.output_token_ids, *[x.output_token_ids for x in o.others]]
    want = samples()
    table = llm.engine.worker.model_runner.page_cache._desc
    kept = table.cpu()
    assert llm.sleep(1) > 0
    assert torch.equal(table.cpu(), kept)                    # readable while the pool is away
    llm.wake_up()
    assert B200MemAllocator.get_instance().stats()["sleeping_bytes"] == 0
    assert samples() == want


def adapter(rank, seed):
    g = torch.Generator().manual_seed(seed)
    shapes = {"self_attn.q_proj": (HEADS * D, H), "mlp.up_proj": (I, H), "mlp.down_proj": (H, I)}
    tensors = {}
    for layer in range(2):
        for part, (out, inp) in shapes.items():
            name = f"base_model.model.model.layers.{layer}.{part}.lora_"
            tensors[name + "A.weight"] = torch.randn(rank, inp, generator=g) / inp ** 0.5
            tensors[name + "B.weight"] = torch.randn(out, rank, generator=g) / 8
    return {"r": rank, "lora_alpha": 2 * rank}, tensors


def test_adapters_after_a_wake_up():
    llm = _llm(enable_lora=True, max_loras=3, max_lora_rank=32)
    m = llm.engine.adapters()
    for i, name in enumerate("ab"):
        config, tensors = adapter(16 - 7 * i, i)
        m.load_tensors(name, config, tensors.items())
    ps, names = [prompt(n) for n in (5, 40, 17, 100)], ["a", None, "b", "a"]
    sp = SamplingParams(max_tokens=8, ignore_eos=True)
    want = [o.output_token_ids for o in llm.generate(ps, sp, adapter=names)]
    llm.sleep(1)
    with pytest.raises(ValueError, match="awake"):
        llm.load_adapter("c", "/nowhere")
    llm.wake_up()
    assert [o.output_token_ids for o in llm.generate(ps, sp, adapter=names)] == want
    # the second level discards the weights as well: what is checked is that no slot holds what was there
    llm.sleep(2)
    assert not m.slots
    llm.wake_up()
    config, tensors = adapter(9, 5)
    assert m.load_tensors("c", config, tensors.items()) == 0
    for name, stack in m.stacks.items():
        ranks = stack.ranks.cpu()
        assert not ranks[1:].any() and set(ranks[0, :-1].tolist()) <= {0, 9}, name
        assert bool(ranks[0].any()) == any(p in name for p in ("qkv_proj", "gate_up_proj", "down_proj"))
