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
