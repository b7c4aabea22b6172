"""Calls that give their arguments by position keep their meaning when fields are added."""
from omni_npu_b200 import SamplingParams
from omni_npu_b200.config import (CacheConfig, CompilationConfig, EngineConfig, ParallelConfig, SchedulerConfig,
                                  SpeculativeConfig, tiny_llama)
from omni_npu_b200.engine.scheduler import SchedulerOutput


def test_sampling_params():
    early = ("max_tokens", "temperature", "top_k", "top_p", "seed", "ignore_eos", "stop_token_ids", "presence_penalty",
             "frequency_penalty", "repetition_penalty", "thinking_token_budget", "logprobs", "prompt_logprobs", "logit_bias",
             "min_tokens", "min_p", "allowed_token_ids", "bad_words_token_ids", "priority", "structured", "extra_args")
    default = SamplingParams()
    sp = SamplingParams(*[getattr(default, k) for k in early[:18]], 5, {"regex": "a"}, {"k": 1})
    assert (sp.priority, sp.structured, sp.extra_args, sp.n) == (5, {"regex": "a"}, {"k": 1}, 1)


def test_engine_config():
    c = EngineConfig(tiny_llama(), CacheConfig(), ParallelConfig(), SchedulerConfig(), CompilationConfig(), None,
                     SpeculativeConfig(), "/weights", "dummy", 7, "cpu")
    assert (c.model_path, c.load_format, c.seed, c.device, c.adapters.max_loras) == ("/weights", "dummy", 7, "cpu", 0)


def test_scheduler_output():
    out = SchedulerOutput("idle", [], 0, 0, [], [], None, 3, [1])
    assert (out.step_index, out.pending_pos, out.block_copies) == (3, [1], [])
