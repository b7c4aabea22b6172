"""Logits kept beside captured decode steps: each step's are those of the graph that ran it."""
import pytest
import torch

from omni_npu_b200 import SamplingParams
from omni_npu_b200.config import ModelConfig
from omni_npu_b200.engine.llm import LLM
from omni_npu_b200.worker import model_runner as module


def _llm(**kw):
    cfg = ModelConfig(hidden_size=64, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=16, intermediate_size=96, vocab_size=97,
                      rope_theta=10000.0, max_position_embeddings=512, dtype=torch.float32)
    return LLM(model=cfg, device="cpu", max_num_seqs=4, max_num_batched_tokens=64, max_model_len=128, num_gpu_blocks=64,
               block_size=4, seed=3, **kw)


class HostGraph:
    """A captured step on the host: replays write into the tensors that the capture left."""
    owner = None
    pool = None

    def __init__(self, fn, device, pool=None):
        self.fn = fn

    def _run(self):
        model, kept = self.owner.model, []
        inner = model.compute_logits
        model.compute_logits = lambda h: kept.append(inner(h)) or kept[-1]
        try:
            return self.fn(), kept[-1]
        finally:
            del model.compute_logits

    def capture(self, warmup=1):
        self.output, self.logits = self._run()

    def replay(self):
        # (no Python of the step runs at a replay)
        rows, self.owner._want_rows, self.owner.keep_logits = self.owner._want_rows, [], False
        with torch.inference_mode():
            out, logits = self._run()
            self.logits.copy_(logits)
        self.owner._want_rows = rows
        return out


@pytest.mark.parametrize("name", [None, "a"])
def test_logits_of_a_captured_step(monkeypatch, name):
    g = torch.Generator().manual_seed(1)
    tensors = {f"model.layers.{i}.self_attn.q_proj.lora_{w}.weight": torch.randn(*s, generator=g)
               for i in range(2) for w, s in (("A", (4, 64)), ("B", (64, 4)))}

    def decode_logits(captured):
        llm = _llm(enable_lora=True, max_loras=1)
        runner = llm.engine.worker.model_runner
        llm.engine.adapters().load_tensors("a", {"r": 4}, tensors.items())
        if captured:
            monkeypatch.setattr(HostGraph, "owner", runner)
            monkeypatch.setattr(module, "CUDAGraphRunner", HostGraph)
            monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
            runner.keep_logits = True
            host, runner.device = runner.device, torch.device("cuda")
            runner.capture_model()
            runner.device = host
            assert runner.graphs and runner.lora_graphs
        llm.engine.add_request([5, 6, 7, 8], SamplingParams(max_tokens=4, ignore_eos=True), adapter=name)
        sched = llm.engine.scheduler
        out = sched.schedule()
        sched.update_from_output(out, runner.execute_model(out))
        out = sched.schedule()
        assert out.kind == "decode"
        return runner.execute_with_logits(out, [0])
    want = decode_logits(False)
    assert torch.equal(decode_logits(True), want)
