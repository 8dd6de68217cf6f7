"""What serving makes of the operators in few bits, on the CPU: errors that their kernels record."""
import pytest
import torch

from connex_b200 import ops
from connex_b200.models.llama import LlamaConfig


def _stage(monkeypatch, layers=(0, 2)):
    """A stage on the CPU whose steps run no kernels."""
    from connex_b200.runtime.pp import StageRuntime
    monkeypatch.setattr(ops, "decode_workspace_int4", lambda *a: torch.zeros(1))      # sized by the GPU's SMs
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t: t)
    rt = StageRuntime(LlamaConfig.tiny(layers=2), *layers, "cpu", num_blocks=16, max_tokens=64, max_batch=4, max_ctx=64,
                      kv_dtype=torch.uint8)
    rt.ran = 0

    def run(inp, *a, **kw):
        rt.ran += 1
        return torch.arange(kw["B"]) if rt.model.is_last else torch.zeros(inp.shape[0], rt.cfg.hidden)
    monkeypatch.setattr(rt.model, "run", run)
    monkeypatch.setattr(ops, "prefill_tile_info", lambda *a, **kw: None)
    return rt


def test_steps_fail_with_what_their_kernels_record(monkeypatch):
    """A stepper raises in the step that went wrong, and serves the next one."""
    from connex_b200.serve.engine import ModelStepper
    rt = _stage(monkeypatch)
    st = object.__new__(ModelStepper)
    st.rt = rt
    assert st.prefill(["a"], [[5, 6, 7]]) == [0]
    run = rt.model.run

    def late(*a, **kw):
        rt.model.status.fill_(1)
        return run(*a, **kw)
    monkeypatch.setattr(rt.model, "run", late)
    for step in (lambda: st.decode(["a"], [[5, 6, 7, 8]]), lambda: st.mixed(["b"], [[5, 6, 7]], [0], [3])):
        with pytest.raises(RuntimeError, match="timeout"):
            step()
    monkeypatch.setattr(rt.model, "run", run)
    assert st.decode(["a"], [[5, 6, 7, 8]]) == [0] and int(rt.model.status) == 0


def test_a_stage_stops_after_a_step_that_went_wrong(monkeypatch):
    """A stage whose rows only go on to the next one raises before its next step, and not for a warm-up."""
    from connex.pp.handover import CX_CTX, REQUEST_IDS
    rt = _stage(monkeypatch, (0, 1))
    td = {"kind": "decode", REQUEST_IDS: ["a"], CX_CTX: [0], "n_new": [1], "ids": torch.tensor([4], dtype=torch.int32)}
    rt.compute(td, [])
    rt.model.status.fill_(2)
    rt.compute({**td, CX_CTX: [1]}, [])
    assert rt.compute({"kind": "warmup", "w": torch.ones(1)}, [])["w"] == 1
    with pytest.raises(RuntimeError, match="bounds"):
        rt.compute({**td, CX_CTX: [2]}, [])
    assert rt.ran == 2 and rt.kv_held("a") == 2
    rt.compute({**td, CX_CTX: [2]}, [])
    assert rt.ran == 3
