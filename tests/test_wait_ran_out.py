"""CPU: the trainer's reaction to a kernel whose wait ran out, with the device's flags stubbed."""
from types import SimpleNamespace

import pytest
import torch


@pytest.fixture
def flags(monkeypatch):
    """The two flags as a device would hold them: read and cleared."""
    from stew_b200 import _lib
    values = {"gemm": 0, "attn": 0}

    def reader(name):
        def read(reset=True):
            v = values[name]
            if reset:
                values[name] = 0
            return v
        return read

    monkeypatch.setattr(_lib, "gemm_error_flag", reader("gemm"))
    monkeypatch.setattr(_lib, "attn_error_flag", reader("attn"))
    return values


@pytest.mark.parametrize("name,value", [("attn", 27), ("gemm", 4)])
def test_flag_raises_once(flags, name, value):
    from stew_b200 import _lib
    _lib.raise_if_wait_ran_out()
    flags[name] = value
    with pytest.raises(RuntimeError, match=f"flag {value}"):
        _lib.raise_if_wait_ran_out()
    _lib.raise_if_wait_ran_out()


@pytest.mark.parametrize("name", ["attn", "gemm"])
def test_trainer_makes_no_step_on_unfinished_gradients(flags, monkeypatch, name):
    """The gradients of a step in which a wait ran out never reach the optimizer."""
    from stew_b200 import _lib
    from stew_b200.qlora_step import QLoRATrainer

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w = torch.nn.Parameter(torch.ones(3))

        def lora_parameters(self):
            return [self.w]

        def forward_packed(self, pb):
            if pb.fail:
                flags[name] = 9
            return (self.w * 2).sum()

    model = Model()
    trainer = QLoRATrainer(model, lr=0.1)
    # (a CUDA device would be asked; here the stubs answer)
    monkeypatch.setattr(QLoRATrainer, "check", lambda self: _lib.raise_if_wait_ran_out())
    pb = SimpleNamespace(n_labels=2, ids=torch.zeros(2, dtype=torch.long), fail=True)
    with pytest.raises(RuntimeError, match="ran out"):
        trainer._eager(pb)
    assert torch.equal(model.w.detach(), torch.ones(3))
    trainer.opt.zero_grad()
    pb.fail = False
    trainer._eager(pb)
    assert bool((model.w < 1).all())


def test_check_asks_no_device_on_the_cpu(flags):
    from stew_b200.qlora_step import QLoRATrainer
    flags["attn"] = 1
    trainer = QLoRATrainer.__new__(QLoRATrainer)
    trainer.params = [torch.zeros(1)]
    trainer.check()
    assert flags["attn"] == 1
