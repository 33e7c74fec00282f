"""GPU: attention kernels whose waits give up early.  Every row is then either the answer or NaN, none is
left as the memory was; the flag tells; the next call is not affected."""
import pytest
import torch

pytestmark = pytest.mark.gpu

LENS = [300, 1, 0, 517, 64]


def _inputs(dtype, d, pad=7):
    g = torch.Generator(device="cuda").manual_seed(d)
    n = sum(LENS) + pad
    q, k, v, dout = (torch.randn(n, h, d, device="cuda", generator=g).to(dtype) for h in (6, 2, 2, 6))
    cu = torch.tensor([0] + LENS, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)
    return q, k, v, cu, dout


def _fill_free_memory():
    """What torch.empty will find: 0x5555, no NaN of any type."""
    kept = [torch.full((1 << s,), 0x5555, dtype=torch.int16, device="cuda") for s in range(9, 22) for _ in range(6)]
    del kept


@pytest.fixture
def limit(monkeypatch):
    from stew_b200 import _lib
    _lib.attn_error_flag()

    def set_limit(cycles):
        if cycles is None:
            monkeypatch.delenv("STEW_ATTN_WAIT_CYCLES", raising=False)
        else:
            monkeypatch.setenv("STEW_ATTN_WAIT_CYCLES", str(cycles))
    yield set_limit
    set_limit(None)
    torch.cuda.synchronize()
    _lib.attn_error_flag()


def _answer_or_nan(got, want, what):
    both = (got == want) | torch.isnan(got)
    assert bool(both.all()), f"{what}: {int((~both).sum())} values are neither"


@pytest.mark.parametrize("dtype,d", [(torch.float16, 128), (torch.bfloat16, 64)])
def test_forward(cuda_lib, limit, dtype, d):
    from stew_b200 import _lib
    from stew_b200.step_ops import _attn_forward
    q, k, v, cu, _ = _inputs(dtype, d)

    def run():
        out, rest, lse, *_ = _attn_forward(q, k, v, cu, -1, 0, d ** -0.5, True)
        return out, rest, lse

    want = run()
    _fill_free_memory()
    limit(0)
    got = run()
    torch.cuda.synchronize()
    assert _lib.attn_error_flag() != 0
    for name, a, b in zip(("out", "rest", "lse"), got, want):
        _answer_or_nan(a, b, name)
    assert torch.isnan(got[0]).any() and not got[0][-7:].any()
    limit(None)
    del got
    for a, b in zip(run(), want):
        assert torch.equal(a, b)
    assert _lib.attn_error_flag() == 0


@pytest.mark.parametrize("split", ["1", "3"])
@pytest.mark.parametrize("dtype,d", [(torch.float16, 128), (torch.bfloat16, 64)])
@pytest.mark.parametrize("cycles", [0, 200])
def test_backward(cuda_lib, limit, monkeypatch, dtype, d, split, cycles):
    """(With 200 clocks only the sums over shares give up, where their shares take longer.)"""
    from stew_b200 import _lib
    from stew_b200.step_ops import packed_attention
    monkeypatch.setenv("STEW_ATTN_SPLIT", split)
    q, k, v, cu, dout = _inputs(dtype, d)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = packed_attention(*leaves, cu)
    want = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    _fill_free_memory()
    limit(cycles)
    got = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    torch.cuda.synchronize()
    gave_up = _lib.attn_error_flag() != 0
    assert gave_up or cycles > 0
    for name, a, b in zip(("dq", "dk", "dv"), got, want):
        _answer_or_nan(a, b, name)
        assert not a[-7:].any()
    assert gave_up == any(bool(torch.isnan(a).any()) for a in got)
    limit(None)
    del got
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, dout), want))
    assert _lib.attn_error_flag() == 0


def test_trainer_raises(cuda_lib, limit):
    """An eager step whose attention gives up raises and leaves the adapters as they were."""
    from stew_b200.qlora_step import QLoRATrainer, QwenConfig, QwenQLoRA, synthetic_batch
    trainer = QLoRATrainer(QwenQLoRA(QwenConfig(layers=1, vocab=4096), device="cuda", seed=3))
    tokens, lengths = synthetic_batch(batch=3, seq=160, vocab=4096, seed=1)
    before = [p.detach().clone() for p in trainer.params]
    limit(0)
    with pytest.raises(RuntimeError, match="ran out"):
        trainer.step(tokens, lengths)
    assert all(torch.equal(a, b) for a, b in zip(before, trainer.params))
    limit(None)
    trainer.opt.zero_grad(set_to_none=True)
    loss, _, _ = trainer.step(tokens, lengths)
    assert bool(torch.isfinite(loss))
    trainer.check()
