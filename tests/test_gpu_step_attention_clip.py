"""GPU: the QLoRA step with its own attention and with clipping: the attention against torch's
variable-length attention through a layer's forward and backward, and clipped steps (eager and
captured, one buffer and buckets) against unclipped gradients scaled by hand."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(seed=3):
    from stew_b200.qlora_step import QwenConfig, QwenQLoRA
    return QwenQLoRA(QwenConfig(layers=2, vocab=4096), device="cuda", seed=seed)


def _batch(seed=1):
    from stew_b200.qlora_step import synthetic_batch
    return synthetic_batch(batch=3, seq=160, vocab=4096, seed=seed)


def test_other_head_sizes_keep_torch_attention(cuda_lib):
    """Head sizes outside the kernels' go where they went before; inside, both agree to rounding."""
    from torch.nn.attention.varlen import varlen_attn

    from stew_b200.qlora_step import packed_causal_attention
    cu = torch.tensor([0, 70, 190], dtype=torch.int32, device="cuda")
    for d in (128, 256):
        q = torch.randn(190, 4, d, device="cuda").half()
        k, v = (torch.randn(190, 2, d, device="cuda").half() for _ in range(2))
        a = packed_causal_attention(q, k, v, (cu, 120))
        b = varlen_attn(q, k, v, cu, cu, 120, 120, window_size=(-1, 0))
        # each within its own rounding of p and of the output: 2 half steps each, values up to ~4
        assert float((a.float() - b.float()).abs().max()) <= 4 * 2.0 ** -11 * float(b.abs().max())


def _grads(model, tokens, lengths):
    loss, n = model(tokens, lengths)
    loss.backward()
    grads = [p.grad.clone() / n for p in model.lora_parameters()]
    for p in model.lora_parameters():
        p.grad = None
    return grads


def _norm(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("bucketed", [False, True])
def test_clipped_step(cuda_lib, graph, bucketed):
    """One step of plain gradient-descent-like size: the norm that the trainer reports is that of the
    normalised gradients, and AdamW sees them scaled: its first moment after a step is
    (1 - beta1) times the clipped gradient."""
    from stew_b200.qlora_step import QLoRATrainer
    model = _model()
    tokens, lengths = _batch()
    model.refresh_lora_half()
    grads = _grads(model, tokens, lengths)
    norm = _norm(grads)
    limit = 0.25 * norm
    tr = QLoRATrainer(model, lr=1e-4, cuda_graph=graph, max_grad_norm=limit, buckets_on_one_rank=bucketed)
    tr.step(tokens, lengths)
    # the same kernels on the same values: fp32 rounding of the sums and factors only
    assert abs(float(tr.grad_norm) - norm) <= 1e-5 * norm
    c = limit / (norm + 1e-6)
    for p, g in zip(tr.params, grads):
        m = tr.opt.state[p]["exp_avg"]
        want = 0.1 * c * g
        assert float((m - want).abs().max()) <= 1e-5 * float(want.abs().max()) + 1e-12
    tr.release()


def test_limit_that_is_not_reached_changes_nothing(cuda_lib):
    """With a limit above the norm the step is the unclipped one, up to the rounding of one division
    as a multiplication (2 x 2^-24 relative on a gradient)."""
    from stew_b200.qlora_step import QLoRATrainer
    tokens, lengths = _batch(2)
    states = []
    for limit in (None, 1e9):
        model = _model()
        tr = QLoRATrainer(model, lr=1e-4, max_grad_norm=limit)
        tr.step(tokens, lengths)
        states.append([tr.opt.state[p]["exp_avg"].clone() for p in tr.params])
    for a, b in zip(*states):
        assert bool(((a - b).abs() <= 4 * 2.0 ** -24 * a.abs() + 1e-30).all())


def test_step_repeats_bit_for_bit(cuda_lib):
    """Forward, backward, clipping: the gradients of two runs are the same bits."""
    model = _model()
    tokens, lengths = _batch(3)
    first = _grads(model, tokens, lengths)
    assert all(torch.equal(a, b) for a, b in zip(first, _grads(model, tokens, lengths)))


def test_refused_limit(cuda_lib):
    from stew_b200.qlora_step import QLoRATrainer
    with pytest.raises(ValueError):
        QLoRATrainer(_model(), max_grad_norm=-1.0)
