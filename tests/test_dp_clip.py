"""CPU: the exchange's clipping -- what dp hands to clip_grads and writes back, on one rank and on two
gloo ranks, with clip_grads' definition in torch standing in for the kernel."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from stew_b200 import dp


def torch_clip(grads, max_norm, divisor=None, out=None):
    """clip_grads' definition."""
    grads = list(grads)
    div = 1.0 if divisor is None else float(divisor)
    norm = sum(float((g.double() / div).square().sum()) for g in grads) ** 0.5
    c = min(1.0, max_norm / (norm + 1e-6))
    for g, o in zip(grads, grads if out is None else out):
        assert o.shape == g.shape and o.dtype == g.dtype
        o.copy_((g.double() / div * c).to(g.dtype))
    return torch.tensor(norm)


def _params(seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter(torch.zeros(n, dtype=dtype)) for n in (6, 1, 20)]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g).to(dtype)
    return ps


def _want(sums, count, limit):
    full = [s / count for s in sums]
    norm = sum(float(f.double().square().sum()) for f in full) ** 0.5
    return [f * min(1.0, limit / (norm + 1e-6)) for f in full], norm


@pytest.mark.parametrize("limit", [0.1, 1e6])
def test_one_rank(monkeypatch, limit):
    monkeypatch.setattr(dp, "clip_grads", torch_clip)
    ps = _params(1)
    want, norm = _want([p.grad.clone() for p in ps], 7.0, limit)
    total, got = dp.allreduce_lora_grads_device(ps, torch.tensor([7.0]), max_norm=limit)
    assert float(total) == 7.0 and abs(float(got) - norm) < 1e-6 * norm
    for p, w in zip(ps, want):
        assert torch.allclose(p.grad, w, rtol=1e-5)
    ps = _params(1)
    red = dp.BucketedGradAllReduce([[p] for p in ps], n_buckets=2)
    red.count = torch.tensor([7.0])
    total, got = red.finish(limit)
    assert float(total) == 7.0 and abs(float(got) - norm) < 1e-6 * norm
    for p, w in zip(ps, want):
        assert torch.allclose(p.grad, w, rtol=1e-5)


def _rank(rank, world, path, port):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    dp.clip_grads = torch_clip
    res = {}
    for dtype in (torch.float32, torch.float16):
        ps = _params(10 + rank, dtype)
        total, norm = dp.allreduce_lora_grads_device(ps, torch.tensor([3.0 + rank]), max_norm=0.05)
        res[str(dtype)] = (float(total), float(norm), [p.grad.clone() for p in ps])
    ps = _params(10 + rank)
    red = dp.BucketedGradAllReduce([[p] for p in ps], n_buckets=3)
    red.count = torch.tensor([3.0 + rank])
    total, norm = red.finish(0.05)
    res["buckets"] = (float(total), float(norm), [p.grad.clone() for p in ps])
    torch.save(res, f"{path}.{rank}")
    dist.destroy_process_group()


def test_two_ranks(tmp_path):
    import socket
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    path = str(tmp_path / "out")
    mp.spawn(_rank, args=(2, path, port), nprocs=2, join=True)
    a, b = (torch.load(f"{path}.{r}") for r in (0, 1))
    for name, dtype, rtol in (("torch.float32", torch.float32, 1e-5), ("buckets", torch.float32, 1e-5),
                              ("torch.float16", torch.float16, 2.0 ** -10)):
        sums = [x.grad.float() + y.grad.float() for x, y in zip(_params(10, dtype), _params(11, dtype))]
        want, norm = _want(sums, 7.0, 0.05)
        for total, got, grads in (a[name], b[name]):
            assert total == 7.0 and abs(got - norm) <= 1e-5 * norm
            for g, w in zip(grads, want):
                assert g.dtype == dtype and torch.allclose(g.float(), w, rtol=rtol, atol=1e-7)
