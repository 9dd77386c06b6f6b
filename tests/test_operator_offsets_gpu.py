"""Rows and weights that lie more than 2^32 bytes and more than 2^31 elements apart."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def far(rows, cols, dtype, dev):
    """A matrix whose rows are over 2^31 elements apart."""
    apart = (1 << 31) + 8
    return torch.empty((rows - 1) * apart + cols, dtype=dtype, device=dev).as_strided((rows, cols), (apart, 1))


def test_route_of_rows_far_apart(cuda_device):
    from execution_ucx_b200.ops import moe
    logits = far(3, 200, torch.bfloat16, cuda_device).copy_(torch.randn(3, 200, device=cuda_device))
    for kw in ({}, {"groups": 4, "topk_groups": 2}):
        for a, b in zip(moe.route(logits, 6, **kw), moe.route(logits.contiguous(), 6, **kw)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t", [3, 12])
def test_experts_far_apart(cuda_device, fp8, t):
    from execution_ucx_b200.ops import moe
    from test_moe_experts_gpu import plain, weights
    h, i, count = 4096, 4096, 200 if fp8 else 100  # 6.7 GB of gate and up, more than 2^31 elements
    used = [0, 1, count // 2, count - 1]
    small = weights(4, h, i, fp8, cuda_device)
    large = []
    for part in small:
        if part is not None:
            flat = torch.empty(count, *part.shape[1:], dtype=part.dtype, device=cuda_device)
            (flat.view(torch.uint8) if fp8 else flat).zero_()
            for a, b in enumerate(used):
                flat[b].copy_(part[a])
            large.append(flat)
    layer = moe.MoeExperts(*large)
    x = torch.randn(t, h, device=cuda_device).to(torch.bfloat16)
    idx = torch.stack([torch.randperm(4)[:2] for _ in range(t)])
    w = torch.rand(t, 2, device=cuda_device)
    out = layer(x, torch.tensor(used)[idx].to(torch.int32).to(cuda_device), w)
    want, tol = plain(x, idx.to(torch.int32).to(cuda_device), w, *small)
    assert bool(((out.double() - want).abs() <= tol).all())
    layer.check_status()


def test_experts_and_adapters_of_rows_far_apart(cuda_device):
    from execution_ucx_b200.ops import lora, moe
    from test_lora_gpu import adapters
    from test_moe_experts_gpu import weights
    x = far(3, 1024, torch.bfloat16, cuda_device)
    dense = torch.randn(3, 1024, device=cuda_device).to(torch.bfloat16)
    layer, some = moe.MoeExperts(*weights(4, 1024, 64, False, cuda_device)), lora.LoraAdapters(*adapters(3, 1024, 1024, 16, cuda_device))
    idx, w = torch.tensor([[0, 1], [2, 3], [1, 2]], dtype=torch.int32, device=cuda_device), torch.rand(3, 2, device=cuda_device)
    ids = torch.tensor([0, -1, 2], dtype=torch.int32, device=cuda_device)
    for call in (lambda a, **kw: layer(a, idx, w, **kw), lambda a, **kw: some(a, ids, a, **kw)):
        x.copy_(dense)
        want = call(dense)
        assert torch.equal(call(x), want)
        assert torch.equal(call(x, out=x), want) and torch.equal(x, want)
    layer.check_status()


@pytest.mark.parametrize("t", [2, 600])
def test_adapters_far_apart(cuda_device, t):
    from execution_ucx_b200.ops import lora
    from test_lora_gpu import adapters, check
    count, k, n, rank = 2100, 8192, 8200, 128  # 2.2e9 elements in each
    a, b, scale = adapters(3, k, n, rank, cuda_device)
    large_a, large_b = (torch.zeros(count, *p.shape[1:], dtype=torch.bfloat16, device=cuda_device) for p in (a, b))
    large_scale = torch.zeros(count, device=cuda_device)
    used = [0, count - 2, count - 1]
    for i, j in enumerate(used):
        large_a[j], large_b[j], large_scale[j] = a[i], b[i], scale[i]
    ids = torch.randint(0, 3, (t,))
    x, y = (torch.randn(t, c, device=cuda_device).to(torch.bfloat16) for c in (k, n))
    want = check(lora.LoraAdapters(a, b, scale), x, ids.to(torch.int32).to(cuda_device), y)
    assert torch.equal(lora.LoraAdapters(large_a, large_b, large_scale)(x, torch.tensor(used)[ids].to(torch.int32).to(cuda_device), y), want)
