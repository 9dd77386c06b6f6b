"""Adapters of many requests against a plain statement in 64 bits.

Bounds are derived, element by element: the result is rounded to bfloat16 once (2^-8 of it); the first product's sums of K
terms in float32 are off by at most K * 2^-24 of the sum of the magnitudes, and what is kept of one between the products by
2^-16 of it; the second product's by rank * 2^-24 likewise, the scale and the addition by a few roundings."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F = 2.0 ** -8, 2.0 ** -24


def adapters(count, k, n, rank, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    a = (torch.randn(count, rank, k, generator=g, device=dev) * k ** -0.5).to(torch.bfloat16)
    b = (torch.randn(count, n, rank, generator=g, device=dev) * rank ** -0.5).to(torch.bfloat16)
    return a, b, 0.5 + torch.rand(count, generator=g, device=dev)


def plain(x, ids, y, a, b, scale):
    """(the result, the bound of its error), both in 64 bits."""
    out = y.double().clone()
    tol = torch.zeros_like(out)
    k, r = x.shape[1], a.shape[1]
    for i in range(a.shape[0]):
        rows = (ids == i).nonzero().squeeze(1)
        if rows.numel():
            xi, ai, bi, s = x[rows].double(), a[i].double(), b[i].double(), scale[i].double()
            v = xi @ ai.t()
            dv = (k + 8) * F * (xi.abs() @ ai.abs().t()) + 2.0 ** -16 * v.abs()
            out[rows] += s * (v @ bi.t())
            tol[rows] += s.abs() * (dv @ bi.abs().t() + (2 * r + 16) * F * ((v.abs() + dv) @ bi.abs().t()))
    return out, tol + 2 * F * out.abs() + BF * (out.abs() + tol) + 2.0 ** -134


def check(layer, x, ids, y, **kw):
    y0 = y.clone()
    out = layer(x, ids, y, **kw)
    want, tol = plain(x, ids, y0, layer.a, layer.b, layer.scale)
    off = (out.double() - want).abs()
    assert bool((off <= tol).all()), f"off by up to {(off / tol).max().item():.3g} of the bound"
    none = (ids < 0) | (ids >= layer.n_adapters)
    assert torch.equal(out[none], y0[none])
    return out


def bf(*shape, dev):
    return torch.randn(*shape, device=dev).to(torch.bfloat16)


@pytest.mark.parametrize("t,k,n,rank,count,run", [
    (1, 4096, 4096, 16, 32, 1), (1, 8, 8, 8, 1, 1), (2, 1000, 24, 24, 3, 1), (3, 64, 8200, 128, 2, 1), (17, 520, 264, 40, 5, 1), (64, 2048, 1024, 16, 64, 1),
    (65, 256, 136, 8, 4, 1), (130, 72, 2056, 64, 300, 1), (200, 8192, 512, 16, 3, 7), (500, 136, 1032, 32, 9, 33), (1000, 1024, 512, 56, 2, 300),
    (1025, 512, 520, 96, 4, 100), (4097, 256, 128, 16, 16, 1), (2048, 128, 72, 120, 1, 1)])
def test_against_plain(cuda_device, t, k, n, rank, count, run):
    from execution_ucx_b200.ops import lora
    layer = lora.LoraAdapters(*adapters(count, k, n, rank, cuda_device, seed=t))
    g = torch.Generator(device=cuda_device).manual_seed(t)
    ids = torch.randint(-1 if count > 1 else 0, count, (-(-t // run),), generator=g, device=cuda_device).repeat_interleave(run)[:t].to(torch.int32)
    x, y = bf(t, k, dev=cuda_device), bf(t, n, dev=cuda_device)
    out = check(layer, x, ids, y)
    assert torch.equal(out, layer(x, ids, y)), "the same arguments give the same bits"


@pytest.mark.parametrize("rank", [40, 64, 104, 128])
@pytest.mark.parametrize("count", [3, 80])
def test_larger_ranks_with_few_and_with_many_adapters(cuda_device, rank, count):
    from execution_ucx_b200.ops import lora
    layer = lora.LoraAdapters(*adapters(count, 2056, 200, rank, cuda_device, seed=rank))
    g = torch.Generator(device=cuda_device).manual_seed(count)
    ids = torch.randint(-1, count, (650,), generator=g, device=cuda_device, dtype=torch.int32)
    x, y = bf(650, 2056, dev=cuda_device), bf(650, 200, dev=cuda_device)
    out = check(layer, x, ids, y)
    assert torch.equal(out, layer(x, ids, y))


@pytest.mark.parametrize("t", [1, 40, 300])
def test_tokens_without_an_adapter(cuda_device, t):
    from execution_ucx_b200.ops import lora
    layer = lora.LoraAdapters(*adapters(4, 256, 264, 16, cuda_device))
    ids = torch.randint(-1, 4, (t,), device=cuda_device, dtype=torch.int32)
    ids[0] = 4
    if t > 30:
        ids[5], ids[6], ids[30] = 2 ** 31 - 1, -2 ** 31, -7
    x, y = bf(t, 256, dev=cuda_device), bf(t, 264, dev=cuda_device)
    x[0] = float("nan")
    y[0, 3] = float("nan")  # kept as it is
    out = layer(x, ids, y)
    want, tol = plain(x[1:], ids[1:], y[1:], layer.a, layer.b, layer.scale)
    assert torch.equal(out[0].view(torch.int16), y[0].view(torch.int16))
    assert bool(((out[1:].double() - want).abs() <= tol).all())
    ids[:] = -1
    assert torch.equal(layer(x, ids, y).view(torch.int16), y.view(torch.int16))
    assert layer(x[:0], ids[:0], y[:0]).shape == (0, 264)


@pytest.mark.parametrize("t", [20, 300])
def test_numbers_that_are_none_stay_with_their_token(cuda_device, t):
    from execution_ucx_b200.ops import lora
    layer = lora.LoraAdapters(*adapters(2, 256, 264, 16, cuda_device))
    ids = torch.zeros(t, dtype=torch.int32, device=cuda_device)
    x, y = bf(t, 256, dev=cuda_device), bf(t, 264, dev=cuda_device)
    x[3, 7], x[11, 0], y[12, 5] = float("inf"), float("nan"), float("inf")
    out = layer(x, ids, y)
    fine = torch.ones(t, dtype=torch.bool, device=cuda_device)
    fine[[3, 11, 12]] = False
    want, tol = plain(x[fine], ids[fine], y[fine], layer.a, layer.b, layer.scale)
    assert bool(((out[fine].double() - want).abs() <= tol).all())
    assert bool(out[11].isnan().all()) and not bool(out[3].isfinite().any()) and bool(out[12, 5].isinf()) and bool(out[12, 6:].isfinite().all())


@pytest.mark.parametrize("t", [20, 300])
def test_rows_that_lie_apart_and_in_place(cuda_device, t):
    from execution_ucx_b200.ops import lora
    layer = lora.LoraAdapters(*adapters(4, 256, 264, 16, cuda_device))
    ids = torch.randint(0, 4, (t,), device=cuda_device, dtype=torch.int32)
    xw, yw = bf(t, 512, dev=cuda_device), bf(t, 288, dev=cuda_device)
    x, y = xw[:, 64:320], yw[:, 8:272]
    want = layer(x.contiguous(), ids, y.contiguous())
    room = torch.full((t, 272), 7.0, dtype=torch.bfloat16, device=cuda_device)
    got = layer(x, ids, y, out=room[:, :264])
    assert torch.equal(got, want) and bool((room[:, 264:] == 7).all())
    before = yw.clone()
    assert torch.equal(layer(x, ids, y, out=y), want)
    assert torch.equal(yw[:, :8], before[:, :8]) and torch.equal(yw[:, 272:], before[:, 272:])


@pytest.mark.parametrize("t", [8, 300])
def test_captured_beside_other_streams(cuda_device, t):
    from execution_ucx_b200.ops import lora
    layer = lora.LoraAdapters(*adapters(6, 512, 264, 16, cuda_device))
    args = [(bf(t, 512, dev=cuda_device), torch.randint(-1, 6, (t,), device=cuda_device, dtype=torch.int32), bf(t, 264, dev=cuda_device)) for _ in range(3)]
    want = [layer(*a) for a in args]
    graphs, outs = [], []
    for s in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(*args[s]))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                graphs[s].replay()
        third = layer(*args[2])
        torch.cuda.synchronize()
        assert torch.equal(third, want[2]) and all(torch.equal(outs[s], want[s]) for s in range(2))


@pytest.mark.parametrize("t", [3, 300])
def test_what_a_graph_writes_in_front_of_a_call_is_seen(cuda_device, t):
    """ids, y and the adapters, written by kernels that run just before the call, replay after replay."""
    from execution_ucx_b200.ops import lora
    layer = lora.LoraAdapters(*adapters(6, 512, 264, 16, cuda_device))
    x, y, ids = bf(t, 512, dev=cuda_device), bf(t, 264, dev=cuda_device), torch.zeros(t, dtype=torch.int32, device=cuda_device)
    new = [torch.empty_like(v) for v in (x, y, ids, layer.a, layer.b)]
    layer(x, ids, y)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for old, v in zip((x, y, ids, layer.a, layer.b), new):
            old.copy_(v)
        out = layer(x, ids, y)
        out2 = layer(x, ids, out)
    for rnd in range(5):
        for v in new:
            v.copy_(torch.randint(-1, 6, v.shape, device=cuda_device) if v.dtype == torch.int32 else torch.randn(v.shape, device=cuda_device))
        g.replay()
        torch.cuda.synchronize()
        want, tol = plain(new[0], new[2], new[1], new[3], new[4], layer.scale)
        assert bool(((out.double() - want).abs() <= tol).all())
        want, tol = plain(new[0], new[2], out, new[3], new[4], layer.scale)
        assert bool(((out2.double() - want).abs() <= tol).all())


def test_beside_a_shared_projection(cuda_device):
    """The remote GEMM's result for tokens of several requests, and each request's adapter added to it in place."""
    from execution_ucx_b200.ops import lora
    from execution_ucx_b200.ops.remote_gemm import RemoteGemm
    t, k, n = 128, 512, 512
    w = (torch.randn(k, n, device=cuda_device) * k ** -0.5).to(torch.bfloat16)
    x, y = bf(t, k, dev=cuda_device), torch.empty(t, n, dtype=torch.bfloat16, device=cuda_device)
    gemm = RemoteGemm(w, t)
    layer = lora.LoraAdapters(*adapters(5, k, n, 16, cuda_device))
    ids = torch.randint(-1, 5, (t,), device=cuda_device, dtype=torch.int32)
    gemm(x.data_ptr(), t, y.data_ptr(), x_is_local=True)
    shared = y.clone()
    out = layer(x, ids, y, out=y)
    torch.cuda.synchronize()
    gemm.check_status()
    base = x.double() @ w.double()
    dshared = BF * base.abs() + (k * F) * (1 + BF) * (x.double().abs() @ w.double().abs())
    assert bool(((shared.double() - base).abs() <= dshared).all())
    want, tol = plain(x, ids, shared, layer.a, layer.b, layer.scale)
    assert bool(((out.double() - want).abs() <= tol).all())


def test_more_adapters_than_counts_fit_shared_memory(cuda_device):
    """Tokens are then counted by adapter in the workspace, which in a graph may be memory that the call in front still uses."""
    from execution_ucx_b200.ops import lora, moe
    from test_moe_experts_gpu import routing, weights
    t, count, width, rank = 600, 60000, 256, 8
    layer = lora.LoraAdapters(*adapters(count, width, width, rank, cuda_device))
    experts = moe.MoeExperts(*weights(4, width, 1024, False, cuda_device))
    x, y = bf(t, width, dev=cuda_device), bf(t, width, dev=cuda_device)
    before = lora.launch_count()
    for last in (count, 40, 1):  # a tile for nearly every token, many tokens of an adapter, one adapter
        ids = torch.randint(-1, last, (t,), device=cuda_device, dtype=torch.int32)
        ids[7], ids[8], ids[9] = count - 1, count, -1
        out = layer(x, ids, y)
        named = ids.unique()
        named = named[(named >= 0) & (named < count)]
        at = torch.where((ids >= 0) & (ids < count), torch.searchsorted(named, ids), -1)
        want, tol = plain(x, at, y, layer.a[named], layer.b[named], layer.scale[named])
        assert bool(((out.double() - want).abs() <= tol).all()) and torch.equal(out[at < 0], y[at < 0])
        assert torch.equal(out, layer(x, ids, y))
    assert lora.launch_count() - before == 6 * 3, "three launches each: ordered by adapter"
    idx, w = routing(128, 4, 4, cuda_device, 1)
    want_experts = experts(x[:128], idx, w)
    want = layer(x, ids, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = []
        for _ in range(3):
            o = experts(x[:128], idx, w)
            outs.append((o, layer(x, ids, y)))
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
        experts.check_status()
        for o, a in outs:
            assert torch.equal(o, want_experts) and torch.equal(a, want)
