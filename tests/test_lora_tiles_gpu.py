"""Adapters of so many tokens that they are ordered by adapter and go in tiles (three launches): what the smaller calls are tested for too.
Bounds are those of the smaller calls' tests. Every call here is counted, so that a change of the rule that chooses between the forms
shows here."""
import contextlib

import pytest
import torch

from test_lora_gpu import adapters, bf, check, plain

pytestmark = pytest.mark.gpu

T = 600  # more than stand for themselves, whatever their bytes


@contextlib.contextmanager
def in_tiles(calls):
    from execution_ucx_b200.ops import lora
    before = lora.launch_count()
    yield
    assert lora.launch_count() - before == 3 * calls, "order, shrink and expand for each call"


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 48, 72, 128])
@pytest.mark.parametrize("t,k,n,count,run", [(513, 2048, 264, 5, 1), (900, 72, 8, 2, 200), (520, 4096, 1032, 100, 3), (1111, 8, 136, 1, 1), (4000, 264, 512, 8, 777)])
def test_every_size_of_rank(cuda_device, rank, t, k, n, count, run):
    from execution_ucx_b200.ops import lora
    layer = lora.LoraAdapters(*adapters(count, k, n, rank, cuda_device, seed=rank))
    g = torch.Generator(device=cuda_device).manual_seed(t)
    ids = torch.randint(-1, count, (-(-t // run),), generator=g, device=cuda_device).repeat_interleave(run)[:t].to(torch.int32)
    x, y = bf(t, k, dev=cuda_device), bf(t, n, dev=cuda_device)
    with in_tiles(2):
        out = check(layer, x, ids, y)
        assert torch.equal(out, layer(x, ids, y)), "the same arguments give the same bits"


def test_tokens_without_an_adapter(cuda_device):
    from execution_ucx_b200.ops import lora
    layer = lora.LoraAdapters(*adapters(4, 256, 264, 16, cuda_device))
    ids = torch.randint(-1, 4, (T,), device=cuda_device, dtype=torch.int32)
    ids[0], ids[5], ids[6], ids[30], ids[T - 1] = 4, 2 ** 31 - 1, -2 ** 31, -7, 5
    x, y = bf(T, 256, dev=cuda_device), bf(T, 264, dev=cuda_device)
    x[0] = float("nan")
    y[0, 3] = float("nan")  # kept as it is
    with in_tiles(2):
        out = layer(x, ids, y)
        want, tol = plain(x[1:], ids[1:], y[1:], layer.a, layer.b, layer.scale)
        assert torch.equal(out[0].view(torch.int16), y[0].view(torch.int16))
        assert bool(((out[1:].double() - want).abs() <= tol).all())
        ids[:] = -1
        assert torch.equal(layer(x, ids, y).view(torch.int16), y.view(torch.int16))


@pytest.mark.parametrize("rank", [8, 16, 40, 128])
def test_numbers_that_are_none_stay_with_their_token(cuda_device, rank):
    from execution_ucx_b200.ops import lora
    layer = lora.LoraAdapters(*adapters(2, 256, 264, rank, cuda_device))
    ids = torch.zeros(T, dtype=torch.int32, device=cuda_device)
    x, y = bf(T, 256, dev=cuda_device), bf(T, 264, dev=cuda_device)
    x[3, 7], x[11, 0], y[12, 5] = float("inf"), float("nan"), float("inf")
    with in_tiles(1):
        out = layer(x, ids, y)
    fine = torch.ones(T, dtype=torch.bool, device=cuda_device)
    fine[[3, 11, 12]] = False
    want, tol = plain(x[fine], ids[fine], y[fine], layer.a, layer.b, layer.scale)
    assert bool(((out[fine].double() - want).abs() <= tol).all())
    assert bool(out[11].isnan().all()) and not bool(out[3].isfinite().any()) and bool(out[12, 5].isinf()) and bool(out[12, 6:].isfinite().all())


def test_rows_that_lie_apart_and_in_place(cuda_device):
    from execution_ucx_b200.ops import lora
    layer = lora.LoraAdapters(*adapters(4, 256, 264, 16, cuda_device))
    ids = torch.randint(-1, 4, (T,), device=cuda_device, dtype=torch.int32)
    xw, yw = bf(T, 512, dev=cuda_device), bf(T, 288, dev=cuda_device)
    x, y = xw[:, 64:320], yw[:, 8:272]
    with in_tiles(3):
        want = check(layer, x.contiguous(), ids, y.contiguous())
        room = torch.full((T, 272), 7.0, dtype=torch.bfloat16, device=cuda_device)
        got = layer(x, ids, y, out=room[:, :264])
        assert torch.equal(got, want) and bool((room[:, 264:] == 7).all())
        before = yw.clone()
        assert torch.equal(layer(x, ids, y, out=y), want)
    assert torch.equal(yw[:, :8], before[:, :8]) and torch.equal(yw[:, 272:], before[:, 272:])


def test_captured_beside_other_streams(cuda_device):
    from execution_ucx_b200.ops import lora
    layer = lora.LoraAdapters(*adapters(6, 512, 264, 16, cuda_device))
    args = [(bf(T, 512, dev=cuda_device), torch.randint(-1, 6, (T,), device=cuda_device, dtype=torch.int32), bf(T, 264, dev=cuda_device)) for _ in range(3)]
    with in_tiles(3 + 2 + 10):
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


@pytest.mark.parametrize("rank", [16, 72])
def test_what_a_graph_writes_in_front_of_a_call_is_seen(cuda_device, rank):
    """ids, y and the adapters, written by kernels that run just before the call, replay after replay."""
    from execution_ucx_b200.ops import lora
    layer = lora.LoraAdapters(*adapters(6, 512, 264, rank, cuda_device))
    x, y, ids = bf(T, 512, dev=cuda_device), bf(T, 264, dev=cuda_device), torch.zeros(T, dtype=torch.int32, device=cuda_device)
    new = [torch.empty_like(v) for v in (x, y, ids, layer.a, layer.b)]
    with in_tiles(3):
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


def test_threads_that_share_a_stream(cuda_device):
    import threading
    from execution_ucx_b200.ops import lora
    parts = adapters(5, 1024, 512, 24, cuda_device)
    layer = lora.LoraAdapters(*parts)
    args = []
    for t in (513, 700, 1500, 4100):
        args.append((bf(t, 1024, dev=cuda_device), torch.randint(-1, 5, (t,), device=cuda_device, dtype=torch.int32), bf(t, 512, dev=cuda_device)))
    got = [[] for _ in args]
    with in_tiles(4 + 4 * 30):
        want = [layer(*a) for a in args]
        torch.cuda.synchronize()
        fresh = lora.LoraAdapters(*parts)  # whose workspaces have yet to grow

        def run(s):
            for _ in range(30):
                got[s].append(fresh(*args[s]))
        threads = [threading.Thread(target=run, args=(s,)) for s in range(4)]
        [t.start() for t in threads]
        [t.join() for t in threads]
        torch.cuda.synchronize()
    for s in range(4):
        assert len(got[s]) == 30 and all(torch.equal(o, want[s]) for o in got[s])


def test_on_a_stream_of_ones_own(cuda_device):
    from execution_ucx_b200.ops import lora
    layer = lora.LoraAdapters(*adapters(3, 512, 264, 32, cuda_device))
    x, y, ids = bf(T, 512, dev=cuda_device), bf(T, 264, dev=cuda_device), torch.randint(-1, 3, (T,), device=cuda_device, dtype=torch.int32)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with in_tiles(2), torch.cuda.stream(side):
        out = layer(x, ids, y)
        again = layer(x, ids, out)
    side.synchronize()
    want, tol = plain(x, ids, y, layer.a, layer.b, layer.scale)
    assert bool(((out.double() - want).abs() <= tol).all())
    want, tol = plain(x, ids, out, layer.a, layer.b, layer.scale)
    assert bool(((again.double() - want).abs() <= tol).all())


def same_kind(got, want, tol, either):
    """Infinities where the statement has infinities of that sign, NaN where it has NaN, numbers within the bound."""
    got, fine = got.double(), want.isfinite()
    assert torch.equal(got.isnan(), want.isnan())
    # an infinite scale times a sum that is within its own error of zero: of either sign
    assert torch.equal(got[want.isinf()].abs(), want[want.isinf()].abs()) and torch.equal(got[want.isinf() & ~either], want[want.isinf() & ~either])
    assert bool(((got - want).abs()[fine] <= tol[fine]).all())


@pytest.mark.parametrize("t", [20, T])
@pytest.mark.parametrize("rank", [8, 16, 40, 128])
def test_infinities_in_an_adapter(cuda_device, rank, t):
    """An adapter's infinities make infinities, and NaN only where the formula does, whatever the number of tokens."""
    from execution_ucx_b200.ops import lora
    k, n = 256, 264
    a, b, scale = adapters(3, k, n, rank, cuda_device)
    inf = float("inf")
    b[0, 7, 0], b[0, 9, rank - 1], b[0, 200, 3], b[0, 200, 5], b[0, 263, 1] = inf, -inf, inf, -inf, float("nan")
    a[1, 2, 5], b[1, 11, 4], scale[2] = inf, inf, -inf
    layer = lora.LoraAdapters(a, b, scale)
    ids = (torch.arange(t, device=cuda_device) % 4 - 1).to(torch.int32)
    x, y = bf(t, k, dev=cuda_device), bf(t, n, dev=cuda_device)
    x[1] = 0      # of the first adapter: its products are zeros, which times infinity is NaN
    y[5, 7] = -inf  # and here an infinity meets one
    out = layer(x, ids, y)
    want = lora.reference(x, ids, y, a, b, scale)
    clean = lambda v: torch.where(v.isfinite(), v, 0.0)  # noqa: E731
    _, tol = plain(x, ids, clean(y), clean(a), clean(b), clean(scale))
    assert bool(want.isinf().any()) and bool(want.isnan().any())
    sums, of_sums = plain(x, ids, torch.zeros_like(y), clean(a), clean(b), torch.ones_like(scale))
    either = (ids == 2).unsqueeze(1) & (sums.abs() <= of_sums)
    same_kind(out, want, tol, either)


@pytest.mark.parametrize("t", [20, T])
def test_products_that_only_float32_can_hold(cuda_device, t):
    """A x is a number of float32 that rounds to an infinity of bfloat16; what it is multiplied with brings it back."""
    from execution_ucx_b200.ops import lora
    a, b = torch.zeros(1, 16, 64, dtype=torch.bfloat16, device=cuda_device), torch.zeros(1, 64, 16, dtype=torch.bfloat16, device=cuda_device)
    a[0, :, 0], a[0, :, 1], b[0, :, 3] = 1, 2.0 ** -7, 2.0 ** -20
    x, y = torch.zeros(t, 64, dtype=torch.bfloat16, device=cuda_device), bf(t, 64, dev=cuda_device)
    x[2, 0] = x[2, 1] = torch.finfo(torch.bfloat16).max * 0.99609375
    x[2, 1] *= 0.9921875
    layer = lora.LoraAdapters(a, b)
    v = float(x[2, 0]) + float(x[2, 1]) * 2.0 ** -7
    assert torch.tensor(v).isfinite() and torch.tensor(v).to(torch.bfloat16).isinf()
    check(layer, x, torch.zeros(t, dtype=torch.int32, device=cuda_device), y)
