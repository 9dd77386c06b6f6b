"""The expert layer for a few tokens against a plain statement in 64 bits.

Bounds are derived, element by element: the result is rounded to bfloat16 (2^-8 of it), what lies between the two products
is rounded to bfloat16 (2^-8 of each term of the second product), and sums of n terms in float32 are off by at most n * 2^-24
of the sum of the terms' magnitudes, whatever their order (products of bfloat16 values are exact in float32). With e4m3
weights a block's sum is multiplied by its scale: one more rounding of 2^-24."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F = 2.0 ** -8, 2.0 ** -24


def weights(e, h, i, fp8, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    out = []
    for rows, cols in ((2 * i, h), (h, i)):
        w = torch.randn(e, rows, cols, generator=g, device=dev)
        if fp8:
            q = (w * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
            s = (0.5 + torch.rand(e, -(-rows // 128), -(-cols // 128), generator=g, device=dev)) * cols ** -0.5 / 100
            out += [q, s]
        else:
            out += [(w * cols ** -0.5).to(torch.bfloat16), None]
    return out[0], out[2], out[1], out[3]


def plain(x, idx, w, gu, down, gus=None, ds=None, between=BF):
    """(the result, the bound of its error), both in 64 bits. `between`: of the rounding between the products."""
    def full(m, s):
        m = m.double()
        return m if s is None else m * s.double().repeat_interleave(128, 0)[:m.shape[0]].repeat_interleave(128, 1)[:, :m.shape[1]]
    e, h, i = down.shape
    out = torch.zeros(x.shape[0], h, dtype=torch.float64, device=x.device)
    tol = torch.zeros_like(out)
    for j in range(e):
        tok, slot = (idx == j).nonzero(as_tuple=True)
        if not tok.numel():
            continue
        a, b = full(gu[j], None if gus is None else gus[j]), full(down[j], None if ds is None else ds[j])
        xj, wj = x[tok].double(), w[tok, slot].double().unsqueeze(1)
        v, dv = xj @ a.t(), (h + 2) * F * (xj.abs() @ a.abs().t())
        g, u, dg, du = v[:, :i], v[:, i:], dv[:, :i], dv[:, i:]
        s = g * torch.sigmoid(g)
        hid = s * u
        # silu has a slope of at most 1.1; exp, a division and two products in float32
        dh = 1.1 * dg * u.abs() + s.abs() * du + dg * du * 1.1 + 16 * F * hid.abs()
        dh = dh + between * (hid.abs() + dh) + 2.0 ** -134
        out.index_add_(0, tok, wj * (hid @ b.t()))
        tol.index_add_(0, tok, wj.abs() * (dh @ b.abs().t() + (i + 40) * F * ((hid.abs() + dh) @ b.abs().t())))
    tol = tol + BF * (out.abs() + tol) + 2.0 ** -134
    return out, tol


def routing(t, k, total, dev, seed, absent=0.0):
    g = torch.Generator().manual_seed(seed)
    idx = torch.rand(t, total, generator=g).topk(k, -1).indices.to(torch.int32)
    idx[torch.rand(t, k, generator=g) < absent] = -1
    w = torch.softmax(torch.randn(t, k, generator=g), -1)
    return idx.to(dev), w.to(dev)


def check(layer, x, idx, w, **kw):
    out = layer(x, idx, w, **kw)
    torch.cuda.synchronize()
    layer.check_status()
    want, tol = plain(x, idx, w, layer.w_gate_up, layer.w_down, layer.gate_up_scale, layer.down_scale)
    off = (out.double() - want).abs()
    assert out.dtype == torch.bfloat16 and bool((off <= tol).all()), f"off by up to {(off / tol).max().item():.3g} of the bound"
    return out


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t,h,i,e,k,total", [
    (1, 128, 64, 1, 1, 1), (1, 16, 16, 3, 2, 3), (1, 2048, 768, 16, 8, 16), (2, 1928 // 16 * 16, 1008, 40, 6, 40), (7, 256, 80, 5, 3, 5),
    (9, 144, 304, 12, 4, 12), (37, 512, 272, 8, 2, 8), (64, 640, 128, 4, 2, 4), (65, 272, 208, 2, 1, 2), (128, 1024, 96, 2, 2, 2),
    (128, 320, 64, 32, 8, 256), (100, 4096, 16, 3, 3, 3), (33, 16, 2064, 2, 2, 2), (16, 7168, 256, 8, 8, 64), (31, 400, 144, 300, 32, 300)])
def test_against_plain(cuda_device, fp8, t, h, i, e, k, total):
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(e, h, i, fp8, cuda_device, seed=h + i))
    x = torch.randn(t, h, device=cuda_device).to(torch.bfloat16)
    for rnd in range(2):  # scratch must be reusable
        idx, w = routing(t, k, total, cuda_device, 10 * t + rnd)
        out = check(layer, x, idx - (total - e) // 2, w)
        assert torch.equal(out, layer(x, idx - (total - e) // 2, w)), "the same arguments give the same bits"


@pytest.mark.parametrize("h,i", [(8, 8), (24, 40), (1000, 56), (136, 1096)])
def test_bf16_sizes_that_are_multiples_of_8_only(cuda_device, h, i):
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(6, h, i, False, cuda_device))
    x = torch.randn(13, h, device=cuda_device).to(torch.bfloat16)
    check(layer, x, *routing(13, 3, 6, cuda_device, 5))


@pytest.mark.parametrize("fp8", [False, True])
def test_all_tokens_to_one_expert_and_the_same_expert_twice(cuda_device, fp8):
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(4, 256, 144, fp8, cuda_device))
    x = torch.randn(128, 256, device=cuda_device).to(torch.bfloat16)
    w = torch.rand(128, 3, device=cuda_device) - 0.3
    check(layer, x, torch.full((128, 3), 2, dtype=torch.int32, device=cuda_device), w)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t", [7, 8, 9, 15, 16, 17, 24, 25, 31, 32, 33, 45, 48, 49, 63, 64, 65, 97, 128])
def test_every_number_of_tokens_that_an_expert_can_have(cuda_device, fp8, t):
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(3, 272, 208, fp8, cuda_device))
    idx = torch.ones(t, 1, dtype=torch.int32, device=cuda_device)
    idx[:2] = 2  # and another expert with two
    x = torch.randn(t, 272, device=cuda_device).to(torch.bfloat16)
    check(layer, x, idx, torch.rand(t, 1, device=cuda_device))
    layer.check_status()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t,k,e", [(1, 8, 16), (3, 2, 4), (4, 4, 4), (8, 2, 16), (8, 32, 100)])
def test_few_tokens_lose_nothing_between_the_products(cuda_device, fp8, t, k, e):
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(e, 384, 1040, fp8, cuda_device))
    g = torch.Generator().manual_seed(t)
    idx = (torch.arange(t * k).reshape(t, k) % e)[torch.randperm(t, generator=g)].to(torch.int32).to(cuda_device)  # no expert more than four times
    assert int(torch.bincount(idx.flatten().long()).max()) <= 4
    x, w = torch.randn(t, 384, device=cuda_device).to(torch.bfloat16), torch.rand(t, k, device=cuda_device)
    out = check(layer, x, idx, w)
    # two bfloat16 numbers: the second is off by 2^-8 of what the first left, 2^-8 of the value
    want, tol = plain(x, idx, w, layer.w_gate_up, layer.w_down, layer.gate_up_scale, layer.down_scale, between=2.0 ** -16)
    assert bool(((out.double() - want).abs() <= tol).all())
    x[0, 5] = float("inf")  # stays with its token
    rest = layer(x, idx, w)
    assert torch.equal(rest[1:], out[1:])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t,k,e,h,i", [(1, 8, 16, 1936, 1040), (1, 1, 1, 16, 1000 // 16 * 16), (4, 4, 4, 400, 656), (8, 2, 16, 144, 2064), (8, 32, 100, 80, 304), (7, 4, 30, 208, 64)])
def test_few_tokens_lose_nothing_between_the_products_whatever_the_width(cuda_device, fp8, t, k, e, h, i):
    """As above, with rows whose width is no multiple of 128."""
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(e, h, i, fp8, cuda_device))
    idx = (torch.arange(t * k).reshape(t, k) % e).to(torch.int32)
    idx[t // 2:, 0] = torch.where(torch.arange(t - t // 2) % 3 == 2, -1, idx[t // 2:, 0])  # and entries without an expert
    idx = idx.to(cuda_device)
    assert int(torch.bincount(idx[idx >= 0].long()).max()) <= 4
    x, w = torch.randn(t, h, device=cuda_device).to(torch.bfloat16), torch.rand(t, k, device=cuda_device)
    out = check(layer, x, idx, w)
    assert torch.equal(out, layer(x, idx, w))
    want, tol = plain(x, idx, w, layer.w_gate_up, layer.w_down, layer.gate_up_scale, layer.down_scale, between=2.0 ** -16)
    assert bool(((out.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("counts", [(128, 1, 1, 1), (20, 9, 3, 33, 1, 0, 17, 8), (12,) + (1,) * 39, (1,) * 39 + (64,), (40, 128, 100, 70)])
def test_experts_with_very_different_numbers_of_tokens(cuda_device, fp8, counts):
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(len(counts), 400, 336, fp8, cuda_device))
    idx = torch.full((128, 4), -1, dtype=torch.int32)
    at = 0
    for e, n in enumerate(counts):  # entries one after the other, the tokens in turn
        for j in range(n):
            idx[at % 128, at // 128] = e
            at += 1
    idx = idx[torch.randperm(128, generator=torch.Generator().manual_seed(at))].to(cuda_device)
    x, w = torch.randn(128, 400, device=cuda_device).to(torch.bfloat16), torch.rand(128, 4, device=cuda_device)
    out = check(layer, x, idx, w)
    assert torch.equal(out, layer(x, idx, w))
    layer.check_status()


@pytest.mark.parametrize("fp8", [False, True])
def test_entries_without_an_expert(cuda_device, fp8):
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(6, 256, 144, fp8, cuda_device))
    x = torch.randn(40, 256, device=cuda_device).to(torch.bfloat16)
    idx, w = routing(40, 4, 6, cuda_device, 3, absent=0.4)
    idx[0], idx[7], idx[39] = -1, 6, 2 ** 31 - 1
    idx[8, 0] = -2 ** 31
    out = check(layer, x, idx, w)
    assert not out[[0, 7, 39]].any()
    idx[:] = -1
    assert not layer(x, idx, w, out=torch.full_like(x, 3.0)).any()
    assert layer(x[:0], idx[:0], w[:0]).shape == (0, 256)


def test_numbers_that_are_none_stay_with_their_token(cuda_device):
    """A token of infinities and NaN gives such results for itself alone, also beside tokens of the same expert; the weight
    of an entry without an expert may be NaN."""
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(2, 256, 144, False, cuda_device))
    x = torch.randn(20, 256, device=cuda_device).to(torch.bfloat16)
    idx, w = routing(20, 2, 2, cuda_device, 3)
    idx[5, 1], w[5, 1] = -1, float("nan")
    x[3, 7], x[11, 0] = float("inf"), float("nan")
    out = layer(x, idx, w)
    fine = torch.ones(20, dtype=torch.bool, device=cuda_device)
    fine[[3, 11]] = False
    want, tol = plain(x[fine], idx[fine], w[fine], layer.w_gate_up, layer.w_down)
    assert bool(((out[fine].double() - want).abs() <= tol).all())
    assert bool(out[11].isnan().all()) and not bool(out[3].isfinite().all())


def test_rows_that_lie_apart_and_out_given(cuda_device):
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(8, 256, 144, False, cuda_device))
    idx, w = routing(21, 3, 8, cuda_device, 9)
    wide = torch.randn(21, 512, device=cuda_device).to(torch.bfloat16)
    x = wide[:, 128:384]
    room = torch.full((21, 264), 7.0, dtype=torch.bfloat16, device=cuda_device)
    want = layer(x.contiguous(), idx, w)
    got = layer(x, idx, w, out=room[:, :256])
    assert got.data_ptr() == room.data_ptr() and torch.equal(got, want) and bool((room[:, 256:] == 7).all())
    rest = wide.clone()
    assert torch.equal(layer(x, idx, w, out=x), want), "in place"
    assert torch.equal(wide[:, :128], rest[:, :128]) and torch.equal(wide[:, 384:], rest[:, 384:])


@pytest.mark.parametrize("t", [129, 300])
def test_more_tokens_than_one_pass(cuda_device, t):
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(8, 256, 144, False, cuda_device))
    x = torch.randn(t, 256, device=cuda_device).to(torch.bfloat16)
    check(layer, x, *routing(t, 3, 8, cuda_device, 9))
    check(layer, x, *routing(t, 3, 8, cuda_device, 9), out=x.clone())


def test_e4m3_weights_of_every_code(cuda_device):
    """Every e4m3 value, subnormal ones among them, as a weight that a unit vector picks out."""
    from execution_ucx_b200.ops import moe
    codes = torch.tensor([c for c in range(256) if c & 0x7f != 0x7f], dtype=torch.uint8)
    h = i = 256
    gu = torch.zeros(1, 2 * i, h, dtype=torch.uint8)
    gu[0, torch.arange(i), 0] = 0x7e          # gate: 448 * x0, silu of which is itself
    gu[0, i + torch.arange(254), 1] = codes   # up: the code
    down = torch.zeros(1, h, i, dtype=torch.uint8)
    down[0, torch.arange(h), torch.arange(i)] = 0x38  # one
    one = torch.ones(1, 4, 2, device=cuda_device)
    as_e4m3 = lambda v: v.to(cuda_device).view(torch.float8_e4m3fn)  # noqa: E731
    layer = moe.MoeExperts(as_e4m3(gu), as_e4m3(down), one, torch.ones(1, 2, 2, device=cuda_device))
    x = torch.zeros(1, h, dtype=torch.bfloat16, device=cuda_device)
    x[0, 0], x[0, 1] = 1.0, 1.0
    out = layer(x, torch.zeros(1, 1, dtype=torch.int32, device=cuda_device), torch.ones(1, 1, device=cuda_device))
    want = 448 * as_e4m3(codes).float()
    assert torch.equal(out[0, :254].float(), want.to(torch.bfloat16).float())  # 7 bits of 448 times 4 bits: exact before the rounding


def test_e4m3_weights_that_are_nan_are_refused(cuda_device):
    from execution_ucx_b200.ops import moe
    for which, code in ((0, 0x7f), (1, 0xff)):
        gu, down, gus, ds = weights(3, 256, 144, True, cuda_device)
        (gu, down)[which].view(torch.uint8)[2, 5, 9] = code
        with pytest.raises(ValueError, match="NaN"):
            moe.MoeExperts(gu, down, gus, ds)


def test_two_streams_at_once(cuda_device):
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(8, 1024, 256, False, cuda_device))
    streams = [torch.cuda.Stream() for _ in range(3)]
    args = []
    for s in range(3):
        args.append((torch.randn(5 + 9 * s, 1024, device=cuda_device).to(torch.bfloat16), *routing(5 + 9 * s, 3, 8, cuda_device, s)))
    want = [layer(*a) for a in args]
    torch.cuda.synchronize()
    got = [[] for _ in range(3)]
    for _ in range(20):
        for s in range(3):
            with torch.cuda.stream(streams[s]):
                got[s].append(layer(*args[s]))
    torch.cuda.synchronize()
    layer.check_status()
    for s in range(3):
        assert all(torch.equal(o, want[s]) for o in got[s])


def test_threads_that_share_a_stream(cuda_device):
    import threading
    from execution_ucx_b200.ops import lora, moe
    layer = moe.MoeExperts(*weights(8, 1024, 256, False, cuda_device))
    adapters = lora.LoraAdapters(torch.randn(4, 16, 1024, device=cuda_device).to(torch.bfloat16), torch.randn(4, 1024, 16, device=cuda_device).to(torch.bfloat16))
    args, want, got = [], [], [[] for _ in range(4)]
    for s in range(4):
        t = (3, 17, 40, 100)[s]
        x = torch.randn(t, 1024, device=cuda_device).to(torch.bfloat16)
        ids = torch.randint(0, 4, (t,), device=cuda_device, dtype=torch.int32)
        args.append((x, *routing(t, 3, 8, cuda_device, s), ids))
    both = lambda a: adapters(a[0], a[3], layer(*a[:3]))  # noqa: E731
    for a in args:
        want.append(both(a))
    layer2 = moe.MoeExperts(layer.w_gate_up, layer.w_down)  # whose workspaces have yet to grow
    both2 = lambda a: adapters(a[0], a[3], layer2(*a[:3]))  # noqa: E731

    def run(s):
        for _ in range(50):
            got[s].append(both2(args[s]))
    threads = [threading.Thread(target=run, args=(s,)) for s in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    layer2.check_status()
    for s in range(4):
        assert len(got[s]) == 50 and all(torch.equal(o, want[s]) for o in got[s])


def test_threads_that_call_an_object_for_the_first_time_share_one_workspace(cuda_device):
    import threading
    from execution_ucx_b200.ops import _workspace
    scratch = _workspace.CallScratch(8, cuda_device)
    made, begin = [], threading.Barrier(8)
    ordinary = torch.zeros

    def slow(*a, **kw):  # the other threads come while the first is making its words
        import time
        time.sleep(0.05)
        return ordinary(*a, **kw)

    def run():
        begin.wait()
        made.append(scratch.get(1 << 16))
    threads = [threading.Thread(target=run) for _ in range(8)]
    torch.zeros = slow
    try:
        [t.start() for t in threads]
        [t.join() for t in threads]
    finally:
        torch.zeros = ordinary
    assert len(made) == 8 and len(set(made)) == 1


def test_captured_calls_replayed_beside_each_other_and_plain_ones(cuda_device):
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(8, 1024, 256, False, cuda_device))
    args = [(torch.randn(12, 1024, device=cuda_device).to(torch.bfloat16), *routing(12, 3, 8, cuda_device, s)) for s in range(3)]
    want = [layer(*a) for a in args]
    graphs, outs = [], []
    for s in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = layer(*args[s])
            o2 = layer(o, *args[s][1:])
        graphs.append(g), outs.append((o, o2))
    want2 = [layer(want[s], *args[s][1:]) for s in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                graphs[s].replay()
        plain_one = layer(*args[2])
        torch.cuda.synchronize()
        assert torch.equal(plain_one, want[2])
        for s in range(2):
            assert torch.equal(outs[s][0], want[s]) and torch.equal(outs[s][1], want2[s])
    layer.check_status()


def test_more_captured_calls_than_words_zeroed_beforehand(cuda_device):
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(4, 512, 128, False, cuda_device))
    x = torch.randn(6, 512, device=cuda_device).to(torch.bfloat16)
    idx, w = routing(6, 2, 4, cuda_device, 1)
    want = x
    for _ in range(20):
        want = layer(want, idx, w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = x
        for _ in range(20):
            got = layer(got, idx, w)
    for _ in range(3):
        g.replay()
        assert torch.equal(got, want)


def test_weights_written_in_place_hold_for_the_next_call(cuda_device):
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(4, 256, 144, False, cuda_device))
    x = torch.randn(6, 256, device=cuda_device).to(torch.bfloat16)
    idx, w = routing(6, 2, 4, cuda_device, 1)
    check(layer, x, idx, w)
    layer.w_gate_up.mul_(0.5)
    layer.w_down.neg_()
    check(layer, x, idx, w)


@pytest.mark.parametrize("t", [2, 60])
def test_what_a_graph_writes_in_front_of_a_call_is_seen(cuda_device, t):
    """Tokens, choices, weights of choices and of experts, written by kernels that run just before the call, replay after replay."""
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(8, 256, 144, False, cuda_device))
    x = torch.randn(t, 256, device=cuda_device).to(torch.bfloat16)
    idx, w = routing(t, 3, 8, cuda_device, 1)
    old = (x, idx, w, layer.w_gate_up, layer.w_down)
    new = [v.clone() for v in old]
    layer(x, idx, w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for a, b in zip(old, new):
            a.copy_(b)
        out = layer(x, idx, w)
    for rnd in range(5):
        new[0].copy_(torch.randn(t, 256, device=cuda_device))
        for a, b in zip(new[1:3], routing(t, 3, 8, cuda_device, 20 + rnd, absent=0.2)):
            a.copy_(b)
        for b in new[3:]:
            b.copy_(torch.randn(b.shape, device=cuda_device) * 0.07)
        g.replay()
        torch.cuda.synchronize()
        layer.check_status()
        want, tol = plain(*new)
        assert bool(((out.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("fp8_rows", [False])
def test_route_dispatch_experts_combine(cuda_device, fp8_rows):
    """The parts as they are used across GPUs, with logical ranks on one: the router's choice, the rows sent to the experts'
    ranks, every rank's experts over what it received, in place, and the gate-weighted rows back."""
    from execution_ucx_b200.ops import moe
    world, t, h, i, e, k = 2, 24, 256, 144, 8, 3
    ranks = moe.MoeAllToAll.emulated(world, t, h, k, e)
    gu, down, _, _ = weights(e, h, i, False, cuda_device)
    epr = e // world
    layers = [moe.MoeExperts(gu[r * epr:(r + 1) * epr], down[r * epr:(r + 1) * epr]) for r in range(world)]
    xs = [torch.randn(t, h, device=cuda_device).to(torch.bfloat16) for _ in range(world)]
    chosen = [moe.route(torch.randn(t, e, device=cuda_device), k) for _ in range(world)]
    for r in range(world):
        ranks[r].dispatch(xs[r], *chosen[r])
    torch.cuda.synchronize()
    for r in range(world):
        for src in range(world):
            n = int(ranks[r].recv_counts()[src])
            rows = ranks[r].recv_rows(src, n).view(torch.bfloat16)
            local = (ranks[r].recv_meta(src, n)[:, 1] >> 16).view(n, 1).contiguous()
            layers[r](rows, local, torch.ones(n, 1, device=cuda_device), out=rows)
        ranks[r].expert_ready()
    for r in range(world):
        got = ranks[r].combine()
        torch.cuda.synchronize()
        ranks[r].check_status()
        want, tol = plain(xs[r], *chosen[r], gu, down)
        # each expert's row is rounded to bfloat16 before the combine
        idx, w = chosen[r]
        for slot in range(k):
            one, _ = plain(xs[r], idx[:, slot:slot + 1], torch.ones(t, 1, device=cuda_device), gu, down)
            tol = tol + BF * w[:, slot:slot + 1].double().abs() * one.abs() * (1 + BF)
        assert bool(((got.double() - want).abs() <= tol).all())
        # the whole layer on one GPU says the same
        whole = moe.MoeExperts(gu, down)(xs[r], idx, w)
        assert bool(((got.double() - whole.double()).abs() <= 2 * tol).all())


@pytest.mark.parametrize("t,k,h,what", [(1, 2, 256, "bf16"), (8, 1, 144, "bf16"), (9, 1, 256, "bf16"), (40, 3, 256, "bf16"), (128, 2, 144, "bf16"),
                                        (1, 2, 256, "scale"), (8, 1, 144, "scale"), (40, 3, 256, "scale")])
def test_infinities_in_the_weights(cuda_device, t, k, h, what):
    """A weight (or a block's scale) that is infinite makes infinities, and NaN only where the formula does, whatever the number of tokens."""
    from execution_ucx_b200.ops import moe
    i, e, inf = 256, 4, float("inf")
    gu, down, gus, ds = weights(e, h, i, what == "scale", cuda_device)
    x = torch.randn(t, h, device=cuda_device).abs().to(torch.bfloat16)
    idx, w = routing(t, k, e, cuda_device, 5)
    idx[:, 0] = torch.arange(1, t + 1, device=cuda_device) % e  # the second expert first: one token meets an infinity
    if what == "bf16":
        gu[:, 7], gu[:, i + 7] = 0.125, 0.125  # h[7] is well above zero for every token, and so is h[200]
        gu[:, 200], gu[:, i + 200] = 0.25, 0.125
        gu[2, 9] = gu[2, i + 9] = 0            # and h[9] of the third expert is zero
        down[0, 3, 7], down[1, 5, 7], down[1, 5, 200], down[1, 6, 7] = inf, inf, -inf, -inf
        down[2, 8, 9], down[2, 11, 7], down[3, 12, 7] = inf, -inf, float("nan")
    else:
        gu.view(torch.uint8)[:] = gu.view(torch.uint8) & 0x7f  # all is positive: h, and with an infinite scale what it makes
        down.view(torch.uint8)[:] = (down.view(torch.uint8) & 0x7f).clamp(min=1)
        ds[1, 0, 0], ds[2, (h - 1) // 128, 1] = inf, -inf
    layer = moe.MoeExperts(gu, down, gus, ds)
    out = layer(x, idx, w).double()
    torch.cuda.synchronize()
    layer.check_status()
    want = moe.reference_experts(x, idx, w, gu, down, gus, ds)
    clean = lambda v: v if v is None else torch.where(v.float().isfinite(), v, 0.0) if what == "bf16" else v  # noqa: E731
    _, tol = plain(x, idx, w, clean(gu), clean(down), gus, ds if ds is None else torch.where(ds.isfinite(), ds, 0.0))
    fine = want.isfinite()
    assert bool(want.isinf().any()) and torch.equal(out.isnan(), want.isnan()) and torch.equal(out[want.isinf()], want[want.isinf()])
    assert bool(((out - want).abs()[fine] <= tol[fine]).all())


@pytest.mark.parametrize("fp8", [False, True])
def test_as_many_experts_and_entries_as_there_may_be(cuda_device, fp8):
    from execution_ucx_b200.ops import moe
    layer = moe.MoeExperts(*weights(1024, 64, 32, fp8, cuda_device))
    x = torch.randn(128, 64, device=cuda_device).to(torch.bfloat16)
    check(layer, x, *routing(128, 32, 1024, cuda_device, 3))
    idx, w = routing(128, 32, 1024, cuda_device, 4)
    idx[:, :] = 1023
    check(layer, x, idx, w)
