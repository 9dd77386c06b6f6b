"""What the choice of experts, the expert layer and the adapters refuse, before anything runs on a GPU."""
import pytest
import torch


def test_route_refuses():
    from execution_ucx_b200.ops import moe
    ok = torch.randn(4, 16)
    for bad, match in [(dict(logits=ok[0]), "matrix"), (dict(logits=ok.half()), "float32 or bfloat16"), (dict(logits=torch.randn(2, 1025)), "1 to 1024"),
                       (dict(logits=torch.randn(16, 4).t()), "side by side"), (dict(topk=0), "topk"), (dict(topk=17), "topk"),
                       (dict(logits=torch.randn(2, 40), topk=33), "topk"), (dict(scoring="relu"), "scoring"), (dict(groups=3), "groups"),
                       (dict(groups=0), "groups"), (dict(groups=4, topk_groups=5), "topk_groups"), (dict(groups=4, topk_groups=0), "topk_groups"),
                       (dict(bias=torch.zeros(15)), "bias"), (dict(bias=torch.zeros(16).double()), "bias"), (dict(bias=torch.zeros(32)[::2]), "contiguous"),
                       (dict(logits=torch.randn(2, 0)), "experts"), (dict(), "CUDA")]:
        with pytest.raises(ValueError, match=match):
            moe.route(**{"logits": ok, "topk": 4, **bad})


def test_experts_refuse():
    from execution_ucx_b200.ops import moe
    gu, down = torch.zeros(2, 32, 16, dtype=torch.bfloat16), torch.zeros(2, 16, 16, dtype=torch.bfloat16)
    f8 = torch.float8_e4m3fn
    s = torch.ones(2, 1, 1)
    for args, match in [((gu[0], down), "w_gate_up"), ((gu, down[0]), "w_down"), ((gu.half(), down.half()), "bfloat16 or float8"), ((gu.float(), down), "w_gate_up"),
                        ((gu[:, :30], down), "shape"), ((gu[:1], down), "shape"), ((gu.transpose(1, 2), down.transpose(1, 2)), "shape"),
                        ((torch.zeros(2, 24, 16, dtype=torch.bfloat16), torch.zeros(2, 16, 12, dtype=torch.bfloat16)), "multiples of 8"),
                        ((gu, down, s, s), "scales"), ((gu.to(f8), down.to(f8)), "scales"), ((gu.to(f8), down.to(f8), s, None), "scales"),
                        ((gu.to(f8), down.to(f8), s, torch.ones(2, 1, 2)), "down_scale"), ((gu.to(f8), down.to(f8), s.double(), s), "gate_up_scale"),
                        ((torch.zeros(2, 48, 16).to(f8), torch.zeros(2, 16, 24).to(f8), s, s), "multiples of 16"),
                        ((torch.zeros(2, 32, 32, dtype=torch.bfloat16)[:, :, ::2], down), "contiguous"), ((torch.zeros(0, 32, 16, dtype=torch.bfloat16), down[:0]), "experts"),
                        ((gu, down), "CUDA")]:
        with pytest.raises(ValueError, match=match):
            moe.MoeExperts(*args)


def test_adapters_refuse():
    from execution_ucx_b200.ops import lora
    a, b = torch.zeros(3, 16, 32, dtype=torch.bfloat16), torch.zeros(3, 24, 16, dtype=torch.bfloat16)
    for args, match in [((a[0], b), "a must be"), ((a, b[0]), "b must be"), ((a.half(), b), "a must be"), ((a, b.float()), "b must be"), ((a, b[:2]), "shape"),
                        ((a[:, :12], b[:, :, :12]), "rank"), ((torch.zeros(1, 136, 32, dtype=torch.bfloat16), torch.zeros(1, 24, 136, dtype=torch.bfloat16)), "rank"),
                        ((a[:, :, :20], b), "multiples of 8"), ((a, b[:, :20]), "multiples of 8"), ((a, b, torch.ones(2)), "scale"), ((a, b, torch.ones(3).double()), "scale"),
                        ((a[:, :, :24], b), "contiguous"), ((a[:0], b[:0]), "adapter"), ((a, b), "CUDA")]:
        with pytest.raises(ValueError, match=match):
            lora.LoraAdapters(*args)


def test_launches_refuse_without_a_gpu(native_build):
    """The C entry points check what they are given before the first CUDA call."""
    import ctypes as C
    from execution_ucx_b200.ops import _native as n
    lib = n.load()
    bad = 100001
    for launch, size in ((lib.eux_route_launch, None), (lib.eux_experts_launch, lib.eux_experts_workspace_bytes), (lib.eux_lora_launch, lib.eux_lora_workspace_bytes)):
        assert launch(None, None) == bad
        assert lib.eux_experts_maps(None, None) == bad
        assert lib.eux_experts_find_nan(None, 16, None, None) == bad
        assert size is None or size(None) == 0
    good = dict(n_tokens=2, n_experts=16, topk=2, dtype=n.DT_F32, groups=1, topk_groups=1)
    for change in (dict(n_experts=0), dict(n_experts=1025), dict(topk=17), dict(topk=33, n_experts=64), dict(groups=3), dict(groups=2, topk_groups=3), dict(dtype=n.DT_F16),
                   dict(n_tokens=-1), dict()):
        assert lib.eux_route_launch(C.byref(n.RouteDesc(**{**good, **change})), None) == bad   # the last: no pointers
    assert lib.eux_route_launch(C.byref(n.RouteDesc(**{**good, "n_tokens": 0})), None) == 0
    good = dict(n_tokens=2, hidden=64, inner=32, n_experts=4, topk=2)
    for change in (dict(n_tokens=129), dict(n_tokens=-1), dict(hidden=0), dict(hidden=60), dict(inner=33), dict(inner=24, fp8=1), dict(n_experts=0), dict(topk=0), dict(topk=33),
                   dict(x_stride=4), dict(out_stride=-4), dict()):
        assert lib.eux_experts_launch(C.byref(n.ExpertsDesc(**{**good, **change})), None) == bad
    assert lib.eux_experts_launch(C.byref(n.ExpertsDesc(**{**good, "n_tokens": 0})), None) == 0
    assert lib.eux_experts_workspace_bytes(C.byref(n.ExpertsDesc(**good))) > 0
    good = dict(n_tokens=2, k=64, n=32, rank=16, n_adapters=2)
    for change in (dict(n_tokens=-1), dict(k=60), dict(n=0), dict(rank=4), dict(rank=136), dict(rank=20), dict(n_adapters=0), dict(y_stride=2), dict()):
        assert lib.eux_lora_launch(C.byref(n.LoraDesc(**{**good, **change})), None) == bad
    assert lib.eux_lora_launch(C.byref(n.LoraDesc(**{**good, "n_tokens": 0})), None) == 0


def test_experts_refuse_passes_that_32_bits_cannot_number(native_build):
    """The blocks of a pass, times what each may cost, are numbered in 32 bits."""
    import ctypes as C
    from execution_ucx_b200.ops import _native as n
    lib = n.load()
    size = lambda **kw: lib.eux_experts_workspace_bytes(C.byref(n.ExpertsDesc(**kw)))  # noqa: E731
    large = dict(hidden=1 << 18, inner=1 << 18, n_experts=1)  # 4096 x 2048 blocks of e4m3 gate and up rows, 137 GB
    assert size(**large, n_tokens=1, topk=1, fp8=1) > 0 and size(**large, n_tokens=128, topk=1, fp8=1) > 0
    assert size(**large, n_tokens=128, topk=32, fp8=1) == 0  # 128 chunks of 32 entries that cost 9: 9.7e9
    wide = dict(hidden=1 << 17, inner=1 << 17, n_experts=1)  # 2048 x 2048 blocks in bfloat16, 69 GB
    assert size(**wide, n_tokens=128, topk=1) > 0 and size(**wide, n_tokens=128, topk=32) > 0  # 64 chunks: 2.7e8
    assert size(**{**wide, "n_experts": 1024}, n_tokens=128, topk=32) == 0
    assert size(hidden=7168, inner=2048, n_experts=1024, n_tokens=128, topk=32, fp8=1) > 0  # 45 GB, every expert named
    assert size(hidden=16384, inner=16384, n_experts=200, n_tokens=128, topk=32, fp8=1) > 0


def test_memory_that_a_result_may_share():
    """Itself row for row, or none: also where rows lie between another's rows."""
    from execution_ucx_b200.ops import _workspace as ws
    room = torch.zeros(4096, dtype=torch.bfloat16)
    rows = lambda first, count, cols, apart: room.as_strided((count, cols), (apart, 1), first)  # noqa: E731
    y = rows(512, 10, 24, 64)
    for out in (y, rows(512, 10, 24, 64), rows(536, 10, 40, 64), rows(544, 10, 8, 64), rows(488, 10, 24, 64), rows(0, 10, 24, 48), rows(1112, 10, 24, 64),
                rows(536, 3, 40, 128), rows(536, 5, 24, 40 + 88), rows(8, 5, 32, 32), torch.zeros(10, 24, dtype=torch.bfloat16)):
        ws.require_apart(out, y, "y")
    for out in (rows(520, 10, 24, 64), rows(576, 10, 24, 64), rows(448, 10, 24, 64), rows(536, 10, 48, 64), rows(512, 10, 24, 32), rows(512, 10, 24, 128),
                rows(512, 10, 16, 64), rows(1104, 10, 24, 64), rows(0, 10, 24, 64), rows(496, 1, 24, 24), rows(536, 2, 24, 48)):
        with pytest.raises(ValueError, match="share"):
            ws.require_apart(out, y, "y")
    one = rows(512, 1, 24, 24)
    ws.require_apart(rows(512, 1, 24, 8), one, "y")  # one row: the distance of rows says nothing
    ws.require_apart(rows(536, 1, 24, 8), one, "y")
    with pytest.raises(ValueError, match="share"):
        ws.require_apart(rows(528, 1, 24, 8), one, "y")


@pytest.mark.gpu
def test_results_that_share_a_part_of_what_is_read(cuda_device):
    from execution_ucx_b200.ops import lora, moe
    g = torch.Generator(device=cuda_device).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda_device).to(torch.bfloat16)  # noqa: E731
    ad = lora.LoraAdapters(r(3, 16, 32), r(3, 24, 16))
    layer = moe.MoeExperts(r(4, 128, 64) * 0.1, r(4, 64, 64) * 0.1)
    for t in (5, 600):
        room, x, ids = r(t + 1, 48), r(t, 32), torch.randint(-1, 3, (t,), generator=g, device=cuda_device, dtype=torch.int32)
        y = room[1:, :24]
        want = ad(x, ids, y)
        for bad in (room[:-1, :24], room[1:, 8:32], room.view(-1)[48:].as_strided((t, 24), (24, 1))):
            with pytest.raises(ValueError, match="share"):
                ad(x, ids, y, out=bad)
        assert torch.equal(ad(x, ids, y, out=room[1:, 24:]), want)
        assert torch.equal(ad(x, ids, y, out=room[1:, :24]), want)
    for t in (100, 300):
        room, w = r(t + 1, 128), torch.rand(t, 2, generator=g, device=cuda_device)
        idx = torch.randint(0, 4, (t, 2), generator=g, device=cuda_device, dtype=torch.int32)
        x = room[:-1, :64]
        want = layer(x, idx, w)
        assert torch.equal(layer(x, idx, w, out=room[:-1, 64:]), want)
        if t > layer.MAX_TOKENS:  # a later pass would read what an earlier one wrote
            with pytest.raises(ValueError, match="share"):
                layer(x, idx, w, out=room[1:, :64])
        else:
            assert torch.equal(layer(x.clone(), idx, w), layer(x, idx, w, out=room[1:, :64]))
        room[:-1, :64] = x0 = r(t, 64)
        assert torch.equal(layer(x0, idx, w), layer(room[:-1, :64], idx, w, out=room[:-1, :64]))
    layer.check_status()


@pytest.mark.gpu
def test_calls_refuse(cuda_device):
    from execution_ucx_b200.ops import lora, moe
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device=cuda_device)  # noqa: E731
    layer = moe.MoeExperts(z(2, 32, 16), z(2, 16, 16))
    x, idx, w = z(4, 16), z(4, 2, dt=torch.int32), z(4, 2, dt=torch.float32)
    layer(x, idx, w)
    for args, kw, match in [((x.half(), idx, w), {}, "x must be"), ((z(4, 24), idx, w), {}, "columns"), ((x, idx.long(), w), {}, "topk_idx"), ((x, idx, w.half()), {}, "topk_w"),
                            ((x, idx[:3], w), {}, "topk_idx"), ((x, idx, w[:, :1]), {}, "topk_w"), ((x, z(4, 0, dt=torch.int32), w), {}, "topk"),
                            ((x, z(4, 33, dt=torch.int32), z(4, 33, dt=torch.float32)), {}, "topk"), ((z(16, 4).t(), idx, w), {}, "side by side"), ((z(4, 20)[:, :16], idx, w), {}, "aligned"),
                            ((z(4, 32)[:, 4:20], idx, w), {}, "16 bytes"), ((x, z(2, 4, dt=torch.int32).t(), w), {}, "contiguous"), ((x, idx, w), dict(out=z(3, 16)), "rows"),
                            ((x, idx, w), dict(out=z(1, 16).expand(4, 16)), "apart"), ((x.cpu(), idx, w), {}, "is on"), ((x, idx.cpu(), w), {}, "is on")]:
        with pytest.raises(ValueError, match=match):
            layer(*args, **kw)
    ad = lora.LoraAdapters(z(3, 16, 32), z(3, 24, 16))
    x, ids, y = z(4, 32), z(4, dt=torch.int32), z(4, 24)
    ad(x, ids, y)
    for args, kw, match in [((x.float(), ids, y), {}, "x must be"), ((z(4, 40), ids, y), {}, "columns"), ((x, ids.long(), y), {}, "ids"), ((x, ids[:3], y), {}, "ids"),
                            ((x, ids, z(4, 32)), {}, "columns"), ((x, ids, z(3, 24)), {}, "rows"), ((x, ids, y), dict(out=z(4, 24, dt=torch.float32)), "out"),
                            ((x, z(8, dt=torch.int32)[::2], y), {}, "contiguous"), ((x, ids, y.cpu()), {}, "is on"), ((z(4, 40)[:, 4:36], ids, y), {}, "16 bytes")]:
        with pytest.raises(ValueError, match=match):
            ad(*args, **kw)
