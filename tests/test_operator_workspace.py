"""The memory of calls that are captured: whose it is, how long it lives, and that it does not grow with the number of captures."""
import contextlib
import gc
import time
import weakref

import pytest
import torch


class Graphs:
    """The native library's side: tokens of graphs that are there, and of those that are gone."""

    def __init__(self):
        self.there, self.gone, self.refuse = [], [], 0

    def eux_graph_hold(self, stream, token):
        if not self.refuse:
            self.there.append(token)
        return self.refuse

    def eux_graphs_gone(self, tokens, most):
        n = min(most, len(self.gone))
        for i in range(n):
            tokens[i] = self.gone.pop()
        return n

    def eux_error_string(self, rc):
        return b"refused"

    def destroy(self, tokens):
        for t in list(tokens):
            self.there.remove(t)
            self.gone.append(t)


@pytest.fixture
def graphs(monkeypatch):
    """CallScratch on the CPU, on one stream that is being captured."""
    from execution_ucx_b200.ops import _native, _workspace as ws
    fake = Graphs()
    monkeypatch.setattr(_native, "load", lambda: fake)
    monkeypatch.setattr(ws, "on_device", lambda index: contextlib.nullcontext(7))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: type("S", (), {"synchronize": lambda self: None})())
    for name, value in (("_cuda_getDevice", 0), ("_cuda_getCurrentRawStream", 7), ("_cuda_isCurrentStreamCapturing", True)):
        monkeypatch.setattr(torch._C, name, lambda *a, value=value: value, raising=False)
    yield fake
    fake.destroy(fake.there)
    ws._collect()


def scratch(words, **kw):
    from execution_ucx_b200.ops import _workspace as ws
    return ws.CallScratch(words, torch.device("cpu", 0), **kw)


def test_words_of_graphs_that_are_gone_are_given_out_again(graphs):
    s = scratch(8)
    first = [s.get(64)[1] for _ in range(s.SLOTS)]
    assert len(set(first)) == s.SLOTS and len(graphs.there) == s.SLOTS
    graphs.destroy(graphs.there[:5])
    again = [s.get(64)[1] for _ in range(5)]
    assert set(again) <= set(first) and len(set(again)) == 5
    for _ in range(100):  # captured anew for one size after another: no more is held than graphs are there
        graphs.destroy(graphs.there[:1])
        assert s.get(64)[1] in first
    from execution_ucx_b200.ops import _workspace as ws
    assert len(ws._held) == s.SLOTS


def test_words_that_a_graph_zeroes_itself_are_not_kept(graphs):
    s = scratch(8)
    for _ in range(s.SLOTS):
        s.get(64)
    gc.collect()
    before = sum(type(o) is torch.Tensor for o in gc.get_objects())
    for _ in range(50):
        s.get(64)
    gc.collect()
    assert sum(type(o) is torch.Tensor for o in gc.get_objects()) == before
    assert len(graphs.there) == s.SLOTS  # nothing of the object's own in the others


def test_an_object_without_words_keeps_nothing(graphs):
    s = scratch(0)
    assert [s.get(64)[1] for _ in range(30)] == [0] * 30
    assert not graphs.there


@pytest.mark.parametrize("words", [0, 8])
def test_memory_of_an_object_lives_as_long_as_the_graphs_that_use_it(graphs, words):
    from execution_ucx_b200.ops import _workspace as ws
    status = torch.zeros(1)
    s = scratch(words, keep=(status,))
    s.get(64), s.get(64)
    there, status = weakref.ref(status), None
    gone = weakref.ref(s)
    s = None
    gc.collect()
    assert gone() is None and there() is not None
    tokens = list(graphs.there)
    graphs.destroy(tokens[:1])
    ws._collect()
    assert there() is not None
    graphs.destroy(tokens[1:])
    ws._collect()
    assert there() is None


def test_a_hold_that_fails_is_an_error_and_loses_nothing(graphs):
    from execution_ucx_b200.ops import _workspace as ws
    s = scratch(8, keep=(torch.zeros(1),))
    graphs.refuse = 100001
    for _ in range(s.SLOTS + 3):
        with pytest.raises(RuntimeError, match="eux_graph_hold"):
            s.get(64)
    assert len(s._spare) == s.SLOTS and not ws._held


def test_the_library_refuses_what_is_no_capture(native_build):
    import ctypes as C
    from execution_ucx_b200.ops import _native
    lib = _native.load()
    assert lib.eux_graphs_gone(None, 4) == 0 and lib.eux_graphs_gone((C.c_uint64 * 4)(), -1) == 0
    assert lib.eux_graph_hold(None, 1) != 0  # no device here, or the stream is not captured


def experts(dev, **kw):
    from execution_ucx_b200.ops import moe
    from test_moe_experts_gpu import routing, weights
    parts = weights(4, 256, 144, False, dev)
    x = torch.randn(12, 256, device=dev).to(torch.bfloat16)
    return moe, parts, (x, *routing(12, 2, 4, dev, 1))


@pytest.mark.gpu
def test_captured_again_and_again(cuda_device):
    from execution_ucx_b200.ops import _workspace as ws
    moe, parts, args = experts(cuda_device)
    layer = moe.MoeExperts(*parts)
    want = layer(*args)
    kept = []
    held = lambda: sum(owner() is layer._scratch for _, _, owner in ws._held.values())  # noqa: E731
    for rnd in range(3 * layer._scratch.SLOTS):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(*args)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        if rnd % 8 == 0:
            kept.append((graph, out))
        del graph, out
        deadline = time.monotonic() + 5  # what is gone is told of by a thread of CUDA's
        while held() > len(kept) and time.monotonic() < deadline:
            time.sleep(0.001)
            ws._collect()
        assert held() == len(kept) and len(layer._scratch._spare) == layer._scratch.SLOTS - len(kept)
    for _ in range(3):
        for graph, out in kept:
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
    layer.check_status()


@pytest.mark.gpu
def test_a_graph_outlives_the_object(cuda_device):
    """The weights are the caller's to keep; what the object made for itself the graph keeps."""
    from execution_ucx_b200.ops import _workspace as ws, lora
    moe, parts, args = experts(cuda_device)
    a, b = (torch.randn(*s, device=cuda_device).to(torch.bfloat16) for s in ((3, 16, 256), (3, 256, 16)))
    ids = torch.randint(-1, 3, (12,), device=cuda_device, dtype=torch.int32)
    layer, adapters = moe.MoeExperts(*parts), lora.LoraAdapters(a, b)  # scales of one, made by the object
    want = adapters(args[0], ids, layer(*args))
    torch.cuda.synchronize()
    before = set(ws._held)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = adapters(args[0], ids, layer(*args))
    held = set(ws._held) - before
    assert len(held) == 2
    del layer, adapters
    gc.collect()
    others = [torch.full((n,), -1, dtype=torch.int32, device=cuda_device) for n in (1, 3, 320, 320 * 16) for _ in range(100)]
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert all(bool((o == -1).all()) for o in others)
    del graph
    deadline = time.monotonic() + 5
    while held & set(ws._held) and time.monotonic() < deadline:
        time.sleep(0.001)
        ws._collect()
    assert not held & set(ws._held)


@pytest.mark.gpu
def test_a_call_that_gave_up_is_told_and_leaves_nothing(cuda_device, monkeypatch):
    """A status word and counts as a kernel leaves them whose wait has run out, here written by hand: told once, when nothing is in flight
    any more, and the calls that follow, captured ones too, are right."""
    moe, parts, args = experts(cuda_device)
    layer = moe.MoeExperts(*parts)
    want = layer(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(*args)
    graph.replay()
    torch.cuda.synchronize()
    layer.check_status()
    layer.status.fill_(1 | 2 << 8)
    layer._scratch._all.fill_(3)
    for _, words, *_ in layer._scratch._of_stream.values():
        words.fill_(5)
    done, whole, zero = [], torch.cuda.synchronize, layer._scratch.reset
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: (done.append("waited"), whole(*a)))
    monkeypatch.setattr(layer._scratch, "reset", lambda: (done.append("zeroed"), zero()))
    with pytest.raises(RuntimeError, match="code=1 where=2"):
        layer.check_status()
    assert done == ["waited", "zeroed"]
    layer.check_status()
    graph.replay()
    assert torch.equal(layer(*args), want) and torch.equal(out, want)
    layer.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("t", [12, 600])
def test_an_object_dropped_while_its_call_on_another_stream_is_under_way(cuda_device, t):
    from execution_ucx_b200.ops import lora
    a, b = (torch.randn(*s, device=cuda_device).to(torch.bfloat16) for s in ((3, 16, 256), (3, 256, 16)))
    x, y = (torch.randn(t, 256, device=cuda_device).to(torch.bfloat16) for _ in range(2))
    ids = torch.randint(-1, 3, (t,), device=cuda_device, dtype=torch.int32)
    want = lora.LoraAdapters(a, b, torch.ones(3, device=cuda_device))(x, ids, y)
    adapters, side = lora.LoraAdapters(a, b), torch.cuda.Stream()  # scales of one, made by the object, on this stream
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # the call's kernels begin some ten milliseconds later
        out = adapters(x, ids, y)
    del adapters
    others = [torch.full((3,), 7.0, device=cuda_device) for _ in range(50)]
    torch.cuda.synchronize()
    assert torch.equal(out, want) and all(bool((o == 7).all()) for o in others)


@pytest.mark.gpu
def test_parameters_that_are_given_other_memory(cuda_device):
    """The object keeps the memory it was given, also where a parameter's ``data`` is set to other memory, as moving a module does."""
    from execution_ucx_b200.ops import lora
    moe, parts, args = experts(cuda_device)
    given = [torch.nn.Parameter(p) for p in parts[:2]]
    a, b = (torch.nn.Parameter(torch.randn(*s, device=cuda_device).to(torch.bfloat16)) for s in ((3, 16, 256), (3, 256, 16)))
    scale = torch.nn.Parameter(torch.rand(3, device=cuda_device))
    ids = torch.randint(-1, 3, (12,), device=cuda_device, dtype=torch.int32)
    layer, adapters = moe.MoeExperts(*given), lora.LoraAdapters(a, b, scale)
    want = adapters(args[0], ids, layer(*args))
    del parts
    for p in (*given, a, b, scale):
        p.data = torch.zeros_like(p)
    others = [torch.full_like(p, 3.0) for p in (*given, a, b, scale) for _ in range(3)]
    assert torch.equal(adapters(args[0], ids, layer(*args)), want)
    assert all(bool((o == 3).all()) for o in others)
    layer.w_down.mul_(2)  # the memory that is used
    got = layer(*args)
    from test_moe_experts_gpu import plain
    want, tol = plain(*args, layer.w_gate_up, layer.w_down)
    assert bool(((got.double() - want).abs() <= tol).all())
    assert not layer.w_down.requires_grad and not got.requires_grad
