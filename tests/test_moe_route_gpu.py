"""The choice of experts against a plain statement in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def plain(logits, topk, scoring="softmax", bias=None, groups=1, topk_groups=1, renormalize=True, scale=1.0):
    """Row by row, with Python's sort: its order of equal keys is the lowest index first."""
    t, e = logits.shape
    idx, w = torch.full((t, topk), -1, dtype=torch.int32), torch.zeros(t, topk, dtype=torch.float64)
    l64 = logits.cpu().double()
    b = bias.cpu().double() if bias is not None else torch.zeros(e, dtype=torch.float64)
    big = torch.finfo(torch.float32).max
    for r in range(t):
        row = l64[r]
        there = [i for i in range(e) if row[i] > -math.inf and b[i] > -math.inf]
        some = row > -math.inf
        v = row.clamp(max=big)
        if scoring == "softmax":
            m = v[some].max() if some.any() else 0.0
            ex = torch.where(some, torch.exp(v - m), 0.0)
            s = ex / ex.sum() if some.any() else ex
        else:
            s = torch.sigmoid(v)
        c = s + b
        if bias is None and groups == 1:
            c = row
        if groups > 1:
            size = e // groups
            inside = [sorted((float(c[i]) for i in there if i // size == g), reverse=True)[:2] for g in range(groups)]
            order = sorted((g for g in range(groups) if inside[g]), key=lambda g: -sum(inside[g]))[:topk_groups]
            there = [i for i in there if i // size in order]
        pick = sorted(there, key=lambda i: -float(c[i]))[:topk]
        for j, i in enumerate(pick):
            idx[r, j], w[r, j] = i, s[i]
        if renormalize and w[r].sum() > 0:
            w[r] /= w[r].sum()
    return idx, w * scale


def check(logits, topk, **kw):
    from execution_ucx_b200.ops import moe
    idx, w = moe.route(logits, topk, **kw)
    want_idx, want_w = plain(logits, topk, **kw)
    assert idx.dtype == torch.int32 and w.dtype == torch.float32 and idx.shape == w.shape == (logits.shape[0], topk)
    assert torch.equal(idx.cpu(), want_idx)
    # exp of a difference that is rounded once (the relative error of exp is the absolute one of its argument, at most 2^-24 of
    # 40 here), two roundings of exp itself, a sum of up to 32 + 5 steps, two divisions and a product, 2^-24 each
    tol = (40 + 2 * 2 + 37 + 4) * 2.0 ** -24
    torch.testing.assert_close(w.cpu().double(), want_w, rtol=tol, atol=1e-30)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,e,topk,dtype", [(1, 256, 8, torch.float32), (5, 8, 2, torch.bfloat16), (3, 1, 1, torch.float32), (7, 33, 32, torch.float32),
                                            (130, 100, 6, torch.bfloat16), (2, 1024, 8, torch.float32), (9, 600, 4, torch.float32), (6, 64, 8, torch.bfloat16)])
def test_choice_without_bias(cuda_device, scoring, t, e, topk, dtype):
    g = torch.Generator().manual_seed(t * 1000 + e)
    logits = (torch.randn(t, e, generator=g) * 3).clamp(-15, 15).to(dtype).to(cuda_device)  # bfloat16 has many equal ones
    check(logits, topk, scoring=scoring)
    check(logits, topk, scoring=scoring, renormalize=False, scale=2.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,e,topk,groups,topk_groups,bias", [(33, 256, 8, 8, 4, True), (4, 256, 8, 8, 1, False), (17, 96, 5, 32, 7, True), (9, 40, 3, 1, 1, True),
                                                              (5, 12, 2, 12, 3, False), (3, 1024, 8, 16, 4, True), (6, 512, 32, 2, 1, True), (8, 20, 4, 5, 5, False)])
def test_choice_with_bias_and_groups(cuda_device, scoring, t, e, topk, groups, topk_groups, bias):
    g = torch.Generator().manual_seed(e + groups)
    logits = (torch.randn(t, e, generator=g) * 2).clamp(-15, 15).to(cuda_device)
    b = (torch.randn(e, generator=g) * 0.1).to(cuda_device) if bias else None
    check(logits, topk, scoring=scoring, bias=b, groups=groups, topk_groups=topk_groups, scale=1.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("groups,topk_groups", [(1, 1), (4, 2), (8, 3)])
@pytest.mark.parametrize("apart", [1e-9, 1e-7, 2e-7, 1e-6, 1e-5, 1e-4])
def test_scores_that_32_bits_cannot_tell_apart(cuda_device, scoring, renormalize, groups, topk_groups, apart):
    g = torch.Generator().manual_seed(int(1e9 * apart) + groups)
    e = 64
    # every expert's score is near another's, and with a bias every group's: the same logits with a bias that is `apart` times a small number
    logits = torch.randn(40, 8, generator=g).repeat(1, e // 8)
    bias = apart * torch.randint(-3, 4, (e,), generator=g).float()
    for order in (torch.arange(e), torch.randperm(e, generator=g)):
        check(logits[:, order].contiguous().to(cuda_device), 6, scoring=scoring, bias=bias.to(cuda_device), groups=groups, topk_groups=topk_groups,
              renormalize=renormalize)


def test_biases_that_cancel_in_a_group(cuda_device):
    # each group of two has the sum of its two scores, of which 32 bits lose all next to 2^20; what is left decides
    g = torch.Generator().manual_seed(3)
    logits = torch.randn(50, 16, generator=g).to(cuda_device)
    bias = torch.tensor([2.0 ** 20, -(2.0 ** 20)] * 8, device=cuda_device)
    check(logits, 2, scoring="sigmoid", bias=bias, groups=8, topk_groups=2)
    bias = torch.tensor([math.inf, 1.0] * 8, device=cuda_device)
    check(logits, 3, scoring="sigmoid", bias=bias, groups=8, topk_groups=2)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("wide", [False, True])
def test_masks_and_values_that_are_no_numbers(cuda_device, scoring, wide):
    """Rows with fewer experts than places, with none, with NaN among them, with the type's lowest value, with zeros of both
    signs (equal, so the lowest index goes first) and with equal scores throughout."""
    inf, nan, low = math.inf, math.nan, torch.finfo(torch.float32).min
    rows = [[-inf] * 8, [1, -inf, nan, -inf, 2, -inf, -inf, -inf], [nan] * 8, [low] * 8, [low, low, 0, low, low, low, 0, low],
            [-0.0, 0.0, -0.0, 0.0, -1, -1, -1, -1], [5] * 8, [-inf, -inf, -inf, -inf, 1, 1, -inf, -inf], [low, 3, -inf, nan, 1, 0, low, 2]]
    logits = torch.tensor(rows, device=cuda_device)
    kw = dict(bias=torch.zeros(8, device=cuda_device), groups=4, topk_groups=3) if wide else {}
    check(logits, 4, scoring=scoring, **kw)
    if wide:
        b = torch.tensor([0, -inf, 0, nan, 0.5, 0, 0, 0], device=cuda_device)
        from execution_ucx_b200.ops import moe
        idx, _ = moe.route(logits, 8, scoring=scoring, bias=b)
        assert not ((idx == 1) | (idx == 3)).any()
        want, _ = plain(logits, 8, scoring=scoring, bias=torch.where(b.isnan(), -inf, b))
        assert torch.equal(idx.cpu(), want)


def test_infinite_logits_share_the_weight(cuda_device):
    from execution_ucx_b200.ops import moe
    logits = torch.tensor([[0, math.inf, 3, math.inf]], device=cuda_device)
    idx, w = moe.route(logits, 3, renormalize=False)
    assert idx.tolist() == [[1, 3, 2]] and w.tolist() == [[0.5, 0.5, 0.0]]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("low", [-90.0, -200.0, -700.0, -800.0, -3e38])
def test_scores_too_small_for_a_number_of_64_bits_have_no_weight(cuda_device, wide, low):
    from execution_ucx_b200.ops import moe
    logits = torch.full((2, 4), low, device=cuda_device)
    logits[1, 2] = 0
    idx, w = moe.route(logits, 2, scoring="sigmoid", bias=torch.zeros(4, device=cuda_device) if wide else None)
    each = 0.5 if low > -745 else 0.0
    assert idx.tolist() == [[0, 1], [2, 0]] and w.cpu().tolist() == [[each, each], [1.0, pytest.approx(2 * math.exp(low), abs=1e-37)]]
    idx, w = moe.route(torch.full((1, 3), -math.inf, device=cuda_device), 2, scoring="sigmoid", bias=torch.zeros(3, device=cuda_device) if wide else None)
    assert idx.tolist() == [[-1, -1]] and w.tolist() == [[0, 0]]


def test_rows_that_lie_apart_and_no_rows(cuda_device):
    from execution_ucx_b200.ops import moe
    wide = torch.randn(11, 50, device=cuda_device)
    check(wide[:, 3:40], 4)
    check(wide[::2, 1:34], 4, scoring="sigmoid", groups=3, topk_groups=2)
    check(wide[:1, 5:30].expand(4, 25), 3)
    idx, w = moe.route(wide[:0], 4)
    assert idx.shape == w.shape == (0, 4)


def test_captured_and_replayed(cuda_device):
    from execution_ucx_b200.ops import moe
    logits = torch.randn(40, 64, device=cuda_device)
    moe.route(logits, 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        idx, w = moe.route(logits, 4)
    for _ in range(3):
        logits.copy_(torch.randn(40, 64, device=cuda_device))
        graph.replay()
        want_idx, want_w = moe.route(logits, 4)
        assert torch.equal(idx, want_idx) and torch.equal(w, want_w)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("wide", [False, True])
def test_weights_far_below_the_largest(cuda_device, scoring, renormalize, wide):
    """Chosen experts whose scores are so far apart that 32 bits have no number for the quotient's parts, but one for the quotient."""
    from execution_ucx_b200.ops import moe
    rows = [[-60, -95, -97, -100], [-88, -91, -120, -150], [0, -20, -80, -102], [-300, -310, -330, -380], [-700, -705, -708, -700], [30, -30, -60, -70], [-89, -89, -89, -89]]
    logits = torch.tensor(rows, dtype=torch.float32, device=cuda_device)
    kw = dict(scoring=scoring, renormalize=renormalize, bias=torch.zeros(4, device=cuda_device) if wide else None)
    idx, w = moe.route(logits, 4, **kw)
    want_idx, want = plain(logits, 4, **kw)
    # in 64 bits but for a softmax's sum (as above: 37 steps, and the exponentials of it are off by 2 * 2^-24), then rounded once, where there
    # may be no more than a subnormal number
    tol = (37 + 2 + 2) * 2.0 ** -24
    assert bool(((w.cpu().double() - want).abs() <= tol * want + 2.0 ** -149).all())
    if wide and scoring == "sigmoid":  # equal scores in 64 bits go by their index
        assert torch.equal(idx.cpu(), want_idx)
