"""``route_topk`` against the 64-bit oracle: ids equal, weights within f32 error.

Weight tolerance: a score is one expf (2 ulp), a sum (chains of at most 37
f32 additions) and two quotients, under 4e-6 relative altogether; the
renormalised weight of two such numbers under 8e-6.
"""
import numpy as np
import pytest
import torch

from oracle.route_topk import route_topk as oracle

pytestmark = pytest.mark.gpu
TOL = 8e-6


def check(logits, k, bias=None, **kw):
    from aeo_quant_b200.gpu.routing import route_topk
    w, ids = route_topk(logits, k, bias=bias, **kw)
    T = logits.shape[0]
    assert w.shape == ids.shape == (T, k) and w.dtype == torch.float32 and ids.dtype == torch.int64
    rw, ri = oracle(logits.double().cpu().numpy(), k, bias=None if bias is None else bias.double().cpu().numpy(), **kw)
    assert np.array_equal(ids.cpu().numpy(), ri)
    w = w.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(w), np.isnan(rw))
    ok = ~np.isnan(rw)
    assert np.all(np.abs(w - rw)[ok] <= TOL * np.abs(rw[ok]) + 1e-37)
    return w, ri


def gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,E,k", [(1, 128, 8), (1, 1, 1), (3, 7, 7), (5, 33, 4), (130, 128, 8), (9, 160, 6),
                                   (67, 256, 8), (4, 512, 10), (2, 1000, 32), (3, 1024, 16)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_sizes_and_types(dtype, T, E, k, score):
    l = (torch.randn(T, E, generator=gen(T + E)) * 2).to(dtype).cuda()
    check(l, k, score=score)
    check(l, k, score=score, renormalize=False, scale=2.5)


@pytest.mark.parametrize("E,n_group,topk_group,k", [(256, 8, 4, 8), (64, 8, 3, 6), (160, 8, 3, 6), (96, 32, 5, 4),
                                                    (60, 4, 1, 15), (12, 6, 2, 4), (128, 2, 2, 8), (16, 16, 3, 3)])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_groups(E, n_group, topk_group, k, group_score, with_bias):
    g = gen(E + k)
    l = (torch.randn(70, E, generator=g) * 1.5).cuda()
    b = (torch.randn(E, generator=g) * 0.1).cuda() if with_bias else None
    for score in ("softmax", "sigmoid"):
        check(l, k, bias=b, score=score, n_group=n_group, topk_group=topk_group, group_score=group_score, scale=2.5)


def test_many_rows_with_bias():
    """Enough rows that close choices occur: without the second, 64-bit look
    at them some ids would differ."""
    g = gen(1)
    l = (torch.randn(20000, 256, generator=g) * 1.5).cuda()
    b = (torch.randn(256, generator=g) * 0.05).cuda()
    from aeo_quant_b200.gpu.routing import route_topk
    for score in ("softmax", "sigmoid"):
        w, ids = route_topk(l, 8, score=score, bias=b, n_group=8, topk_group=4, group_score="top2")
        x = l.double()
        s = torch.softmax(x, -1) if score == "softmax" else torch.sigmoid(x)
        c = s + b.double()
        gs = c.view(-1, 8, 32).topk(2, -1).values.sum(-1)
        keep = torch.zeros_like(gs, dtype=torch.bool).scatter_(1, gs.topk(4, -1).indices, True)
        c = c.masked_fill(~keep.repeat_interleave(32, 1), -np.inf)
        v, want = c.sort(dim=-1, descending=True, stable=True)
        assert torch.equal(ids, want[:, :8])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k", [(4096, 128, 8), (5003, 256, 3), (4100, 8, 8), (4097, 512, 1), (4099, 136, 5),
                                   (8193, 256, 3), (16390, 512, 1), (4359, 136, 5),
                                   (4096, 520, 4), (4098, 130, 8)])
def test_many_16_bit_rows(dtype, T, E, k):
    """The row counts at which one thread takes a row: ties, masks, NaN and
    infinite rows among them."""
    from aeo_quant_b200.gpu.routing import route_topk
    inf = float("inf")
    l = (torch.randn(T, E, generator=gen(E)) * 2).to(dtype)
    l[torch.rand(T, E, generator=gen(E + 1)) < 0.05] = -inf
    l[7] = -inf
    l[8, 2:] = -inf
    l[9] = 0.0
    l[10] = -0.0
    l[11, ::2] = -0.0
    l[12, E // 2] = float("nan")
    l[13, E - 1] = inf
    l[14] = -300.0
    l[15, 3:] = torch.finfo(dtype).min
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            w, ids = route_topk(l.cuda(), k, score=score, renormalize=renorm, scale=2.0)
            x = l.double().numpy()
            bad = np.isnan(x).any(1) | (np.isposinf(x).any(1) if score == "softmax" else False)
            order = np.argsort(-np.where(np.isnan(x), -inf, x), 1, kind="stable")[:, :k]
            v = np.take_along_axis(x, order, 1)
            with np.errstate(all="ignore"):
                top = np.where(np.isneginf(x).all(1), 0.0, x.max(1))[:, None]
                s = np.exp(v - top) / np.exp(x - top).sum(1, keepdims=True) if score == "softmax" else 1 / (1 + np.exp(-v))
                s = np.where(np.isneginf(v), 0.0, s)
                if renorm:
                    s = np.where(s.sum(1, keepdims=True) > 0, s / s.sum(1, keepdims=True), 0.0)
            want = np.where(bad[:, None], np.arange(k), np.where(np.isneginf(v), E, order))
            got, w = ids.cpu().numpy(), w.cpu().numpy().astype(np.float64)
            assert np.array_equal(got, want)
            assert np.isnan(w[bad]).all() and not np.isnan(w[~bad]).any()
            assert np.all(np.abs(w - 2 * s)[~bad] <= TOL * 2 * s[~bad] + 1e-37)


def test_ties_go_to_the_lower_index():
    l = torch.zeros(4, 128).cuda()
    _, ids = check(l, 8)
    assert ids[0].tolist() == list(range(8))
    l = torch.randint(0, 3, (200, 128), generator=gen(2)).float().cuda()
    check(l, 8)
    check(l, 8, score="sigmoid", bias=torch.zeros(128).cuda())
    check(l, 6, score="sigmoid", bias=torch.zeros(128).cuda(), n_group=8, topk_group=2, group_score="top2")
    check(l.bfloat16(), 6, score="softmax", n_group=8, topk_group=2, group_score="max")


def test_close_values_are_told_apart_exactly():
    """Choice values one f32 step apart, and equal in f32 but not in 64 bits."""
    E = 64
    l = torch.zeros(8, E)
    l[:, 10], l[:, 50] = 1.0, float(np.nextafter(np.float32(1.0), np.float32(2.0)))
    l[:, 3], l[:, 4] = 8.0, 8.0 + 2.0 ** -20      # sigmoids equal in f32
    l = l.cuda()
    check(l, 4)
    for score in ("softmax", "sigmoid"):
        check(l, 4, score=score, bias=torch.zeros(E).cuda())
        check(l, 4, score=score, bias=torch.full((E,), 0.25).cuda(), n_group=4, topk_group=3, group_score="top2")


def test_masked_infinite_and_nan_rows():
    inf, nan = float("inf"), float("nan")
    g = gen(3)
    l = torch.randn(12, 32, generator=g)
    l[0] = -inf                        # nothing left
    l[1, 3:] = -inf                    # fewer than k left
    l[2, ::2] = -inf
    l[3, 5] = nan
    l[4] = nan
    l[5, 7] = inf
    l[6] = torch.finfo(torch.float32).min
    l[7, :16] = torch.finfo(torch.float32).min
    l[8] = -200.0                      # sigmoids below the f32 range
    l[8, 4] = -190.0
    l[9] = -1000.0
    l[10] = 100.0
    l[11, :] = -inf
    l[11, 31] = -3.0
    for bias in (None, torch.linspace(-0.1, 0.1, 32).cuda()):
        for score in ("softmax", "sigmoid"):
            for kw in (dict(), dict(n_group=4, topk_group=2, group_score="top2"), dict(n_group=4, topk_group=2)):
                check(l.cuda(), 6, bias=bias, score=score, **kw)
    b = torch.zeros(32)
    b[4], b[9] = -inf, inf
    check(l.cuda(), 6, bias=b.cuda(), score="sigmoid")
    b[0] = nan
    w, ids = check(l.cuda(), 6, bias=b.cuda())
    seen = (l[:, 0] != -inf).numpy()   # a masked expert's bias is not looked at
    assert np.isnan(w[seen]).all() and (ids[seen] < 32).all() and not np.isnan(w[~seen]).any()


def test_strides_offsets_and_empty():
    from aeo_quant_b200.gpu.routing import route_topk
    big = torch.randn(40, 300, generator=gen(4)).cuda()
    for l in (big[:, :128], big[:, 1:129], big[::2, 7:71], big.t()[:64], big[3:4, 5:21], big.bfloat16()[:, 3:131]):
        check(l, 4)
    check(big[:1, :16].expand(5, 16), 3)
    w, ids = route_topk(big[:0, :16], 3)
    assert w.shape == ids.shape == (0, 3)


def test_refused_on_gpu():
    from aeo_quant_b200 import AeoqError
    from aeo_quant_b200.gpu.routing import route_topk
    l = torch.zeros(2, 16, device="cuda")
    with pytest.raises(AeoqError, match="CUDA tensors only"):
        route_topk(l, 2, bias=torch.zeros(16))
    for bad in (0, -1, 17):
        with pytest.raises(ValueError, match="route_topk: k"):
            route_topk(l, bad)
    with pytest.raises(ValueError, match="topk_group"):
        route_topk(l, 2, n_group=4, topk_group=5)


def test_streams_and_graph():
    from aeo_quant_b200.gpu.routing import route_topk
    l = torch.randn(64, 128, generator=gen(5)).cuda()
    b = (torch.randn(128, generator=gen(6)) * 0.1).cuda()
    want = route_topk(l, 8, score="sigmoid", bias=b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = route_topk(l, 8, score="sigmoid", bias=b)
    s.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    x = torch.zeros_like(l)
    graph = torch.cuda.CUDAGraph()
    route_topk(x, 8, score="sigmoid", bias=b)
    with torch.cuda.graph(graph):
        out = route_topk(x, 8, score="sigmoid", bias=b)
    for seed in (7, 8):
        y = torch.randn(64, 128, generator=gen(seed)).cuda()
        x.copy_(y)
        graph.replay()
        assert all(torch.equal(a, c) for a, c in zip(out, route_topk(y, 8, score="sigmoid", bias=b)))


@pytest.mark.parametrize("E", [20, 64, 128, 256, 1000])
def test_a_better_expert_behind_equal_ones(E):
    """More equal experts than slots, then one whose score is larger by less
    than f32 holds: it goes first. (A step of f32 at 20 is 2^-19: the sigmoids
    differ by 4e-15.)"""
    up = float(np.nextafter(np.float32(20), np.float32(21)))
    l = torch.full((6, E), 20.0)
    l[0, E - 1] = l[1, E // 2] = l[2, E - 2] = l[2, E - 3] = up
    l[3, : E // 2] = up
    l[4, ::3] = up
    l = l.cuda()
    for k in (1, 3, 8):
        for bias in (torch.zeros(E).cuda(), torch.full((E,), 0.5).cuda()):
            _, ids = check(l, k, score="sigmoid", bias=bias)
            assert ids[0, 0] == E - 1 and ids[1, 0] == E // 2 and ids[2, 0] == E - 3
        check(l, k, score="sigmoid", n_group=4, topk_group=2, group_score="top2")


def test_saturated_scores_keep_the_order_of_their_logits():
    """Sigmoids from about 37 on are 1 in 64 bits, and small scores vanish
    beside a bias: with equal choice values the larger logit goes first, then
    the lower index, so that a bias that is the same for all changes nothing."""
    from aeo_quant_b200.gpu.routing import route_topk
    inf = float("inf")
    for E, low, high in ((8, 2, 5), (64, 1, 40), (256, 3, 4), (1000, 7, 999)):
        l = torch.zeros(1, E)
        l[0, low], l[0, high] = 40.0, 45.0
        l = l.cuda()
        rest = next(e for e in range(E) if e not in (low, high))
        for bias in (None, torch.zeros(E).cuda(), torch.full((E,), 0.25).cuda(), torch.full((E,), inf).cuda()):
            assert route_topk(l, 3, score="sigmoid", bias=bias)[1].tolist() == [[high, low, rest]]
    # groups: the better of two saturated ones, and the sums of their two best
    l = torch.zeros(1, 32)
    l[0, 3], l[0, 9], l[0, 10] = 40.0, 45.0, -5.0
    l = l.cuda()
    for bias in (None, torch.zeros(32).cuda()):
        kw = dict(score="sigmoid", bias=bias, n_group=4, topk_group=1)
        assert route_topk(l, 2, **kw)[1].tolist() == [[9, 8]]
        assert route_topk(l, 2, group_score="top2", **kw)[1].tolist() == [[9, 8]]
    # equal logits still go by index
    l = torch.full((2, 64), 50.0).cuda()
    assert route_topk(l, 4, score="sigmoid", bias=torch.zeros(64).cuda())[1].tolist() == [[0, 1, 2, 3]] * 2


@pytest.mark.parametrize("E,n_group,topk_group,k", [(64, 1, 1, 6), (256, 8, 4, 8), (60, 4, 1, 15), (1000, 1, 1, 32),
                                                    (96, 32, 5, 4)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_a_bias_that_is_the_same_for_all_changes_no_choice(E, n_group, topk_group, k, score):
    from aeo_quant_b200.gpu.routing import route_topk
    l = (torch.randn(500, E, generator=gen(E)) * 30).cuda()
    l[:20] = l[:20].round()                # equal logits among them
    kw = dict(score=score, n_group=n_group, topk_group=topk_group)
    w, ids = route_topk(l, k, **kw)
    for b in (0.0, 0.1):
        check(l, k, bias=torch.full((E,), b).cuda(), **kw)
        w2, ids2 = route_topk(l, k, bias=torch.full((E,), b).cuda(), **kw)
        assert torch.equal(ids, ids2)
    check(l, k, bias=(torch.randn(E, generator=gen(1)) * 0.1).cuda(), **kw)
    check(l, k, bias=torch.zeros(E).cuda(), group_score="top2", **kw)
