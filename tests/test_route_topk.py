"""Refusals of the routing entry points, checked before any GPU call (CPU)."""
import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from aeo_quant_b200 import _capi
    return _capi.load()


def call(lib, **kw):
    a = dict(logits=None, dtype=0, ld=128, T=4, E=128, k=8, score=0, bias=None, n_group=1, topk_group=1, gs=0,
             renorm=1, scale=1.0, w=None, ids=None)
    a.update(kw)
    return lib.aeoq_route_topk(a["logits"], a["dtype"], a["ld"], a["T"], a["E"], a["k"], a["score"], a["bias"],
                               a["n_group"], a["topk_group"], a["gs"], a["renorm"], a["scale"], a["w"], a["ids"], None)


@pytest.mark.parametrize("bad,msg", [
    (dict(E=0), b"num_experts"), (dict(E=1025, ld=1025), b"num_experts"), (dict(k=0), b"k (0)"),
    (dict(k=33), b"k (33)"), (dict(E=4, ld=4, k=5), b"k (5)"), (dict(n_group=3), b"n_group"),
    (dict(n_group=64), b"n_group"), (dict(n_group=0), b"n_group"), (dict(n_group=8, topk_group=9), b"topk_group"),
    (dict(topk_group=0), b"topk_group"), (dict(score=2), b"bad score"), (dict(gs=2), b"group score"),
    (dict(ld=100), b"bad shape"), (dict(T=-1), b"bad shape"), (dict(), b"null pointer")])
def test_c_entry_refuses(lib, bad, msg):
    assert call(lib, **bad) == -1
    assert msg in lib.aeoq_last_error()


def test_no_tokens_is_no_work(lib):
    assert call(lib, T=0) == 0


def test_python_refusals():
    from aeo_quant_b200 import AeoqError
    from aeo_quant_b200.gpu.routing import route_topk
    l = torch.zeros(2, 16)
    with pytest.raises(AeoqError):
        route_topk(l, 2)                                     # no CPU path
    with pytest.raises(ValueError, match="must be 2D"):
        route_topk(l[0], 2)
    with pytest.raises(ValueError, match="bfloat16, float16 or float32"):
        route_topk(l.double(), 2)
    with pytest.raises(ValueError, match="'softmax' or 'sigmoid'"):
        route_topk(l, 2, score="relu")
    with pytest.raises(ValueError, match="'max' or 'top2'"):
        route_topk(l, 2, group_score="sum")
    with pytest.raises(ValueError, match=r"bias must have shape \(16,\)"):
        route_topk(l, 2, bias=torch.zeros(8))
    with pytest.raises(ValueError, match="bias must be"):
        route_topk(l, 2, bias=torch.zeros(16, dtype=torch.int32))
