"""CPU checks of the decode step's few-row operators: the C entries refuse bad
arguments before any device work, the wrappers refuse CPU tensors, and the
4-bit quantiser's codes stand for the weights."""

import pytest
import torch

from vllm_ernie_b200 import _lib, ops

P = 256  # a placeholder pointer: nothing is launched


def test_w4_linear_statuses():
    f = _lib.lib().hca_w4_linear
    ok = dict(out=P, os=64, x=P, xs=128, q=P, s=P, z=None, t=1, n=64, k=128, g=64, half=0)

    def status(**change):
        a = {**ok, **change}
        return f(a["out"], a["os"], a["x"], a["xs"], a["q"], a["s"], a["z"], a["t"], a["n"], a["k"], a["g"], a["half"], None)

    assert status(g=16) == -2 and status(g=96) == -2
    assert status(t=0) == 0
    for bad in (dict(t=-1), dict(n=0), dict(k=0), dict(k=96, g=64), dict(out=None), dict(x=None), dict(q=None), dict(s=None),
                dict(x=P + 8), dict(q=P + 4), dict(s=P + 1), dict(out=P + 1), dict(xs=132, t=2)):
        assert status(**bad) == -1, bad


def _moe(f, route=False, **change):
    a = dict(out=P, x=P, xs=128, router=P, ids=P, w=P, fmt=0, g=0, w13=P, s13=None, w2=P, s2=None, sh13=None, sh2=None, t=2, e=8,
             h=128, i=64, si=0, k=2, ws=P, bytes=1 << 20)
    a.update(change)
    weights = (a["w13"], a["s13"], None, a["w2"], a["s2"], None, a["sh13"], None, None, a["sh2"], None, None)
    sizes = (a["t"], a["e"], a["h"], a["i"], a["si"], a["k"], a["ws"], a["bytes"], None)
    if route:
        return f(a["out"], 128, a["x"], a["xs"], a["router"], 0, None, 0, 1, 1.0, None, a["fmt"], a["g"], *weights, *sizes)
    return f(a["out"], 128, a["x"], a["xs"], a["ids"], a["w"], None, a["fmt"], a["g"], *weights, *sizes)


@pytest.mark.parametrize("route", [False, True])
def test_moe_statuses(route):
    lib = _lib.lib()
    f = lib.hca_moe_decode if route else lib.hca_moe_experts
    assert _moe(f, route, t=0) == 0
    for bad in (dict(t=-1), dict(e=0), dict(k=0), dict(i=0), dict(si=-32), dict(w13=None), dict(w2=P + 8), dict(fmt=1),
                dict(fmt=2, g=128, s13=P, s2=P), dict(si=64), dict(ws=None), dict(ws=P + 8), dict(out=None), dict(x=P + 2),
                dict(xs=100)):
        assert _moe(f, route, **bad) == -1, bad
    for bad in (dict(e=513, k=2), dict(k=17, e=20), dict(h=100), dict(i=48), dict(si=16), dict(fmt=3), dict(fmt=2, g=48)):
        assert _moe(f, route, **bad) == -2, bad
    assert _moe(f, route, bytes=100) == -4
    if route:
        assert _moe(f, route, k=9) == -1 and _moe(f, route, router=None) == -1
    else:
        assert _moe(f, route, ids=None) == -1 and _moe(f, route, w=None) == -1


def test_moe_workspace_is_for_one_pass_and_the_routing():
    f = _lib.lib().hca_moe_workspace_bytes
    assert f(0, 64, 8, 4096, 1024, 0) == 0 and f(1, 64, 8, 4096, 0, 0) == 0
    assert f(1, 64, 8, 4096, 1024, 0) >= 8 * 1024 * 2 + 9 * 4096 * 4 + 64 * 4
    # the intermediates of 64 tokens at most, however many tokens follow
    assert f(1000, 64, 8, 4096, 1024, 512) < f(64, 64, 8, 4096, 1024, 512) + 1000 * (64 + 2 * 8) * 4 + 1024


def test_route_statuses():
    f = _lib.lib().hca_moe_route

    def status(ids=P, x=P, xs=128, router=P, t=2, e=8, h=128, k=2, ws=P, size=4096):
        return f(ids, P, x, xs, router, 0, None, None, t, e, h, k, 0, 1, 1.0, ws, size, None)

    assert status(t=0) == 0
    assert [status(ids=None), status(x=P + 8), status(xs=4), status(router=P + 8), status(k=9), status(e=0, k=0),
            status(ws=None), status(ws=P + 8)] == [-1] * 8
    assert status(size=60) == -4
    assert [status(e=600), status(e=20, k=17), status(h=48)] == [-2] * 3


def test_logit_statuses():
    f = _lib.lib().hca_logit_penalties

    def status(logits=P, type=0, index=None, reqs=4, ids=P, lens=P, bias=0, bids=None, rows=4, vocab=100):
        return f(logits, 100, type, index, reqs, ids, 8, 8, lens, lens, None, None, None, bids, bids, bias, bias, None, 0, rows,
                 vocab, None)

    assert status(rows=0) == 0
    assert status(type=3) == -2
    assert [status(logits=None), status(logits=P + 2), status(reqs=3), status(lens=None), status(bias=2), status(rows=-1),
            status(vocab=0)] == [-1] * 7


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros((1, 64), dtype=torch.bfloat16)
    q, s, _ = ops.quantize_weight_w4(torch.zeros((4, 64)), 32)
    with pytest.raises(ValueError):
        ops.w4_linear(x, q, s)
    w = ops.MoEWeights(torch.zeros((2, 64, 64), dtype=torch.bfloat16), torch.zeros((2, 64, 32), dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        ops.moe_decode(x, torch.zeros((2, 64)), w, 1)
    with pytest.raises(ValueError):
        ops.apply_logit_penalties(torch.zeros((1, 8)))


@pytest.mark.parametrize("asymmetric", [False, True])
def test_quantize_weight_w4_codes(asymmetric):
    w = torch.linspace(-1, 2, 2 * 3 * 128).view(2, 3, 128)
    w[0, 0] = 0
    q, s, z = ops.quantize_weight_w4(w, 64, asymmetric, dtype=torch.float16)
    assert q.shape == (2, 3, 64) and s.shape == (2, 3, 2) and s.dtype == torch.float16 and (z is not None) == asymmetric
    codes = torch.stack((q & 15, q >> 4), -1).flatten(-2).float()
    zero = 8.0 if z is None else z.float().repeat_interleave(64, -1)
    step = s.float().repeat_interleave(64, -1)
    assert (((codes - zero) * step - w).abs() <= (0.5 + 15 * 2.0 ** -11) * step + 1e-6).all()
    assert (q[0, 0] == (0 if asymmetric else 0x88)).all()


@pytest.mark.parametrize("group,k", [(48, 96), (64, 96)])
def test_quantize_weight_w4_refuses(group, k):
    with pytest.raises(ValueError):
        ops.quantize_weight_w4(torch.zeros((2, k)), group)
