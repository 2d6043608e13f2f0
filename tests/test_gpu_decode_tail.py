"""GPU parity of the operators of a decode step after its attention --
``w4_linear``, ``moe_route`` / ``moe_experts`` / ``moe_decode`` and
``apply_logit_penalties`` -- against their definitions in 64 bits.

Tolerances.  A result that is summed in fp32 and rounded once to a type with
unit roundoff u (2^-8 bf16, 2^-11 fp16, as a bound on the relative error of
one rounding) is within ``u |ref| + 2^-24 n S`` of the exact sum, S the sum of
the magnitudes of its n terms; tensor sums may truncate, so 2^-22 stands for
2^-24.  With the offset trick of 4-bit codes a term's magnitude is taken with
|q - z| <= 15.  The experts' gated product is rounded to bf16 in between,
which adds 2^-8 sum_i |W2_i h_i|; its own fp32 error is far below that.
Whole numbers (expert ids, which logits are -inf) have to be equal.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
FP8 = torch.float8_e4m3fn
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -23}


def _ops():
    from vllm_ernie_b200 import ops

    return ops


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _within(got, ref, bound):
    got = got.double()
    assert torch.isfinite(got).all()
    over = (got - ref).abs() - bound
    assert (over <= 0).all(), (over.max().item(), int((over > 0).sum()), got.numel())


# ---------------------------------------------------------------------------
# weights
# ---------------------------------------------------------------------------


def _w4(shape, group, zeros, gen, dtype=torch.bfloat16):
    """(codes, scales, zeros, the weights in 64 bits)."""
    *lead, n, k = shape
    codes = torch.randint(0, 16, shape, generator=gen, device=DEV)
    q = (codes[..., 0::2] + 16 * codes[..., 1::2]).to(torch.uint8)
    s = ((0.5 + torch.rand((*lead, n, k // group), generator=gen, device=DEV)) / (4.6 * math.sqrt(k))).to(dtype)
    z = torch.randint(0, 16, s.shape, generator=gen, device=DEV, dtype=torch.uint8) if zeros else None
    zero = torch.full(s.shape, 8.0, device=DEV, dtype=torch.float64) if z is None else z.double()
    w = (codes.double() - zero.repeat_interleave(group, -1)) * s.double().repeat_interleave(group, -1)
    return q.contiguous(), s, z, w


def _matrix(kind, shape, gen):
    """(data, scales, zeros, 64-bit weights) of a weight format."""
    *lead, n, k = shape
    if kind.startswith("w4"):
        return _w4(shape, int(kind.split("-")[1].rstrip("z")), kind.endswith("z"), gen)
    w = torch.randn(shape, generator=gen, device=DEV) / math.sqrt(k)
    if kind == "bf16":
        w = w.to(torch.bfloat16)
        return w, None, None, w.double()
    s = torch.exp2(torch.randint(-3, 1, (*lead, -(-n // 128), -(-k // 128)), generator=gen, device=DEV).float()) / 37
    full = s.double().repeat_interleave(128, -2).repeat_interleave(128, -1)[..., :n, :k]
    d = (w * 37).to(FP8)
    return d, s, None, d.double() * full


# ---------------------------------------------------------------------------
# 4-bit linear
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens,n,groups,zeros", [
    (1, 1, 1, False),       # one value from one group
    (1, 129, 3, True),      # ragged row tile, fewer groups than warps
    (2, 16, 8, False),
    (8, 257, 9, True),      # a full block of columns
    (9, 100, 16, False),    # second block with one column
    (17, 48, 33, True),
    (32, 1000, 12, False),
    (33, 31, 5, True),      # a second grid column of rows
    (150, 64, 4, False),
])
def test_w4_linear(tokens, n, groups, group, zeros, dtype):
    gen = _gen(tokens * 1000 + n)
    k = groups * group
    x = torch.randn((tokens, k), generator=gen, device=DEV).to(dtype)
    q, s, z, w = _w4((n, k), group, zeros, gen, dtype)
    got = _ops().w4_linear(x, q, s, z)
    assert got.dtype == dtype and got.shape == (tokens, n)
    xd = x.double()
    size = xd.abs() @ (s.double().repeat_interleave(group, 1) * 15).T
    _within(got, xd @ w.T, U[dtype] * (xd @ w.T).abs() + 2.0 ** -22 * k * size + 1e-6)


def test_w4_linear_strided_rows_and_out():
    gen = _gen(5)
    base = torch.randn((6, 520), generator=gen, device=DEV).to(torch.bfloat16)
    x = base[::2, 8:264]  # rows 1040 elements apart, 16 bytes in
    q, s, z, w = _w4((77, 256), 64, True, gen)
    buf = torch.full((3, 90), 7.0, device=DEV, dtype=torch.bfloat16)
    out = buf[:, 5:82]
    got = _ops().w4_linear(x, q, s, z, out=out)
    assert got is out
    assert torch.equal(out, _ops().w4_linear(x.contiguous(), q, s, z))
    assert (buf[:, :5] == 7).all() and (buf[:, 82:] == 7).all()


def test_w4_linear_keeps_a_rows_values_to_itself():
    """NaN and infinity in one row of x reach that row's results only."""
    gen = _gen(6)
    x = torch.randn((5, 128), generator=gen, device=DEV).to(torch.bfloat16)
    q, s, _, _ = _w4((40, 128), 32, False, gen)
    clean = _ops().w4_linear(x, q, s)
    bad = x.clone()
    bad[1, 3], bad[3, 100] = math.nan, math.inf
    got = _ops().w4_linear(bad, q, s)
    assert torch.isnan(got[1]).all()
    assert torch.equal(got[[0, 2, 4]], clean[[0, 2, 4]])


def test_w4_linear_same_bits_each_time_and_on_another_stream():
    gen = _gen(7)
    x = torch.randn((12, 1024), generator=gen, device=DEV).to(torch.float16)
    q, s, z, _ = _w4((500, 1024), 128, True, gen, torch.float16)
    first = _ops().w4_linear(x, q, s, z)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        other = _ops().w4_linear(x, q, s, z)
        torch.cuda.current_stream().synchronize()
    assert torch.equal(first, other)


@pytest.mark.parametrize("asymmetric", [False, True])
@pytest.mark.parametrize("group", [32, 128])
def test_quantize_weight_w4_is_within_half_a_step(group, asymmetric):
    ops = _ops()
    w = torch.randn((3, 50, 256), generator=_gen(8), device=DEV) + (0.5 if asymmetric else 0.0)
    w[0, 0] = 0
    q, s, z = ops.quantize_weight_w4(w, group, asymmetric)
    assert q.shape == (3, 50, 128) and s.shape == (3, 50, 256 // group)
    eye = torch.eye(256, device=DEV, dtype=torch.bfloat16)
    for e in range(3):
        back = ops.w4_linear(eye, q[e], s[e], None if z is None else z[e]).T.float()
        step = s[e].float().repeat_interleave(group, 1)
        # half a step, the bf16 scale's rounding at the range's end (7 or 15
        # steps), and the result's own
        assert ((back - w[e]).abs() <= (0.5 + 15 * 2.0 ** -8) * step + 2.0 ** -8 * back.abs() + 1e-6).all()


@pytest.mark.parametrize("change", ["cpu", "type", "group", "short", "strided", "misaligned", "scales", "zeros", "out"])
def test_w4_linear_refuses(change):
    x = torch.randn((2, 256), device=DEV).to(torch.bfloat16)
    q, s, z, _ = _w4((10, 256), 64, True, _gen(9))
    out = None
    if change == "cpu":
        q = q.cpu()
    elif change == "type":
        x = x.float()
    elif change == "group":
        s = torch.ones((10, 16), device=DEV, dtype=torch.bfloat16)
        z = None
    elif change == "short":
        q = q[:, :-1].contiguous()
    elif change == "strided":
        q = q.T.contiguous().T
    elif change == "misaligned":
        x = torch.randn((2, 257), device=DEV).to(torch.bfloat16)[:, 1:]
    elif change == "scales":
        s = s.half()
    elif change == "zeros":
        z = z.int()
    elif change == "out":
        out = torch.empty((2, 11), device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        _ops().w4_linear(x, q, s, z, out=out)


# ---------------------------------------------------------------------------
# router
# ---------------------------------------------------------------------------


def _route_ref(x, wr, k, score, bias, renormalize, scale):
    logits = x.double() @ wr.double().T
    p = torch.softmax(logits, 1) if score == "softmax" else torch.sigmoid(logits)
    by = p if bias is None else p + bias.double()
    ids = torch.sort(by, dim=1, descending=True, stable=True).indices[:, :k]
    w = torch.gather(p, 1, ids)
    if renormalize:
        w = w / w.sum(1, keepdim=True)
    return ids.int(), w * scale, by


@pytest.mark.parametrize("score,renormalize,with_bias,router", [
    ("softmax", True, False, torch.bfloat16), ("softmax", False, True, torch.float32),
    ("sigmoid", True, True, torch.float32), ("sigmoid", False, False, torch.bfloat16)])
@pytest.mark.parametrize("tokens,experts,k,hidden", [
    (1, 1, 1, 32), (1, 8, 8, 64), (2, 33, 5, 2080), (3, 64, 6, 4096), (7, 9, 2, 96), (8, 512, 16, 512), (64, 128, 8, 1024),
    (100, 60, 4, 256)])
def test_moe_route(tokens, experts, k, hidden, score, renormalize, with_bias, router):
    gen = _gen(tokens + experts)
    x = torch.randn((tokens, hidden), generator=gen, device=DEV).to(torch.bfloat16)
    wr = (torch.randn((experts, hidden), generator=gen, device=DEV) * 1.5 / math.sqrt(hidden)).to(router)
    bias = torch.randn(experts, generator=gen, device=DEV) * 0.2 if with_bias else None
    ids, weights = _ops().moe_route(x, wr, k, score=score, router_bias=bias, renormalize=renormalize, routed_scale=2.5)
    ref_ids, ref_w, by = _route_ref(x, wr, k, score, bias, renormalize, 2.5)
    # an id may differ only where the two experts' scores are a rounding apart
    gap = (torch.gather(by, 1, ids.long()) - torch.gather(by, 1, ref_ids.long())).abs()
    assert (gap <= 1e-5).all() and (ids != ref_ids).double().mean() <= 0.01
    same = ids == ref_ids
    assert ((weights.double() - ref_w).abs() <= 2e-5 * ref_w.abs() + 1e-7)[same].all()


def test_moe_route_ties_go_to_the_lower_expert():
    x = torch.ones((3, 64), device=DEV, dtype=torch.bfloat16)
    wr = torch.zeros((70, 64), device=DEV)
    wr[[5, 40, 41, 69]] = 0.125
    ids, w = _ops().moe_route(x, wr, 6)
    assert ids.tolist() == [[5, 40, 41, 69, 0, 1]] * 3
    bias = torch.zeros(70, device=DEV)
    bias[7] = -0.0
    ids, _ = _ops().moe_route(torch.zeros_like(x), wr, 4, score="sigmoid", router_bias=bias)
    assert ids.tolist() == [[0, 1, 2, 3]] * 3


def test_moe_route_extreme_logits():
    ops = _ops()
    wr = torch.zeros((16, 32), device=DEV)
    wr[3, 0], wr[9, 0], wr[4, 1] = 1e4, 1e4, math.nan
    x = torch.zeros((4, 32), device=DEV, dtype=torch.bfloat16)
    x[0, 0], x[1, 0], x[2, 2] = 100.0, -100.0, math.nan
    ids, w = ops.moe_route(x, wr, 3, score="sigmoid")
    # rows of x times expert 4's NaN are NaN: that expert is chosen last
    assert ids[0].tolist() == [3, 9, 0] and 4 not in ids[1].tolist()
    assert ids[2].tolist() == [0, 1, 2]  # all NaN: every expert ties
    assert ((ids >= 0) & (ids < 16)).all()
    low = torch.full((16, 32), -1e4, device=DEV)
    ids, w = ops.moe_route(torch.ones_like(x), low, 3, score="sigmoid")  # every score underflows to 0
    assert ids.tolist() == [[0, 1, 2]] * 4 and (w == 0).all()


def test_moe_route_mask():
    x = torch.randn((11, 256), generator=_gen(3), device=DEV).to(torch.bfloat16)
    wr = torch.randn((20, 256), generator=_gen(4), device=DEV)
    mask = torch.tensor([1, 0, 1, 1, 0, 0, 1, 1, 1, 0, 1], device=DEV, dtype=torch.bool)
    ids, w = _ops().moe_route(x, wr, 4)
    got, gw = _ops().moe_route(x, wr, 4, token_mask=mask)
    assert torch.equal(got[mask], ids[mask]) and torch.equal(gw[mask], w[mask])
    assert (got[~mask] == -1).all() and (gw[~mask] == 0).all()


# ---------------------------------------------------------------------------
# experts
# ---------------------------------------------------------------------------

FORMATS = ["bf16", "fp8", "w4-32", "w4-64z", "w4-128"]


def _stack(kind, lead, hidden, inner, gen):
    d13, s13, z13, w13 = _matrix(kind, (*lead, 2 * inner, hidden), gen)
    d2, s2, z2, w2 = _matrix(kind, (*lead, hidden, inner), gen)
    return _ops().MoEWeights(d13, d2, s13, s2, z13, z2), w13, w2


def _expert_ref(x, w13, w2, weight):
    """(y, the size of its bf16 rounding of h) of rows x with weights [rows]."""
    gate, up = (x @ w13.T).chunk(2, -1)
    h = gate * torch.sigmoid(gate) * up * weight.unsqueeze(1)
    return h @ w2.T, h.abs() @ w2.abs().T


def _experts_ref(x, ids, weights, w13, w2, mask=None, shared=None):
    x, weights = x.double(), weights.double()
    y, size = torch.zeros_like(x), torch.zeros_like(x)
    if mask is not None:
        x = torch.where(mask.unsqueeze(1), x, 0.0)
    for e in range(w13.shape[0]):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if t.numel():
            a, b = _expert_ref(x[t], w13[e], w2[e], weights[t, j])
            y.index_add_(0, t, a)
            size.index_add_(0, t, b)
    if shared is not None:
        a, b = _expert_ref(x, *shared, torch.ones(x.shape[0], device=DEV, dtype=torch.float64))
        y, size = y + a, size + b
    if mask is not None:
        y, size = (torch.where(mask.unsqueeze(1), v, 0.0) for v in (y, size))
    return y, size


def _moe_bound(ref, size, terms):
    # one rounding of the result, one of h, and fp32 sums of both products
    return 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -22 * terms) * size + 1e-6


@pytest.mark.parametrize("kind", FORMATS)
@pytest.mark.parametrize("tokens,experts,k,hidden,inner,shared", [
    (1, 1, 1, 128, 128, 0),
    (1, 16, 4, 256, 128, 256),
    (3, 7, 2, 384, 256, 0),
    (8, 40, 8, 512, 128, 128),
    (9, 3, 3, 256, 384, 0),       # every expert gets every token: two blocks
    (31, 20, 5, 256, 128, 128),
    (9, 2, 1, 256, 1536, 0),      # the products' warps grouped differently, groups without a tile
    (1, 1, 1, 256, 512, 0),
    (64, 4, 3, 128, 256, 128),    # far more tokens an expert than columns
    (70, 33, 2, 256, 128, 0),     # a second pass with six tokens
])
def test_moe_experts(tokens, experts, k, hidden, inner, shared, kind):
    gen = _gen(tokens * 31 + experts)
    x = torch.randn((tokens, hidden), generator=gen, device=DEV).to(torch.bfloat16)
    stack, w13, w2 = _stack(kind, (experts,), hidden, inner, gen)
    ids = torch.rand((tokens, experts), generator=gen, device=DEV).argsort(1)[:, :k].int().contiguous()
    weights = torch.rand((tokens, k), generator=gen, device=DEV) * 2 - 0.5
    one, ref_shared = None, None
    if shared:
        one, a, b = _stack(kind, (), hidden, shared, gen)
        ref_shared = (a, b)
    got = _ops().moe_experts(x, ids, weights, stack, shared=one)
    ref, size = _experts_ref(x, ids, weights, w13, w2, shared=ref_shared)
    _within(got, ref, _moe_bound(ref, size, hidden + k * inner + shared))


@pytest.mark.parametrize("kind", ["bf16", "fp8", "w4-32"])
@pytest.mark.parametrize("hidden,inner,shared", [(32, 32, 0), (2080, 736, 96), (96, 160, 32), (4096, 32, 4096)])
def test_moe_experts_odd_sizes(hidden, inner, shared, kind):
    """Multiples of 32 that end inside a 64-wide piece, a 128-wide block or a
    warp's share."""
    gen = _gen(hidden + inner)
    x = torch.randn((5, hidden), generator=gen, device=DEV).to(torch.bfloat16)
    stack, w13, w2 = _stack(kind, (6,), hidden, inner, gen)
    one, a, b = _stack(kind, (), hidden, shared, gen) if shared else (None, None, None)
    ids = torch.randint(0, 6, (5, 3), generator=gen, device=DEV, dtype=torch.int32)
    weights = torch.rand((5, 3), generator=gen, device=DEV)
    got = _ops().moe_experts(x, ids, weights, stack, shared=one)
    ref, size = _experts_ref(x, ids, weights, w13, w2, shared=(a, b) if shared else None)
    _within(got, ref, _moe_bound(ref, size, hidden + 3 * inner + shared))


def test_moe_experts_skipped_repeated_and_all_alike():
    """Ids of other ranks are skipped; an id may repeat in a row; all tokens may
    choose one expert (more pairs than any block holds)."""
    ops, gen = _ops(), _gen(11)
    x = torch.randn((64, 128), generator=gen, device=DEV).to(torch.bfloat16)
    stack, w13, w2 = _stack("bf16", (5,), 128, 64, gen)
    weights = torch.rand((64, 16), generator=gen, device=DEV)
    ids = torch.randint(-3, 9, (64, 16), generator=gen, device=DEV, dtype=torch.int32)
    ids[0], ids[1] = -1, 2 ** 31 - 1  # rows with nothing
    for i in (ids, torch.full_like(ids, 4), torch.full_like(ids, 5)):
        got = ops.moe_experts(x, i, weights, stack)
        ref, size = _experts_ref(x, i, weights, w13, w2)
        _within(got, ref, _moe_bound(ref, size, 128 + 16 * 64))
    assert (ops.moe_experts(x, torch.full_like(ids, 5), weights, stack) == 0).all()


@pytest.mark.parametrize("tokens", [1, 6, 40])
def test_moe_masked_rows_are_zero_whatever_they_hold(tokens):
    ops, gen = _ops(), _gen(12)
    x = torch.randn((tokens, 256), generator=gen, device=DEV).to(torch.bfloat16)
    wr = torch.randn((12, 256), generator=gen, device=DEV).to(torch.bfloat16)
    stack, w13, w2 = _stack("fp8", (12,), 256, 128, gen)
    shared, a, b = _stack("fp8", (), 256, 128, gen)
    mask = torch.arange(tokens, device=DEV) % 3 != 0
    ids, weights = ops.moe_route(x, wr, 3)
    ref, size = _experts_ref(x, ids, weights, w13, w2, mask=mask, shared=(a, b))
    bad = torch.where(mask.unsqueeze(1), x, math.nan)
    got = ops.moe_decode(bad, wr, stack, 3, shared=shared, token_mask=mask)
    _within(got, ref, _moe_bound(ref, size, 256 + 4 * 128))
    assert (got[~mask] == 0).all()
    got = ops.moe_decode(bad, wr, stack, 3, shared=shared, token_mask=torch.zeros_like(mask))
    assert (got == 0).all()


def test_moe_nan_stays_in_its_token():
    ops, gen = _ops(), _gen(13)
    x = torch.randn((9, 256), generator=gen, device=DEV).to(torch.bfloat16)
    wr = torch.randn((12, 256), generator=gen, device=DEV)
    stack, w13, w2 = _stack("bf16", (12,), 256, 96, gen)
    ref, size = _experts_ref(x, *ops.moe_route(x, wr, 4), w13, w2)
    bad = x.clone()
    bad[4, 17] = math.nan
    got = ops.moe_decode(bad, wr, stack, 4)
    keep = [t for t in range(9) if t != 4]
    assert torch.isnan(got[4]).all()
    _within(got[keep], ref[keep], _moe_bound(ref, size, 256 + 4 * 96)[keep])


@pytest.mark.parametrize("kind", FORMATS)
@pytest.mark.parametrize("tokens", [1, 5, 64, 65])
def test_moe_decode_is_route_then_experts(tokens, kind):
    ops, gen = _ops(), _gen(14)
    base = torch.randn((tokens, 600), generator=gen, device=DEV).to(torch.bfloat16)
    x = base[:, 40:552]  # strided rows
    wr = torch.randn((24, 512), generator=gen, device=DEV) * 0.1
    bias = torch.randn(24, generator=gen, device=DEV) * 0.1
    stack, _, _ = _stack(kind, (24,), 512, 128, gen)
    shared, _, _ = _stack(kind, (), 512, 256, gen)
    mask = torch.rand(tokens, generator=gen, device=DEV) < 0.8
    how = dict(score="sigmoid", router_bias=bias, routed_scale=2.5, token_mask=mask)
    ids, weights = ops.moe_route(x, wr, 4, **how)
    buf = torch.full((tokens, 530), 3.0, device=DEV, dtype=torch.bfloat16)
    got = ops.moe_decode(x, wr, stack, 4, shared=shared, out=buf[:, 9:521], **how)
    assert torch.equal(got, ops.moe_experts(x, ids, weights, stack, shared=shared, token_mask=mask))
    assert (buf[:, :9] == 3).all() and (buf[:, 521:] == 3).all()


def test_moe_decode_in_a_graph_and_on_two_streams():
    ops, gen = _ops(), _gen(15)
    x = torch.randn((4, 512), generator=gen, device=DEV).to(torch.bfloat16)
    wr = torch.randn((16, 512), generator=gen, device=DEV)
    stack, _, _ = _stack("w4-64z", (16,), 512, 256, gen)
    first = ops.moe_decode(x, wr, stack, 2)
    other = ops.moe_decode(x.flip(0).contiguous(), wr, stack, 2)
    torch.cuda.synchronize()
    graph, held = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        y = ops.moe_decode(held, wr, stack, 2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, first)
    held.copy_(x.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, other)
    streams, flipped, got = [torch.cuda.Stream() for _ in range(2)], x.flip(0).contiguous(), []
    torch.cuda.synchronize()
    for _ in range(20):
        for s, v in zip(streams, (x, flipped)):
            with torch.cuda.stream(s):
                got.append(ops.moe_decode(v, wr, stack, 2))
    torch.cuda.synchronize()
    for i, v in enumerate(got):
        assert torch.equal(v, first if i % 2 == 0 else other)


@pytest.mark.parametrize("change", ["type", "format", "scales", "no_scales", "extra_scales", "zeros", "inner", "shared_format", "mask",
                                    "top_k", "score", "router", "bias", "out", "strided"])
def test_moe_refuses(change):
    ops, gen = _ops(), _gen(16)
    x = torch.randn((3, 128), generator=gen, device=DEV).to(torch.bfloat16)
    wr = torch.randn((8, 128), generator=gen, device=DEV)
    w, _, _ = _stack("fp8", (8,), 128, 64, gen)
    shared, _, _ = _stack("fp8", (), 128, 64, gen)
    top_k, how = 2, {}
    if change == "type":
        x = x.float()
    elif change == "format":
        w = w._replace(w2=w.w2.to(torch.bfloat16))
    elif change == "scales":
        w = w._replace(s13=w.s13[:, :, :0])
    elif change == "no_scales":
        w = w._replace(s2=None)
    elif change == "extra_scales":
        w = _stack("bf16", (8,), 128, 64, gen)[0]._replace(s13=w.s13)
        shared = None
    elif change == "zeros":
        w = w._replace(z13=torch.zeros((8, 128, 1), device=DEV, dtype=torch.uint8))
    elif change == "inner":
        w = w._replace(w2=w.w2[:, :, :32].contiguous())
    elif change == "shared_format":
        shared = _stack("bf16", (), 128, 64, gen)[0]
    elif change == "mask":
        how["token_mask"] = torch.ones(4, device=DEV, dtype=torch.bool)
    elif change == "top_k":
        top_k = 9
    elif change == "score":
        how["score"] = "tanh"
    elif change == "router":
        wr = wr[:, :64].contiguous()
    elif change == "bias":
        how["router_bias"] = torch.zeros(8, device=DEV, dtype=torch.bfloat16)
    elif change == "out":
        how["out"] = torch.empty((3, 128), device=DEV)
    elif change == "strided":
        w = w._replace(w2=w.w2.transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(ValueError):
        ops.moe_decode(x, wr, w, top_k, shared=shared, **how)


def test_moe_refuses_sizes_that_are_not_built():
    from vllm_ernie_b200 import HcaError

    ops, gen = _ops(), _gen(17)
    x = torch.randn((2, 48), generator=gen, device=DEV).to(torch.bfloat16)
    w, _, _ = _stack("bf16", (4,), 48, 32, gen)
    with pytest.raises(HcaError) as e:
        ops.moe_decode(x, torch.randn((4, 48), device=DEV), w, 2)
    assert e.value.status == -2
    x = torch.randn((2, 32), generator=gen, device=DEV).to(torch.bfloat16)
    with pytest.raises(HcaError) as e:
        ops.moe_route(x, torch.randn((600, 32), device=DEV), 2)
    assert e.value.status == -2


def test_empty_batches():
    ops, gen = _ops(), _gen(18)
    w, _, _ = _stack("bf16", (4,), 64, 32, gen)
    x = torch.empty((0, 64), device=DEV, dtype=torch.bfloat16)
    wr = torch.randn((4, 64), device=DEV)
    assert ops.moe_decode(x, wr, w, 2).shape == (0, 64)
    assert ops.moe_route(x, wr, 2)[0].shape == (0, 2)
    q, s, _, _ = _w4((10, 64), 32, False, gen)
    assert ops.w4_linear(x, q, s).shape == (0, 10)
    assert ops.apply_logit_penalties(torch.empty((0, 50), device=DEV)).shape == (0, 50)


# ---------------------------------------------------------------------------
# logits
# ---------------------------------------------------------------------------


def _logits_ref(x, ids, prompt, seq, rep, freq, pres, bias_ids, bias_values, allowed, index):
    """The definition row by row in 64 bits, and the size of what it adds."""
    y, size = x.double().clone(), x.double().abs()
    v = x.shape[1]
    for r in range(x.shape[0]):
        q = r if index is None else int(index[r])
        tables = [t for t in (ids, rep, bias_ids) if t is not None]
        if index is not None and not 0 <= q < tables[0].shape[0]:
            continue
        if bias_ids is not None:
            for i, b in zip(bias_ids[q].tolist(), bias_values[q].tolist()):
                if 0 <= i < v:
                    y[r, i] = float(x[r, i]) + b
                    size[r, i] = abs(float(x[r, i])) + abs(b)
        if ids is not None:
            n = min(int(seq[r]), ids.shape[1])
            t = ids[q, :n].long()
            at = torch.arange(n, device=DEV)
            answer, t_all = t[(at >= int(prompt[r])) & (t >= 0) & (t < v)], t[(t >= 0) & (t < v)]
            seen = torch.zeros(v, dtype=torch.bool, device=DEV)
            seen[t_all] = True
            count = torch.bincount(answer, minlength=v).double()
            if rep is not None:
                p = float(rep[q])
                y[r] = torch.where(seen, torch.where(y[r] > 0, y[r] / p, y[r] * p), y[r])
                size[r] *= max(p, 1 / p)
            if freq is not None:
                y[r] -= float(freq[q]) * count
                size[r] += abs(float(freq[q])) * count
            if pres is not None:
                y[r] -= float(pres[q]) * (count > 0)
                size[r] += abs(float(pres[q]))
        if allowed is not None:
            bits = torch.arange(v, device=DEV)
            y[r][(allowed[r, bits // 32] >> (bits % 32)) & 1 == 0] = -math.inf
    return y, size


def _check_logits(got, ref, size, dtype):
    inf = torch.isinf(ref)
    assert torch.equal(torch.isinf(got) & (got < 0), inf & (ref < 0))
    # four fp32 operations and one rounding of the result
    bound = U[dtype] * ref.abs() + 4 * 2.0 ** -24 * size + 1e-9
    _within(torch.where(inf, 0.0, got.double()), torch.where(inf, 0.0, ref), torch.where(inf, 0.0, bound))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab,length,bias,mask", [
    (1, 1, 1, 0, False),
    (1, 31, 40, 3, True),
    (3, 1000, 0, 5, False),       # no history
    (2, 32000, 300, 0, False),
    (5, 50257, 5000, 17, True),
    (2, 262147, 1000, 40, True),  # two slices' worth with biases
    (1, 600011, 9000, 0, False),  # more than the cluster's counts hold
    (40, 129281, 700, 0, True),
])
def test_logit_penalties(rows, vocab, length, bias, mask, dtype):
    gen = _gen(rows + vocab)
    x = (torch.randn((rows, vocab), generator=gen, device=DEV) * 4).to(dtype)
    rand = lambda *s: torch.rand(s, generator=gen, device=DEV)  # noqa: E731
    # the ends of every slice are hit, and ids outside the vocabulary
    ids = torch.cat([(rand(rows, length) ** 2 * vocab).int(), torch.tensor([[-1, vocab, vocab - 1, 0, 2 ** 31 - 1]], device=DEV)
                     .int().expand(rows, 5)], 1)[:, torch.randperm(length + 5, generator=gen, device=DEV)].contiguous()
    seq = (rand(rows) * (length + 7)).int()  # some past the table's width
    prompt = (seq * rand(rows)).int()
    seq[0], prompt[-1] = 2 ** 31 - 1, 0
    rep, freq, pres = 0.5 + rand(rows), rand(rows) - 0.3, rand(rows) - 0.3
    bias_ids = (torch.rand((rows, vocab), generator=gen, device=DEV).argsort(1)[:, :bias].int().contiguous() if bias else None)
    bias_values = rand(rows, bias) * 6 - 3 if bias else None
    if bias:
        bias_ids[0, 0] = -1
        bias_ids[-1, -1] = vocab
    allowed = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=gen, device=DEV).int() if mask else None
    ref, size = _logits_ref(x, ids, prompt, seq, rep, freq, pres, bias_ids, bias_values, allowed, None)
    got = _ops().apply_logit_penalties(x, ids, prompt, seq, repetition=rep, frequency=freq, presence=pres, bias_ids=bias_ids,
                                       bias_values=bias_values, allowed_bitmask=allowed)
    assert got.data_ptr() == x.data_ptr()
    _check_logits(x, ref, size, dtype)


def test_logit_penalties_draft_rows_share_a_request():
    """Rows of one request with lengths of their own; rows outside the requests stay."""
    gen = _gen(21)
    x = torch.randn((8, 999), generator=gen, device=DEV)
    ids = torch.randint(0, 999, (3, 64), generator=gen, device=DEV, dtype=torch.int32)
    index = torch.tensor([0, 0, 0, 2, 2, -1, 1, 3], device=DEV, dtype=torch.int32)
    seq = torch.tensor([10, 11, 12, 64, 63, 20, 0, 9], device=DEV, dtype=torch.int32)
    prompt = torch.tensor([4, 4, 4, 64, 0, 3, 0, 1], device=DEV, dtype=torch.int32)
    rep, freq = torch.tensor([1.3, 0.7, 2.0], device=DEV), torch.tensor([0.5, -0.5, 0.1], device=DEV)
    pres = torch.tensor([0.2, 0.0, -1.0], device=DEV)
    before = x.clone()
    ref, size = _logits_ref(x, ids, prompt, seq, rep, freq, pres, None, None, None, index)
    _ops().apply_logit_penalties(x, ids, prompt, seq, repetition=rep, frequency=freq, presence=pres, req_index=index)
    _check_logits(x, ref, size, torch.float32)
    assert torch.equal(x[[5, 6, 7]], before[[5, 6, 7]])


def test_logit_penalties_special_values():
    """Infinities and NaN go through the arithmetic; a masked place is -inf
    whatever it held; a row whose mask leaves nothing is all -inf; of an id
    listed twice the later bias counts."""
    x = torch.zeros((2, 70), device=DEV)
    x[0, 0], x[0, 1], x[0, 2], x[0, 3], x[0, 69] = math.nan, math.inf, -math.inf, 2.0, math.nan
    ids = torch.tensor([[0, 1, 2, 3, 3, 69], [0, 1, 2, 3, 3, 69]], device=DEV, dtype=torch.int32)
    lens = lambda a: torch.full((2,), a, device=DEV, dtype=torch.int32)  # noqa: E731
    two = lambda a: torch.full((2,), a, device=DEV)  # noqa: E731
    allowed = torch.full((2, 3), -1, device=DEV, dtype=torch.int32)
    allowed[0, 2], allowed[1] = 0, 0
    bias_ids = torch.tensor([[3, 5, 3], [1, -1, 70]], device=DEV, dtype=torch.int32)
    bias_values = torch.tensor([[100.0, 1.0, 2.0], [math.inf, 1.0, 1.0]], device=DEV)
    _ops().apply_logit_penalties(x, ids, lens(1), lens(6), repetition=two(2.0), frequency=two(0.25), presence=two(0.5),
                                 bias_ids=bias_ids, bias_values=bias_values, allowed_bitmask=allowed)
    assert math.isnan(x[0, 0]) and x[0, 1] == math.inf and x[0, 2] == -math.inf
    assert x[0, 3] == (2.0 + 2.0) / 2 - 0.25 * 2 - 0.5 and x[0, 5] == 1.0
    assert (x[0, 64:] == -math.inf).all() and (x[0, 6:64] == 0).all()
    assert (x[1] == -math.inf).all()


def test_logit_penalties_each_part_alone_and_strided_rows():
    ops, gen = _ops(), _gen(22)
    wide = torch.randn((4, 1203), generator=gen, device=DEV).to(torch.bfloat16)
    table = torch.randint(0, 1001, (4, 90), generator=gen, device=DEV, dtype=torch.int32)
    ids = table[:, 7:57]
    seq, prompt = (torch.full((4,), n, device=DEV, dtype=torch.int32) for n in (50, 20))
    part = torch.full((4,), 1.25, device=DEV)
    words = torch.randint(-2 ** 31, 2 ** 31, (4, 40), generator=gen, device=DEV).int()
    bias_ids = torch.arange(12, device=DEV, dtype=torch.int32).view(4, 3).contiguous()
    bias_values = torch.ones((4, 3), device=DEV)
    for how in ({"repetition": part}, {"frequency": part}, {"presence": part}, {"allowed_bitmask": words[:, 3:35]},
                {"bias_ids": bias_ids, "bias_values": bias_values}, {}):
        buf = wide.clone()
        x = buf[:, 101:1102]
        history = () if "allowed_bitmask" in how or "bias_ids" in how else (ids, prompt, seq)
        a = (*history, None, None, None)[:3]
        ref, size = _logits_ref(x, *a, how.get("repetition"), how.get("frequency"), how.get("presence"), how.get("bias_ids"),
                                how.get("bias_values"), how.get("allowed_bitmask"), None)
        ops.apply_logit_penalties(x, *history, **how)
        _check_logits(x, ref, size, torch.bfloat16)
        assert torch.equal(buf[:, :101], wide[:, :101]) and torch.equal(buf[:, 1102:], wide[:, 1102:])


@pytest.mark.parametrize("change", ["type", "ids", "lens", "rep", "rows", "bias", "mask", "index", "strided"])
def test_logit_penalties_refuse(change):
    x = torch.zeros((3, 100), device=DEV)
    ids = torch.zeros((3, 8), device=DEV, dtype=torch.int32)
    n = torch.full((3,), 4, device=DEV, dtype=torch.int32)
    how = dict(prompt_lens=n, seq_lens=n, repetition=torch.ones(3, device=DEV))
    if change == "type":
        x = x.double()
    elif change == "ids":
        ids = ids.long()
    elif change == "lens":
        how["seq_lens"] = None
    elif change == "rep":
        how["repetition"] = torch.ones(2, device=DEV)
    elif change == "rows":
        ids = ids[:2]
        how["repetition"] = None
    elif change == "bias":
        how["bias_ids"] = ids
    elif change == "mask":
        how["allowed_bitmask"] = torch.zeros((3, 3), device=DEV, dtype=torch.int32)
    elif change == "index":
        how["req_index"] = torch.zeros(3, device=DEV, dtype=torch.int64)
    elif change == "strided":
        x = torch.zeros((100, 3), device=DEV).T
    with pytest.raises(ValueError):
        _ops().apply_logit_penalties(x, ids, **how)


# ---------------------------------------------------------------------------
# the ends of the ranges
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("tokens,n,k", [
    (3, 70, 640), (4, 16, 8192), (5, 100, 4224), (7, 33, 128), (10, 40, 8192),
    (8, 50, 16384),   # shared memory holds four rows: two passes over the weights
    (11, 20, 16384),
    (3, 24, 32768),   # two rows
    (1, 40, 65536),   # pieces of a row
    (11, 2400, 61568),
])
def test_w4_linear_few_rows_and_long_ones(tokens, n, k, group, zeros, dtype):
    gen = _gen(tokens + n + k)
    x = torch.randn((tokens, k), generator=gen, device=DEV).to(dtype)
    q, s, z, w = _w4((n, k), group, zeros, gen, dtype)
    got = _ops().w4_linear(x, q, s, z)
    xd = x.double()
    size = xd.abs() @ (s.double().repeat_interleave(group, 1) * 15).T
    _within(got, xd @ w.T, U[dtype] * (xd @ w.T).abs() + 2.0 ** -22 * k * size + 1e-6)


@pytest.mark.parametrize("dtype,exponents", [(torch.bfloat16, [-60, -20, 0, 20, 40]), (torch.float16, [-14, -7, 0, 7, 11])])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_linear_magnitudes(group, dtype, exponents):
    """Rows of very different sizes, each exact to its own size."""
    gen = _gen(31)
    x = torch.randn((len(exponents), 1280), generator=gen, device=DEV).clamp(-4, 4)
    x = (x * torch.exp2(torch.tensor(exponents, device=DEV, dtype=torch.float32)).unsqueeze(1)).to(dtype)
    q, s, z, _ = _w4((90, 1280), group, True, gen, dtype)
    z.copy_(torch.randint(0, 256, z.shape, generator=gen, device=DEV))  # any byte
    s /= 64  # keeps fp16 results in range
    w = (q.long().unsqueeze(-1) >> torch.tensor([0, 4], device=DEV) & 15).flatten(-2).double()
    w = (w - z.double().repeat_interleave(group, 1)) * s.double().repeat_interleave(group, 1)
    s64 = s.double().repeat_interleave(group, 1)
    got, ref = _ops().w4_linear(x, q, s, z), x.double() @ w.T
    size = x.double().abs() @ (s64 * 255).T
    least = 2.0 ** -25 if dtype is torch.float16 else 0.0  # half a step of the smallest results
    # the group sum of x and its product with the zero point round as well
    _within(got, ref, U[dtype] * ref.abs() + 2.0 ** -22 * 1280 * size + least)


def test_w4_linear_refuses_misaligned_scales_and_overlapping_rows():
    from vllm_ernie_b200 import HcaError

    gen = _gen(32)
    x, (q, s, _, _) = torch.zeros((1, 96), device=DEV, dtype=torch.bfloat16), _w4((3, 96), 32, False, gen)
    odd = torch.ones(10, device=DEV, dtype=torch.bfloat16)[1:].view(3, 3)  # two bytes past a word
    with pytest.raises(HcaError) as e:
        _ops().w4_linear(x, q, odd)
    assert e.value.status == -1
    two = torch.zeros((2, 96), device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        _ops().w4_linear(two, q, s, out=torch.zeros((1, 3), device=DEV, dtype=torch.bfloat16).expand(2, 3))


@pytest.mark.parametrize("kind", FORMATS)
@pytest.mark.parametrize("tokens,hidden,inner,shared", [
    (9, 8192, 128, 256),    # shared memory holds one block of columns
    (16, 512, 8192, 0),
    (6, 16384, 128, 128),   # four columns
    (12, 8192, 1024, 128),
])
def test_moe_experts_long_rows(tokens, hidden, inner, shared, kind):
    gen = _gen(tokens + hidden)
    x = torch.randn((tokens, hidden), generator=gen, device=DEV).to(torch.bfloat16)
    stack, w13, w2 = _stack(kind, (3,), hidden, inner, gen)
    one, a, b = _stack(kind, (), hidden, shared, gen) if shared else (None, None, None)
    ids = torch.rand((tokens, 3), generator=gen, device=DEV).argsort(1)[:, :2].int().contiguous()
    weights = torch.rand((tokens, 2), generator=gen, device=DEV)
    got = _ops().moe_experts(x, ids, weights, stack, shared=one)
    ref, size = _experts_ref(x, ids, weights, w13, w2, shared=(a, b) if shared else None)
    _within(got, ref, _moe_bound(ref, size, hidden + 2 * inner + shared))


@pytest.mark.parametrize("kind", ["bf16", "fp8", "w4-32z"])
@pytest.mark.parametrize("hidden,inner,shared", [(512, 64, 16384), (16384, 16384, 32), (64, 32, 8192)])
def test_moe_experts_of_very_different_lengths(hidden, inner, shared, kind):
    gen = _gen(hidden + shared)
    x = torch.randn((3, hidden), generator=gen, device=DEV).to(torch.bfloat16)
    stack, w13, w2 = _stack(kind, (2,), hidden, inner, gen)
    one, a, b = _stack(kind, (), hidden, shared, gen)
    ids = torch.tensor([[0], [1], [0]], device=DEV, dtype=torch.int32)
    weights = torch.rand((3, 1), generator=gen, device=DEV)
    got = _ops().moe_experts(x, ids, weights, stack, shared=one)
    ref, size = _experts_ref(x, ids, weights, w13, w2, shared=(a, b))
    _within(got, ref, _moe_bound(ref, size, hidden + inner + shared))


@pytest.mark.parametrize("tokens", [1, 3, 16, 17, 64])
@pytest.mark.parametrize("experts,k", [(129, 6), (512, 16)])
def test_moe_decode_of_many_experts_is_route_then_experts(experts, k, tokens):
    ops, gen = _ops(), _gen(33)
    x = torch.randn((tokens, 256), generator=gen, device=DEV).to(torch.bfloat16)
    wr = torch.randn((experts, 256), generator=gen, device=DEV) * 0.1
    stack, _, _ = _stack("w4-32", (experts,), 256, 64, gen)
    shared, _, _ = _stack("w4-32", (), 256, 96, gen)
    ids, weights = ops.moe_route(x, wr, k)
    got = ops.moe_decode(x, wr, stack, k, shared=shared)
    assert torch.equal(got, ops.moe_experts(x, ids, weights, stack, shared=shared))


def test_moe_result_does_not_depend_on_the_batchs_other_tokens():
    ops, gen = _ops(), _gen(34)
    x = torch.randn((11, 512), generator=gen, device=DEV).to(torch.bfloat16)
    wr = torch.randn((24, 512), generator=gen, device=DEV) * 0.1
    stack, _, _ = _stack("w4-64z", (24,), 512, 192, gen)
    first = ops.moe_decode(x, wr, stack, 3)
    other = torch.randn((11, 512), generator=gen, device=DEV).to(torch.bfloat16)
    other[7] = x[2]
    assert torch.equal(ops.moe_decode(other, wr, stack, 3)[7], first[2])


@pytest.mark.parametrize("change", ["one", "other", "overlapping"])
def test_moe_refuses_half_a_format(change):
    """Zero points for the experts and none for the shared one, or the other
    way round; rows of a result on top of each other."""
    ops, gen = _ops(), _gen(35)
    x = torch.randn((3, 128), generator=gen, device=DEV).to(torch.bfloat16)
    wr = torch.randn((8, 128), generator=gen, device=DEV)
    stack, _, _ = _stack("w4-64z", (8,), 128, 64, gen)
    shared, _, _ = _stack("w4-64z", (), 128, 64, gen)
    out = None
    if change == "one":
        shared = shared._replace(z13=None)
    elif change == "other":
        stack = stack._replace(z2=None)
    else:
        out = torch.zeros((1, 128), device=DEV, dtype=torch.bfloat16).expand(3, 128)
    with pytest.raises(ValueError):
        ops.moe_decode(x, wr, stack, 2, shared=shared, out=out)


@pytest.mark.parametrize("zeros", ["z13", "z2"])
def test_moe_zero_points_of_one_product(zeros):
    ops, gen = _ops(), _gen(36)
    x = torch.randn((4, 256), generator=gen, device=DEV).to(torch.bfloat16)
    q13, s13, z13, w13 = _w4((5, 384, 256), 64, zeros == "z13", gen)
    q2, s2, z2, w2 = _w4((5, 256, 192), 64, zeros == "z2", gen)
    ids = torch.randint(0, 5, (4, 1), generator=gen, device=DEV, dtype=torch.int32)
    weights = torch.rand((4, 1), generator=gen, device=DEV)
    got = ops.moe_experts(x, ids, weights, ops.MoEWeights(q13, q2, s13, s2, z13, z2))
    ref, size = _experts_ref(x, ids, weights, w13, w2)
    _within(got, ref, _moe_bound(ref, size, 256 + 192))


@pytest.mark.parametrize("shift", [2, 4, 6, 8])
def test_4_bit_scales_that_start_off_16_bytes(shift):
    """Rows of whole 16 bytes whose arrays start elsewhere."""
    ops, gen = _ops(), _gen(37)

    def moved(v, by):
        flat = torch.zeros(v.numel() + by, device=DEV, dtype=v.dtype)
        flat[by:] = v.flatten()
        return flat[by:].view(v.shape)

    x = torch.randn((3, 4096), generator=gen, device=DEV).to(torch.bfloat16)
    q, s, z, _ = _w4((100, 4096), 32, True, gen)
    assert torch.equal(ops.w4_linear(x, q, moved(s, shift), moved(z, 2 * shift)), ops.w4_linear(x, q, s, z))
    x = x[:, :1024].contiguous()
    stack, _, _ = _stack("w4-64z", (5,), 1024, 512, gen)
    one, _, _ = _stack("w4-64z", (), 1024, 512, gen)
    wr = torch.randn((5, 1024), generator=gen, device=DEV) * 0.1
    first = ops.moe_decode(x, wr, stack, 2, shared=one)

    def off(w):
        return w._replace(s13=moved(w.s13, shift), s2=moved(w.s2, shift), z13=moved(w.z13, 2 * shift), z2=moved(w.z2, 2 * shift))

    assert torch.equal(ops.moe_decode(x, wr, off(stack), 2, shared=one), first)
    assert torch.equal(ops.moe_decode(x, wr, stack, 2, shared=off(one)), first)


def test_logit_penalties_refuse_rows_on_top_of_each_other():
    x = torch.zeros((1, 64), device=DEV).expand(3, 64)
    with pytest.raises(ValueError):
        _ops().apply_logit_penalties(x, frequency=torch.zeros(3, device=DEV))


def test_no_wait_gave_up():
    assert _ops().device_error() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,length,bias,mask", [
    (200, 5003, 300, 6, True),     # more rows than SMs, small tables
    (150, 32000, 40, 0, False),
    (300, 17, 0, 2, True),
    (2, 3000, 70000, 4, True),     # counts past 16 bits
    (170, 900, 66000, 0, False),
])
def test_logit_penalties_many_rows_and_long_histories(rows, vocab, length, bias, mask, dtype):
    test_logit_penalties(rows, vocab, length, bias, mask, dtype)
