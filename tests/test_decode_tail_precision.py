"""How exact the few-row operators are: relative errors over a whole result,
which a term left out or rounded once too often cannot hide in.

Tolerances.  The last rounding leaves |e| <= u |y| with u = 2^-8 (bf16) or
2^-11 (fp16).  Over n normally distributed results its relative L2 error is
0.425 u whatever their size (the same within 0.002 at sixteen sizes of an
octave), and with a second rounding to the same type anywhere before, 0.60 u.
The limit between them is (0.48 + 0.8 / sqrt(n)) u.

Sums: within a group at most 16 additions by the tensor instructions, which may
truncate (2^-22 of the group's terms each), then one rounding to nearest for
each further group, warp and piece (2^-24 of all terms).  With S = sum |x| |w|,
codes taken as 15 at most for q and for z each, that is
(16 2^-22 + (groups + 32) 2^-24) 2 S, which the L2 check leaves unused.
"""

import math

import pytest
import torch

gpu = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _ops():
    from vllm_ernie_b200 import ops

    return ops


def _rounded_once(got, ref, dtype):
    error = ((got.double() - ref).norm() / ref.norm()).item()
    return error <= (0.48 + 0.8 / math.sqrt(ref.numel())) * U[dtype]


def _w4_weights(n, k, group, zeros, dtype, gen, device):
    q = torch.randint(0, 256, (n, k // 2), generator=gen, device=device, dtype=torch.uint8)
    s = ((0.5 + torch.rand((n, k // group), generator=gen, device=device)) / (4.6 * math.sqrt(k))).to(dtype)
    z = torch.randint(0, 16, s.shape, generator=gen, device=device, dtype=torch.uint8) if zeros else None
    return q, s, z


def _w4_rows(q, s, z, group):
    """Rows of 4-bit weights in 64 bits."""
    codes = torch.stack((q & 15, q >> 4), -1).flatten(-2).double()
    zero = 8.0 if z is None else z.double().repeat_interleave(group, -1)
    return (codes - zero) * s.double().repeat_interleave(group, -1)


def _w4_ref(x, q, s, z, group):
    """The product in 64 bits and the size 2 S of its terms, some rows at a time."""
    xd, step = x.double(), 2048
    y = torch.cat([xd @ _w4_rows(q[a:a + step], s[a:a + step], None if z is None else z[a:a + step], group).T
                   for a in range(0, q.shape[0], step)], 1)
    sums = xd.abs().unflatten(1, (s.shape[1], group)).sum(2)
    return y, 30 * (sums @ s.double().T)


def _w4_holds(got, ref, size, dtype, groups):
    bound = U[dtype] * ref.abs() + 1.01 * (16 * 2.0 ** -22 + (groups + 32) * 2.0 ** -24) * size + 2.0 ** -25
    return bool(((got.double() - ref).abs() <= bound).all()) and _rounded_once(got, ref, dtype)


# ---------------------------------------------------------------------------
# the checks themselves, on the CPU: what they have to let through and not
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group,k", [(32, 29568), (128, 43136)])
def test_the_long_row_check_tells_mistakes_apart(group, k, dtype):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn((2, k), generator=gen).to(dtype)
    q, s, z = _w4_weights(600, k, group, True, dtype, gen, "cpu")
    ref, size = _w4_ref(x, q, s, z, group)
    groups = k // group

    def holds(y):
        return _w4_holds(y.to(dtype), ref, size, dtype, groups)

    assert holds(ref)
    assert not holds(torch.zeros_like(ref))
    some = x.clone()
    some[:, -group:] = 0  # the last group left out
    assert not holds(_w4_ref(some, q, s, z, group)[0])
    other = s.clone()
    other[:, 4096 // group] = s[:, 4096 // group + 1]  # a neighbour's scales
    assert not holds(_w4_ref(x, q, other, z, group)[0])
    other = z.clone()
    other[:, -1] = z[:, -2]
    assert not holds(_w4_ref(x, q, s, other, group)[0])
    part = _w4_ref(x[:, :4096], q[:, :2048], s[:, :4096 // group], z[:, :4096 // group], group)[0]
    assert not holds(part.to(dtype) + (ref - part).to(dtype))  # rounded between the pieces


@pytest.mark.parametrize("inner", [128, 384, 16384])
def test_the_rounding_check_tells_one_bf16_number_from_two(inner):
    gen = torch.Generator().manual_seed(2)
    h = torch.randn((3, inner), generator=gen).double()
    w2 = torch.randn((1024, inner), generator=gen).double()
    ref = h @ w2.T
    first = h.bfloat16()
    second = (h - first.double()).bfloat16()
    assert _rounded_once(((first.double() + second.double()) @ w2.T).bfloat16(), ref, torch.bfloat16)
    assert not _rounded_once((first.double() @ w2.T).bfloat16(), ref, torch.bfloat16)
    swapped = first.double() + second.double().roll(1, 0)  # another token's second part
    assert not _rounded_once((swapped @ w2.T).bfloat16(), ref, torch.bfloat16)


# ---------------------------------------------------------------------------
# 4-bit products of long rows
# ---------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("tokens,n,k,group", [
    (1, 40, 65536, 128),      # whole pieces of 4096
    (11, 2400, 61568, 32),
    # a short last piece, and several groups of warps with a tile in each block
    (3, 8192, 29568, 32),
    (1, 20000, 29568, 32),
    (2, 10000, 37504, 64),
    (9, 8192, 43136, 128),
    (2, 8192, 33792, 32),     # the last piece's scales in whole 16 bytes
])
def test_w4_linear_of_long_rows(tokens, n, k, group, zeros, dtype):
    gen = torch.Generator(device="cuda").manual_seed(n + k)
    x = torch.randn((tokens, k), generator=gen, device="cuda").to(dtype)
    q, s, z = _w4_weights(n, k, group, zeros, dtype, gen, "cuda")
    got = [_ops().w4_linear(x, q, s, z) for _ in range(6)]
    ref, size = _w4_ref(x, q, s, z, group)
    assert _w4_holds(got[0], ref, size, dtype, k // group)
    for again in got[1:]:
        assert torch.equal(again, got[0])


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (64, True), (128, True)])
@pytest.mark.parametrize("tokens,n,k", [
    (1, 3000, 640), (2, 2500, 4224), (3, 2000, 8192), (4, 1500, 16384), (5, 1003, 8192), (8, 800, 16384), (9, 700, 4096),
    (16, 513, 8192), (17, 300, 2176), (33, 200, 8192), (3, 1201, 24576), (2, 700, 32768)])
def test_w4_linear_rounds_once(tokens, n, k, group, zeros, dtype):
    gen = torch.Generator(device="cuda").manual_seed(n + k)
    x = torch.randn((tokens, k), generator=gen, device="cuda").to(dtype)
    q, s, z = _w4_weights(n, k, group, zeros, dtype, gen, "cuda")
    ref, size = _w4_ref(x, q, s, z, group)
    assert _w4_holds(_ops().w4_linear(x, q, s, z), ref, size, dtype, k // group)


# ---------------------------------------------------------------------------
# experts
# ---------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _matrix(kind, shape, gen):
    """(data, scales, zero points, 64-bit weights) of a weight format."""
    *lead, n, k = shape
    if kind.startswith("w4"):
        group, zeros = int(kind.split("-")[1].rstrip("z")), kind.endswith("z")
        q, s, z = _w4_weights(math.prod(lead) * n, k, group, zeros, torch.bfloat16, gen, "cuda")
        w = _w4_rows(q, s, z, group).view(shape)
        return q.view(*lead, n, -1), s.view(*lead, n, -1), None if z is None else z.view(*lead, n, -1), w
    w = torch.randn(shape, generator=gen, device="cuda") / math.sqrt(k)
    if kind == "bf16":
        return w.bfloat16(), None, None, w.bfloat16().double()
    s = torch.exp2(torch.randint(-3, 1, (*lead, -(-n // 128), -(-k // 128)), generator=gen, device="cuda").float()) / 37
    d = (w * 37).to(FP8)
    return d, s, None, d.double() * s.double().repeat_interleave(128, -2).repeat_interleave(128, -1)[..., :n, :k]


def _stack(kind, lead, hidden, inner, gen):
    d13, s13, z13, w13 = _matrix(kind, (*lead, 2 * inner, hidden), gen)
    d2, s2, z2, w2 = _matrix(kind, (*lead, hidden, inner), gen)
    return _ops().MoEWeights(d13, d2, s13, s2, z13, z2), w13, w2


def _mlp(x, w13, w2):
    gate, up = (x @ w13.transpose(-1, -2)).chunk(2, -1)
    return (gate * torch.sigmoid(gate) * up) @ w2.transpose(-1, -2)


def _experts_ref(x, ids, weights, w13, w2, shared=None):
    x, weights = x.double(), weights.double()
    y = torch.zeros_like(x) if shared is None else _mlp(x, *shared)
    for e in range(w13.shape[0]):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        y.index_add_(0, t, _mlp(x[t], w13[e], w2[e]) * weights[t, j].unsqueeze(1))
    return y


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "w4-32", "w4-64z", "w4-128"])
@pytest.mark.parametrize("tokens,experts,hidden,inner,shared", [
    (1, 4, 1024, 256, 384), (2, 4, 1024, 384, 128), (3, 4, 1024, 256, 384), (4, 6, 1024, 384, 128), (5, 6, 1024, 256, 384),
    (8, 6, 512, 384, 640), (9, 20, 512, 256, 384), (16, 3, 512, 384, 256), (40, 6, 512, 256, 384), (70, 12, 512, 128, 0), (5, 6, 8192, 256, 0), (12, 4, 1024, 8192, 384)])
def test_moe_experts_round_once(tokens, experts, hidden, inner, shared, kind):
    """The gated product between the two products is not rounded to bf16: with it
    in one number the error is that of two roundings.  All widths of columns, with
    a shared expert of another length."""
    gen = _gen(tokens + inner)
    x = torch.randn((tokens, hidden), generator=gen, device="cuda").bfloat16()
    stack, w13, w2 = _stack(kind, (experts,), hidden, inner, gen)
    one, a, b = _stack(kind, (), hidden, shared, gen) if shared else (None, None, None)
    ids = torch.rand((tokens, experts), generator=gen, device="cuda").argsort(1)[:, :3].int().contiguous()
    weights = torch.rand((tokens, 3), generator=gen, device="cuda")
    got = _ops().moe_experts(x, ids, weights, stack, shared=one)
    assert _rounded_once(got, _experts_ref(x, ids, weights, w13, w2, (a, b) if shared else None), torch.bfloat16)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "w4-32"])
@pytest.mark.parametrize("tokens,hidden,inner,shared", [(5, 2080, 736, 96), (2, 2080, 160, 736), (13, 1056, 96, 32), (3, 4128, 32, 4096)])
def test_moe_experts_of_odd_sizes_round_once(tokens, hidden, inner, shared, kind):
    gen = _gen(tokens + hidden)
    x = torch.randn((tokens, hidden), generator=gen, device="cuda").bfloat16()
    stack, w13, w2 = _stack(kind, (4,), hidden, inner, gen)
    one, a, b = _stack(kind, (), hidden, shared, gen)
    ids = torch.randint(-1, 4, (tokens, 3), generator=gen, device="cuda", dtype=torch.int32)  # skipped and repeated ones too
    weights = torch.rand((tokens, 3), generator=gen, device="cuda")
    got = _ops().moe_experts(x, ids, weights, stack, shared=one)
    assert _rounded_once(got, _experts_ref(x, ids, weights, w13, w2, (a, b)), torch.bfloat16)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "w4-32", "w4-32z", "w4-64z", "w4-128z"])
@pytest.mark.parametrize("tokens,inner,shared", [(1, 16384, 0), (5, 16384, 256), (3, 256, 16384), (9, 14336, 64 * 6)])
def test_moe_experts_round_once_whatever_the_length(tokens, inner, shared, kind):
    gen = _gen(tokens + inner)
    x = torch.randn((tokens, 2048), generator=gen, device="cuda").bfloat16()
    stack, w13, w2 = _stack(kind, (2,), 2048, inner, gen)
    one, a, b = _stack(kind, (), 2048, shared, gen) if shared else (None, None, None)
    ids = torch.randint(0, 2, (tokens, 1), generator=gen, device="cuda", dtype=torch.int32)
    weights = torch.rand((tokens, 1), generator=gen, device="cuda") + 0.5
    got = _ops().moe_experts(x, ids, weights, stack, shared=one)
    assert _rounded_once(got, _experts_ref(x, ids, weights, w13, w2, (a, b) if shared else None), torch.bfloat16)


@gpu
@pytest.mark.parametrize("value", [0x7F, 0xFF])
@pytest.mark.parametrize("tokens,hidden,inner", [(2, 256, 128), (5, 2080, 736), (12, 512, 256)])
def test_an_e4m3_nan_is_a_nan(tokens, hidden, inner, value):
    """In an expert's first product it makes the expert's tokens NaN, in the second
    its row of the result; others keep their bits."""
    gen = _gen(tokens)
    x = torch.randn((tokens, hidden), generator=gen, device="cuda").bfloat16()
    stack, _, _ = _stack("fp8", (4,), hidden, inner, gen)
    ids = torch.randint(0, 4, (tokens, 1), generator=gen, device="cuda", dtype=torch.int32)
    ids[0] = 2
    ids[1] = 1
    weights = torch.rand((tokens, 1), generator=gen, device="cuda")
    clean = _ops().moe_experts(x, ids, weights, stack)
    has = ids[:, 0] == 2
    for k in (0, 77, hidden - 1):
        for row in (0, inner - 1, 2 * inner - 3):
            bad = stack.w13.clone()
            bad.view(torch.uint8)[2, row, k] = value
            got = _ops().moe_experts(x, ids, weights, stack._replace(w13=bad))
            assert torch.isnan(got[has]).all() and torch.equal(got[~has], clean[~has])
    for k in (0, inner - 1):
        bad = stack.w2.clone()
        bad.view(torch.uint8)[2, hidden - 9, k] = value
        got = _ops().moe_experts(x, ids, weights, stack._replace(w2=bad))
        want = clean.clone()
        want[has, hidden - 9] = math.nan
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(0), want.nan_to_num(0))


# ---------------------------------------------------------------------------
# the range of bf16 activations
# ---------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("tokens,experts", [(1, 3), (4, 3), (40, 20), (64, 4), (70, 5)])
def test_an_e4m3_nan_in_any_block_and_in_the_shared_expert(tokens, experts):
    gen = _gen(tokens + experts)
    hidden, inner, shared = 384, 256, 160
    x = torch.randn((tokens, hidden), generator=gen, device="cuda").bfloat16()
    stack, _, _ = _stack("fp8", (experts,), hidden, inner, gen)
    one, _, _ = _stack("fp8", (), hidden, shared, gen)
    ids = torch.randint(0, experts, (tokens, 2), generator=gen, device="cuda", dtype=torch.int32)
    weights = torch.rand((tokens, 2), generator=gen, device="cuda")

    def run(w, sh):
        return _ops().moe_experts(x, ids, weights, w, shared=sh)

    def with_nan(w, *at):
        w = w.clone()
        w.view(torch.uint8)[at] = 0x7F
        return w

    clean = run(stack, one)
    e = int(ids[tokens // 2, 1])
    has = (ids == e).any(1)
    got = run(stack._replace(w13=with_nan(stack.w13, e, 11, 300)), one)
    assert torch.isnan(got[has]).all() and torch.equal(got[~has], clean[~has])
    got = run(stack._replace(w2=with_nan(stack.w2, e, 380, 31)), one)
    assert torch.isnan(got[has, 380]).all() and torch.isnan(got).sum() == has.sum()
    keep = ~torch.isnan(got)
    assert torch.equal(got[keep], clean[keep])
    assert torch.isnan(run(stack, one._replace(w13=with_nan(one.w13, 2 * shared - 1, 5)))).all()
    got = run(stack, one._replace(w2=with_nan(one.w2, 7, 159)))
    assert torch.isnan(got[:, 7]).all() and torch.isnan(got).sum() == tokens
    # two experts at once, and none left over for the next call
    bad = with_nan(with_nan(stack.w13, 0, 0, 0), experts - 1, 2 * inner - 1, hidden - 1)
    has = (ids == 0).any(1) | (ids == experts - 1).any(1)
    got = run(stack._replace(w13=bad), one)
    assert torch.equal(torch.isnan(got).all(1), has) and torch.equal(got[~has], clean[~has])
    assert torch.equal(run(stack, one), clean)


@gpu
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("tokens,k", [(1, 640), (4, 1152), (8, 640), (11, 4096), (9, 29952)])
def test_w4_linear_over_the_range_of_activations(tokens, k, group, zeros):
    """Rows of sizes from 2^-40 to just below 2^48 are all as exact as any; from
    2^48 on a value makes its own row infinite or NaN, never a wrong number."""
    gen = _gen(tokens + k)
    size = torch.tensor([45, 0, 47, 20, -40], device="cuda").repeat(3)[:tokens].float()
    x = (torch.randn((tokens, k), generator=gen, device="cuda").clamp(-1.9, 1.9) * torch.exp2(size).unsqueeze(1)).bfloat16()
    q, s, z = _w4_weights(2000, k, group, zeros, torch.bfloat16, gen, "cuda")
    got = _ops().w4_linear(x, q, s, z)
    ref, _ = _w4_ref(x, q, s, z, group)
    for t in range(tokens):
        assert _rounded_once(got[t], ref[t], torch.bfloat16)
    for value in (2.0 ** 52, -2.0 ** 100, math.inf, -math.inf, math.nan):
        bad = x.clone()
        bad[tokens // 2, k // 3] = value
        out = _ops().w4_linear(bad, q, s, z)
        assert not torch.isfinite(out[tokens // 2]).any()
        keep = [t for t in range(tokens) if t != tokens // 2]
        assert torch.equal(out[keep], got[keep])


@gpu
@pytest.mark.parametrize("kind", ["fp8", "w4-32", "w4-64z", "w4-128"])
@pytest.mark.parametrize("tokens", [1, 2, 3, 6, 12, 30])
def test_moe_experts_over_the_range_of_activations(tokens, kind):
    gen = _gen(tokens)
    size = torch.tensor([22, 0, -20, 10], device="cuda").repeat(8)[:tokens].float()  # products of two below 2^48
    x = (torch.randn((tokens, 640), generator=gen, device="cuda").clamp(-3, 3) * torch.exp2(size).unsqueeze(1)).bfloat16()
    stack, w13, w2 = _stack(kind, (5,), 640, 384, gen)
    one, a, b = _stack(kind, (), 640, 256, gen)
    ids = torch.rand((tokens, 5), generator=gen, device="cuda").argsort(1)[:, :3].int().contiguous()
    weights = torch.rand((tokens, 3), generator=gen, device="cuda")
    got = _ops().moe_experts(x, ids, weights, stack, shared=one)
    ref = _experts_ref(x, ids, weights, w13, w2, (a, b))
    for t in range(tokens):
        assert _rounded_once(got[t], ref[t], torch.bfloat16), t
    for value in (2.0 ** 52, math.inf, math.nan):
        bad = x.clone()
        bad[tokens // 2, 333] = value
        out = _ops().moe_experts(bad, ids, weights, stack, shared=one)
        assert not torch.isfinite(out[tokens // 2]).any()
        keep = [t for t in range(tokens) if t != tokens // 2]
        assert torch.equal(out[keep], got[keep])


# ---------------------------------------------------------------------------
# router
# ---------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts", [16, 60, 300])
def test_route_weights_are_those_of_32_bit_functions(score, experts):
    """One activation of 1 a token and logits of 11 bits, so that they and their
    differences are exact.  What rounds, in units of 2^-24: the exponential (2), a
    sum of up to 300 of them (2 of the terms, 10 additions of a lane and 5 of the
    tree), the division (1): 20 units, and in the subnormals one of their steps for
    the exponential and one for the division."""
    gen = _gen(4)
    wr = torch.randint(-60 * 16, 60 * 16, (experts, 32), generator=gen, device="cuda") / 16.0
    x = torch.eye(32, device="cuda").bfloat16()
    ids, w = _ops().moe_route(x, wr, 16, score=score, renormalize=False)
    l = wr.T.double()
    p = torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l)
    want = torch.gather(p, 1, ids.long())
    assert ((w.double() - want).abs() <= 20 * 2.0 ** -24 * want + 2 * 2.0 ** -149).all()


# ---------------------------------------------------------------------------
# logits
# ---------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("value", [1.1, 0.7, 3.0, 2.0 ** -130])
def test_the_repetition_penalty_divides(value):
    """fp32 logits have the bits of the division and the product of the definition
    (the reciprocal of a penalty below 2^-128 is infinite, quotients are not)."""
    x = torch.randn((4, 5000), generator=_gen(3), device="cuda") * (2.0 ** -20 if value < 1e-30 else 5.0)
    ids = torch.arange(5000, device="cuda", dtype=torch.int32).repeat(4, 1)
    lens = torch.full((4,), 5000, device="cuda", dtype=torch.int32)
    r = torch.full((4,), value, device="cuda")
    want = torch.where(x > 0, x / r[:, None], x * r[:, None])
    assert torch.isfinite(want).all()
    assert torch.equal(_ops().apply_logit_penalties(x, ids, lens, lens, repetition=r), want)


# ---------------------------------------------------------------------------
# more rows than a grid has columns
# ---------------------------------------------------------------------------


@gpu
def test_w4_linear_of_very_many_rows():
    gen = _gen(1)
    x = torch.randn((65536 + 70, 32), generator=gen, device="cuda").bfloat16()
    q, s, z = _w4_weights(16, 32, 32, True, torch.bfloat16, gen, "cuda")
    got = _ops().w4_linear(x, q, s, z)
    assert torch.equal(got[65530:], _ops().w4_linear(x[65530:], q, s, z)) and torch.equal(got[:9], _ops().w4_linear(x[:9], q, s, z))


@gpu
def test_moe_route_of_very_many_rows():
    x = torch.randn((65536 * 8 + 20, 32), generator=_gen(1), device="cuda").bfloat16()
    wr = torch.randn((3, 32), generator=_gen(2), device="cuda")
    ids, w = _ops().moe_route(x, wr, 2)
    last, lw = _ops().moe_route(x[-40:], wr, 2)
    assert torch.equal(ids[-40:], last) and torch.equal(w[-40:], lw)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("name", ["repetition", "frequency", "presence", "bias_ids"])
def test_a_number_for_all_requests_is_refused(name):
    """As the other arguments are, with a ValueError and the logits untouched."""
    x = torch.ones((3, 40), device="cuda")
    one = torch.tensor(1, dtype=torch.int32 if name == "bias_ids" else torch.float32, device="cuda")
    with pytest.raises(ValueError):
        _ops().apply_logit_penalties(x, **{name: one}, **({"bias_values": one.float()} if name == "bias_ids" else {}))
    assert (x == 1).all()


@gpu
def test_experts_without_a_stack_are_refused():
    x = torch.zeros((2, 64), device="cuda", dtype=torch.bfloat16)
    ids, weights = torch.zeros((2, 1), device="cuda", dtype=torch.int32), torch.ones((2, 1), device="cuda")
    for w13 in (torch.tensor(1.0, device="cuda", dtype=torch.bfloat16), torch.zeros((128, 64), device="cuda", dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            _ops().moe_experts(x, ids, weights, _ops().MoEWeights(w13, torch.zeros((64, 64), device="cuda", dtype=torch.bfloat16)))
