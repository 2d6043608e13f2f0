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
