"""How far packed attention's gradients lie from the formula's in 64 bits, as norms, for incoming gradients of any size.

The exact gradient rounded to its type is off by r of its norm.  A kernel's is further off by what it rounds on the way, errors of the same relative size and of signs that have nothing to do with each other, so that
squares add: dV's probabilities, and dK's dS, once each, sqrt(2) r; dQ's dS is two values, whose error is below r's by as many bits again as a value has, r.  What fp32 leaves, the forward's probabilities, which lse and delta are
of, and how evenly values lie between two powers of two are allowed 15 in a hundred more: 1.3 r for dQ (where those of the forward show most) and 1.65 r for dK and dV.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _exact(q, k, v, dout, lengths, causal):
    """The output and the gradients in 64 bits."""
    H, Hk, D = q.shape[1], k.shape[1], q.shape[2]
    outs = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, q, k, v)]
    at = 0
    for n in lengths:
        rows = slice(at, at + n)
        for h in range(H):
            hk = h // (H // Hk)
            Q, K, V, dO = (t[rows, i].double() for t, i in ((q, h), (k, hk), (v, hk), (dout, h)))
            S = Q @ K.T / math.sqrt(D)
            if causal:
                S = S.masked_fill(~torch.ones(n, n, dtype=torch.bool, device=q.device).tril(), -math.inf)
            P = S.softmax(-1)
            outs[0][rows, h] = P @ V
            dP = dO @ V.T
            dS = P * (dP - (P * dP).sum(-1, keepdim=True)) / math.sqrt(D)
            outs[1][rows, h] = dS @ K
            outs[2][rows, hk] += dS.T @ Q
            outs[3][rows, hk] += P.T @ dO
        at += n
    return outs


def _inputs(dtype, lengths, H, Hk, D, size, sharp=1.0):
    g = torch.Generator(device="cuda:0").manual_seed(11)
    T = sum(lengths)
    made = [torch.randn(T, h, D, device="cuda:0", generator=g) * s for h, s in ((H, sharp), (Hk, 1.0), (Hk, 1.0), (H, size))]
    return [t.to(dtype) for t in made]


def _off(lengths):
    return torch.tensor([0] + lengths, device="cuda:0").cumsum(0).to(torch.int32)


# lengths, H, Hk, D, causal: walks in parts, two groups of waves to a tile, one
SHAPES = [
    ([4096], 1, 1, 64, False),
    ([256], 2, 2, 128, False),
    ([1900, 77], 2, 1, 32, True),
    ([1500], 4, 1, 96, True),
    ([1024, 1000, 900], 12, 6, 128, False),
    ([300] * 9, 24, 12, 128, True),
    ([700, 33, 900] * 3, 16, 16, 64, True),
    ([51, 768, 300, 120] * 6, 16, 16, 32, False),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("size", [1e-4, 1e-2, 1.0, 8000.0])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(x).replace(" ", "") for x in (len(s[0]), s[0][0], *s[1:])))
def test_small_and_large_gradients_keep_their_bits(gpu_device, dtype, size, shape):
    from evoformer_triton_amd import packed_attention
    lengths, H, Hk, D, causal = shape
    q, k, v, dout = _inputs(dtype, lengths, H, Hk, D, size)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(packed_attention(*leaves, _off(lengths), causal=causal), leaves, dout)
    for name, a, want, most in zip(("dq", "dk", "dv"), got, _exact(*(t.detach() for t in leaves), dout, lengths, causal)[1:], (1.3, 1.65, 1.65)):
        fits = want.abs() < 0.99 * torch.finfo(dtype).max      # (of what lies beyond the type, an infinity or nearly one)
        assert torch.isfinite(a[fits]).all() and (a.double() * want.sign())[~fits].ge(0.98 * torch.finfo(dtype).max).all(), name
        a, want = a[fits], want[fits]
        off, rounded = (a.double() - want).norm(), (want.to(dtype).double() - want).norm()
        assert off <= most * rounded, f"{name}: {float(off / rounded):.3f} times the error of the exact gradient rounded"


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(x).replace(" ", "") for x in (len(s[0]), s[0][0], *s[1:])))
@pytest.mark.parametrize("size,values", [(100.0, 512.0), (8000.0, 4096.0)])
def test_values_far_from_one_leave_theirs(gpu_device, dtype, shape, size, values):
    """dS grows with the values: what brings it down for its own rounding takes no bits of the probabilities that dV is formed of.  (Small queries and keys keep dQ and dK within the type, mostly.)  They also make a row's
    probabilities nearly alike, which are rounded alike then: off together by up to half a step, 1 / 0.425 times what a rounding is off by on average (r is 0.00166 in bf16, half a step 0.0039), so that dV may be off by
    sqrt(1 + 2.35^2) r = 2.55 r; 5 in a hundred for the rest."""
    from evoformer_triton_amd import packed_attention
    lengths, H, Hk, D, causal = shape
    q, k, v, dout = _inputs(dtype, lengths, H, Hk, D, size)
    q, k, v = q * 2.0 ** -6, k * 2.0 ** -6, v * values
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(packed_attention(*leaves, _off(lengths), causal=causal), leaves, dout)
    for name, a, want, most in zip(("dq", "dk", "dv"), got, _exact(*(t.detach() for t in leaves), dout, lengths, causal)[1:], (1.3, 1.65, 2.68)):
        fits = want.abs() < 0.99 * torch.finfo(dtype).max
        if fits.double().mean() < 0.999:      # (what is left of a sum's values when the larger ones do not fit are those whose terms cancel: off by what their terms are, not by what they are)
            assert name != "dv"
            continue
        _near(a[fits], want[fits], most, dtype, name)


def _near(got, want, most, dtype, name):
    off, rounded = (got.double() - want).norm(), (want.to(dtype).double() - want).norm()
    assert off <= most * rounded, f"{name}: {float(off / rounded):.3f} times the error of the exact result rounded"


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(x).replace(" ", "") for x in (len(s[0]), s[0][0], *s[1:])))
def test_sharp_scores_keep_theirs(gpu_device, dtype, shape):
    """Where few keys have most of the probability, what rounding leaves of the output, dS as two values and the sums' corrections decide: without one of them dQ or dK is beyond these bounds (test_packed_precision.py)."""
    from evoformer_triton_amd import packed_attention
    lengths, H, Hk, D, causal = shape
    q, k, v, dout = _inputs(dtype, lengths, H, Hk, D, 1.0, sharp=6.0)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(packed_attention(*leaves, _off(lengths), causal=causal), leaves, dout)
    for name, a, want, most in zip(("dq", "dk", "dv"), got, _exact(*(t.detach() for t in leaves), dout, lengths, causal)[1:], (1.3, 1.65, 1.65)):
        _near(a, want, most, dtype, name)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", SHAPES + [([5] * 40, 8, 2, 64, True)], ids=lambda s: "-".join(str(x).replace(" ", "") for x in (len(s[0]), s[0][0], *s[1:])))
def test_what_rounding_left_of_the_output(gpu_device, dtype, shape):
    """It is at most half a step, and with it the output is off by what the rounded probabilities leave alone: as much as one rounding (their errors are as large as the output's, value by value), where without it there are
    two, sqrt(2) times that.  15 in a hundred for how values lie between two powers of two."""
    lengths, H, Hk, D, causal = shape
    q, k, v, dout = _inputs(dtype, lengths, H, Hk, D, 1.0)
    o, _, left = torch.ops.evoattn.packed(q, k, v, _off(lengths), None, causal, None)
    assert (left.double().abs() <= torch.finfo(dtype).eps / 2 * o.double().abs() + torch.finfo(dtype).tiny * torch.finfo(dtype).eps).all()
    _near(o.double() + left.double(), _exact(q, k, v, dout, lengths, causal)[0], 1.15, dtype, "o and what is left")
