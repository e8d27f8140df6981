"""What the bounds of test_gpu_packed_gradients.py hold packed attention to: its roundings one by one in 64 bits, and each of the steps that keep its gradients' precision left out.  No GPU."""
import math

import pytest
import torch

BF16, F16 = torch.bfloat16, torch.float16
MOST = {"dq": 1.3, "dk": 1.65, "dv": 1.65}


def _errors(dtype, L, D, causal, sharp, left=True, two=True, shift=True, mended=True, size=1.0):
    """Errors of dQ, dK and dV in those of the exact results rounded.  left: delta of the output and of what rounding left of it; two: dS as two values for dQ; mended: lse and delta by the sums of P and dS; shift: fp16's
    operands of the backward times a power of two."""
    g = torch.Generator().manual_seed(5)

    def rounded(x):
        return x.to(dtype).double()

    q, k, v, dout = (rounded(torch.randn(L, D, generator=g, dtype=torch.float64) * s) for s in (sharp, 1.0, 1.0, size))
    S = q @ k.T / math.sqrt(D)
    if causal:
        S = S.masked_fill(~torch.ones(L, L, dtype=torch.bool).tril(), -math.inf)
    P, dP = S.softmax(-1), dout @ v.T
    dS = P * (dP - (P * dP).sum(-1, keepdim=True)) / math.sqrt(D)
    want = {"dq": dS @ k, "dk": dS.T @ q, "dv": P.T @ dout}
    top = S.amax(-1, keepdim=True)
    e = rounded(torch.exp(S - top))
    total = e.sum(-1, keepdim=True)
    o, lse = e @ v / total, top + total.log()
    delta = (dout * (rounded(o) + (rounded(o - rounded(o)) if left else 0.0))).sum(-1, keepdim=True)
    e = torch.exp(S - lse)
    ds = e * (dP - delta)

    def power(x, dim):        # that takes the largest to some 2^12
        return 2.0 ** (12 - torch.frexp(x.abs().amax(dim, keepdim=True))[1]) if shift and dtype == F16 else torch.ones(())

    by = power(ds, 1)
    high = rounded(ds * by)
    dq = (high + (rounded(ds * by - high) if two else 0.0)) / by @ k
    total, rest = e.sum(-1, keepdim=True), ds.sum(-1, keepdim=True)
    if mended:
        dq, lse, delta = dq / total, lse + total.log(), delta + rest / total
    e = torch.exp(S - lse)
    ds = e * (dP - delta)
    by, up = power(ds, 0), 2.0 ** 13 if shift and dtype == F16 else 1.0
    got = {"dq": dq / math.sqrt(D), "dk": (rounded(ds * by) / by).T @ q / math.sqrt(D), "dv": (rounded(e * up) / up).T @ dout}
    return {n: float((rounded(got[n]) - w).norm() / (rounded(w) - w).norm()) for n, w in want.items()}


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("L,D,causal,sharp", [(300, 32, False, 1.0), (300, 64, True, 6.0), (700, 32, False, 6.0), (200, 128, True, 1.0)])
def test_the_steps_together_stay_within_the_bounds(dtype, L, D, causal, sharp):
    for name, error in _errors(dtype, L, D, causal, sharp).items():
        assert error <= MOST[name], (name, error)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("L,D,causal", [(300, 64, True), (700, 32, False)])
def test_without_one_of_them_they_do_not(dtype, L, D, causal):
    assert _errors(dtype, L, D, causal, 6.0, left=False)["dq"] > MOST["dq"]
    assert _errors(dtype, L, D, causal, 6.0, two=False)["dq"] > MOST["dq"]
    assert _errors(dtype, L, D, causal, 6.0, left=False, mended=False)["dk"] > MOST["dk"]
    if dtype == F16:
        small = _errors(dtype, 2000, 64, False, 1.0, shift=False, size=1e-3)
        assert small["dq"] > MOST["dq"] and small["dk"] > MOST["dk"]
        assert all(e <= MOST[n] for n, e in _errors(dtype, 2000, 64, False, 1.0, size=1e-3).items())
