"""Packed attention of inputs that are no numbers: what a row sees decides about its results, column by column, and how long a call takes does not depend on it."""
import math

import pytest
import torch

from test_gpu_packed import BF16, F16, F32, _inputs, _offsets

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


def _formula(q, k, v, dout, queries, keys, causal):
    """([o, dq, dk, dv], [sums of their terms' absolute values]) in 64 bits, each row from the rows alone that it sees."""
    (_, H, D), Hk = q.shape, k.shape[1]
    q, k, v, dout = (t.double().cpu() for t in (q, k, v, dout))
    outs = [torch.zeros_like(t) for t in (q, q, k, v)]
    sizes = [torch.zeros_like(t) for t in outs]
    a = b = 0
    for n, m in zip(queries, keys):
        for h in range(H):
            hk = h // (H // Hk)
            for i in range(n):
                seen = max(0, min(m, m - n + i + 1)) if causal else m
                if not seen:
                    continue
                K, V, row, s = k[b:b + seen, hk], v[b:b + seen, hk], (a + i, h), slice(b, b + seen)
                x = (K * q[row]).sum(-1) / math.sqrt(D)
                e = torch.exp(x - x.max())
                P = e / e.sum()
                outs[0][row] = (P[:, None] * V).sum(0)
                dP = (V * dout[row]).sum(-1)
                dS = P * (dP - (P * dP).sum()) / math.sqrt(D)
                outs[1][row] = (dS[:, None] * K).sum(0)
                outs[2][s, hk] += dS[:, None] * q[row]
                outs[3][s, hk] += P[:, None] * dout[row]
                size = (V.abs() * dout[row].abs()).sum(-1)
                size = P * (size + (P * size).sum()) / math.sqrt(D)
                sizes[0][row] = (P[:, None] * V.abs()).sum(0)
                sizes[1][row] = (size[:, None] * K.abs()).sum(0)
                sizes[2][s, hk] += size[:, None] * q[row].abs()
                sizes[3][s, hk] += P[:, None] * dout[row].abs()
        a, b = a + n, b + m
    return outs, sizes


def _same(q, k, v, dout, queries, keys, causal, what):
    """Numbers where the formula has numbers, each term of a sum within eight roundings, and none where it has none."""
    from evoformer_triton_amd import packed_attention
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = packed_attention(*leaves, _offsets(queries)[1], _offsets(keys)[1], causal=causal)
    got = [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    few = packed_attention(q, k, v, _offsets(queries)[1], _offsets(keys)[1], causal=causal)
    assert torch.equal(few.nan_to_num(1.0), got[0].nan_to_num(1.0))
    eps = max(torch.finfo(q.dtype).eps, 2.0 ** -18)      # (fp32: 128 products and as many sums)
    for name, g, w, size in zip(("o", "dq", "dk", "dv"), got, *_formula(q, k, v, dout, queries, keys, causal)):
        g = g.double().cpu()
        assert torch.equal(torch.isfinite(g), torch.isfinite(w)), (what, name, int((torch.isfinite(g) != torch.isfinite(w)).sum()))
        fine = torch.isfinite(w)
        assert ((g - w).abs()[fine] <= 8 * eps * size[fine] + 1e-6).all(), (what, name)


# dtype, queries, keys, H, Hk, D, causal: whole sequences by one group of waves and by parts of a walk, the last queries, few of them
PATHS = [
    (BF16, [75, 131], None, 2, 1, 64, True), (F16, [75, 131], None, 2, 2, 128, True), (F16, [333], None, 2, 1, 32, False), (BF16, [90, 75], [170, 110], 2, 2, 96, True),
    (F32, [75, 131], None, 2, 1, 64, True), (F32, [60], [333], 2, 2, 40, True), (BF16, [3, 2], [210, 77], 4, 2, 64, True), (F32, [3, 2], [210, 77], 4, 2, 64, True),
    (F16, [1050], None, 1, 1, 64, True), (F32, [1050], None, 1, 1, 32, True), (BF16, [4, 9], [900, 1400], 2, 1, 128, True),
]


@pytest.mark.parametrize("path", PATHS, ids=lambda c: "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c))
def test_numbers_where_the_formula_has_them(gpu_device, path):
    dtype, queries, keys, H, Hk, D, causal = path
    keys = keys or queries
    base = _inputs(dtype, queries, keys, H, Hk, D)
    g = torch.Generator(device="cuda:0").manual_seed(2)
    Tq, Tk = sum(queries), sum(keys)

    def spoilt(which, change):
        x = [t.clone() for t in base]
        change(x[which])
        _same(*x, queries, keys, causal, (which, change.__name__))

    def some_infinities(t):        # of either sign, in a third of the rows
        hit = (torch.rand(t.shape, device=t.device, generator=g) < 0.1) & (torch.rand(t.shape[0], 1, 1, device=t.device, generator=g) < 0.33)
        t[hit] = torch.where(torch.rand(int(hit.sum()), device=t.device, generator=g) < 0.5, INF, -INF).to(t.dtype)

    def one_row(t):
        t[t.shape[0] // 3] = NAN

    def one_infinity(t):
        t[t.shape[0] // 2, 0, 3] = INF

    def the_end(t):
        t[-2:, :, 1] = -INF

    def a_column(t):
        t[:, :, 2] = NAN

    def everything(t):
        t.fill_(NAN)

    for change in (some_infinities, one_row, one_infinity, the_end, a_column, everything):
        spoilt(3, change)
        spoilt(2, change)
    for change in (one_row, everything):
        spoilt(0, change)
        spoilt(1, change)
    # keys that a score of minus infinity takes out: probabilities of zero, no NaN but in the column where zero meets the infinity (dq's)
    x = [t.clone() for t in base]
    x[0][..., 0] = x[0][..., 0].abs() + 0.25
    x[1][Tk // 3, :, 0] = x[1][Tk - 3, :, 0] = -INF
    _same(*x, queries, keys, causal, "minus infinity")
    # seen and unseen ones in different columns
    x = [t.clone() for t in base]
    x[2][Tk // 4, :, 1] = INF
    x[2][Tk // 4 + 2:, :, 5] = NAN
    x[3][Tq // 4:, :, 4] = INF
    x[3][:Tq // 4, :, 6] = NAN
    _same(*x, queries, keys, causal, "columns")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_a_step_without_numbers_takes_no_longer(gpu_device, dtype):
    """An incoming gradient that has overflowed as a whole, one whose row has, and values that have: a few times what a step of numbers takes, where rows that are formed one by one took hundreds of times."""
    from evoformer_triton_amd import packed_attention
    lengths = [2048, 1024]
    q, k, v, dout = _inputs(dtype, lengths, lengths, 8, 8, 64)
    off = _offsets(lengths)[1]

    def step(q, k, v, dout):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        return torch.autograd.grad(packed_attention(*leaves, off), leaves, dout)

    def time(*x):
        step(*x)
        times = []
        for _ in range(3):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            step(*x)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    clean = max(time(q, k, v, dout), 0.1)
    nothing = torch.full_like(dout, NAN)
    overflown = torch.where(torch.rand(dout.shape, device="cuda:0") < 0.5, INF, -INF).to(dtype)
    last = dout.clone()
    last[2047] = NAN
    for what, x in (("all", (q, k, v, nothing)), ("infinities", (q, k, v, overflown)), ("the last query", (q, k, v, last)), ("values", (q, k, nothing, dout)), ("keys", (q, nothing, v, dout))):
        assert time(*x) <= 8 * clean, (what, time(*x), clean)
