"""Rotary positions on the GPU against their formula in 64 bits.

Sine and cosine are off by up to 2^-23 (their argument's and their own rounding, and the polynomials' 2e-9), the scale and two products and a sum round once more
each: 6 * 2^-24 of |x_i| + |x_j|; the result is rounded to its type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _formula(x, positions, turns, interleaved, scale, inverse=False):
    """(the turned values, how far from them a result may lie) in 64 bits; positions [N] or [B,N]."""
    R = 2 * turns.numel()
    fraction = (positions.long()[..., None] * turns).double() / 2.0 ** 64 * (2 * math.pi)     # (int64 wraps around)
    while fraction.dim() < x.dim() - 1:
        fraction = fraction.unsqueeze(-3 if positions.dim() == 2 else 0)
    fraction = fraction.unsqueeze(-2)
    c, s = scale * fraction.cos(), scale * fraction.sin() * (-1 if inverse else 1)
    at = torch.arange(R // 2, device=x.device)
    i, j = (2 * at, 2 * at + 1) if interleaved else (at, at + R // 2)
    y, size = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    a, b = x[..., i].double(), x[..., j].double()
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    size[..., i] = size[..., j] = (a.abs() + b.abs()) * abs(scale)
    f = torch.finfo(x.dtype)
    return y, size * 6 * 2.0 ** -24 + (y.abs() * f.eps / 2 + f.tiny * f.eps / 2) * (x.dtype != F32 or 1)


def _close(got, want_bound):
    want, bound = want_bound
    assert got.shape == want.shape and got.is_contiguous()
    off = (got.double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())


# dtype, shape before the heads, H, Hk (0: no keys), D, R, interleaved, positions' type, batches of positions, how far they reach, scale
CASES = [
    (F32, (1,), 1, 1, 2, 2, False, torch.int64, 0, 0, 1.0),
    (F32, (3,), 1, 2, 7, 4, True, torch.int32, 0, 10, 1.0),
    (BF16, (5,), 2, 1, 8, 8, False, torch.int64, 0, 100, 1.0),
    (BF16, (4,), 8, 8, 32, 32, False, torch.int64, 0, 8192, 1.0),
    (F16, (67,), 4, 1, 40, 20, True, torch.int64, 0, 200000, 1.1),
    (F16, (67,), 4, 1, 40, 20, False, torch.int64, 0, 200000, 0.7),
    (F32, (130,), 12, 4, 80, 40, True, torch.int32, 0, 20000, 1.2),
    (BF16, (3, 41), 5, 0, 64, 64, True, torch.int64, 3, 1000, 1.0),
    (BF16, (2, 5, 33), 8, 8, 32, 24, False, torch.int64, 2, 300, 1.0),
    (BF16, (2, 5, 33), 8, 8, 32, 32, False, torch.int16, 1, 300, 1.0),
    (F16, (2, 5, 33), 3, 2, 128, 128, False, torch.int64, 0, 2 ** 31, 1.0),
    (F32, (999,), 33, 7, 96, 96, False, torch.int64, 0, 2 ** 38, 1.0),      # some heads to a thread
    (BF16, (2100,), 32, 8, 128, 128, False, torch.int64, 0, 100000, 1.0),
    (BF16, (2100,), 32, 8, 128, 64, True, torch.uint8, 0, 200, -2.0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c))
def test_the_formula_and_its_gradient(gpu_device, case):
    from evoformer_triton_amd import rotary_positions, rotary_turns
    dtype, lead, H, Hk, D, R, interleaved, index, batches, reach, scale = case
    g = torch.Generator(device="cuda:0").manual_seed(3)
    turns = rotary_turns(R, device="cuda:0")
    low = 0 if index == torch.uint8 else -reach
    at = torch.randint(low, reach + 1, ((batches,) if batches else ()) + lead[-1:], device="cuda:0", generator=g).to(index)
    q, k = (torch.randn((*lead, h, D), device="cuda:0", generator=g).to(dtype) if h else None for h in (H, Hk))
    leaves = [t.requires_grad_() for t in (q, k) if t is not None]
    out = rotary_positions(q, k, at, turns, interleaved=interleaved, scale=scale)
    outs = [out] if k is None else list(out)
    douts = [torch.randn(t.shape, device="cuda:0", generator=g).to(dtype) for t in leaves]
    grads = torch.autograd.grad(outs, leaves, douts)
    for x, y, dy, dx in zip(leaves, outs, douts, grads):
        assert y.dtype == dtype and dx.dtype == dtype
        _close(y, _formula(x.detach(), at, turns, interleaved, scale))
        _close(dx, _formula(dy, at, turns, interleaved, scale, inverse=True))
        assert torch.equal(y[..., R:], x[..., R:]) and torch.equal(dx[..., R:], dy[..., R:])


def test_strides_and_alignment(gpu_device):
    from evoformer_triton_amd import rotary_positions, rotary_turns
    g = torch.Generator(device="cuda:0").manual_seed(4)
    turns, at = rotary_turns(32, device="cuda:0"), torch.arange(50, device="cuda:0") * 3
    for dtype in (BF16, F32):
        for interleaved in (False, True):
            q, k = (torch.randn((50, h, 32), device="cuda:0", generator=g).to(dtype) for h in (4, 2))

            def turn(a, b, p=at):
                return rotary_positions(a, b, p, turns, interleaved=interleaved)

            want = turn(q, k)
            P = torch.cat([q, k], 1)
            wide = torch.zeros((50, 6, 35), dtype=dtype, device="cuda:0")     # rows at odd addresses
            wide[..., 1:33] = P
            every = torch.zeros((50, 6, 64), dtype=dtype, device="cuda:0")
            every[..., ::2] = P
            for x in (P, wide[..., 1:33], every[..., ::2], P.transpose(0, 1).contiguous().transpose(0, 1)):
                for a, b in zip(turn(x[:, :4], x[:, 4:]), want):
                    assert torch.equal(a, b)
            # even addresses that are no multiples of 16 bytes
            even = torch.zeros((50, 6, 36), dtype=dtype, device="cuda:0")[..., 2:34]
            even.copy_(P)
            for a, b in zip(turn(even[:, :4], even[:, 4:]), want):
                assert torch.equal(a, b)
            for p in (torch.stack([at, at * 0], 1)[:, 0], at.to(torch.int32)):
                for a, b in zip(turn(q, k, p), want):
                    assert torch.equal(a, b)
            one = k[:, :1].expand(-1, 4, -1)
            assert torch.equal(turn(one, None) if False else rotary_positions(one, None, at, turns, interleaved=interleaved), turn(one.contiguous(), k)[0])


def test_turned_there_and_back(gpu_device):
    """Products depend on the difference of positions, also far out where fp32 angles have lost their fraction."""
    from evoformer_triton_amd import RotaryPositions
    r = RotaryPositions(64, base=500000.0).to("cuda:0")
    g = torch.Generator(device="cuda:0").manual_seed(5)
    q, k = (torch.randn((40, 2, 64), device="cuda:0", generator=g) for _ in range(2))
    at = torch.randint(0, 300, (40,), device="cuda:0", generator=g)
    near = [(a * b).double().sum(-1) for a, b in [r(q, k, at)]]
    # the key turned as far as the query: the products are those of the unturned
    assert (near[0] - (q.double() * k.double()).sum(-1)).abs().max() < 64 * 16 * 2.0 ** -22
    for far in (2 ** 20, 2 ** 34, -2 ** 34):
        a = r(q, None, at + far), r(k, None, at * 0 + far)
        b = r(q, None, at), r(k, None, at * 0)
        x, y = ((u.double() * w.double()).sum(-1) for u, w in (a, b))
        # (angles to 2^-24 turns: some 4e-7 of each product)
        assert (x - y).abs().max() < 64 * 16 * 2.0 ** -20


def test_one_gradient_only_and_many(gpu_device):
    from evoformer_triton_amd import rotary_positions, rotary_turns
    g = torch.Generator(device="cuda:0").manual_seed(6)
    turns, at = rotary_turns(16, device="cuda:0"), torch.arange(30, device="cuda:0")
    q, k, dq, dk = (torch.randn((30, h, 16), device="cuda:0", generator=g) for h in (3, 2, 3, 2))
    leaves = [q.requires_grad_(), k.requires_grad_()]
    a, b = rotary_positions(*leaves, at, turns)
    want = torch.autograd.grad([a, b], leaves, [dq, dk], retain_graph=True)
    assert torch.equal(torch.autograd.grad(a, q, dq, retain_graph=True)[0], want[0])
    assert torch.equal(torch.autograd.grad(b, k, dk, retain_graph=True)[0], want[1])
    only = rotary_positions(q.detach(), k, at, turns)[1]
    assert torch.equal(torch.autograd.grad(only, k, dk)[0], want[1])
    a.sum().backward()
    assert torch.isfinite(q.grad).all()
    (d,) = torch.autograd.grad(rotary_positions(q, None, at, turns), q, dq, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        d.sum().backward()
    out = rotary_positions(q, None, at, turns)
    with torch.no_grad():
        at.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_a_captured_step_replays(gpu_device):
    from evoformer_triton_amd import rotary_positions, rotary_turns
    turns, at = rotary_turns(32, device="cuda:0"), torch.arange(300, device="cuda:0")
    q, k = (torch.randn((300, h, 64), device="cuda:0", dtype=BF16) for h in (8, 2))

    def step(leaves):
        outs = rotary_positions(*leaves, at, turns)
        return [*outs, *torch.autograd.grad(outs, leaves, [q * 0.5, k * 0.5])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.detach().requires_grad_() for t in (q, k)])
    torch.cuda.current_stream().wait_stream(side)
    leaves = [t.detach().requires_grad_() for t in (q, k)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = step(leaves)
    for shift in (0, 1000, -7):
        at.copy_(torch.arange(300) + shift)
        q.normal_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step([t.detach().requires_grad_() for t in (q, k)])):
            assert torch.equal(a, b)


def test_compiled_and_registered(gpu_device):
    from evoformer_triton_amd import RotaryPositions, rotary_positions
    r = RotaryPositions(32, rotary_dim=16, interleaved=True).to("cuda:0")
    q, k = (torch.randn((2, 20, h, 32), device="cuda:0").requires_grad_() for h in (4, 2))
    at = torch.arange(20, device="cuda:0")

    def step(q, k):
        a, b = r(q * 1.0, k, at)
        return a.sum() + (b * b).sum()

    want = torch.autograd.grad(step(q, k), [q, k])
    got = torch.autograd.grad(torch.compile(step, fullgraph=True, backend="aot_eager")(q, k), [q, k])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    torch.library.opcheck(torch.ops.evoattn.rotary, (q, k, at, r.turns, True, 1.0, False), test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_static"))
    with pytest.raises(NotImplementedError, match="forward mode"):
        with torch.autograd.forward_ad.dual_level():
            rotary_positions(torch.autograd.forward_ad.make_dual(q.detach(), q.detach()), None, at, r.turns)
    assert rotary_positions(q[:, :0], k[:, :0], at[:0], r.turns)[0].shape == (2, 0, 4, 32)
