"""Attention within packed sequences on the GPU against its formula in 64 bits (oracle/packed.py, which also says how far a result may lie from it)."""
import math

import pytest
import torch

from oracle.packed import packed

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _offsets(lengths, device="cuda:0", dtype=torch.int32):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at, torch.tensor(at, device=device, dtype=dtype)


def _inputs(dtype, queries, keys, H, Hk, D, padding=0, seed=1, sharp=1.0):
    g = torch.Generator(device="cuda:0").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device="cuda:0", generator=g)

    T, Tk = sum(queries) + padding, sum(keys) + padding
    return [(normal(T, H, D) * sharp).to(dtype), normal(Tk, Hk, D).to(dtype), normal(Tk, Hk, D).to(dtype), normal(T, H, D).to(dtype)]


def _close(got, want, bound, what):
    for name, g, w, b in zip(what, got, want, bound):
        assert g.shape == w.shape, name
        off = (g.double() - w).abs()
        bad = ~(off <= b)
        assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} beyond the bound, the worst {float((off / b).nan_to_num(math.inf).max()):.3g} times it"


def _check(q, k, v, dout, queries, keys, causal, scale=None, grad=True, index=torch.int32):
    from evoformer_triton_amd import packed_attention
    D = q.shape[2]
    a, off = _offsets(queries, dtype=index)
    b, koff = _offsets(keys, dtype=index)
    same = queries == keys
    leaves = [t.detach().requires_grad_() for t in (q, k, v)] if grad else [q, k, v]
    out = packed_attention(*leaves, off, None if same else koff, causal=causal, scale=scale)
    got = [out, *torch.autograd.grad(out, leaves, dout)] if grad else [out]
    want, bound = packed(q, k, v, a, b, causal, D ** -0.5 if scale is None else scale, dout if grad else None)
    assert all(t.dtype == q.dtype and t.is_contiguous() for t in got)
    _close(got, want, bound, ("o", "dq", "dk", "dv"))
    return got


# dtype, queries' lengths, keys' lengths (None: the queries'), H, Hk, D, causal, rows of no sequence
CASES = [
    (F32, [1], None, 1, 1, 1, True, 0),
    (F32, [5, 0, 70, 1], None, 4, 2, 24, True, 3),
    (F32, [65, 130], [70, 131], 3, 1, 128, True, 0),
    (F32, [33], [7], 2, 2, 65, False, 1),
    (BF16, [1], None, 1, 1, 8, True, 0),
    (BF16, [2, 3, 1], None, 2, 1, 32, True, 0),
    (F16, [31, 32, 33], None, 4, 4, 32, False, 5),
    (BF16, [63, 64, 65, 0, 0, 1], None, 4, 2, 64, True, 2),
    (F16, [127, 128, 129], None, 3, 3, 64, True, 0),
    (BF16, [255, 257, 10], None, 8, 2, 128, True, 0),
    (F16, [300], None, 6, 2, 128, False, 0),
    (BF16, [200, 71], None, 4, 1, 96, True, 40),
    (F16, [200, 71], None, 4, 1, 80, False, 40),
    (BF16, [190], None, 2, 1, 40, True, 0),
    (BF16, [190, 3], None, 2, 1, 13, True, 1),            # a head dim that is padded
    (F16, [77], None, 2, 2, 128, False, 300),             # whole tiles of no sequence
    (BF16, [700, 20], None, 4, 4, 32, False, 0),
    (BF16, [600], None, 4, 2, 128, True, 0),
    # fewer queries than keys, and more (rows that see no key)
    (BF16, [1, 1, 1], [1, 100, 1000], 8, 2, 64, True, 0),
    (F16, [1] * 9, [3, 64, 65, 127, 128, 129, 500, 0, 2000], 8, 8, 128, True, 0),
    (BF16, [1], [5000], 16, 2, 128, True, 0),
    (F16, [3, 0, 5], [300, 7, 5], 12, 4, 80, True, 0),
    (BF16, [17, 2], [900, 40], 8, 1, 64, True, 0),
    (BF16, [130], [400], 4, 2, 128, True, 0),
    (F16, [130, 1], [40, 64], 4, 2, 64, True, 7),         # 90 queries see nothing
    (BF16, [10, 200], [3, 1], 2, 2, 32, True, 0),
    (BF16, [40, 9], [0, 9], 2, 2, 128, False, 0),         # a sequence without keys
    (F16, [4, 4], [64, 250], 32, 4, 64, False, 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c))
def test_the_formula_and_its_gradients(gpu_device, case):
    dtype, queries, keys, H, Hk, D, causal, padding = case
    keys = keys or queries
    q, k, v, dout = _inputs(dtype, queries, keys, H, Hk, D, padding)
    got = _check(q, k, v, dout, queries, keys, causal)
    alone = _check(q, k, v, dout, queries, keys, causal, grad=False)     # (the forward without a backward: the same bits)
    assert torch.equal(got[0], alone[0])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_sharp_scores_and_other_scales(gpu_device, dtype):
    q, k, v, dout = _inputs(dtype, [150, 90], [150, 90], 4, 2, 64, sharp=12.0)
    _check(q, k, v, dout, [150, 90], [150, 90], True)
    _check(q, k, v, dout, [150, 90], [150, 90], False, scale=0.01)
    q, k, v, _ = _inputs(dtype, [1, 1], [900, 90], 4, 2, 64, sharp=12.0)
    _check(q, k, v, None, [1, 1], [900, 90], True, grad=False)


@pytest.mark.parametrize("queries", [[200], [1]])
def test_scores_that_grow_and_fall_along_the_keys(gpu_device, queries):
    """The running maximum moves at every tile, or is that of the first one."""
    for sign in (1.0, -1.0):
        q, k, v, dout = _inputs(BF16, queries, [1500], 2, 1, 64)
        q[..., 0] = 30.0
        k[..., 0] = (sign * torch.linspace(-20, 20, 1500, device=k.device))[:, None].to(BF16)
        _check(q, k, v, dout, queries, [1500], True)
    # scores far below zero, all alike
    q, k, v, dout = _inputs(BF16, queries, [300], 2, 1, 64)
    q[..., 0], k[..., 0] = 60.0, -60.0
    _check(q, k, v, dout, queries, [300], True)


def test_64_bit_offsets(gpu_device):
    q, k, v, dout = _inputs(BF16, [40, 90], [40, 90], 2, 2, 32)
    _check(q, k, v, dout, [40, 90], [40, 90], True, index=torch.int64)
    from evoformer_triton_amd import packed_attention
    mixed = packed_attention(q, k, v, _offsets([40, 90])[1], _offsets([40, 90], dtype=torch.int64)[1])
    assert torch.equal(mixed, packed_attention(q, k, v, _offsets([40, 90])[1]))


def test_many_sequences(gpu_device):
    """More than a wave asks for at once, empty ones among them, and single rows."""
    from evoformer_triton_amd import packed_attention
    for lengths in ([1] * 5000, [i % 7 for i in range(700)], [0] * 4200 + [9] + [0] * 100):
        q, k, v, dout = _inputs(BF16, lengths, lengths, 2, 1, 32)
        _check(q, k, v, dout, lengths, lengths, True)
    lengths = [1] * 300
    q, k, v, _ = _inputs(F16, lengths, [5] * 300, 8, 2, 64)
    _check(q, k, v, None, lengths, [5] * 300, True, grad=False)
    out = packed_attention(q, k, v, torch.zeros(1, device="cuda:0", dtype=torch.int32), torch.zeros(1, device="cuda:0", dtype=torch.int32))
    assert not out.any()      # no sequence: zeros


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64), (BF16, 32), (F32, 40)])
def test_what_is_not_seen_does_not_reach_a_result(gpu_device, dtype, D):
    """Infinities and NaN in rows of no sequence, in other sequences and in rows that causal queries do not see: the same bits as with numbers there."""
    from evoformer_triton_amd import packed_attention
    lengths = [70, 130, 45]
    q, k, v, dout = _inputs(dtype, lengths, lengths, 4, 2, D, padding=30)
    _, off = _offsets(lengths)
    bad = [float("nan"), float("inf"), -float("inf")]

    def step(q, k, v, dout):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = packed_attention(*leaves, off)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    want = step(q, k, v, dout)
    # rows behind the last sequence: everything else stays, and theirs are zeros
    for value in bad:
        spoilt = [t.clone() for t in (q, k, v, dout)]
        for t in spoilt:
            t[245:] = value
        got = step(*spoilt)
        for g, w in zip(got, want):
            assert torch.equal(g, w) and not g[245:].any()
    # the middle sequence's rows: the others' stay
    for value in bad:
        spoilt = [t.clone() for t in (q, k, v, dout)]
        for t in spoilt:
            t[70:200] = value
        for g, w in zip(step(*spoilt), want):
            assert torch.equal(g[:70], w[:70]) and torch.equal(g[200:], w[200:])
    # the last key and value of the middle sequence: only its last query sees them
    a, _ = _offsets(lengths)
    for value in bad:
        for which in (1, 2):
            spoilt = [q, k.clone(), v.clone(), dout]
            spoilt[which][199] = value
            got = step(*spoilt)
            keep = [i for i in range(245) if i != 199]
            exact, bounds = packed(q, k, v, a, a, True, D ** -0.5, dout)
            for i in (0, 1):     # o, dq of the queries that do not see it (by way of another kernel: within the bound, not bit for bit)
                _close([got[i][keep]], [exact[i][keep]], [bounds[i][keep]], [f"result {i}, input {which}"])
    # the first query's and its gradient: only the first key sees them, the others' gradients stay
    for value in bad:
        for which in (0, 3):
            spoilt = [q.clone(), k, v, dout.clone()]
            spoilt[which][70] = value
            got = step(*spoilt)
            keep = [i for i in range(245) if i != 70]
            exact, bounds = packed(q, k, v, a, a, True, D ** -0.5, dout)
            for i in (0, 1, 2, 3):
                if i == 0 and which == 3:
                    continue
                _close([got[i][keep]], [exact[i][keep]], [bounds[i][keep]], [f"result {i}, input {which}"])


def test_single_tokens_do_not_see_other_rows(gpu_device):
    from evoformer_triton_amd import packed_attention
    q, k, v, _ = _inputs(BF16, [1, 1], [70, 700], 8, 2, 128, padding=0)
    _, off = _offsets([1, 1])
    koff = torch.tensor([0, 70, 770], device="cuda:0", dtype=torch.int32)
    big = [torch.cat([t, torch.full_like(t[:50], float("nan"))]) for t in (k, v)]
    assert torch.equal(packed_attention(q, *big, off, koff), packed_attention(q, k, v, off, koff))
    big[1][:70] = float("inf")
    assert torch.equal(packed_attention(q, *big, off, koff)[1], packed_attention(q, k, v, off, koff)[1])


def test_infinite_values_that_are_seen(gpu_device):
    from evoformer_triton_amd import packed_attention
    q, k, v, _ = _inputs(BF16, [100], [100], 2, 1, 64)
    v[50, 0, 3] = float("inf")
    v[60, 0, 5] = float("nan")
    out = packed_attention(q, k, v, _offsets([100])[1])
    assert torch.isposinf(out[50:, :, 3]).all() and torch.isnan(out[60:, :, 5]).all()
    assert torch.isfinite(out[:50]).all() and torch.isfinite(out[..., 6:]).all()


def test_bad_offsets_stay_in_bounds(gpu_device):
    """Offsets beyond the rows, negative or descending: no access leaves the tensors (what the rows hold is not specified), and good rows' neighbours are not asked for."""
    from evoformer_triton_amd import packed_attention
    for dtype in (BF16, F32):
        q, k, v, dout = (t.requires_grad_() for t in _inputs(dtype, [100], [100], 2, 1, 32))
        for bad in ([0, 1000], [-5, 100], [50, 20, 100], [0, 2 ** 31 - 1], [-2 ** 31, 2 ** 31 - 1], [100, 0]):
            off = torch.tensor(bad, device="cuda:0", dtype=torch.int64)
            out = packed_attention(q, k, v, off)
            torch.autograd.grad(out, [q, k, v], dout)
        torch.cuda.synchronize()


def test_strides_and_alignment(gpu_device):
    """Slices of a projection's result, heads before rows, odd addresses, heads that are expanded."""
    from evoformer_triton_amd import packed_attention
    lengths = [60, 77]
    _, off = _offsets(lengths)
    for dtype in (BF16, F32):
        q, k, v, dout = _inputs(dtype, lengths, lengths, 4, 4, 64)
        want = packed_attention(q, k, v, off)
        P = torch.stack([q, k, v], 1)
        assert torch.equal(packed_attention(P[:, 0], P[:, 1], P[:, 2], off), want)
        heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
        assert torch.equal(packed_attention(*heads_first, off), want)

        def odd(t):
            x = torch.empty(t.numel() + 1, dtype=dtype, device=t.device)[1:].view(t.shape)
            return x.copy_(t)

        assert torch.equal(packed_attention(odd(q), odd(k), odd(v), off), want)
        wide = torch.zeros(137, 4, 130, dtype=dtype, device="cuda:0")
        wide[..., 1:65] = q
        assert torch.equal(packed_attention(wide[..., 1:65], k, v, off), want)
        step2 = torch.zeros(137, 4, 128, dtype=dtype, device="cuda:0")
        step2[..., ::2] = k
        assert torch.equal(packed_attention(q, step2[..., ::2], v, off), want)
        # a key head for all, expanded: its gradient is the sum over the heads
        one, one_v = k[:, :1].detach().requires_grad_(), v[:, :1].detach().requires_grad_()
        a = packed_attention(q, one.expand(-1, 4, -1), one_v.expand(-1, 4, -1), off)
        b = packed_attention(q, one, one_v, off)
        assert torch.equal(a, b)
        ga, gb = torch.autograd.grad(a, [one, one_v], dout), torch.autograd.grad(b, [one, one_v], dout)
        for x, y in zip(ga, gb):
            assert (x.float() - y.float()).abs().max() <= 8 * torch.finfo(dtype).eps * y.float().abs().max() + 1e-5
        # the result's gradient in other layouts
        t = dout.transpose(0, 1).contiguous().transpose(0, 1)
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = packed_attention(*leaves, off)
        first = torch.autograd.grad(out, leaves, dout, retain_graph=True)
        for other in (t, odd(dout)):
            for x, y in zip(torch.autograd.grad(out, leaves, other, retain_graph=True), first):
                assert torch.equal(x, y)
        out.sum().backward()      # (a gradient that is expanded from one number)
        assert all(torch.isfinite(x.grad).all() for x in leaves)


def test_gradients_are_the_differences(gpu_device):
    from evoformer_triton_amd import packed_attention
    lengths = [9, 30]
    q, k, v, dout = _inputs(F32, lengths, lengths, 4, 2, 16)
    _, off = _offsets(lengths)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = packed_attention(*leaves, off)
    grads = torch.autograd.grad(out, leaves, dout)
    g = torch.Generator(device="cuda:0").manual_seed(9)
    for i, (x, d) in enumerate(zip(leaves, grads)):
        way = torch.randn(x.shape, device=x.device, generator=g)
        h = 2.0 ** -7
        ends = []
        for s in (h, -h):
            moved = [t.detach() for t in leaves]
            moved[i] = moved[i] + s * way
            ends.append((packed_attention(*moved, off).double() * dout.double()).sum())
        slope, want = float((ends[0] - ends[1]) / (2 * h)), float((d.double() * way.double()).sum())
        # the differences' error: fp32 roundings (some 2^-20 of the sum over h) and the third derivative's h^2
        assert abs(slope - want) <= 2e-3 * max(1.0, float((d.double().abs() * way.double().abs()).sum())), (i, slope, want)


def test_two_calls_give_the_same_bits_and_streams_are_kept(gpu_device):
    from evoformer_triton_amd import packed_attention
    lengths = [500, 300, 3]
    q, k, v, dout = _inputs(BF16, lengths, lengths, 8, 2, 64)
    _, off = _offsets(lengths)

    def step():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = packed_attention(*leaves, off)
        return [out, *torch.autograd.grad(out, leaves, dout)]

    first = step()
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, other):
        assert torch.equal(a, b)


def test_a_captured_call_replays_with_other_offsets(gpu_device):
    """Everything that depends on the lengths is read on the device: a graph follows what its tensors hold."""
    from evoformer_triton_amd import packed_attention
    g = torch.cuda.CUDAGraph()
    q, k, v, dout = _inputs(BF16, [400], [400], 4, 2, 64)
    lists = [[400], [0, 100, 400], [0, 3, 4, 400]]
    off = torch.tensor([0, 100, 250, 400], device="cuda:0", dtype=torch.int32)

    def step(leaves):
        out = packed_attention(*leaves, off)
        return [out, *torch.autograd.grad(out, leaves, dout)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step([t.detach().requires_grad_() for t in (q, k, v)])
    torch.cuda.current_stream().wait_stream(side)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    with torch.cuda.graph(g):
        held = step(leaves)
    for at in ([0, 100, 250, 400], [0, 0, 399, 400], [0, 133, 133, 350], [0, 100, 250, 400]):
        off.copy_(torch.tensor(at, dtype=torch.int32))
        q.normal_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step([t.detach().requires_grad_() for t in (q, k, v)])):
            assert torch.equal(a, b)
    assert lists


def test_captured_single_tokens_share_no_scratch(gpu_device):
    """Two graphs of split keys, replayed in turn, with eager calls between."""
    from evoformer_triton_amd import packed_attention
    calls = []
    for seed in (1, 2):
        q, k, v, _ = _inputs(BF16, [1, 1], [3000 * seed, 77], 8, 2, 64, seed=seed)
        off, koff = _offsets([1, 1])[1], _offsets([3000 * seed, 77])[1]
        calls.append(lambda q=q, k=k, v=v, off=off, koff=koff: packed_attention(q, k, v, off, koff))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    graphs = []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = c()
        graphs.append((g, out))
    for _ in range(3):
        for (g, out), w, c in zip(graphs, want, calls):
            out.zero_()
            g.replay()
            assert torch.equal(c(), w)
            torch.cuda.synchronize()
            assert torch.equal(out, w)


def test_compiled_and_registered(gpu_device):
    from evoformer_triton_amd import packed_attention
    q, k, v, dout = _inputs(BF16, [50, 60], [50, 60], 4, 2, 32)
    _, off = _offsets([50, 60])

    def step(q, k, v):
        return packed_attention(q * 1.0, k, v, off)

    leaves = [t.requires_grad_() for t in (q, k, v)]
    want = step(*leaves)
    grads = torch.autograd.grad(want, leaves, dout)
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(*leaves)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, leaves, dout), grads):
        assert torch.equal(a, b)
    torch.library.opcheck(torch.ops.evoattn.packed, (*leaves, off, None, True, None), test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_static"))


def test_refusals_on_the_gpu(gpu_device):
    from evoformer_triton_amd import packed_attention
    q, k, v, dout = _inputs(BF16, [50], [50], 4, 2, 32)
    _, off = _offsets([50])
    with pytest.raises(ValueError, match="one device"):
        packed_attention(q, k, v, off.cpu())
    with pytest.raises(NotImplementedError, match="forward mode"):
        with torch.autograd.forward_ad.dual_level():
            packed_attention(torch.autograd.forward_ad.make_dual(q, q), k, v, off)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = packed_attention(*leaves, off)
    (d,) = torch.autograd.grad(out, [q], dout, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        d.sum().backward()
    out = packed_attention(*leaves, off)
    with torch.no_grad():
        off.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(dout)
    # no rows
    empty = packed_attention(q[:0], k[:0], v[:0], off)
    assert empty.shape == (0, 4, 32)


def test_some_gradients_only(gpu_device):
    from evoformer_triton_amd import packed_attention
    q, k, v, dout = _inputs(BF16, [90], [90], 4, 2, 64)
    _, off = _offsets([90])
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(packed_attention(*leaves, off), leaves, dout)
    for i in range(3):
        some = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        (g,) = torch.autograd.grad(packed_attention(*some, off), [some[i]], dout)
        assert torch.equal(g, want[i])
