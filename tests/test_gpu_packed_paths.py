"""Packed attention where the kernels split their work: long walks shared by groups of waves and by workgroups, few queries in all their arrangements, tensors beyond 32 bits."""
import pytest
import torch

from oracle.packed import packed
from test_gpu_packed import BF16, F16, F32, _check, _close, _inputs, _offsets

pytestmark = pytest.mark.gpu

# dtype, queries' lengths, keys' lengths (None: the queries'), H, Hk, D, causal
LONG = [
    # parts of a walk in workgroups of their own, joined
    (BF16, [2200], None, 2, 1, 64, True),
    (F16, [1500], None, 2, 2, 128, False),
    (BF16, [1900], None, 2, 1, 32, True),
    (F16, [1700, 1], None, 2, 1, 80, True),
    (BF16, [130], [4100], 2, 1, 128, True),        # few rows, a long walk
    (F16, [2500], [100], 2, 1, 64, False),          # and the other way around
    # two groups of waves to a tile
    (BF16, [1000, 900, 1100, 777], None, 10, 10, 64, True),
    (F16, [1024, 1000, 900], None, 12, 6, 96, False),
    (BF16, [1200, 0, 1300], None, 12, 12, 128, True),
    (BF16, [800] * 4, None, 16, 16, 32, True),
    # one
    (F16, [300] * 9, None, 12, 4, 128, True),
    (BF16, [520, 3, 700] * 4, None, 12, 12, 64, False),
    # fp32: in parts, in many of them for one token, without parts, vectors that are not 16 bytes long
    (F32, [2200], None, 2, 1, 128, True),
    (F32, [300, 0, 700, 1], None, 4, 2, 64, False),
    (F32, [1], [20000], 2, 1, 96, True),
    (F32, [130], [4100], 2, 2, 40, True),
    (F32, [2000], [90], 2, 1, 32, False),
    (F32, [700] * 12, None, 16, 8, 32, True),
    (F32, [1000, 33], None, 3, 3, 77, True),
]


@pytest.mark.parametrize("case", LONG, ids=lambda c: "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c))
def test_long_walks(gpu_device, case):
    dtype, queries, keys, H, Hk, D, causal = case
    keys = queries if keys is None else keys
    _check(*_inputs(dtype, queries, keys, H, Hk, D, padding=3), queries, keys, causal)


@pytest.mark.parametrize("dtype,D,H,Hk,lengths", [(BF16, 64, 2, 1, [2200, 40]), (F16, 128, 2, 2, [1500, 40]), (BF16, 96, 12, 12, [1200, 1300]), (F16, 32, 2, 1, [2000, 9]),
                                                   (F32, 64, 2, 1, [1500, 40]), (F32, 33, 12, 12, [1200, 1300])])
def test_long_walks_past_infinities_and_nan(gpu_device, dtype, D, H, Hk, lengths):
    """In rows of no sequence and in the second sequence: the same bits.  In the first one's last key: the queries that do not see it stay within their bounds."""
    from evoformer_triton_amd import packed_attention
    q, k, v, dout = _inputs(dtype, lengths, lengths, H, Hk, D, padding=70)
    at, off = _offsets(lengths)

    def step(q, k, v, dout):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = packed_attention(*leaves, off)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    want, first = step(q, k, v, dout), lengths[0]
    for value in (float("nan"), float("inf")):
        spoilt = [t.clone() for t in (q, k, v, dout)]
        for t in spoilt:
            t[first:] = value
        for g, w in zip(step(*spoilt), want):
            assert torch.equal(g[:first], w[:first]) and not g[at[-1]:].any()
    exact, bounds = packed(q, k, v, at, at, True, D ** -0.5, dout)
    for value in (float("nan"), float("inf")):
        for which in (1, 2):
            spoilt = [q, k.clone(), v.clone(), dout]
            spoilt[which][first - 1] = value
            got = step(*spoilt)
            for i in (0, 1):
                _close([got[i][:first - 1]], [exact[i][:first - 1]], [bounds[i][:first - 1]], [f"result {i}, input {which}, {value}"])


# dtype, queries, keys, H, Hk, D: by how many sequences and key heads there are (128 and more), by the queries that share a key head (16 and more of them), by the longest's length
FEW = [(dtype, [q] * n, [1 + (i * 37) % most for i in range(n)], H, Hk, D)
       for dtype, q, n, most, H, Hk, D in [
           (BF16, 1, 2, 9000, 4, 2, 64), (F16, 1, 2, 9000, 32, 1, 128), (BF16, 3, 3, 5000, 8, 1, 96), (F16, 1, 1, 20000, 8, 8, 32), (BF16, 5, 2, 700, 8, 2, 80),
           (F16, 1, 70, 300, 8, 2, 64), (BF16, 1, 70, 3000, 8, 2, 128), (F16, 2, 70, 2000, 32, 2, 96), (BF16, 1, 200, 1000, 24, 1, 32), (F16, 1, 64, 5000, 2, 2, 40),
           (F32, 1, 2, 9000, 4, 2, 64), (F32, 3, 3, 5000, 16, 1, 96), (F32, 1, 70, 300, 40, 2, 13), (F32, 1, 300, 100, 8, 8, 128), (F32, 2, 1, 33, 2, 2, 30)]]


@pytest.mark.parametrize("case", FEW, ids=lambda c: f"{c[0]}-{c[1][0]}x{len(c[1])}-{c[3:]}".replace("torch.", "").replace(" ", ""))
@pytest.mark.parametrize("causal", [True, False])
def test_few_queries(gpu_device, case, causal):
    dtype, queries, keys, H, Hk, D = case
    keys = [max(keys)] + keys[1:]
    q, k, v, _ = _inputs(dtype, queries, keys, H, Hk, D, padding=5)
    out, = _check(q, k, v, None, queries, keys, causal, grad=False)
    assert not out[sum(queries):].any()


def test_few_queries_with_gradients(gpu_device):
    for dtype, queries, keys, H, Hk, D in ((BF16, [1, 2], [3000, 500], 8, 2, 64), (F16, [1] * 40, [60] * 40, 4, 4, 128)):
        q, k, v, dout = _inputs(dtype, queries, keys, H, Hk, D)
        _check(q, k, v, dout, queries, keys, True)


def test_room_between_a_caches_sequences(gpu_device):
    """Sequences that have grown into the room that was left for them: what is left is a sequence without queries."""
    from evoformer_triton_amd import packed_attention
    room, lengths = 500, [137, 1, 499, 260]
    q, k, v, _ = _inputs(BF16, [1] * 4, [room] * 4, 8, 2, 64)
    koff = [x for i, n in enumerate(lengths) for x in (i * room, i * room + n)] + [4 * room]
    off = [0] + [(i + 1) // 2 for i in range(1, 9)]
    for i, n in enumerate(lengths):       # what lies in the room is not read
        k[i * room + n:(i + 1) * room] = float("nan")
        v[i * room + n:(i + 1) * room] = float("nan")
    out = packed_attention(q, k, v, *(torch.tensor(x, device="cuda:0", dtype=torch.int32) for x in (off, koff)))
    want, bound = packed(q, k, v, off, koff, True, 64 ** -0.5)
    _close([out], want, bound, ["o"])


@pytest.mark.parametrize("few", [True, False])
def test_a_cache_beyond_32_bits(gpu_device, few):
    """Keys and values whose last sequence lies more than 2^32 bytes from the first."""
    from evoformer_triton_amd import packed_attention
    H, Hk, D, queries = 4, 2, 128, [1, 1] if few else [300, 200]
    keys = [9_000_000, 3000]
    q = torch.randn(sum(queries), H, D, device="cuda:0").to(BF16)
    k, v = (torch.zeros(sum(keys), Hk, D, device="cuda:0", dtype=BF16) for _ in range(2))
    assert k.numel() * 2 > 2 ** 32
    for t in (k, v):
        t[keys[0]:] = torch.randn(keys[1], Hk, D, device="cuda:0").to(BF16)
    koff = torch.tensor([0, keys[0], sum(keys)], device="cuda:0", dtype=torch.int32)
    off = torch.tensor([0, queries[0], sum(queries)], device="cuda:0", dtype=torch.int32)
    out = packed_attention(q, k, v, off, koff)
    last = slice(queries[0], None)
    want, bound = packed(q[last], k[keys[0]:], v[keys[0]:], [0, queries[1]], [0, keys[1]], True, D ** -0.5)
    _close([out[last]], want, bound, ["o"])
    assert not out[:queries[0]].any()            # (values of zero)


def test_rows_beyond_32_bits_and_their_gradients(gpu_device):
    """Queries, and keys, whose last sequence lies more than 2^32 bytes from the first: before it one that has nothing on the other side."""
    from evoformer_triton_amd import packed_attention
    H, D, many, last = 16, 64, 2_200_000, 200
    for long in ("queries", "keys"):
        n = many + last
        q = torch.zeros(n if long == "queries" else last, H, D, device="cuda:0", dtype=BF16)
        k, v = (torch.zeros(n if long == "keys" else last, H, D, device="cuda:0", dtype=BF16) for _ in range(2))
        dout = torch.zeros_like(q)
        assert max(q.numel(), k.numel()) * 2 > 2 ** 32
        g = torch.Generator(device="cuda:0").manual_seed(4)
        for t in (q, k, v, dout):
            t[-last:] = torch.randn(last, H, D, device="cuda:0", generator=g).to(BF16)
        ends = [0, many, n], [0, 0, last]
        off, koff = (torch.tensor(x, device="cuda:0", dtype=torch.int32) for x in (ends if long == "queries" else ends[::-1]))
        leaves = [t.requires_grad_() for t in (q, k, v)]
        out = packed_attention(*leaves, off, koff)
        got = [out, *torch.autograd.grad(out, leaves, dout)]
        want, bound = packed(*(t.detach()[-last:] for t in (q, k, v)), [0, last], [0, last], True, D ** -0.5, dout[-last:])
        _close([t[-last:] for t in got], want, bound, ("o", "dq", "dk", "dv"))
        assert not any(t[:-last].any() for t in got)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_side_is_empty(gpu_device, dtype):
    """No queries, no keys, and neither: zeros of the right shapes."""
    from evoformer_triton_amd import packed_attention
    for Tq, Tk in ((0, 70), (200, 0), (3, 0), (0, 0)):
        for n in (0, 1, 70):
            q, k, v, dout = _inputs(dtype, [Tq], [Tk], 4, 2, 40)
            dout = dout[:Tq]
            off, koff = (torch.tensor([0] + [t] * n, device="cuda:0") for t in (Tq, Tk))
            leaves = [t[:m].requires_grad_() for t, m in ((q, Tq), (k, Tk), (v, Tk))]
            out = packed_attention(*leaves, off, koff)
            got = [out, *torch.autograd.grad(out, leaves, dout)]
            assert [g.shape for g in got] == [t.shape for t in (leaves[0], *leaves)] and not any(g.any() for g in got)
