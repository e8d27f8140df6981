"""The relative position bias on the GPU against its formula in 64 bits.

The forward rounds an fp32 sum of two numbers once: half a step of the result and, with 16 bits, half a step of the sum.  The
gradient's tests use whole numbers whose sums fp32 holds, so that it has to be the formula's, rounded to the table's type; one with
other numbers allows each of the additions half a step of what it may have added up to then."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _formula(table, lut, q, k, cq, ck, pair):
    """(out, bucket [B,Nq,Nk]) in 64 bits, on the CPU."""
    q, k = (t if t.dim() == 2 else t[None] for t in (q, k))
    reach = lut.numel() // 2
    q, k = q.to(torch.int64), k.to(torch.int64)
    d = torch.tensor([[[max(-reach, min(reach, int(a) - int(b))) for b in kk] for a in qq] for qq, kk in zip(q.expand(max(len(q), len(k)), -1).tolist(), k.expand(max(len(q), len(k)), -1).tolist())])
    bucket = lut.long()[d + reach]
    if cq is not None:
        cq, ck = (t if t.dim() == 2 else t[None] for t in (cq, ck))
        bucket = torch.where(cq[:, :, None] != ck[:, None, :], len(table) - 1, bucket)
    padded = torch.cat([table.double(), torch.zeros(256 - len(table) + 1, table.shape[1], dtype=torch.float64)])
    out = padded[bucket].permute(0, 3, 1, 2).unsqueeze(1)
    return (out + pair.double() if pair is not None else out), bucket


def _grad(bucket, dout, rows):
    dout = dout.double().squeeze(1)                                                   # [B,H,Nq,Nk]
    hot = (bucket.expand(len(dout), -1, -1)[..., None] == torch.arange(rows)).double()  # [B,Nq,Nk,rows]
    return torch.stack([torch.stack([(dout[:, h] * hot[..., r]).sum() for h in range(dout.shape[1])]) for r in range(rows)])


def _half_step(want, dt):
    f = torch.finfo(dt)
    return want.abs() * (f.eps / 2) + f.tiny * f.eps / 2


# B, Nq, Nk, H, reach, buckets, chains, pair batches (0: none), dtype, table's dtype, positions' dtype
CASES = [
    (1, 1, 1, 1, 0, None, 0, 0, F32, F32, torch.int64),
    (1, 1, 130, 3, 2, None, 0, 0, BF16, F32, torch.int32),         # a row of queries; a last piece that steps back
    (2, 3, 5, 2, 4, None, 2, 2, F16, F16, torch.int64),            # rows shorter than a piece
    (2, 3, 3, 2, 4, None, 2, 1, F32, BF16, torch.int32),
    (1, 33, 8, 4, 32, None, 0, 1, BF16, BF16, torch.int64),        # one piece a row
    (3, 17, 61, 5, 32, None, 3, 1, BF16, F32, torch.int64),        # a pair bias that batches share
    (2, 64, 64, 8, 16, 16, 0, 2, F16, F32, torch.int32),
    (1, 70, 513, 2, 128, 32, 2, 1, BF16, BF16, torch.int64),       # a strip and a key more
    (1, 40, 257, 2, 100, None, 0, 0, F32, F32, torch.int64),       # 201 rows: lanes take turns
    (1, 37, 100, 2, 60, None, 3, 0, BF16, F32, torch.int16),       # 122 rows
    (1, 9, 77, 2, 4096, 64, 0, 1, F16, F16, torch.int64),
]


def _inputs(case, seed=5):
    from evoformer_triton_amd import relative_buckets
    B, Nq, Nk, H, reach, num, chains, pb, dt, tdt, index = case
    g = torch.Generator().manual_seed(seed)
    lut = relative_buckets(reach, num)
    rows = int(lut.max()) + 1 + (chains > 0)
    q = torch.randint(-2 * reach - 3, 2 * reach + 4, (B, Nq), generator=g).to(index)
    k = torch.randint(-2 * reach - 3, 2 * reach + 4, (B, Nk), generator=g).to(index)
    cq, ck = (torch.randint(0, chains, (B, n), generator=g).to(index) for n in (Nq, Nk)) if chains else (None, None)
    table = torch.randn((rows, H), generator=g).to(tdt)
    pair = torch.randn((pb, 1, H, Nq, Nk), generator=g).to(dt) if pb else None
    dout = torch.randint(-8, 9, (B, 1, H, Nq, Nk), generator=g).to(dt)
    return lut, q, k, cq, ck, table, pair, dout


def _dev(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_the_formula_and_its_gradients(gpu_device, case):
    from evoformer_triton_amd import relative_position_bias
    lut, q, k, cq, ck, table, pair, dout = _inputs(case)
    want, bucket = _formula(table, lut, q, k, cq, ck, pair)
    t, p = _dev(gpu_device, table, pair)
    t.requires_grad_()
    if p is not None:
        p.requires_grad_()
    leaves = [t] + ([p] if p is not None else [])
    args = _dev(gpu_device, lut, q, k, cq, ck)
    out = relative_position_bias(t, *args[:3], chains=args[3], key_chains=args[4], pair_bias=p, dtype=case[8])
    assert out.grad_fn.name() == "RelativePositionBiasBackward" and out.dtype == case[8]
    assert ((out.detach().cpu().double() - want).abs() <= _half_step(want, case[8]) + (want.abs() + 2 * table.double().abs().max()) * 2 ** -24).all()
    got = torch.autograd.grad(out, leaves, dout.to(gpu_device), retain_graph=True)
    dtable = _grad(bucket, dout, len(table))
    assert torch.equal(got[0].cpu(), dtable.to(case[9])) and got[0].dtype == case[9]
    if p is not None:
        assert torch.equal(got[1].cpu(), dout.double().sum(0, keepdim=True).to(case[8]) if len(pair) < len(dout) else dout)
    again = torch.autograd.grad(out, leaves, dout.to(gpu_device))
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_gradients_are_the_differences(gpu_device):
    """Linear in the table: what a step of one entry adds to <dout, out> is the step times its gradient, in whole numbers."""
    from evoformer_triton_amd import relative_position_bias
    lut, q, k, cq, ck, table, _, dout = _inputs((2, 19, 45, 3, 6, None, 2, 0, F32, F32, torch.int64))
    lut, q, k, cq, ck, table, dout = _dev(gpu_device, lut, q, k, cq, ck, table.round(), dout)
    call = lambda t: relative_position_bias(t, lut, q, k, chains=cq, key_chains=ck)  # noqa: E731
    t = table.clone().requires_grad_()
    grad, = torch.autograd.grad(call(t), t, dout)
    base = (call(table) * dout).double().sum()
    for r in range(len(table)):
        for h in range(3):
            step = table.clone()
            step[r, h] += 4
            assert (call(step) * dout).double().sum() - base == 4 * grad[r, h].double()


def test_any_numbers_within_the_additions_roundings(gpu_device):
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    g = torch.Generator().manual_seed(3)
    N, H = 300, 2
    lut, pos = relative_buckets(32), torch.arange(N)
    dout = torch.randn((2, 1, H, N, N), generator=g)
    d = (pos[:, None] - pos[None]).clamp(-32, 32) + 32
    t = torch.zeros(65, H, device=gpu_device, requires_grad=True)
    out = relative_position_bias(t, lut.to(gpu_device), pos.to(gpu_device).expand(2, -1))
    got, = torch.autograd.grad(out, t, dout.to(gpu_device))
    for r in range(65):
        at = dout.double().squeeze(1)[:, :, d == r]                       # [2, H, n]
        n, total = at.shape[0] * at.shape[2], at.abs().sum((0, 2))
        assert ((got[r].cpu().double() - at.sum((0, 2))).abs() <= min(n, 4096) * 2 ** -24 * total).all(), r


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_positions_at_the_ends_of_their_type(gpu_device, index):
    """Differences that the type does not hold are far, not near."""
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    i = torch.iinfo(index)
    q = torch.tensor([[i.min, i.max, 0, i.min + 3, i.max - 2, -1, 2 ** 30, -2 ** 30 - 1]], dtype=index)
    k = torch.tensor([[i.max, i.min, i.min + 1, i.max - 1, 0, 1, 2 ** 30 + 2, -2 ** 30, 5, i.min]], dtype=index)
    lut, table = relative_buckets(4), torch.arange(1, 19, dtype=F32).view(9, 2)
    want, bucket = _formula(table, lut, q, k, None, None, None)
    t = table.to(gpu_device).requires_grad_()
    out = relative_position_bias(t, *_dev(gpu_device, lut, q, k))
    assert torch.equal(out.cpu().double(), want)
    dout = torch.arange(160.).view(1, 1, 2, 8, 10)
    assert torch.equal(torch.autograd.grad(out, t, dout.to(gpu_device))[0].cpu().double(), _grad(bucket, dout, 9))


def test_a_bucket_beyond_the_table_takes_nothing(gpu_device):
    from evoformer_triton_amd import relative_position_bias
    lut = torch.tensor([0, 255, 1], dtype=torch.uint8, device=gpu_device)
    t = torch.tensor([[1.0], [2.0]], device=gpu_device, requires_grad=True)
    pos = torch.arange(3, device=gpu_device)
    out = relative_position_bias(t, lut, pos)
    assert out.tolist() == [[[[[0, 1, 1], [2, 0, 1], [2, 2, 0]]]]]
    assert torch.autograd.grad(out.sum(), t)[0].tolist() == [[3], [3]]


def test_infinities_and_nan_stay_where_they_belong(gpu_device):
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    lut, pos = relative_buckets(2).to(gpu_device), torch.arange(40, device=gpu_device)
    table = torch.zeros(5, 2, device=gpu_device)
    table[4, 1] = float("inf")
    pair = torch.zeros(1, 1, 2, 40, 40, device=gpu_device)
    pair[0, 0, 0, 3, 7] = float("nan")
    pair[0, 0, 1, :, 5] = float("-inf")
    t = table.clone().requires_grad_()
    out = relative_position_bias(t, lut, pos, pair_bias=pair)
    want = pair.clone()
    want[0, 0, 1][(pos[:, None] - pos[None]) >= 2] += float("inf")
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(), want.nan_to_num())
    dout = torch.ones_like(out)
    dout[0, 0, 0, 10, 10], dout[0, 0, 1, 10, 9] = float("nan"), float("inf")
    got, = torch.autograd.grad(out, t, dout)
    bad = ~torch.isfinite(got)
    assert bad.nonzero().tolist() == [[2, 0], [3, 1]] and got[3, 1] == float("inf")


def test_strides_devices_streams(gpu_device):
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    g = torch.Generator().manual_seed(9)
    lut = relative_buckets(8).to(gpu_device)
    wide = torch.randn((2, 1, 30, 4, 50), generator=g).to(F16).to(gpu_device)
    pair = wide.permute(0, 1, 3, 2, 4)[..., 1:42]                                   # rows of 41 keys, heads apart, off any boundary
    pos = torch.randint(0, 30, (2, 82), generator=g).to(gpu_device)
    k, q = pos[:, ::2], pos[:, 1:31]
    table = torch.randn((4, 17), generator=g).to(gpu_device).t()
    want = relative_position_bias(table.contiguous(), lut, q.contiguous(), k.contiguous(), pair_bias=pair.contiguous())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = relative_position_bias(table, lut, q, k, pair_bias=pair)
        crossed = relative_position_bias(table, lut, q, k, pair_bias=pair.transpose(3, 4).contiguous().transpose(3, 4))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(crossed, want)
    # gradients that autograd hands over with strides of their own
    t = table.contiguous().requires_grad_()
    out = relative_position_bias(t, lut, q, k, pair_bias=pair)
    a, = torch.autograd.grad(out.sum(), t, retain_graph=True)
    b, = torch.autograd.grad(out, t, torch.ones_like(out).transpose(3, 4).contiguous().transpose(3, 4), retain_graph=True)
    c, = torch.autograd.grad(out, t, torch.ones_like(out))
    assert torch.equal(a, c) and torch.equal(b, c)
    with torch.autograd.graph.save_on_cpu():
        out = relative_position_bias(t, lut, q, k, pair_bias=pair)
    assert torch.equal(torch.autograd.grad(out, t, torch.ones_like(out))[0], c)


def test_empty_calls(gpu_device):
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    lut = relative_buckets(2).to(gpu_device)
    t = torch.ones(5, 3, device=gpu_device, requires_grad=True)
    for q, k in ((0, 4), (4, 0), (0, 0)):
        out = relative_position_bias(t, lut, torch.arange(q, device=gpu_device), torch.arange(k, device=gpu_device))
        assert out.shape == (1, 1, 3, q, k)
        assert torch.equal(torch.autograd.grad(out.sum(), t)[0], torch.zeros_like(t))


def test_a_captured_step_replays(gpu_device):
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    g = torch.Generator().manual_seed(2)
    lut, pos = relative_buckets(16).to(gpu_device), torch.arange(160, device=gpu_device)
    t = torch.randn((33, 4), generator=g).to(gpu_device).requires_grad_()
    pair = torch.randn((1, 1, 4, 160, 160), generator=g).to(gpu_device)
    dout = torch.randn((1, 1, 4, 160, 160), generator=g).to(gpu_device)

    def step():
        out = relative_position_bias(t, lut, pos, pair_bias=pair)
        return out.detach(), torch.autograd.grad(out, t, dout)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(4):
        pair.copy_(torch.randn((1, 1, 4, 160, 160), generator=torch.Generator().manual_seed(seed)))
        dout.copy_(pair.flip(3))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_compiled_and_watched_calls(gpu_device):
    from torch.utils._python_dispatch import TorchDispatchMode
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    lut, pos = relative_buckets(4).to(gpu_device), torch.arange(24, device=gpu_device)
    t = torch.randn((9, 2), device=gpu_device, requires_grad=True)
    pair = torch.randn((1, 1, 2, 24, 24), device=gpu_device, requires_grad=True)
    call = lambda t, p: relative_position_bias(t, lut, pos, pair_bias=p)  # noqa: E731
    want = call(t, pair)
    want_g = torch.autograd.grad(want, [t, pair], torch.ones_like(want))
    seen = []

    class Recorder(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    with Recorder():
        watched = call(t, pair)
    compiled = torch.compile(call, fullgraph=True, backend="aot_eager")(t, pair)
    assert any("relative_bias" in s for s in seen)
    for out in (watched, compiled):
        assert torch.equal(out, want)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, [t, pair], torch.ones_like(out)), want_g))


def test_transforms_are_refused_not_dropped(gpu_device):
    from torch.autograd import forward_ad
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    lut, pos = relative_buckets(4).to(gpu_device), torch.arange(24, device=gpu_device)
    t = torch.randn((9, 2), device=gpu_device)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: relative_position_bias(x, lut, pos))(t.expand(3, 9, 2))
    with forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        relative_position_bias(forward_ad.make_dual(t, torch.ones_like(t)).requires_grad_(), lut, pos)
    x = t.clone().requires_grad_()
    g, = torch.autograd.grad(relative_position_bias(x, lut, pos).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
