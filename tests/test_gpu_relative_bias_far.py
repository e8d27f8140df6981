"""The relative position bias far from zero and at the ends of its numbers: positions and chains as far apart as their type allows, gradients near
the smallest and without a number."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _sums(bucket, dout, rows):
    """The table's gradient in 64 bits: bucket [Nq,Nk], dout [B,1,H,Nq,Nk]."""
    per_pair = dout.double().sum((0, 1)).flatten(1).t()
    return torch.zeros(rows, dout.shape[2], dtype=torch.float64, device=dout.device).index_add_(0, bucket.flatten(), per_pair)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("far", [2 ** 30 - 4097, 2 ** 30 - 4096, 2 ** 30 - 5, 2 ** 30 - 2, 2 ** 30 - 1, 2 ** 30])
@pytest.mark.parametrize("reach", [1, 2, 4, 4096])
def test_positions_within_a_workgroups_reach(gpu_device, index, far, reach):
    """Queries and keys on either side of the first query: differences of up to 2^31, in the forward and in the gradient's buckets."""
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    lut = relative_buckets(reach, None if reach < 128 else 64).to(gpu_device)
    q = torch.tensor([0, far, -far, 3, far - 1], dtype=index, device=gpu_device)
    k = torch.tensor([-far, far, 0, -far + 1, far - 2, 5, 1, -far + 2, far], dtype=index, device=gpu_device)
    rows = int(lut.max()) + 1
    bucket = lut.long()[(q.long()[:, None] - k.long()[None]).clamp(-reach, reach) + reach]
    table = torch.arange(1.0, 1 + 2 * rows, device=gpu_device).view(rows, 2).requires_grad_()
    out = relative_position_bias(table, lut, q, k)
    assert torch.equal(out[0, 0], table.detach()[bucket].permute(2, 0, 1))
    dout = torch.arange(1.0, 91, device=gpu_device).view(1, 1, 2, 5, 9)
    assert torch.equal(torch.autograd.grad(out, table, dout)[0].double(), _sums(bucket, dout, rows))


@pytest.mark.parametrize("ids,index", [((0, 2 ** 40), torch.int64), ((-2 ** 63, 2 ** 63 - 1), torch.int64), ((5, 5 + 2 ** 32), torch.int64), ((-2 ** 31, 2 ** 31 - 1), torch.int32),
                                       ((0, 2 ** 30), torch.int32), ((7, 7 + 2 ** 62), torch.int64)])
@pytest.mark.parametrize("N,dt", [(37, F32), (200, BF16), (203, F16), (5, F32)])
def test_chains_are_told_apart_by_any_numbers(gpu_device, ids, index, N, dt):
    """A chain's number is a name: which one it is changes no bit."""
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    g = torch.Generator().manual_seed(N)
    lut, at = relative_buckets(8).to(gpu_device), torch.arange(N, device=gpu_device).expand(2, N)
    which = torch.randint(0, 2, (2, N), generator=g).to(gpu_device)
    named = torch.where(which == 1, torch.tensor(ids[1], device=gpu_device), torch.tensor(ids[0], device=gpu_device)).to(index)
    table = torch.randn((18, 3), generator=g).to(gpu_device).requires_grad_()
    dout = torch.randn((2, 1, 3, N, N), generator=g).to(dt).to(gpu_device)
    results = []
    for chains in (which, named):
        out = relative_position_bias(table, lut, at, chains=chains, dtype=dt)
        results.append((out, torch.autograd.grad(out, table, dout)[0]))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    bucket = torch.where(which[:, :, None] == which[:, None, :], lut.long()[(at[:, :, None] - at[:, None, :]).clamp(-8, 8) + 8], 17)
    want = _sums(bucket[0], dout[:1], 18) + _sums(bucket[1], dout[1:], 18)
    size = _sums(bucket[0], dout[:1].abs(), 18) + _sums(bucket[1], dout[1:].abs(), 18)
    # (each addition may lose half a step of what it has added up: of 203^2 pairs in sums of 64 keys, 203 rows, two batches and strips; a chain of 600 at most)
    assert ((results[1][1].double() - want).abs() <= 600 * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("exponent", [-100, -126, -133, -135, -140, -149])
def test_small_gradients_keep_their_bits(gpu_device, exponent):
    """Whole numbers of up to 8 bits in units down to fp32's smallest: their sums are exact."""
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    g = torch.Generator().manual_seed(4)
    lut, at = relative_buckets(4).to(gpu_device), torch.arange(70, device=gpu_device)
    whole = torch.randint(-127, 128, (1, 1, 2, 70, 70), generator=g).to(gpu_device)
    dout = (whole.double() * 2.0 ** exponent).float()
    assert torch.equal(dout.double() * 2.0 ** -exponent, whole.double())
    table = torch.zeros(9, 2, device=gpu_device, requires_grad=True)
    got, = torch.autograd.grad(relative_position_bias(table, lut, at), table, dout)
    bucket = lut.long()[(at[:, None] - at[None]).clamp(-4, 4) + 4]
    assert torch.equal(got.double() * 2.0 ** -exponent, _sums(bucket, whole, 9))


@pytest.mark.parametrize("size", [2.0 ** 100, 2.0 ** 110, 2.0 ** 120])
def test_large_gradients_are_no_infinities(gpu_device, size):
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    lut, at = relative_buckets(2).to(gpu_device), torch.arange(9, device=gpu_device)
    whole = torch.randint(-3, 4, (1, 1, 2, 9, 9), generator=torch.Generator().manual_seed(4)).to(gpu_device)
    table = torch.zeros(5, 2, device=gpu_device, requires_grad=True)
    got, = torch.autograd.grad(relative_position_bias(table, lut, at), table, whole.float() * size)
    bucket = lut.long()[(at[:, None] - at[None]).clamp(-2, 2) + 2]
    assert torch.equal(got.double() / size, _sums(bucket, whole, 5))


@pytest.mark.parametrize("size", [2.0 ** -126, 2.0 ** -118, 2.0 ** -110, 1.0, 2.0 ** 103, 2.0 ** 106, 2.0 ** 126])
def test_a_gradient_of_one_pair_comes_out_as_it_went_in(gpu_device, size):
    """Each bucket has one pair: all 24 bits of its gradient, from the smallest normal number to the largest."""
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    g = torch.Generator().manual_seed(7)
    lut = relative_buckets(50).to(gpu_device)
    q, k = torch.zeros(1, dtype=torch.int64, device=gpu_device), torch.arange(-50, 51, device=gpu_device)
    dout = ((1 + torch.rand((1, 1, 5, 1, 101), generator=g)) * (torch.randint(0, 2, (1, 1, 5, 1, 101), generator=g) * 2 - 1)).to(gpu_device) * size
    table = torch.zeros(101, 5, device=gpu_device, requires_grad=True)
    got, = torch.autograd.grad(relative_position_bias(table, lut, q, k), table, dout)
    assert torch.equal(got, dout[0, 0, :, 0].flip(1).t())


def test_sums_beside_one_without_a_number_are_as_good(gpu_device):
    """One infinity makes its workgroups form their sums one by one.  Of equal numbers the roundings of a single chain of additions all go the same way for long stretches; of sums
    by rows they stay within what 64 keys, N rows and the workgroups' parts, one after the other, may lose."""
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    N = 2048
    lut, at = relative_buckets(1).to(gpu_device), torch.arange(N, device=gpu_device)
    table = torch.zeros(3, 16, device=gpu_device, requires_grad=True)
    dout = torch.full((1, 1, 16, N, N), 0.1, device=gpu_device)
    dout[0, 0, 0, ::16, ::16] = float("inf")
    got, = torch.autograd.grad(relative_position_bias(table, lut, at), table, dout)
    pairs = torch.tensor([N * (N - 1) // 2, N, N * (N - 1) // 2], dtype=torch.float64, device=gpu_device)
    want = pairs * dout[0, 0, 1, 0, 0].double()
    assert torch.isinf(got[:, 0]).all()
    assert ((got[:, 1:].double() / want[:, None] - 1).abs() <= (64 + 256 + 32) * 2.0 ** -24).all(), (got[:, 1].double() / want - 1).abs()


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.uint16, torch.uint32, torch.int32, torch.int64], ids=str)
def test_positions_of_any_whole_type(gpu_device, dtype):
    from evoformer_triton_amd import RelativePositionBias
    bias = RelativePositionBias(2, 20, other_chain=True).to(gpu_device)
    bias.weight.data.normal_()
    i = torch.iinfo(dtype)
    values = [0, 1, 5, 100, i.max, i.max - 3] + ([i.min, i.min + 2, -1] if i.min else [])
    at = torch.tensor(values, dtype=dtype, device=gpu_device)
    d = torch.tensor([[max(-20, min(20, a - b)) + 20 for b in values] for a in values], device=gpu_device)
    chains = torch.tensor([2 ** 64 - 1 if k % 2 else 3 for k in range(len(values))], dtype=torch.uint64, device=gpu_device)
    same = torch.tensor([[(a - b) % 2 == 0 for b in range(len(values))] for a in range(len(values))], device=gpu_device)
    for given in (None, chains):
        want = bias.weight[d if given is None else torch.where(same, d, 41)].permute(2, 0, 1)
        assert torch.equal(bias(at, chains=given)[0, 0], want)
        assert torch.equal(bias.plain(at, chains=given)[0, 0], want)


def test_the_registered_backward_gives_what_is_traced(gpu_device):
    """Shapes and strides of the gradients are those that the compiler has been told, also for a gradient that comes with strides of its own or without a batch."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from evoformer_triton_amd import relative_buckets
    lut, at = relative_buckets(4), torch.arange(24)
    table = torch.zeros(9, 2)
    for B, pair_b, crossed in ((1, 1, True), (2, 2, True), (2, 1, True), (2, 1, False), (0, 1, False), (0, 0, False)):
        dout = torch.randn(B, 1, 2, 24, 24)
        dout = dout.transpose(3, 4) if crossed else dout
        args = (dout, table, lut, at.expand(B, 24), at, None, None, torch.zeros(pair_b, 1, 2, 24, 24))
        real = [t if t is None else t.to(gpu_device) for t in args]
        with FakeTensorMode(allow_non_fake_inputs=True) as mode:
            told = torch.ops.evoattn.relative_bias_bwd(*(t if t is None else mode.from_tensor(t) for t in real), True, True)
        got = torch.ops.evoattn.relative_bias_bwd(*real, True, True)
        assert [(t.shape, t.stride(), t.dtype) for t in got] == [(t.shape, t.stride(), t.dtype) for t in told], (B, pair_b, crossed)
        assert torch.equal(got[1], real[0] if pair_b == B else real[0].sum(0, keepdim=True)), (B, pair_b, crossed)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("which", ["positions", "key_positions", "chains", "key_chains", "buckets"])
@pytest.mark.parametrize("shape", [(24,), (1, 24), (2, 24)], ids=str)
def test_what_is_saved_and_changed_before_the_backward_is_noticed(gpu_device, which, shape, index):
    """As of any tensor that a backward needs; what was copied for it may change."""
    from evoformer_triton_amd import relative_buckets, relative_position_bias
    g = torch.Generator().manual_seed(1)
    args = {n: torch.randint(0, 9, shape, generator=g).to(index).to(gpu_device) for n in ("positions", "key_positions", "chains", "key_chains")}
    args["buckets"] = relative_buckets(3).to(gpu_device)
    table = torch.randn(8, 2, device=gpu_device, requires_grad=True)
    dout = torch.randn(shape[0] if len(shape) == 2 else 1, 1, 2, 24, 24, device=gpu_device)
    out = relative_position_bias(table, **args)
    args[which].copy_(args[which].flip(-1))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, table, dout)
    # one row of chains for two batches of positions is copied
    if shape == (2, 24) and which == "chains":
        short = args["chains"][0].clone()
        call = lambda: relative_position_bias(table, **{**args, "chains": short, "key_chains": short})  # noqa: E731
        want, = torch.autograd.grad(call(), table, dout)
        out = call()
        short.zero_()
        assert torch.equal(torch.autograd.grad(out, table, dout)[0], want)
