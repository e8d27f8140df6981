"""Linear layers in 8 bits on the GPU against their definition in 64 bits.

The rounding is exact: bytes and scales are compared as such.  A product is held to the rounding of its result (half a step), and to
that of its sums: in fp32, where every addition may lose a step of what it has added up to, K 2^-23 of the sum of magnitudes; with a
16-bit result the 8-bit matrix instruction's, of which neighbouring products are cut off 13 bits below the largest of
them: each loses up to 2^-13 of a product that is in the sum as well, eight neighbours 2^-10 of the largest."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _rounded(x):
    """Q along the last axis: (values in units of the scale, exponents), 64 bits, on the CPU."""
    k = x.shape[-1]
    v = torch.zeros((*x.shape[:-1], -(-k // 128) * 128), dtype=torch.float64)
    v[..., :k] = x.double().cpu()
    v = v.unflatten(-1, (-1, 128))
    a = torch.where(v.isfinite(), v.abs(), 0).amax(-1, keepdim=True)
    m, e = torch.frexp(a)
    e = torch.where(a == 0, 0, torch.where(m > 0.875, e - 8, e - 9).clamp(-127, 127))
    u = torch.ldexp(v, -e)
    u = torch.where(u.isfinite(), u, float("nan"))
    step = torch.exp2(torch.floor(torch.log2(torch.where((u == 0) | u.isnan(), 1.0, u.abs()))).clamp(-6, 8) - 3)
    return torch.round(u / step) * step, e.squeeze(-1)


def _q(x):
    u, e = _rounded(x)
    return torch.ldexp(u, e.unsqueeze(-1)).flatten(-2)[..., :x.shape[-1]]


def _near(got, want, magnitudes, K):
    """Whether `got` is within its own and its sums' rounding of `want`."""
    f = torch.finfo(got.dtype)
    sums = magnitudes * (K * 2 ** -23 if got.dtype == F32 else 2 ** -10 + K * 2 ** -23)
    bound = sums + (want.abs() + sums) * (f.eps / 2) + f.tiny * f.eps
    d = (got.detach().cpu().double() - want).abs()
    assert (d <= bound).all(), ((d / bound).max().item(), (d > bound).sum().item())


def _data(shape, dt, g, spread=1.0):
    return (torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[-1:], generator=g))).to(dt)


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 128), (5, 129), (127, 40), (128, 512), (130, 641), (300, 200)])
def test_rounding_is_the_definitions(gpu_device, dt, shape):
    from evoformer_triton_amd import Fp8Weight
    g = torch.Generator().manual_seed(1)
    x = _data(shape, dt, g)
    x[0, 0] = 0
    x.view(-1)[-1] = -0.0
    if shape[1] >= 128:
        x[1, :128] = 0                                                       # a block of zeros
        x[2, :4] = torch.tensor([448., 232., 248., 1.0625]).to(dt)            # ties, up and down
        x[2, 4:128] = 0
    w = Fp8Weight.of(x.to(gpu_device))
    u, e = _rounded(x)
    assert w.values.dtype == torch.float8_e4m3fn and w.values.shape == (shape[0], u.shape[1] * 128) and w.scales.shape == (shape[0], -(-u.shape[1] // 4) * 4)
    assert torch.equal(w.values.cpu().double(), u.flatten(-2))
    assert torch.equal(w.scales.cpu()[:, :u.shape[1]].int() - 127, e.int()) and (w.scales[:, u.shape[1]:] == 127).all()
    assert torch.equal(w.dequantize().cpu().double(), _q(x).float().double())


def test_rounding_at_the_ends_of_fp32(gpu_device):
    from evoformer_triton_amd import Fp8Weight
    inf, nan, big, tiny = float("inf"), float("nan"), torch.finfo(F32).max, 2.0 ** -149
    x = torch.zeros(8, 128)
    x[0, :5] = torch.tensor([inf, 3.0, -inf, nan, -448.0])        # found by the finite ones
    x[1, :2] = torch.tensor([inf, nan])                            # nothing finite but zeros
    x[2, :3] = torch.tensor([big, -big, 1.0])
    x[3, :3] = torch.tensor([tiny, -tiny, 3 * tiny])
    x[4, :2] = torch.tensor([448 * 2.0 ** -127, 2.0 ** -136])
    x[5, :2] = torch.tensor([1.75, 1.75 * 2.0 ** -20])
    x[6, :2] = torch.tensor([1.7500001, -1.0])
    w = Fp8Weight.of(x.to(gpu_device))
    u, e = _rounded(x)
    got = w.values.cpu().double()
    assert torch.equal(got.isnan(), u.flatten(-2).isnan()) and torch.equal(got.nan_to_num(), u.flatten(-2).nan_to_num())
    assert torch.equal(w.scales.cpu()[:, :1].int() - 127, e.int())


# rows, k, n, bias, x, weight, bias dtypes
CASES = [
    (1, 1, 1, True, BF16, BF16, BF16),
    (1, 256, 1024, False, BF16, BF16, None),
    (5, 128, 3, True, F32, F32, F32),
    (16, 1200, 33, True, BF16, BF16, F32),            # few rows, rounded on the way: one tile, ten blocks over eight waves
    (33, 5000, 50, False, F16, BF16, None),           # three tiles, five slices of eight blocks
    (50, 513, 200, True, F32, F32, F32),
    (64, 1920, 8200, True, BF16, BF16, BF16),         # the most; 64 outputs to a workgroup, two slices
    (20, 2048, 8192, True, F32, BF16, F32),
    (65, 300, 70, True, BF16, BF16, BF16),            # one more
    (17, 200, 130, True, F16, F32, F16),
    (64, 640, 257, False, F32, BF16, None),
    (129, 129, 127, True, BF16, BF16, F32),           # a tile and a row; a block and a value
    (300, 1100, 96, True, F16, F16, F16),             # three groups of four blocks
    (2500, 96, 40, True, BF16, F32, BF16),            # the weight's gradient in slices of the rows
    (2500, 640, 200, False, F32, F32, None),
    (128, 4224, 64, True, BF16, BF16, BF16),          # the forward in slices of the contraction
    (65537, 130, 200, True, BF16, BF16, BF16),        # strips of 128 rows, the last of one row; two blocks, of which one has two values
    (700, 250, 130, True, F32, F32, F32),             # strips in fp32, three tiles, the last of two columns
    (40000, 400, 100, True, F16, F16, BF16),          # four blocks to a strip
    (200, 512, 1000, False, BF16, BF16, None),        # the same, rounded before: eight pieces to a strip
    (300, 380, 200, True, F32, F32, F32),             # three in fp32
    (66000, 520, 260, True, BF16, BF16, BF16),        # tiles of 256 x 256, the last ones of a few rows and columns
    (33000, 700, 300, False, F16, F16, None),         # two and three of them side by side; more than one group of scales
    (33000, 600, 520, True, F32, F32, F32),           # the same in fp32
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_products_and_gradients(gpu_device, case):
    from evoformer_triton_amd import Fp8Weight, fp8_linear
    rows, k, n, with_bias, dt, wdt, bdt = case
    g = torch.Generator().manual_seed(17)
    x, w = _data((rows, k), dt, g), (_data((n, k), F32, g, 0.5) * k ** -0.5).to(wdt)
    b = torch.randn((n,), generator=g).to(bdt) if with_bias else None
    dy = (torch.randn((rows, n), generator=g) * torch.exp(torch.randn((rows, 1), generator=g) - 4)).to(dt)
    if rows > 4:
        x[3], dy[3] = 0, 0
    leaves = [t.to(gpu_device).requires_grad_() for t in (x, w) + ((b,) if with_bias else ())]
    y = fp8_linear(leaves[0], leaves[1], leaves[2] if with_bias else None)
    assert y.grad_fn.name() == "Fp8LinearBackward" and y.dtype == dt
    got = torch.autograd.grad(y, leaves, dy.to(gpu_device), retain_graph=True)
    assert [t.dtype for t in got] == [t.dtype for t in leaves]

    def product(a, bt):
        return a @ bt.t(), a.abs() @ bt.abs().t()

    want, size = product(_q(x), _q(w))
    if with_bias:
        want, size = want + b.double(), size + b.double().abs()
    _near(y, want, size, k)
    _near(got[0], *product(_q(dy), _q(w.t())), n)
    _near(got[1], *product(_q(dy.t()), _q(x.t())), rows)
    if with_bias:
        _near(got[2].float() if bdt == F32 else got[2], dy.double().sum(0), dy.double().abs().sum(0), rows)
    again = torch.autograd.grad(y, leaves, dy.to(gpu_device))
    assert all(torch.equal(a, c) for a, c in zip(got, again))
    for i, t in enumerate(leaves):      # one gradient at a time
        y1 = fp8_linear(*(u if j == i else u.detach() for j, u in enumerate(leaves)))
        assert torch.equal(y1, y) and torch.equal(torch.autograd.grad(y1, t, dy.to(gpu_device))[0], got[i])
    with torch.no_grad():
        held = fp8_linear(leaves[0], Fp8Weight.of(leaves[1]), leaves[2] if with_bias else None)
    assert torch.equal(held, y)


@pytest.mark.parametrize("rows,k,n", [(9, 150, 11), (140, 150, 70), (140, 700, 33)])
def test_gradients_are_the_differences(gpu_device, rows, k, n):
    """Whole numbers of up to 4 bits are what they are in 8 bits, whatever their block's scale, and so are the steps between them: differences are exact."""
    from evoformer_triton_amd import fp8_linear
    g = torch.Generator().manual_seed(8)
    leaves = [torch.randint(-7, 8, s, generator=g).float().to(gpu_device).requires_grad_() for s in ((rows, k), (n, k), (n,))]
    c = torch.randint(-7, 8, (rows, n), generator=g).float().to(gpu_device)

    def loss():
        return (fp8_linear(*leaves).double() * c).sum()

    grads = torch.autograd.grad(loss(), leaves)
    for t, got in zip(leaves, grads):
        for at in torch.randint(0, t.numel(), (6,), generator=g).tolist() + [0, t.numel() - 1]:
            with torch.no_grad():
                flat, was = t.view(-1), t.view(-1)[at].clone()
                flat[at] = was + 2
                up = loss()
                flat[at] = was - 3
                down = loss()
                flat[at] = was
            assert (up - down) / 5 == got.view(-1)[at]


def test_rows_with_infinities_and_nan_are_theirs_alone(gpu_device):
    from evoformer_triton_amd import Fp8Weight, fp8_linear
    g = torch.Generator().manual_seed(4)
    w = Fp8Weight.of(torch.randn((70, 300), generator=g).to(gpu_device))
    for rows in (5, 200):
        x = torch.randn((rows, 300), generator=g).to(BF16)
        with torch.no_grad():
            want = fp8_linear(x.to(gpu_device), w)
            x[2, 7], x[4, 299] = float("inf"), float("nan")
            got = fp8_linear(x.to(gpu_device), w)
        bad = torch.tensor([2, 4], device=gpu_device)
        assert got[bad].isnan().all()
        keep = torch.ones(rows, dtype=torch.bool, device=gpu_device)
        keep[bad] = False
        assert torch.equal(got[keep], want[keep])


def test_strides_shapes_and_streams(gpu_device):
    from evoformer_triton_amd import Fp8Weight, fp8_linear
    g = torch.Generator().manual_seed(6)
    wide = torch.randn((4, 40, 901), generator=g).to(F16).to(gpu_device)
    wt = torch.randn((333, 300), generator=g).to(gpu_device)                         # the weight as the transpose of a tensor
    bias = torch.randn((601,), generator=g).to(F16).to(gpu_device)[1::2][:300]
    cases = (wide[..., 3:336], wide[:, ::2, 3:336], wide[0, :, 1:334], wide[0, 0, :333], wide.transpose(0, 1)[..., :333], wide[..., ::2][..., 100:433])
    for x in cases:
        def step():
            leaves = [x.detach().requires_grad_(), wt.detach().t().requires_grad_(), bias.detach().requires_grad_()]
            y = fp8_linear(*leaves)
            return [y.detach(), *torch.autograd.grad(y.sum(), leaves)]

        leaves = [x.detach().contiguous().requires_grad_(), wt.detach().t().contiguous().requires_grad_(), bias.detach().contiguous().requires_grad_()]
        y = fp8_linear(*leaves)
        want = [y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        torch.cuda.current_stream().wait_stream(side)
        with torch.autograd.graph.save_on_cpu():
            hooked = step()
        for a, b, c in zip(got, want, hooked):
            assert a.shape == b.shape and torch.equal(a, b) and torch.equal(c, b)
        with torch.no_grad():
            assert torch.equal(fp8_linear(x, Fp8Weight.of(wt.t()), bias), want[0])


def test_a_single_row_of_any_stride(gpu_device):
    from evoformer_triton_amd import Fp8Weight, fp8_linear
    for k in (1, 5, 200):
        x, w = torch.randn(k, 1, device=gpu_device).t(), torch.randn(k, 1, device=gpu_device).t()      # [1, k], strides (1, 1)
        y, want = (fp8_linear(a.detach().requires_grad_(), b, None) for a, b in ((x, w), (x.clone(memory_format=torch.contiguous_format), w.reshape(-1).view(1, k))))
        dy = torch.randn(1, device=gpu_device).expand(1, 1)
        assert torch.equal(y, want) and torch.equal(Fp8Weight.of(w).dequantize(), Fp8Weight.of(w.reshape(-1).view(1, k)).dequantize())
        y.backward(dy)
        z = fp8_linear(torch.randn(300, k, device=gpu_device), w)
        assert z.shape == (300, 1) and torch.isfinite(z).all()


def test_more_rows_than_fit_32_bits(gpu_device):
    """The weight's gradient contracts them; their rounded columns lie 4 MB apart, and a group of 512 of them spans 2^31 bytes."""
    from evoformer_triton_amd import fp8_linear
    g = torch.Generator().manual_seed(3)
    rows, k, n = 2 ** 22 + 133, 5, 600
    x, w = torch.randn((rows, k), generator=g).to(BF16), torch.randn((n, k), generator=g)
    xg, wg = x.to(gpu_device), w.to(gpu_device).requires_grad_()
    y = fp8_linear(xg, wg)
    for part in (slice(0, 300), slice(rows - 300, rows)):
        want = _q(x[part]) @ _q(w).t()
        _near(y[part], want, _q(x[part]).abs() @ _q(w).abs().t(), k)
    dy = torch.zeros((rows, n), dtype=BF16, device=gpu_device)
    at = torch.tensor([0, 127, 5000, 2 ** 22 - 1, 2 ** 22, rows - 1])
    values = torch.randn((len(at), n), generator=g).to(BF16)
    dy[at.to(gpu_device)] = values.to(gpu_device)
    dw, = torch.autograd.grad(y, wg, dy)
    want, size = torch.zeros(n, k, dtype=torch.float64), torch.zeros(n, k, dtype=torch.float64)
    for i, r in enumerate(at.tolist()):        # each alone in its block of 128 rows, but for the two around 2^22
        block = slice(r // 128 * 128, min(r // 128 * 128 + 128, rows))
        one = torch.zeros(block.stop - block.start, n, dtype=torch.float64)
        for j, other in enumerate(at.tolist()):
            if block.start <= other < block.stop:
                one[other - block.start] = values[j].double()
        a, b = _q(one.t())[:, r - block.start], _q(x[block].t())[:, r - block.start]
        want += torch.outer(a, b)
        size += torch.outer(a, b).abs()
    _near(dw, want, size, 8)


def test_empty_calls(gpu_device):
    from evoformer_triton_amd import Fp8Weight, fp8_linear
    for rows, k, n in ((0, 5, 3), (4, 0, 3), (4, 5, 0), (0, 0, 0)):
        x, w, b = (torch.randn(s, device=gpu_device).requires_grad_() for s in ((rows, k), (n, k), (n,)))
        y = fp8_linear(x, w, b)
        assert y.shape == (rows, n)
        if k == 0:
            assert torch.equal(y, b.detach().expand(rows, n))
        dx, dw, db = torch.autograd.grad(y.sum() + 0 * (x.sum() + w.sum() + b.sum()), [x, w, b])
        assert not dx.any() and not dw.any() and dx.shape == x.shape and dw.shape == w.shape and torch.equal(db, torch.full_like(b, float(rows)))
        with torch.no_grad():
            assert torch.equal(fp8_linear(x, Fp8Weight.of(w), b), y)


def test_an_8_bit_weight_takes_no_gradients(gpu_device):
    from evoformer_triton_amd import Fp8Weight, fp8_linear
    w = Fp8Weight.of(torch.randn(8, 16, device=gpu_device))
    x, b = torch.randn(3, 16, device=gpu_device), torch.randn(8, device=gpu_device)
    for args in ((x.clone().requires_grad_(), w), (x, w, b.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="no_grad"):
            fp8_linear(*args)
        with torch.no_grad():
            assert fp8_linear(*args).shape == (3, 8)


@pytest.mark.parametrize("rows", [20, 300])
def test_a_captured_step_replays(gpu_device, rows):
    from evoformer_triton_amd import fp8_linear
    x, w, b = (torch.randn(s, device=gpu_device).to(BF16).requires_grad_() for s in ((rows, 1200), (90, 1200), (90,)))
    dy = torch.randn(rows, 90, device=gpu_device).to(BF16)

    def step():
        y = fp8_linear(x, w, b)
        return [y.detach(), *torch.autograd.grad(y, [x, w, b], dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        for t in (x, w, dy):
            t.data.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(held, step()):
            assert torch.equal(a, c)


def test_compiled_and_watched_calls_and_transforms(gpu_device):
    from torch.autograd import forward_ad
    from torch.utils._python_dispatch import TorchDispatchMode
    from evoformer_triton_amd import Fp8Weight, fp8_linear
    leaves = [torch.randn(s, device=gpu_device).requires_grad_() for s in ((70, 140), (30, 140), (30,))]
    want = fp8_linear(*leaves)
    want_g = torch.autograd.grad(want, leaves, torch.ones_like(want))
    seen = []

    class Recorder(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    with Recorder():
        watched = fp8_linear(*leaves)
    compiled = torch.compile(fp8_linear, fullgraph=True, backend="aot_eager")(*leaves)
    assert any("fp8_linear" in s for s in seen)
    for y in (watched, compiled):
        assert torch.equal(y, want) and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, torch.ones_like(y)), want_g))
    held = Fp8Weight.of(leaves[1])
    with torch.no_grad():
        assert torch.equal(torch.compile(lambda t: fp8_linear(t, held, leaves[2]), fullgraph=True, backend="aot_eager")(leaves[0]), want)
    x, w = leaves[0].detach(), leaves[1].detach()
    pair = torch.stack((x, 2 * x))
    assert torch.equal(torch.func.vmap(lambda t: fp8_linear(t, w))(pair), torch.stack((fp8_linear(x, w), fp8_linear(2 * x, w))))
    with forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        fp8_linear(forward_ad.make_dual(x, torch.ones_like(x)).requires_grad_(), w)
    dx, = torch.autograd.grad(fp8_linear(*leaves).square().sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        dx.sum().backward()
