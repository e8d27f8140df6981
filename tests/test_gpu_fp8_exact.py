"""Linear layers in 8 bits where every number is one that the formats hold: a result has to be the formula's, bit for bit.

Whole numbers of two bits times powers of two from 1 to 8 are what they are in e4m3, whatever their block's scale, and so are their products; neighbouring products
lie within seven bits of each other, sums within 24.  A lost element, a wrong scale or a block that is left out shows in whole units."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _whole(shape, g, dt, dev):
    """-3 .. 3, times a power of two for each row and block of 128 columns."""
    rows, cols = shape
    v = torch.randint(-3, 4, shape, generator=g, device=dev).float()
    s = torch.randint(0, 4, (rows, -(-cols // 128)), generator=g, device=dev)
    return (v * torch.exp2(s.float()).repeat_interleave(128, 1)[:, :cols]).to(dt)


# rows, k, n: few rows (one to four tiles of them, slices, both widths of a workgroup), strips rounded on the way or before, tiles of 128 x 128 with and without slices,
# tiles of 256 x 256; last rows, columns and blocks of every kind
SIZES = [(1, 256, 1024), (17, 1300, 70), (33, 4096, 4100), (64, 1920, 8200), (65, 300, 70), (129, 129, 127), (65537, 130, 200), (40000, 400, 100), (200, 512, 1000),
         (300, 380, 200), (300, 1100, 96), (128, 4224, 64), (5021, 500, 333), (2500, 640, 200), (66000, 520, 260), (33000, 700, 300), (8192, 1030, 2050)]


@pytest.mark.parametrize("dt,wdt", [(BF16, BF16), (F16, F32), (F32, F32), (BF16, F32)], ids=str)
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_whole_numbers_are_exact(gpu_device, rows, k, n, dt, wdt):
    from evoformer_triton_amd import Fp8Weight, fp8_linear
    g = torch.Generator(device=gpu_device).manual_seed(rows + k + n)
    x, w, dy = _whole((rows, k), g, dt, gpu_device), _whole((n, k), g, wdt, gpu_device), torch.randint(-3, 4, (rows, n), generator=g, device=gpu_device).to(dt)
    b = torch.randint(-9, 10, (n,), generator=g, device=gpu_device).to(F32)
    xd, wd, dd = x.double(), w.double(), dy.double()
    for p, q in ((xd, wd.t()), (dd, wd), (dd.t(), xd)):
        assert (p.abs() @ q.abs()).max() < 2 ** 24                       # (no sum of any of the terms needs more than 24 bits)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = fp8_linear(*leaves)
    got = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(y, (xd @ wd.t() + b.double()).to(dt))
    for a, want, t in zip(got, (dd @ wd, dd.t() @ xd, dd.sum(0)), leaves):
        assert torch.equal(a, want.to(t.dtype)), t.shape
    with torch.no_grad():
        assert torch.equal(fp8_linear(x, Fp8Weight.of(w), b), y)


@pytest.mark.parametrize("rows,k,n", [(5, 256, 70), (40, 700, 300), (200, 250, 130), (300, 380, 200), (300, 640, 200), (33000, 600, 520)])
def test_sums_of_fp32_results_lose_no_small_term(gpu_device, rows, k, n):
    """In each block one product is 2^21 times as large as the smallest beside it, which is lost where eight neighbours keep 13 bits of the largest; in fp32 all sums hold both."""
    from evoformer_triton_amd import fp8_linear
    g = torch.Generator(device=gpu_device).manual_seed(rows + k)

    def small(shape, unit):
        sign = torch.randint(0, 2, shape, generator=g, device=gpu_device) * 2 - 1
        return (torch.randint(0, 2, shape, generator=g, device=gpu_device) * 2 + 1).float() * sign * unit

    def signs(shape):
        return (torch.randint(0, 2, shape, generator=g, device=gpu_device) * 2 - 1).float()

    x, w = small((rows, k), 2.0 ** -5), small((n, k), 2.0 ** -4)
    for block in range(0, k, 128):
        at = block + torch.randint(0, min(128, k - block), (1,), generator=g, device=gpu_device)
        x[:, at], w[:, at] = 256 * signs((rows, 1)), 16 * signs((n, 1))
    assert torch.equal(fp8_linear(x, w).double(), x.double() @ w.double().t())
    # the weight's gradient: four rows of the kind, in blocks of their own where there are as many
    x, dy = small((rows, k), 2.0 ** -5), small((rows, n), 2.0 ** -4)
    for at in {0, rows // 3, rows // 2, rows - 1}:
        x[at], dy[at] = 256 * signs((k,)), 16 * signs((n,))
    w.requires_grad_()
    dw, = torch.autograd.grad(fp8_linear(x, w), w, dy)
    assert torch.equal(dw.double(), dy.double().t() @ x.double())


def _rounded(x):
    """Q along the last axis of [rows, 128]: values in units of the scale and exponents, in 64 bits."""
    v = x.double()
    a = torch.where(v.isfinite(), v.abs(), 0).amax(-1, keepdim=True)
    m, e = torch.frexp(a)
    e = torch.where(a == 0, 0, torch.where(m > 0.875, e - 8, e - 9).clamp(-127, 127))
    u = torch.ldexp(v, -e)
    u = torch.where(u.isfinite(), u, float("nan"))
    step = torch.exp2(torch.floor(torch.log2(torch.where((u == 0) | u.isnan(), 1.0, u.abs()))).clamp(-6, 8) - 3)
    return torch.round(u / step) * step, e


@pytest.mark.parametrize("dt", [BF16, F16], ids=str)
def test_every_number_of_16_bits_is_rounded_as_defined(gpu_device, dt):
    """All of them, subnormal ones, infinities and NaN too, beside the largest of a block."""
    from evoformer_triton_amd import Fp8Weight
    every = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dt)
    every = torch.cat([every, torch.zeros(127 * 517 - 65536, dtype=dt)]).view(517, 127)
    for most in (0.0, torch.finfo(dt).max, 2.0 ** -130 if dt == BF16 else 2.0 ** -24, 2.0 ** -120 if dt == BF16 else 2.0 ** -14, 1.75, 1.7578125, 300.0):
        x = torch.cat([torch.full((517, 1), most).to(dt), every], 1)
        if most:
            x = torch.where(x.float().abs() <= x[:1, :1].float(), x, torch.where(x.isfinite(), 0, x))
        w = Fp8Weight.of(x.to(gpu_device))
        u, e = _rounded(x)
        got = w.values.cpu().double()
        assert torch.equal(w.scales.cpu()[:, :1].int() - 127, e.int()), most
        assert torch.equal(got.isnan(), u.isnan()) and torch.equal(got.nan_to_num(), u.nan_to_num()), most


def test_the_values_are_exact_on_the_gpu(gpu_device):
    """What a weight stands for, at every scale there is: e4m3 times a power of two."""
    from evoformer_triton_amd import Fp8Weight
    values = torch.arange(256, dtype=torch.uint8).view(2, 128)
    for byte in range(255):
        for dev in ("cpu", gpu_device):
            got = Fp8Weight(values.to(dev), torch.full((2, 4), byte, dtype=torch.uint8, device=dev), 128).dequantize().cpu()
            want = (values.view(torch.float8_e4m3fn).double() * 2.0 ** (byte - 127)).float()
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7), want.nan_to_num(7)), (byte, dev)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("rows,k,n", [(1, 256, 70), (40, 1300, 300), (200, 250, 130), (300, 640, 200)])
def test_a_scale_that_is_no_number(gpu_device, rows, k, n, dt):
    """A byte of 255: the weight's row has no numbers in that block, and results by it are none."""
    from evoformer_triton_amd import Fp8Weight, fp8_linear
    w = Fp8Weight.of(torch.randn((n, k), generator=torch.Generator().manual_seed(1)).to(gpu_device))
    w.scales[3, 1] = 255
    assert w.dequantize().isnan().nonzero().tolist() == [[3, c] for c in range(128, min(256, k))]
    with torch.no_grad():
        bad = fp8_linear(torch.zeros(rows, k, device=gpu_device, dtype=dt), w).isnan()
    assert bad[:, 3].all() and bad.sum() == rows


@pytest.mark.parametrize("rows", [3000, 9000])
def test_the_registered_backward_fills_no_memory_twice(gpu_device, rows):
    """What a compiled or watched step calls takes the gradients' memory once."""
    import evoformer_triton_amd  # noqa: F401
    k, n = 1024, 768
    x, w, b, dy = (torch.randn(s, device=gpu_device).to(torch.bfloat16) for s in ((rows, k), (n, k), (n,), (rows, n)))
    torch.ops.evoattn.fp8_linear_bwd(dy, x, w, b, True, False, False)

    def taken(need_x):
        before = torch.cuda.memory_stats()["allocated_bytes.all.allocated"]
        grads = torch.ops.evoattn.fp8_linear_bwd(dy, x, w, b, need_x, False, False)
        return torch.cuda.memory_stats()["allocated_bytes.all.allocated"] - before, grads[0]

    total, dx = taken(True)
    up = lambda v: -(-v // 128) * 128  # noqa: E731
    rounded = k * up(n) + rows * up(n) + 16 * (k + rows)                     # w^T and dy along their rows, with scales
    assert dx.shape == x.shape and total < rounded + dx.numel() * 2 * 1.5      # (bytes: less than twice dx's; the product is not cut into slices)
