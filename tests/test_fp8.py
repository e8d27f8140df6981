"""Linear layers in 8 bits without a GPU: their refusals, the C ABI's checks, the traced operators' shapes, the block's options."""
import ctypes

import pytest
import torch

from evoformer_triton_amd import Fp8Weight, _lib, fp8_linear
from evoformer_triton_amd.block import Fp8BlockWeights, GatedAttentionBlock


@pytest.mark.parametrize("x,w,b,match", [
    (torch.zeros(3, 5, dtype=torch.float64), torch.zeros(4, 5), None, "input must be"), (torch.zeros(()), torch.zeros(4, 5), None, "input must be"),
    (torch.zeros(3, 5), torch.zeros(4, 6), None, "last dimension"), (torch.zeros(3, 5), torch.zeros(4, 5, 1), None, "weight must be"),
    (torch.zeros(3, 5), torch.zeros(4, 5, dtype=torch.int8), None, "weight must be"), (torch.zeros(3, 5), torch.zeros(4, 5), torch.zeros(5), "bias must be"),
    (torch.zeros(3, 5), torch.zeros(4, 5), torch.zeros(4, dtype=torch.float64), "bias must be"), (torch.zeros(3, 5), torch.zeros(4, 5), torch.zeros(4, device="meta"), "one device"),
    (torch.zeros(1, 1).expand(2 ** 26 + 1, 1), torch.zeros(4, 1), None, "2.26 rows"), (torch.zeros(1, 1), torch.zeros(1, 1).expand(2 ** 26 + 1, 1), None, "2.26 rows or columns"),
    (torch.zeros(1, 1).expand(1, 2 ** 26 + 1), torch.zeros(1, 1).expand(1, 2 ** 26 + 1), None, "2.26 rows or columns"), (torch.zeros(3, 5), torch.zeros(4, 5), None, "GPU only")])
def test_calls_that_are_refused(x, w, b, match):
    with pytest.raises((ValueError, RuntimeError), match=match):
        fp8_linear(x, w, b)


def _held(n=4, k=300, **change):
    u8 = torch.uint8
    parts = dict(values=torch.zeros(n, 384, dtype=torch.float8_e4m3fn), scales=torch.full((n, 4), 127, dtype=u8), k=k)
    return Fp8Weight(**{**parts, **change})


@pytest.mark.parametrize("change", [dict(values=torch.zeros(4, 300, dtype=torch.uint8)), dict(values=torch.zeros(4, 384)), dict(scales=torch.zeros(4, 3, dtype=torch.uint8)),
                                    dict(scales=torch.zeros(3, 4, dtype=torch.uint8)), dict(k=400), dict(k=-1), dict(values=torch.zeros(384, 4, dtype=torch.uint8).t()),
                                    dict(scales=torch.zeros(4, 4))])
def test_weights_in_8_bits_that_are_refused(change):
    w = _held(**change)
    with pytest.raises(ValueError, match="8 bits"):
        fp8_linear(torch.zeros(2, w.k if w.k > 0 else 300), w)


def test_what_else_is_refused():
    with pytest.raises(TypeError, match="weight"):
        fp8_linear(torch.zeros(2, 3), [[1.0, 2.0, 3.0]])
    with pytest.raises(TypeError, match="bias"):
        fp8_linear(torch.zeros(2, 3), torch.zeros(4, 3), 1.0)
    with pytest.raises(RuntimeError, match="GPU only"):
        fp8_linear(torch.zeros(2, 300), _held())
    with pytest.raises(RuntimeError, match="GPU only"):
        Fp8Weight.of(torch.zeros(2, 300))
    with pytest.raises(ValueError, match="weight must be"):
        Fp8Weight.of(torch.zeros(300))


def test_what_the_bytes_stand_for():
    w = _held(n=2, k=130, values=torch.zeros(2, 256, dtype=torch.uint8), scales=torch.tensor([[127, 130, 127, 127], [0, 119, 127, 127]], dtype=torch.uint8))
    w.values[0, :3] = torch.tensor([0x38, 0xb8, 0x7e])        # 1, -1, 448
    w.values[0, 128] = 0x01                                    # 2^-9, in units of 2^3
    w.values[1, 0], w.values[1, 129] = 0x40, 0x39              # 2, in units of 2^-127; 1.125, of 2^-8
    d = w.dequantize()
    assert d.shape == (2, 130) and d.dtype == torch.float32
    assert d[0, :3].tolist() == [1, -1, 448] and d[0, 128] == 2.0 ** -6 and d[1, 0] == 2.0 ** -126 and d[1, 129] == 1.125 * 2.0 ** -8


def test_the_traced_operators_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, w, b = (torch.empty(s, device="cuda", dtype=torch.bfloat16) for s in ((2, 7, 40), (30, 40), (30,)))
        y = torch.ops.evoattn.fp8_linear(x, w, b)
        assert y.shape == (2, 7, 30) and y.dtype == torch.bfloat16
        assert [tuple(t.shape) for t in torch.ops.evoattn.fp8_linear_bwd(y, x, w.float(), b, True, True, False)] == [(2, 7, 40), (30, 40), (0,)]
        q, s = torch.empty(30, 128, device="cuda", dtype=torch.uint8), torch.empty(30, 4, device="cuda", dtype=torch.uint8)
        assert torch.ops.evoattn.fp8_linear_held(x, q, s, 40, None).shape == (2, 7, 30)


def _product(**change):
    p = _lib.EvoFp8Matmul()
    p.m, p.n, p.k, p.ldo, p.dtype, p.bias_dtype = 300, 200, 5000, 200, _lib.EVO_BF16, _lib.EVO_F32
    for f in ("a", "b", "scales_a", "scales_b", "out", "workspace"):
        setattr(p, f, 0x10000)
    p.workspace_bytes = 1 << 30
    for k, v in change.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,code", [
    (dict(m=0), _lib.EVO_EINVAL), (dict(n=-1), _lib.EVO_EINVAL), (dict(k=0), _lib.EVO_EINVAL), (dict(dtype=5), _lib.EVO_EINVAL), (dict(a=None), _lib.EVO_EINVAL),
    (dict(scales_b=None), _lib.EVO_EINVAL), (dict(out=None), _lib.EVO_EINVAL), (dict(ldo=199), _lib.EVO_EINVAL), (dict(bias=0x10000, bias_dtype=-1), _lib.EVO_EINVAL),
    (dict(a=0x10008), _lib.EVO_EALIGN), (dict(scales_a=0x10002), _lib.EVO_EALIGN), (dict(k=(1 << 26) + 1), _lib.EVO_EUNSUPPORTED), (dict(m=1 << 31), _lib.EVO_EOVERFLOW),
    (dict(workspace=None), _lib.EVO_EWORKSPACE), (dict(workspace_bytes=100), _lib.EVO_EWORKSPACE)])
def test_products_that_the_c_abi_rejects_before_any_launch(change, code):
    assert _lib.load().evoattn_fp8_matmul(ctypes.byref(_product(**change)), None) == code


@pytest.mark.parametrize("change,x,ldx,code", [
    (dict(), 0x10000, 5000, _lib.EVO_EUNSUPPORTED), (dict(m=64), None, 5000, _lib.EVO_EINVAL), (dict(m=64), 0x10000, 4999, _lib.EVO_EINVAL), (dict(m=64, b=0x10001), 0x10000, 5000, _lib.EVO_EALIGN),
    (dict(m=64, workspace=None), 0x10000, 5000, _lib.EVO_EWORKSPACE), (dict(m=0), 0x10000, 5000, _lib.EVO_EINVAL)])
def test_few_rows_that_the_c_abi_rejects_before_any_launch(change, x, ldx, code):
    assert _lib.load().evoattn_fp8_matmul_rounding(ctypes.byref(_product(**change)), x, ldx, None) == code


def test_the_c_abis_workspaces():
    lib = _lib.load()
    need = lib.evoattn_fp8_matmul_workspace_bytes(ctypes.byref(_product()))
    assert need > 0 and need % (300 * 200 * 4) == 0
    assert lib.evoattn_fp8_matmul_workspace_bytes(ctypes.byref(_product(m=8192, n=8192))) == 0 and lib.evoattn_fp8_matmul_workspace_bytes(ctypes.byref(_product(k=0))) == 0
    assert lib.evoattn_fp8_matmul_rounding_workspace_bytes(ctypes.byref(_product(m=65))) == 0 and lib.evoattn_fp8_matmul_rounding_workspace_bytes(ctypes.byref(_product(m=3, k=256))) == 0
    assert lib.evoattn_fp8_matmul_rounding_workspace_bytes(ctypes.byref(_product(m=3))) % (3 * 200 * 4) == 0


@pytest.mark.parametrize("args,code", [
    ((None, 40, 0x10000, 0x10000, None, None, None, 3, 40, 0), _lib.EVO_EINVAL), ((0x10000, 39, 0x10000, 0x10000, None, None, None, 3, 40, 0), _lib.EVO_EINVAL),
    ((0x10000, 40, 0x10000, None, None, None, None, 3, 40, 0), _lib.EVO_EINVAL), ((0x10000, 40, None, None, None, None, None, 3, 40, 0), _lib.EVO_EINVAL),
    ((0x10000, 40, 0x10000, 0x10000, None, None, 0x10000, 3, 40, 0), _lib.EVO_EINVAL), ((0x10000, 40, 0x10000, 0x10000, None, None, None, 0, 40, 0), _lib.EVO_EINVAL),
    ((0x10000, 40, 0x10000, 0x10000, None, None, None, 3, 40, 3), _lib.EVO_EINVAL), ((0x10000, 40, 0x10008, 0x10000, None, None, None, 3, 40, 0), _lib.EVO_EALIGN),
    ((0x10000, 1 << 27, 0x10000, 0x10000, None, None, None, 3, (1 << 26) + 1, 0), _lib.EVO_EUNSUPPORTED)])
def test_rounding_that_the_c_abi_rejects_before_any_launch(args, code):
    assert _lib.load().evoattn_fp8_quantize(*args, None) == code


def test_two_at_once_that_the_c_abi_rejects_before_any_launch():
    lib = _lib.load()

    def two(a, b, dtype=_lib.EVO_BF16):
        r = [_lib.EvoFp8Rounding(0x10000, 40, 3, 40, 0x10000, 0x10000, None, None, None) for _ in range(2)]
        for one, change in zip(r, (a, b)):
            for k, v in change.items():
                setattr(one, k, v)
        return lib.evoattn_fp8_quantize_two(ctypes.byref(r[0]), ctypes.byref(r[1]), dtype, None)
    for change, code in ((dict(x=None), _lib.EVO_EINVAL), (dict(ldx=39), _lib.EVO_EINVAL), (dict(sums=0x10000), _lib.EVO_EINVAL), (dict(q=0x10004), _lib.EVO_EALIGN), (dict(rows=0), _lib.EVO_EINVAL),
                         (dict(cols=(1 << 26) + 1, ldx=1 << 27), _lib.EVO_EUNSUPPORTED)):
        assert two(change, {}) == code and two({}, change) == code
    assert two({}, {}, 7) == _lib.EVO_EINVAL and lib.evoattn_fp8_quantize_two(None, None, 0, None) == _lib.EVO_EINVAL
    for change in (dict(sums=None), dict(rows=0), dict(out=None), dict(dtype=4)):
        args = {**dict(sums=0x10000, rows=300, out=0x10000, dtype=0), **change}
        assert lib.evoattn_fp8_matmul_sums(ctypes.byref(_product()), *args.values(), None) == _lib.EVO_EINVAL
    assert lib.evoattn_fp8_matmul_sums(ctypes.byref(_product(workspace=None)), 0x10000, 300, 0x10000, 0, None) == _lib.EVO_EWORKSPACE
    rounds = [lib.evoattn_fp8_matmul_rounds(ctypes.byref(_product(m=m, n=n, k=k, dtype=t))) for m, n, k, t in ((64, 9, 5000, 0), (65, 9, 5000, 0), (70000, 900, 256, 2), (70000, 900, 257, 2), (70000, 300, 500, 0), (200, 3000, 500, 0))]
    assert rounds == [1, 0, 1, 0, 1, 0]


def test_the_blocks_options():
    plain = GatedAttentionBlock(64, 32, 4, c_z=64)
    block = GatedAttentionBlock(64, 32, 4, c_z=64, fp8=True, relative_distance=16, relative_buckets=8, other_chain=True)
    assert set(block.state_dict()) - set(plain.state_dict()) == {"relative.weight"} and block.relative.weight.shape == (9, 4)
    m, z, at = torch.zeros(1, 2, 5, 64), torch.zeros(1, 5, 5, 64), torch.arange(5)
    for b, args, match in ((block, dict(), "positions"), (plain, dict(positions=at), "relative_distance"), (plain, dict(chains=at), "other_chain"),
                           (plain, dict(weights=Fp8BlockWeights(None, None, None)), "fp8=True"),
                           (GatedAttentionBlock(64, 32, 4, relative_distance=4), dict(positions=at, chains=at), "other_chain")):
        with pytest.raises(ValueError, match=match):
            b(m, z, None, **args)
    with pytest.raises(ValueError, match="relative_distance"):
        GatedAttentionBlock(64, 32, 4, other_chain=True)


def test_a_block_that_was_saved_without_the_options():
    import copy
    torch.manual_seed(2)
    block = GatedAttentionBlock(16, 8, 2, c_z=8)
    old = copy.copy(block)
    old.__dict__ = {k: v for k, v in block.__dict__.items() if k not in ("relative", "fp8")}
    old._modules = {k: v for k, v in block._modules.items() if k != "relative"}
    m, z = torch.randn(1, 3, 7, 16), torch.randn(1, 7, 7, 8)
    assert torch.equal(old.forward_eager(m, z), block.forward_eager(m, z))
    with pytest.raises(ValueError, match="relative_distance"):
        old(m, z, None, torch.arange(7))


def test_the_relative_bias_in_plain_operations_moves_the_blocks_result():
    torch.manual_seed(3)
    block = GatedAttentionBlock(16, 8, 2, c_z=8, relative_distance=4, other_chain=True)
    m, z, at, chain = torch.randn(1, 3, 7, 16), torch.randn(1, 7, 7, 8), torch.arange(7), torch.tensor([[0, 0, 0, 0, 1, 1, 1]])
    with torch.no_grad():
        before = block.forward_eager(m, z, None, at, chain)
        assert torch.equal(before, block.forward_eager(m, z, None, at + 5, chain))      # (a table of zeros; and only differences count)
        block.relative.weight.normal_()
        after = block.forward_eager(m, z, None, at, chain)
        assert not torch.allclose(before, after) and torch.allclose(after, block.forward_eager(m, z, None, at + 5, chain))
        block.relative.weight.copy_(torch.arange(10.).view(10, 1).expand(10, 2))
        bias = block.relative.plain(at, chains=chain)
        assert bias.shape == (1, 1, 2, 7, 7) and bias[0, 0, 0, 0].tolist() == [4, 3, 2, 1, 9, 9, 9] and bias[0, 0, 1, :4, 0].tolist() == [4, 5, 6, 7]
