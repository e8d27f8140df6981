"""The gated block with a relative position bias and with projections in 8 bits: what its parts give one after the other."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _case(dev, dt=torch.bfloat16, c_z=64, gating=True, **options):
    from evoformer_triton_amd.block import GatedAttentionBlock
    torch.manual_seed(12)
    block = GatedAttentionBlock(96, 32, 4, c_z=c_z, gating=gating, **options).to(dev).to(dt)
    if block.relative is not None:
        block.relative.weight.data.normal_()
    B, S, N = 2, 6, 72
    m = torch.randn(B, S, N, 96, device=dev).to(dt).requires_grad_()
    z = torch.randn(B, N, N, c_z, device=dev).to(dt).requires_grad_() if c_z else None
    mask = (torch.rand(B, S, N, device=dev) < 0.9).float()
    mask[1, 2] = 0                                                 # a row without a key
    at = torch.arange(N, device=dev) + (torch.arange(N, device=dev) > 40) * 30
    chains = (torch.arange(N, device=dev) > 50).long().expand(B, N)
    return block, m, z, mask, at.expand(B, N), chains, torch.randn(B, S, N, 96, device=dev).to(dt)


def _leaves(block, m, z):
    return [m] + ([z] if z is not None else []) + list(block.parameters())


def _vanishing(block, m, z, mask, at, chains, dout):
    """What the gradient of layer_norm_z.bias may be off by.  A constant added to a row's scores moves no softmax, so it is
    sum_r W^T g_r = 0 with g_r = the gradient of the row r of linear_z's result: what is computed is the rounding errors of the
    terms alone.  Where each g_r is off by 2e-2 |g_r|, by itself, the squares of the terms' errors add up:
    sqrt(sum_r (2e-2 |W| |g_r|)^2) = 2e-2 |W| |g|.  In fp32, of a copy of the block."""
    import copy
    ref, kept = copy.deepcopy(block).float(), []
    ref.linear_z.register_forward_hook(lambda mod, args, out: (out.retain_grad(), kept.append(out))[0])
    ref.forward_eager(m.detach().float(), z.detach().float(), mask, at, chains).backward(dout.float())
    return 2e-2 * ref.linear_z.weight.norm() * kept[0].grad.norm()


@pytest.mark.parametrize("c_z,gating", [(64, True), (None, False)])
def test_the_relative_bias_in_the_block(gpu_device, c_z, gating):
    """Against plain torch operations in fp32: roundings of 16-bit operands and results, as of the block without it."""
    block, m, z, mask, at, chains, dout = _case(gpu_device, c_z=c_z, gating=gating, relative_distance=32, relative_buckets=16, other_chain=True)
    leaves = _leaves(block, m, z)
    y = block(m, z, mask, at, chains)
    got = torch.autograd.grad(y, leaves, dout)
    vanishing = _vanishing(block, m, z, mask, at, chains, dout) if c_z else None
    names = ["m", "z"][:1 if z is None else 2] + [name for name, _ in block.named_parameters()]
    ref = block.float()
    f = [t.detach().float().requires_grad_() for t in leaves[:1 if z is None else 2]]
    want_y = ref.forward_eager(f[0], f[1] if z is not None else None, mask, at, chains)
    want = torch.autograd.grad(want_y, f + list(ref.parameters()), dout.float())
    assert (y.float() - want_y).norm() <= 1e-2 * want_y.norm()
    for name, a, b in zip(names, got, want):
        bound = vanishing if name == "layer_norm_z.bias" else 2e-2 * b.norm() + 1e-3 * b.numel() ** 0.5
        assert (a.float() - b).norm() <= bound, name
    assert got[names.index("relative.weight")].float().abs().max() > 0


def _by_parts(block, m, z, mask, at, chains):
    """The same from the public functions, one after the other."""
    from evoformer_triton_amd import evoformer_attention, fp8_linear
    B, S, N, _ = m.shape
    x = _norm(block, m)
    w = torch.cat([block.linear_q.weight, block.linear_k.weight, block.linear_v.weight, block.linear_g.weight])
    b = torch.cat([block.linear_g.bias.new_zeros(3 * 128), block.linear_g.bias])
    q, k, v, g = fp8_linear(x, w, b).view(B, S, N, 4, 4, 32).unbind(3)
    bias, add = block._bias_and_mask(z, mask, m.dtype, (B, S, N), *_fns(), at, chains)
    o = evoformer_attention(q.contiguous(), k.contiguous(), v.contiguous(), add, bias, layout="ds4sci", gate=g.contiguous())
    return fp8_linear(o.reshape(B, S, N, 128), block.linear_o.weight, block.linear_o.bias)


def _fns():
    from evoformer_triton_amd import block as b
    return b._layer_norm, b._linear


def _norm(block, m):
    return _fns()[0](block.layer_norm_m, m)


def test_8_bit_projections_and_the_relative_bias_together(gpu_device):
    block, m, z, mask, at, chains, dout = _case(gpu_device, fp8=True, relative_distance=16, other_chain=True)
    leaves = _leaves(block, m, z)
    y = block(m, z, mask, at, chains)
    got = torch.autograd.grad(y, leaves, dout)
    want_y = _by_parts(block, m, z, mask, at, chains)
    want = torch.autograd.grad(want_y, leaves, dout)
    assert torch.equal(y, want_y)
    for (name, _), a, b in zip([("m", 0), ("z", 0)] + list(block.named_parameters()), got, want):
        # (the gated attention on slots of one buffer and on tensors of their own: the same numbers, rounded at other places in the gate's pass)
        bound = _vanishing(block, m, z, mask, at, chains, dout) if name == "layer_norm_z.bias" else 1e-2 * b.float().norm() + 1e-3 * b.numel() ** 0.5
        assert torch.isfinite(a).all() and (a.float() - b.float()).norm() <= bound, name
    with torch.no_grad():
        assert torch.equal(block(m, z, mask, at, chains, weights=block.fp8_weights()), y)


def test_8_bit_projections_in_fp32_and_without_a_gate(gpu_device):
    for options in (dict(dt=torch.float32), dict(gating=False), dict(dt=torch.float16, c_z=None)):
        block, m, z, mask, at, chains, dout = _case(gpu_device, fp8=True, **options)
        y = block(m, z, mask)
        grads = torch.autograd.grad(y, _leaves(block, m, z), dout)
        assert all(torch.isfinite(g).all() for g in grads)
        with torch.no_grad():
            assert torch.equal(block(m, z, mask, weights=block.fp8_weights()), y)
            near = block.forward_eager(m, z, mask)
        # operands within 2^-4 of themselves, twice one after the other: a few parts in a hundred of the result
        assert (y - near).float().norm() <= 0.15 * near.float().norm()


def test_a_captured_step_of_both_replays(gpu_device):
    block, m, z, mask, at, chains, dout = _case(gpu_device, fp8=True, relative_distance=16, other_chain=True)
    leaves = _leaves(block, m, z)

    def step():
        y = block(m, z, mask, at, chains)
        return [y.detach(), *torch.autograd.grad(y, leaves, dout)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        for t in (m, z, dout):
            t.data.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_a_compiled_block(gpu_device):
    block, m, z, mask, at, chains, dout = _case(gpu_device, fp8=True, relative_distance=16, other_chain=True)
    want = block(m, z, mask, at, chains)
    got = torch.compile(block, backend="aot_eager")(m, z, mask, at, chains)
    assert (got.float() - want.float()).norm() <= 1e-2 * want.float().norm()
