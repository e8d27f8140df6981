"""The gated block with rotary positions and on packed sequences, and a prompt whose tokens come one by one: rotary positions and packed attention as they are used together."""
import pytest
import torch

from oracle.packed import packed
from test_gpu_packed import _close

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
LENGTHS = [70, 1, 0, 133, 40]


def _block(dev, dt, gating=True, rotary=None, **options):
    from evoformer_triton_amd import RotaryPositions
    from evoformer_triton_amd.block import GatedAttentionBlock
    torch.manual_seed(3)
    rotary = None if rotary is None else RotaryPositions(32, **rotary)
    return GatedAttentionBlock(96, 32, 4, gating=gating, rotary=rotary, **options).to(dev).to(dt)


def _near(got, want, dt, names):
    """Norms apart by a few times what independent roundings of some six (forward) and twelve (backward) operands and results, 2^-9 of them each for bf16, make of them; in fp32 sums over some hundred
    terms count, 1e-5."""
    eps = max(torch.finfo(dt).eps, 1e-5)
    for i, (name, a, b) in enumerate(zip(names, got, want)):
        assert torch.isfinite(a).all(), name
        assert (a.float() - b).norm() <= (1.28 if i == 0 else 2.56) * eps * b.norm() + (0 if i == 0 else 0.13 * eps * b.numel() ** 0.5), name


@pytest.mark.parametrize("dt,gating,rotary,relative", [
    (BF16, True, {}, None), (F16, False, dict(interleaved=True, rotary_dim=16), None), (BF16, True, dict(scaling="parts", factor=8.0, original_length=64), 16),
    (F32, True, dict(base=500.0), None)])
def test_rotary_positions_in_the_block(gpu_device, dt, gating, rotary, relative):
    block = _block(gpu_device, dt, gating, rotary, relative_distance=relative)
    if relative:
        block.relative.weight.data.normal_()
    B, S, N = 2, 3, 72
    m = torch.randn(B, S, N, 96, device=gpu_device).to(dt).requires_grad_()
    mask = (torch.rand(B, S, N, device=gpu_device) < 0.9).float()
    mask[1, 2] = 0
    at = torch.arange(N, device=gpu_device) + torch.tensor([[0], [1000]], device=gpu_device)
    dout = torch.randn(B, S, N, 96, device=gpu_device).to(dt)
    y = block(m, None, mask, at)
    got = [y, *torch.autograd.grad(y, [m, *block.parameters()], dout)]
    names = ["y", "m"] + [n for n, _ in block.named_parameters()]
    ref, f = block.float(), m.detach().float().requires_grad_()
    y = ref.forward_eager(f, None, mask, at)
    _near(got, [y, *torch.autograd.grad(y, [f, *ref.parameters()], dout.float())], dt, names)
    # with other positions another result
    assert not torch.equal(ref.forward_eager(f, None, mask, at * 3), y)


def _reference(block, m, lengths, positions, causal):
    """Sequence by sequence in plain operations."""
    outs, begin, H, D = [], 0, block.no_heads, block.c_hidden
    for n in lengths:
        rows = slice(begin, begin + n)
        begin += n
        if n == 0:
            continue
        q, k, v, g, _, _ = block.operands(m[rows][None, None], None, None, plain=True, positions=None if block.rotary is None else positions[rows])
        q, k, v = (t[0, 0].transpose(0, 1) for t in (q, k, v))
        s = torch.matmul(q, k.transpose(1, 2).contiguous()) * D ** -0.5
        if causal:
            s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device=s.device).tril(), float("-inf"))
        o = torch.matmul(torch.softmax(s, -1), v).transpose(0, 1)
        if g is not None:
            o = torch.sigmoid(g[0, 0]) * o
        outs.append(o.reshape(n, H * D))
    outs.append(m.new_zeros(m.shape[0] - begin, H * D))
    return block.linear_o(torch.cat(outs))


def _packed_case(dev, dt, padding=3):
    T = sum(LENGTHS) + padding
    g = torch.Generator(device=dev).manual_seed(9)
    off = torch.tensor([0] + LENGTHS, device=dev).cumsum(0)
    return [torch.randn(T, 96, device=dev, generator=g).to(dt) for _ in range(2)] + [off]


@pytest.mark.parametrize("dt,gating,rotary,causal", [(BF16, True, {}, False), (F16, True, None, True), (BF16, False, dict(rotary_dim=8), True), (F32, True, {}, True)])
def test_packed_sequences_in_the_block(gpu_device, dt, gating, rotary, causal):
    from evoformer_triton_amd import packed_positions
    block = _block(gpu_device, dt, gating, rotary)
    m, dout, off = _packed_case(gpu_device, dt)
    m.requires_grad_()
    y = block.packed(m, off, causal=causal)
    got = [y, *torch.autograd.grad(y, [m, *block.parameters()], dout)]
    at = packed_positions(off, m.shape[0])
    if rotary is not None:
        assert torch.equal(block.packed(m, off, at, causal=causal), y)
    names = ["y", "m"] + [n for n, _ in block.named_parameters()]
    ref, f = block.float(), m.detach().float().requires_grad_()
    y = _reference(ref, f, LENGTHS, at, causal)
    _near(got, [y, *torch.autograd.grad(y, [f, *ref.parameters()], dout.float())], dt, names)


def test_the_blocks_packed_rows_are_its_parts_one_after_the_other(gpu_device):
    from evoformer_triton_amd import packed_attention, packed_positions, rotary_positions
    from evoformer_triton_amd import block as b
    block = _block(gpu_device, BF16, rotary=dict(interleaved=True))
    m, dout, off = _packed_case(gpu_device, BF16)
    m.requires_grad_()

    def parts():
        P = b._StackedProjection.apply(b._layer_norm(block.layer_norm_m, m), block.linear_g.bias, block.linear_q.weight, block.linear_k.weight, block.linear_v.weight,
                                       block.linear_g.weight).view(-1, 4, 4, 32)
        q, k = rotary_positions(P[:, 0], P[:, 1], packed_positions(off, m.shape[0]), block.rotary.turns, interleaved=True)
        o = torch.sigmoid(P[:, 3]) * packed_attention(q, k, P[:, 2], off, causal=False)
        return b._linear(block.linear_o, o.reshape(-1, 128))

    leaves = [m, *block.parameters()]
    y, want = block.packed(m, off), parts()
    assert torch.equal(y, want)
    for a, w in zip(torch.autograd.grad(y, leaves, dout), torch.autograd.grad(want, leaves, dout)):
        assert torch.equal(a, w)


def test_packed_rows_in_8_bits_under_autocast_and_compiled(gpu_device):
    block = _block(gpu_device, BF16, rotary={}, fp8=True)
    m, dout, off = _packed_case(gpu_device, BF16)
    with torch.no_grad():
        y = block.packed(m, off)
        assert torch.equal(block.packed(m, off, weights=block.fp8_weights()), y)
        at = torch.arange(m.shape[0], device=gpu_device)
        assert torch.equal(block(m[None, None], None, None, at), block(m[None, None], None, None, at, weights=block.fp8_weights()))
    block = _block(gpu_device, F32, rotary={})
    m = m.float().requires_grad_()
    want = block.packed(m, off)
    with torch.autocast("cuda", torch.bfloat16):
        y = block.packed(m, off)
        grads = torch.autograd.grad(y, [m, *block.parameters()], dout.to(y.dtype))
    assert y.dtype == BF16 and all(g.dtype == F32 and torch.isfinite(g).all() for g in grads)
    assert (y.float() - want).norm() <= 1e-2 * want.norm()
    block = _block(gpu_device, BF16, rotary={})
    m = m.detach().to(BF16).requires_grad_()
    y = block.packed(m, off)
    z = torch.compile(block.packed, backend="aot_eager")(m, off)
    assert (z.float() - y.float()).norm() <= 1e-2 * y.float().norm()
    for a, w in zip(torch.autograd.grad(z, [m, *block.parameters()], dout), torch.autograd.grad(y, [m, *block.parameters()], dout)):
        assert (a.float() - w.float()).norm() <= 2e-2 * w.float().norm() + 1e-3 * w.numel() ** 0.5


def test_captured_steps_replay_with_other_sequences(gpu_device):
    block = _block(gpu_device, BF16, rotary={})
    m, dout, off = _packed_case(gpu_device, BF16)
    m.requires_grad_()
    leaves = [m, *block.parameters()]

    def step():
        y = block.packed(m, off, causal=True)
        return [y.detach(), *torch.autograd.grad(y, leaves, dout)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed, ends in enumerate(([0, 70, 71, 71, 204, 244], [0, 10, 20, 30, 40, 50], [0, 0, 0, 0, 0, 247])):
        g = torch.Generator().manual_seed(seed)
        off.copy_(torch.tensor(ends))
        for t in (m, dout):
            t.data.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_a_prompt_and_its_tokens_one_by_one(gpu_device, dt):
    """Keys turned as they come and kept, a token's query against all that are there: the rows of the prompt taken at once."""
    from evoformer_triton_amd import RotaryPositions, packed_attention
    H, Hk, D, lengths, tokens = 8, 2, 64, [150, 3, 64], 6
    rotary = RotaryPositions(D, scaling="base", factor=4.0).to(gpu_device)
    g = torch.Generator(device=gpu_device).manual_seed(2)
    whole = [[torch.randn(n + tokens, h, D, device=gpu_device, generator=g).to(dt) for h in (H, Hk, Hk)] for n in lengths]
    q, k, v = (torch.cat([w[i] for w in whole]) for i in range(3))
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n + tokens)
    at = torch.cat([torch.arange(n + tokens, device=gpu_device) for n in lengths])
    qr, kr = rotary(q, k, at)
    all_ = packed_attention(qr, kr, v, torch.tensor(ends, device=gpu_device))
    want, bound = packed(qr, kr, v, ends, ends, True, D ** -0.5)
    _close([all_], want, bound, ["at once"])
    # the cache: the prompts' turned keys and values, and room for the tokens behind each
    kc, vc = torch.full_like(kr, float("nan")), torch.full_like(v, float("nan"))
    for begin, n in zip(ends, lengths):
        kc[begin:begin + n], vc[begin:begin + n] = kr[begin:begin + n], v[begin:begin + n]
    off = torch.tensor([0] + [(i + 1) // 2 for i in range(1, 7)], device=gpu_device)
    for t in range(tokens):
        rows = torch.tensor([b + n + t for b, n in zip(ends, lengths)], device=gpu_device)
        qt, kt = rotary(q[rows], k[rows], torch.tensor([n + t for n in lengths], device=gpu_device))
        assert torch.equal(qt, qr[rows]) and torch.equal(kt, kr[rows])
        kc[rows], vc[rows] = kt, v[rows]
        koff = torch.tensor([x for b, n in zip(ends, lengths) for x in (b, b + n + t + 1)] + [ends[-1]], device=gpu_device)
        _close([packed_attention(qt, kc, vc, off, koff)], [want[0][rows]], [bound[0][rows]], [f"token {t}"])


def test_checkpointed_in_inference_mode_and_without_gradients(gpu_device):
    from torch.utils.checkpoint import checkpoint
    block = _block(gpu_device, BF16, rotary={})
    m, dout, off = _packed_case(gpu_device, BF16)
    m.requires_grad_()
    rows, at = m.detach().view(1, 1, *m.shape).requires_grad_(), torch.arange(m.shape[0], device=gpu_device)
    for call, x, d in ((lambda x: block.packed(x, off), m, dout), (lambda x: block(x, None, None, at), rows, dout.view(rows.shape))):
        leaves = [x, *block.parameters()]
        y = call(x)
        want = torch.autograd.grad(y, leaves, d)
        for again in (checkpoint(call, x, use_reentrant=False), checkpoint(call, x, use_reentrant=True)):
            assert torch.equal(again, y)
        y2 = checkpoint(call, x, use_reentrant=False)
        for a, w in zip(torch.autograd.grad(y2, leaves, d), want):
            assert torch.equal(a, w)
        with torch.inference_mode():
            assert torch.equal(call(x), y)
        with torch.no_grad():
            assert torch.equal(call(x.detach()), y)


def test_two_streams_at_once(gpu_device):
    block = _block(gpu_device, F16, rotary={})
    m, _, off = _packed_case(gpu_device, F16)
    with torch.no_grad():
        want = [block.packed(m, off), block.packed(m * 2, off, causal=True)]
        streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
        twice = m * 2
        torch.cuda.synchronize()
        for _ in range(10):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i] = block.packed(twice if i else m, off, causal=bool(i))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_slots_gradient_that_somebody_else_has_stays(gpu_device):
    """The queries' and keys' gradient is turned back where it lies only if nobody else sees it."""
    from evoformer_triton_amd import RotaryPositions, packed_positions, rotary_positions
    rotary = RotaryPositions(32).to(gpu_device)
    T, shape = 40, (40, 3, 4, 32)
    at = torch.arange(T, device=gpu_device)
    x = torch.randn(T, 384, device=gpu_device, requires_grad=True)
    d = torch.randn(shape, device=gpu_device)
    kept = d.clone()

    def plain():
        q, k, v = (x * 2).view(shape).unbind(1)
        return torch.stack((*rotary_positions(q, k, at, rotary.turns), v), 1)

    want, = torch.autograd.grad(plain(), x, d)
    y = x * 2
    out = rotary.rotate_slots(y, shape, at)
    assert torch.equal(out, plain()) and out.data_ptr() == y.data_ptr()
    assert torch.equal(torch.autograd.grad(out, x, d)[0], want) and torch.equal(d, kept)      # the caller's own
    seen = []
    y = x * 2
    out = rotary.rotate_slots(y, shape, at)
    out.register_hook(lambda g: seen.append(g))
    out.retain_grad()
    (out * 1.0).backward(d)
    assert torch.equal(seen[0], kept) and torch.equal(out.grad, kept) and torch.equal(x.grad, want)
    # a leaf and a view cannot be turned where they lie: in a copy
    leaf = x.detach().clone().requires_grad_()
    base = leaf.detach().clone()
    out = rotary.rotate_slots(leaf, shape, at)
    assert torch.equal(leaf, base)
    assert torch.equal(2 * torch.autograd.grad(out, leaf, d)[0], want)
    view = torch.cat((x * 2, x))[:T]
    assert torch.equal(rotary.rotate_slots(view, shape, at), plain())
    # what is in use for another gradient is not overwritten unnoticed
    y = x * 2
    z = y * y
    rotary.rotate_slots(y, shape, at)
    with pytest.raises(RuntimeError, match="inplace"):
        z.sum().backward()


def test_no_rows_and_one(gpu_device):
    for dt in (BF16, F32):
        block = _block(gpu_device, dt, rotary={})
        for T in (0, 1):
            m = torch.randn(T, 96, device=gpu_device).to(dt).requires_grad_()
            y = block.packed(m, torch.tensor([0, T], device=gpu_device))
            g, = torch.autograd.grad(y, m, torch.ones_like(y))
            assert y.shape == g.shape == (T, 96) and torch.isfinite(y).all() and torch.isfinite(g).all()
        assert torch.equal(y, block.packed(m, torch.tensor([0, T], device=gpu_device), torch.tensor([-7], device=gpu_device)))      # (a token alone sees itself, wherever it is)
