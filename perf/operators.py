"""The learned relative position bias and the 8-bit projections of the gated block, as cases that can be timed.

`relative`: a bias per head and bucket of the distance between two residues, [B,1,H,Nq,Nk] as the attention takes it, on its own or
added to the pair bias, and (`grad`) its gradients.  `projection`: a Linear layer whose operands are rounded to e4m3 with a
power-of-two scale for each block of 128 along the contraction; `grad` is a training step, which rounds the weight, the input and the
gradient of each product's two operands along that product's own contraction; without it the weight is held in 8 bits already.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _relative(grad, dtype, B, Nq, Nk, H, reach, buckets, chains, base):
    return {"kind": "relative", "grad": grad, "dtype": dtype, "B": B, "Nq": Nq, "Nk": Nk, "H": H, "reach": reach, "buckets": buckets, "chains": chains,
            "base": base}


def _projection(grad, dtype, rows, k, n, bias, wide):
    return {"kind": "projection", "grad": grad, "dtype": dtype, "rows": rows, "k": k, "n": n, "bias": bias, "wide": wide}


def listed():
    return [
        # One new residue against those before it: a row of the bias. The smallest call there is.
        dict(_relative(False, "bf16", 1, 1, 1000, 8, 32, 0, 0, False), name="relative-row"),
        # A crop in inference (the headline configuration's pairs), added to the pair bias.
        dict(_relative(False, "bf16", 1, 256, 256, 8, 32, 0, 0, True), name="relative-forward"),
        # A batch of complexes in training: a protein's own length, several chains.
        dict(_relative(True, "fp16", 2, 251, 251, 8, 32, 0, 3, True), name="relative-step-ragged"),
        # A long crop in training (triangle attention's heads), added to the pair bias.
        dict(_relative(True, "bf16", 1, 768, 768, 4, 32, 0, 0, True), name="relative-step-long"),
        # The reference's speed benchmark's shapes: a batch of single sequences, many heads, fp32 bias; buckets that widen with the distance.
        dict(_relative(True, "fp32", 4, 1024, 1024, 32, 128, 32, 0, True), name="relative-step-batch"),
        # One token through the block's stacked Q, K, V and gate projections.
        dict(_projection(False, "bf16", 1, 256, 1024, False, False), name="projection-token"),
        # A few tokens through a wide layer, as in serving.
        dict(_projection(False, "fp16", 24, 4096, 4096, True, False), name="projection-tokens"),
        # The stacked projections of 128 alignment rows of a crop, in inference.
        dict(_projection(False, "bf16", 32768, 256, 1024, True, False), name="projection-forward"),
        # The same in training, the weight in the activations' type.
        dict(_projection(True, "bf16", 32768, 256, 1024, True, False), name="projection-step"),
        # Sizes that fill no tile, in training.
        dict(_projection(True, "fp16", 5021, 500, 333, True, False), name="projection-step-ragged"),
        # A wide layer in inference: bound by the matrix cores.
        dict(_projection(False, "bf16", 8192, 4096, 4096, True, False), name="projection-forward-wide"),
        # A transition's first layer in training, its weight in fp32.
        dict(_projection(True, "bf16", 8192, 2048, 8192, True, True), name="projection-step-wide"),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, evenly over the logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def _size(rng, lo, hi):
    """Every other one a multiple of 64 (where the range has one), the others as they fall."""
    n = _spread(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.5 and hi >= 64 else n


def draw(rng):
    kind = rng.choice(("relative-row", "relative-forward", "relative-step", "relative-step", "projection-tokens", "projection-forward", "projection-step",
                       "projection-step"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if kind.startswith("relative"):
        clipped = rng.random() < 0.6
        reach = _spread(rng, 8, 127) if clipped else rng.choice((64, 128, 500))
        buckets = 0 if clipped else rng.choice((16, 32, 64))
        chains = rng.choice((0, 0, 2, 5))
        if kind == "relative-row":
            return _relative(False, dtype, rng.randint(1, 8), 1, _spread(rng, 1, 8192), rng.choice((4, 8, 16)), reach, buckets, chains, rng.random() < 0.5)
        N, H = _size(rng, 16, 1024), rng.choice((4, 8, 12, 32))
        return _relative(kind == "relative-step", dtype, rng.randint(1, 4), N, N, H, reach, buckets, chains, rng.random() < 0.7)
    bias = rng.random() < 0.5
    if kind == "projection-tokens":
        return _projection(False, dtype, _spread(rng, 1, 64), _size(rng, 64, 8192), _size(rng, 64, 8192), bias, False)
    k, n = _size(rng, 32, 4096), _size(rng, 32, 4096)
    rows = _size(rng, 64, max(128, min(65536, (1 << 36) // (k * n), (1 << 27) // max(k, n))))
    return _projection(kind == "projection-step", dtype, rows, k, n, bias, rng.random() < 0.3)


def _lookup(reach, buckets):
    """Bucket of each clipped distance -reach .. reach: one each, or (`buckets`) half of them for either sign, half of those one each
    from distance 0 on and the others ever wider up to `reach`: bucket near + i from the first distance d with
    (d / near)^(half - near) >= (reach / near)^i on, in whole numbers."""
    if not buckets:
        return torch.arange(2 * reach + 1, dtype=torch.uint8)
    half, near = buckets // 2, buckets // 4
    far = half - near
    of = [d if d < near else min(half - 1, near + sum(d ** far * near ** i >= reach ** i * near ** far for i in range(1, far))) for d in range(reach + 1)]
    return torch.tensor([half + of[-d] if d < 0 else of[d] for d in range(-reach, reach + 1)], dtype=torch.uint8)


def _rounded(x):
    """x's values as e4m3 with a scale for each 128 of the last axis hold them, and its scales' exponents, one for each block."""
    k = x.shape[-1]
    v = torch.nn.functional.pad(x.float(), (0, -k % 128)).unflatten(-1, (-1, 128))
    m, e = torch.frexp(v.abs().amax(-1, keepdim=True))
    e = torch.where(m == 0, 0, e - 9 + (m > 0.875).int()).clamp(-127, 127)
    q = torch.ldexp(v, -e).to(torch.float8_e4m3fn)
    return q.flatten(-2), e.squeeze(-1)


def _values(q, e, k):
    return torch.ldexp(q.float().unflatten(-1, (-1, 128)), e.unsqueeze(-1)).flatten(-2)[..., :k].contiguous()


def _held(x):
    return _values(*_rounded(x), x.shape[-1])


def prepare(case, seed):
    dt, dev = _DTYPES[case["dtype"]], torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=dt):
        return torch.randn(shape, device=dev, generator=g).to(dtype)

    state = dict(case)
    if case["kind"] == "relative":
        B, Nq, Nk, H = case["B"], case["Nq"], case["Nk"], case["H"]
        # Residue numbers as a structure file has them: ascending, with a gap now and then, from a number of its own on.
        steps = 1 + (torch.rand((B, Nk), device=dev, generator=g) < 0.02) * torch.randint(1, 40, (B, Nk), device=dev, generator=g)
        at = steps.cumsum(1) + torch.randint(-50, 50, (B, 1), device=dev, generator=g)
        lut = _lookup(case["reach"], case["buckets"]).to(dev)
        rows = int(lut.max()) + 1 + (case["chains"] > 0)
        chain = torch.arange(Nk, device=dev).mul(max(1, case["chains"])).div(Nk, rounding_mode="floor").expand(B, Nk).contiguous()
        state.update(lut=lut, table=normal(rows, H), key_positions=at, positions=at[:, Nk - Nq:].contiguous(),
                     key_chain=chain if case["chains"] else None, chain=chain[:, Nk - Nq:].contiguous() if case["chains"] else None,
                     pair=normal(B, 1, H, Nq, Nk) if case["base"] else None)
        if case["grad"]:
            state["table"].requires_grad_()
            if case["base"]:
                state["pair"].requires_grad_()
            state["dout"] = normal(B, 1, H, Nq, Nk)
        return state
    rows, k, n = case["rows"], case["k"], case["n"]
    # Activations: some channels far larger than the others, some tokens padded away. Gradients: tokens of very different weight.
    channel = torch.exp(0.7 * torch.randn((k,), device=dev, generator=g))
    x = (torch.randn((rows, k), device=dev, generator=g) * channel).to(dt)
    w = normal(n, k, dtype=torch.float32 if case["wide"] else dt) * k ** -0.5
    state.update(x=x, bias=normal(n) if case["bias"] else None)
    if case["grad"]:
        padded = torch.rand((rows, 1), device=dev, generator=g) < 0.05
        dy = torch.randn((rows, n), device=dev, generator=g) * torch.exp(torch.randn((rows, 1), device=dev, generator=g) - 4)
        state.update(x=x.masked_fill_(padded, 0).requires_grad_(), weight=w.requires_grad_(), dy=dy.masked_fill_(padded, 0).to(dt))
        if case["bias"]:
            state["bias"].requires_grad_()
    else:
        # A serving program's weight: e4m3 [n, k up to the next 128], a scale byte (the exponent + 127) for each block, blocks up to the next four.
        q, e = _rounded(w)
        state.update(values=q, scales=torch.nn.functional.pad((e + 127).to(torch.uint8), (0, -e.shape[-1] % 4), value=127))
    return state


def _relative_plain(s):
    """The bias, and a closure for its gradients."""
    o = (s["positions"][:, :, None] - s["key_positions"][:, None, :]).clamp(-s["reach"], s["reach"]) + s["reach"]
    bucket = s["lut"][o].long()
    if s["chain"] is not None:
        bucket = torch.where(s["chain"][:, :, None] != s["key_chain"][:, None, :], s["table"].shape[0] - 1, bucket)
    out = s["table"].detach().float()[bucket].permute(0, 3, 1, 2).unsqueeze(1)
    if s["pair"] is not None:
        out = out + s["pair"].detach().float()
    out = out.to(s["table"].dtype).contiguous()
    if not s["grad"]:
        return [out]
    # a row of pairs at a time in 32 bits, the rows' sums in 64
    one_hot = (bucket[..., None] == torch.arange(s["table"].shape[0], device=bucket.device)).float().flatten(0, 1)        # [B Nq, Nk, rows]
    sums = torch.bmm(s["dout"].float().squeeze(1).transpose(1, 2).flatten(0, 1).contiguous(), one_hot)                     # [B Nq, H, rows]
    return [out, sums.double().sum(0).t().to(s["table"].dtype).contiguous()] + ([s["dout"].clone()] if s["pair"] is not None else [])


def _projection_plain(s):
    if not s["grad"]:
        w = _values(s["values"], s["scales"][:, :s["values"].shape[1] // 128].int() - 127, s["k"])
        y = torch.mm(_held(s["x"]), w.t())
        return [(y + s["bias"].float() if s["bias"] is not None else y).to(s["x"].dtype)]
    x, w, dy = s["x"].detach(), s["weight"].detach(), s["dy"]
    y = torch.mm(_held(x), _held(w).t())
    if s["bias"] is not None:
        y = y + s["bias"].detach().float()
    dx = torch.mm(_held(dy), _held(w.t()).t())
    dw = torch.mm(_held(dy.t()), _held(x.t()).t())
    db = [dy.double().sum(0).to(dy.dtype)] if s["bias"] is not None else []
    return [y.to(x.dtype), dx.to(x.dtype), dw.to(w.dtype), *db]


def run(state):
    s = state
    if not own:
        with torch.no_grad():
            return _relative_plain(s) if s["kind"] == "relative" else _projection_plain(s)
    import evoformer_triton_amd as evo
    if s["kind"] == "relative":
        out = evo.relative_position_bias(s["table"], s["lut"], s["positions"], s["key_positions"], chains=s["chain"], key_chains=s["key_chain"], pair_bias=s["pair"])
        leaves, d = [s["table"]] + ([s["pair"]] if s["pair"] is not None else []), s.get("dout")
    elif s["grad"]:
        out = evo.fp8_linear(s["x"], s["weight"], s["bias"])
        leaves, d = [s["x"], s["weight"]] + ([s["bias"]] if s["bias"] is not None else []), s["dy"]
    else:
        out = evo.fp8_linear(s["x"], evo.Fp8Weight(s["values"], s["scales"], s["k"]), s["bias"])
    return [out, *torch.autograd.grad(out, leaves, d)] if s["grad"] else [out]


def work(case):
    """Each input read once, each output written once; a product of two per element of a projection and product, an addition per pair and head."""
    es = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "relative":
        B, Nq, Nk, H = case["B"], case["Nq"], case["Nk"], case["H"]
        table = ((2 * case["reach"] + 1 if not case["buckets"] else case["buckets"]) + (case["chains"] > 0)) * H * es
        residues = 8 * B * (Nq + Nk) * (2 if case["chains"] else 1)
        # out and the pair bias; in training the output's gradient read, which is the pair bias's as it lies
        arrays = 1 + case["base"] + case["grad"]
        return {"bytes": arrays * B * H * Nq * Nk * es + (2 if case["grad"] else 1) * table + residues, "flops": (1 + case["grad"]) * B * H * Nq * Nk}
    rows, k, n = case["rows"], case["k"], case["n"]
    x, y, bias = rows * k * es, rows * n * es, n * es * case["bias"]
    if not case["grad"]:
        blocks = -(-k // 128)
        return {"bytes": x + n * blocks * 129 + bias + y, "flops": 2 * rows * k * n}
    return {"bytes": 2 * x + 2 * n * k * (4 if case["wide"] else es) + 2 * y + 2 * bias, "flops": 6 * rows * k * n}


def _exact_held(x):
    """e4m3 along the last axis from its definition: four significant bits, no step below 2^-9 of the scale, ties to even."""
    k = x.shape[-1]
    v = torch.zeros((*x.shape[:-1], -(-k // 128) * 128), dtype=torch.float64, device=x.device)
    v[..., :k] = x.double()
    v = v.view(*x.shape[:-1], -1, 128)
    a = v.abs().max(-1, keepdim=True).values
    scale = torch.exp2(torch.ceil(torch.log2(torch.where(a > 0, a, 1.0) / 448.0)))
    scale = torch.where(scale * 224 >= a, scale / 2, torch.where(scale * 448 < a, scale * 2, scale))
    scale = torch.where(a > 0, scale, 1.0).clamp(2.0 ** -127, 2.0 ** 127)
    v = v / scale
    step = torch.exp2(torch.floor(torch.log2(torch.where(v != 0, v.abs(), 1.0))).clamp(-6, 8) - 3)
    return (torch.round(v / step) * step * scale).view(*x.shape[:-1], -1)[..., :k]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "relative":
        table, reach = s["table"].detach().double(), case["reach"]
        half, near = case["buckets"] // 2, case["buckets"] // 4
        of = list(range(-reach, reach + 1))
        for i, d in enumerate(of):
            if not case["buckets"]:
                of[i] = d + reach
                continue
            b = abs(d)
            if b >= near:
                b = near
                while b < half - 1 and abs(d) ** (half - near) >= reach ** (b + 1 - near) * near ** (half - b - 1):
                    b += 1
            of[i] = b + (half if d < 0 else 0)
        of = torch.tensor(of, device=table.device)
        d = s["positions"].unsqueeze(2) - s["key_positions"].unsqueeze(1)
        bucket = of[torch.minimum(torch.maximum(d, torch.tensor(-reach, device=d.device)), torch.tensor(reach, device=d.device)) + reach]
        if s["chain"] is not None:
            bucket[s["chain"].unsqueeze(2) != s["key_chain"].unsqueeze(1)] = table.shape[0] - 1
        out = torch.empty((case["B"], 1, case["H"], case["Nq"], case["Nk"]), dtype=torch.float64, device=table.device)
        for h in range(case["H"]):
            out[:, 0, h] = table[:, h][bucket]
        if s["pair"] is not None:
            out += s["pair"].detach()
        if not case["grad"]:
            return [out]
        dtable = torch.empty_like(table)
        for h in range(case["H"]):
            dtable[:, h] = torch.bincount(bucket.flatten(), s["dout"][:, 0, h].double().flatten(), minlength=table.shape[0])
        return [out, dtable] + ([s["dout"].double()] if s["pair"] is not None else [])
    x = s["x"].detach()
    if case["grad"]:
        w, dy = s["weight"].detach(), s["dy"]
        y = _exact_held(x) @ _exact_held(w).T
        more = [_exact_held(dy) @ _exact_held(w.T).T.contiguous(), _exact_held(dy.T) @ _exact_held(x.T).T.contiguous()] + ([dy.double().sum(0)] if case["bias"] else [])
    else:
        blocks = s["values"].shape[1] // 128
        scale = torch.tensor([math.ldexp(1.0, b - 127) for b in range(255)], dtype=torch.float64, device=x.device)[s["scales"][:, :blocks].long()]
        w = (s["values"].double().view(case["n"], blocks, 128) * scale[:, :, None]).view(case["n"], -1)[:, :case["k"]]
        y, more = _exact_held(x) @ w.T, []
    return [y + s["bias"].detach().double() if case["bias"] else y, *more]
