"""Rotary positions and attention over packed sequences, as cases that can be timed.

`rotary`: queries and keys rotated by their positions, pairs of a head's halves or of neighbours, all of a head or its first part, frequencies as
they are or scaled for long contexts; `grad` is a training step's share, forward and backward.  `packed`: attention within sequences of different
lengths that lie one after the other without padding, causal or not, query heads in groups that share a key and value head; all rows of a sequence as
queries (a prompt, a training step) or its last few (`queries`: single tokens, a few at a time, a piece of a prompt) against all of its keys.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _rotary(grad, dtype, tokens, H, Hk, D, rotary, interleaved, base, factor, far, slots):
    """far: the greatest position that a sequence starts from; slots: queries and keys as slices of one projection's result; factor: of a context
    `factor` times as long as the 4096 positions the frequencies were trained on (0: as they are)."""
    return {"kind": "rotary", "grad": grad, "dtype": dtype, "tokens": tokens, "H": H, "Hk": Hk, "D": D, "rotary": rotary, "interleaved": interleaved,
            "base": base, "factor": factor, "far": far, "slots": slots}


def _packed(grad, causal, dtype, sequences, longest, shortest, queries, H, Hk, D, padding):
    return {"kind": "packed", "grad": grad, "causal": causal, "dtype": dtype, "sequences": sequences, "longest": longest, "shortest": shortest,
            "queries": queries, "H": H, "Hk": Hk, "D": D, "padding": padding}


def listed():
    return [
        # The new tokens of four sequences that are being continued: the smallest call there is.
        dict(_rotary(False, "bf16", 4, 8, 8, 32, 32, False, 10000.0, 0, 8192, True), name="rotary-tokens"),
        # The headline configuration's alignment (128 rows of 256 residues), slices of the block's stacked projection, in inference.
        dict(_rotary(False, "bf16", 32768, 8, 8, 32, 32, False, 10000.0, 0, 0, True), name="rotary-alignment"),
        # Neighbours as pairs, part of the head, scaled for long contexts, a number of tokens that fills no block, in training.
        dict(_rotary(True, "fp32", 5021, 12, 4, 80, 40, True, 10000.0, 8.0, 20000, False), name="rotary-step-part"),
        # A batch of long sequences in training, positions far out.
        dict(_rotary(True, "bf16", 65536, 32, 8, 128, 128, False, 500000.0, 0, 100000, False), name="rotary-step-long"),
        # One token each of a few sequences against what lies before it: where latency counts.
        dict(_packed(False, True, "bf16", 4, 1000, 200, 1, 8, 2, 64, 0), name="packed-tokens-few"),
        # Serving: a token of each of 32 sequences of very different lengths.
        dict(_packed(False, True, "fp16", 32, 8192, 100, 1, 32, 8, 128, 0), name="packed-tokens"),
        # One token of one very long sequence.
        dict(_packed(False, True, "bf16", 1, 131072, 131072, 1, 16, 2, 128, 0), name="packed-token-long"),
        # Prompts of different lengths, in one call.
        dict(_packed(False, True, "fp16", 7, 2011, 90, 0, 16, 4, 64, 0), name="packed-prompts"),
        # One long prompt: bound by the matrix cores.
        dict(_packed(False, True, "bf16", 1, 16384, 16384, 0, 32, 8, 128, 0), name="packed-prompt-long"),
        # Protein chains in training, each residue attends to all of its chain (the headline configuration's heads).
        dict(_packed(True, False, "bf16", 24, 768, 51, 0, 8, 8, 32, 0), name="packed-chains-step"),
        # A head dim and lengths that fill no tile, rows of no sequence at the end, in training.
        dict(_packed(True, True, "fp16", 5, 1777, 333, 0, 12, 4, 80, 45), name="packed-step-ragged"),
        # Long sequences in training: bound by the matrix cores.
        dict(_packed(True, True, "bf16", 4, 4096, 4096, 0, 32, 8, 128, 0), name="packed-step-long"),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, evenly over the logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(("rotary-tokens", "rotary", "rotary-step", "packed-tokens", "packed-tokens", "packed-prompts", "packed-step", "packed-step"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    Hk, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 1, 2, 3, 4, 8))
    H, D = Hk * group, rng.choice((32, 40, 64, 64, 80, 96, 128, 128))
    if kind.startswith("rotary"):
        dtype = rng.choice((dtype, dtype, "fp32"))
        R = rng.choice((D, D, D, D // 2, 24))
        tokens = rng.randint(1, 64) if kind == "rotary-tokens" else _spread(rng, 65, min(65536, (1 << 27) // ((H + Hk) * D)))
        scaled = rng.random() < 0.3
        return _rotary(kind == "rotary-step", dtype, tokens, H, Hk, D, R, rng.random() < 0.4, rng.choice((10000.0, 500000.0)),
                       rng.choice((2.0, 8.0, 40.0)) if scaled else 0, rng.choice((0, 5000, 150000)), rng.random() < 0.4)
    if kind == "packed-tokens":
        queries, sequences = rng.choice((1, 1, 1, 2, 5, 17)), _spread(rng, 1, 64)
        longest = _spread(rng, 20, min(131072, (1 << 28) // (sequences * Hk * D)))
        return _packed(False, True, dtype, sequences, longest, _spread(rng, 1, longest), queries, H, Hk, D, 0)
    # (pairs of a query and a key by heads by head dim: below half of the largest listed case)
    sequences = _spread(rng, 1, 40)
    longest = _spread(rng, 16, min(16384, 131072 // sequences, int(((1 << 38) / (sequences * H * D)) ** 0.5)))
    queries = rng.choice((0, 0, 0, 512))
    step = kind == "packed-step"
    return _packed(step, rng.random() < 0.7, dtype, sequences, longest, _spread(rng, 1, longest), 0 if step else queries, H, Hk, D, rng.choice((0, 0, 1, 70)))


def _lengths(case):
    """The sequences' lengths: spread evenly over the logarithm from the longest to the shortest, in a mixed order."""
    n, longest, shortest = case["sequences"], case["longest"], case["shortest"]
    lengths = [round(longest * (shortest / longest) ** (i / max(1, n - 1))) for i in range(n)]
    step = next(s for s in (7, 11, 13, 17) if math.gcd(s, n) == 1)
    return [lengths[i * step % n] for i in range(n)]


def _frequencies(case):
    """Radians per position of each pair, and what the rotated values are multiplied by.  Scaled (`factor`): a pair that turns 32 times or more over
    the 4096 positions keeps its frequency, one that turns at most once has it divided by the factor, those between are blended by their turns; the values grow by
    0.1 ln(factor) + 1, which sharpens the attention over the longer context."""
    R, factor = case["rotary"], case["factor"]
    f = [case["base"] ** (-2.0 * i / R) for i in range(R // 2)]
    if not factor:
        return f, 1.0
    keep = [min(1.0, max(0.0, (4096 * x / (2 * math.pi) - 1.0) / 31.0)) for x in f]
    return [x * (w + (1.0 - w) / factor) for x, w in zip(f, keep)], 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    dt, dev = _DTYPES[case["dtype"]], torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device=dev, generator=g).to(dt)

    state = dict(case)
    H, Hk, D = case["H"], case["Hk"], case["D"]
    if case["kind"] == "rotary":
        T, R = case["tokens"], case["rotary"]
        # Sequences of 256 residues or tokens, each from a position of its own on; single tokens each where its sequence stands.
        run = 256 if T > 64 else 1
        starts = torch.randint(0, case["far"] + 1, (-(-T // run),), device=dev, generator=g)
        positions = (starts[:, None] + torch.arange(run, device=dev)).flatten()[:T].contiguous()
        frequencies, scale = _frequencies(case)
        if case["slots"]:
            both = normal(T, H + 2 * Hk, D)      # (queries, keys, values side by side)
            q, k = both[:, :H], both[:, H:H + Hk]
        else:
            q, k = normal(T, H, D), normal(T, Hk, D)
        state.update(q=q, k=k, positions=positions, scale=scale, frequencies=torch.tensor(frequencies, dtype=torch.float64, device=dev))
        if own:
            from evoformer_triton_amd import rotary_turns
            scaling = dict(scaling="parts", factor=case["factor"], original_length=4096) if case["factor"] else {}
            state["turns"] = rotary_turns(R, case["base"], device=dev, **scaling)
    else:
        lengths = _lengths(case)
        rows = [min(n, case["queries"]) if case["queries"] else n for n in lengths]
        Tq, Tk = sum(rows) + case["padding"], sum(lengths) + case["padding"]

        def offsets(lens):
            return torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)

        # Normalised queries and keys: scores of about one, heads of different sharpness.
        sharp = torch.exp(0.5 * torch.randn((H, 1), device=dev, generator=g))
        state.update(q=(torch.randn((Tq, H, D), device=dev, generator=g) * sharp).to(dt), k=normal(Tk, Hk, D), v=normal(Tk, Hk, D),
                     offsets=offsets(rows), key_offsets=offsets(lengths) if case["queries"] else None, rows=rows, lengths=lengths)
    if case["grad"]:
        names = ("q", "k") if case["kind"] == "rotary" else ("q", "k", "v")
        for name in names:
            state[name] = state[name].detach().requires_grad_()
        state["dout"] = [normal(*state[name].shape) for name in names[:2]] if case["kind"] == "rotary" else normal(*state["q"].shape)
    return state


def _rotated(x, cos, sin, R, interleaved, scale):
    """x [T, H, D] in 32 bits by angles [T, 1, R / 2]; the gradient's formula with -sin."""
    part = x[..., :R]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :R // 2], part[..., R // 2:])
    y, z = (a * cos - b * sin) * scale, (b * cos + a * sin) * scale
    turned = torch.stack((y, z), -1).flatten(-2) if interleaved else torch.cat((y, z), -1)
    return torch.cat((turned, x[..., R:]), -1)


def _rotary_plain(s):
    angle = (s["positions"].double()[:, None] * s["frequencies"])[:, None, :]
    cos, sin = angle.cos().float(), angle.sin().float()
    outs = [_rotated(s[n].detach().float(), cos, sin, s["rotary"], s["interleaved"], s["scale"]).to(s[n].dtype) for n in ("q", "k")]
    if s["grad"]:
        outs += [_rotated(d.float(), cos, -sin, s["rotary"], s["interleaved"], s["scale"]).to(d.dtype) for d in s["dout"]]
    return outs


def _packed_plain(s):
    q, k, v = (s[n].detach() for n in ("q", "k", "v"))
    (Tq, H, D), Hk, G = q.shape, k.shape[1], q.shape[1] // k.shape[1]
    scale = D ** -0.5
    out = torch.zeros_like(q)
    grads = [torch.zeros_like(t) for t in (q, k, v)] if s["grad"] else []
    at_q = at_k = 0
    for Lq, Lk in zip(s["rows"], s["lengths"]):
        # key and value heads at a time, as many as their scores take two GiB for
        some = max(1, (1 << 29) // max(1, G * Lq * Lk))
        hidden = None
        if s["causal"]:
            hidden = torch.arange(Lk, device=q.device)[None, :] - Lk > torch.arange(Lq, device=q.device)[:, None] - Lq
        for h in range(0, Hk, some):
            e = min(Hk, h + some)
            qs = q[at_q:at_q + Lq, h * G:e * G].float().unflatten(1, (e - h, G)).permute(1, 2, 0, 3).reshape(e - h, G * Lq, D)
            ks, vs = (t[at_k:at_k + Lk, h:e].float().transpose(0, 1).contiguous() for t in (k, v))
            p = torch.bmm(qs, ks.transpose(1, 2)).mul_(scale)
            if hidden is not None:
                p.view(e - h, G, Lq, Lk).masked_fill_(hidden, float("-inf"))
            p.sub_(p.amax(-1, keepdim=True)).exp_()
            p.div_(p.sum(-1, keepdim=True))
            o = torch.bmm(p, vs)

            def placed(x):
                return x.view(e - h, G, Lq, D).permute(2, 0, 1, 3).reshape(Lq, (e - h) * G, D)

            out[at_q:at_q + Lq, h * G:e * G] = placed(o)
            if s["grad"]:
                do = s["dout"][at_q:at_q + Lq, h * G:e * G].float().unflatten(1, (e - h, G)).permute(1, 2, 0, 3).reshape(e - h, G * Lq, D)
                grads[2][at_k:at_k + Lk, h:e] = torch.bmm(p.transpose(1, 2), do).transpose(0, 1)
                ds = torch.bmm(do, vs.transpose(1, 2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
                grads[0][at_q:at_q + Lq, h * G:e * G] = placed(torch.bmm(ds, ks))
                grads[1][at_k:at_k + Lk, h:e] = torch.bmm(ds.transpose(1, 2), qs).transpose(0, 1)
        at_q, at_k = at_q + Lq, at_k + Lk
    return [out, *grads]


def run(state):
    s = state
    if not own:
        with torch.no_grad():
            return _rotary_plain(s) if s["kind"] == "rotary" else _packed_plain(s)
    import evoformer_triton_amd as evo
    if s["kind"] == "rotary":
        outs = list(evo.rotary_positions(s["q"], s["k"], s["positions"], s["turns"], interleaved=s["interleaved"], scale=s["scale"]))
        return [*outs, *torch.autograd.grad(outs, [s["q"], s["k"]], s["dout"])] if s["grad"] else outs
    out = evo.packed_attention(s["q"], s["k"], s["v"], s["offsets"], s["key_offsets"], causal=s["causal"])
    return [out, *torch.autograd.grad(out, [s["q"], s["k"], s["v"]], s["dout"])] if s["grad"] else [out]


def work(case):
    """Each input read once, each output written once.  A rotation of a pair: six operations.  Attention: two products per pair of a query and a key it sees and
    head, forward; four more backward."""
    es, D = 4 if case["dtype"] == "fp32" else 2, case["D"]
    passes = 2 if case["grad"] else 1
    if case["kind"] == "rotary":
        T, heads = case["tokens"], case["H"] + case["Hk"]
        return {"bytes": passes * 2 * T * heads * D * es + 8 * (T + case["rotary"] // 2), "flops": passes * 3 * T * heads * case["rotary"]}
    lengths = _lengths(case)
    pairs = rows = 0
    for n in lengths:
        m = min(n, case["queries"]) if case["queries"] else n
        rows += m
        pairs += m * n - m * (m - 1) // 2 if case["causal"] else m * n
    q, k = (rows + case["padding"]) * case["H"] * D * es, (sum(lengths) + case["padding"]) * case["Hk"] * D * es
    offsets = 4 * (len(lengths) + 1)
    # q, k, v, out; in training dout, dq, dk, dv
    return {"bytes": 2 * q + 2 * k + offsets + (2 * q + 2 * k if case["grad"] else 0), "flops": (12 if case["grad"] else 4) * D * case["H"] * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        R, pairs = case["rotary"], case["rotary"] // 2
        at = torch.arange(pairs, device=s["q"].device)
        first, second = (2 * at, 2 * at + 1) if case["interleaved"] else (at, at + pairs)
        angle = s["positions"].double().outer(s["frequencies"])
        turn = torch.polar(torch.full_like(angle, s["scale"]), angle)

        def turned(x, by):
            z = torch.complex(x[..., first].double(), x[..., second].double()) * by[:, None, :]
            y = x.double()
            y[..., first], y[..., second] = z.real, z.imag
            return y

        outs = [turned(s[n].detach(), turn) for n in ("q", "k")]
        return outs + [turned(d, turn.conj()) for d in s["dout"]] if case["grad"] else outs
    q, k, v = (s[n].detach() for n in ("q", "k", "v"))
    H, Hk, D = case["H"], case["Hk"], case["D"]
    dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device=t.device) for t in (q, k, v))
    out = torch.zeros_like(dq)
    # a sequence, a head and up to 4096 queries at a time
    at_q = at_k = 0
    for Lq, Lk in zip(s["rows"], s["lengths"]):
        for h in range(H):
            K, V = k[at_k:at_k + Lk, h * Hk // H].double(), v[at_k:at_k + Lk, h * Hk // H].double()
            for i in range(0, Lq, 4096):
                n = min(4096, Lq - i)
                seen = Lk - Lq + i + n if case["causal"] else Lk      # (keys that any of these queries sees)
                Q, rows = q[at_q + i:at_q + i + n, h].double(), slice(at_q + i, at_q + i + n)
                score = Q @ K[:seen].T / math.sqrt(D)
                if case["causal"]:
                    score += torch.full_like(score, -math.inf).triu(Lk - Lq + i + 1)
                P = torch.softmax(score, -1)
                out[rows, h] = P @ V[:seen]
                if case["grad"]:
                    dO = s["dout"][rows, h].double()
                    dv[at_k:at_k + seen, h * Hk // H] += P.T @ dO
                    dP = dO @ V[:seen].T
                    dS = P * (dP - (P * dP).sum(-1, keepdim=True)) / math.sqrt(D)
                    dq[rows, h] = dS @ K[:seen]
                    dk[at_k:at_k + seen, h * Hk // H] += dS.T @ Q
        at_q, at_k = at_q + Lq, at_k + Lk
    return [out, dq, dk, dv] if case["grad"] else [out]
