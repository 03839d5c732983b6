"""Packed attention and the weight-only NVFP4 linear, as cases that can be timed.

kind    entry point
step    ``attention.packed_attention``, one query a sequence over a cache
packed  ``attention.packed_attention``, several queries a sequence: whole prompts, prompts
        appended to a cache, and full (unmasked) attention
w4      ``NVFP4Execution(activations="unquantized").linear``

``run`` computes them in elementary torch operations, or with ``own`` through the package.
"""

import math
import random

import torch

own = False

F32, F64 = torch.float32, torch.float64
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
# Scores held at once by the plain forms (elements).
BLOCK = 1 << 28


def listed():
    return [
        # One new token of one sequence over a short prompt: the smallest call, latency alone.
        dict(name="step_1x77", kind="step", batch=1, low=77, high=77, heads=32, kv=8, dim=128, dtype="bf16"),
        # A decoding batch whose sequences are of very different lengths.
        dict(name="step_16x1to8191", kind="step", batch=16, low=1, high=8191, heads=32, kv=8, dim=128, dtype="bf16"),
        # One sequence with a long cache: the keys alone have to fill the card.
        dict(name="step_1x131071_f16", kind="step", batch=1, low=131071, high=131071, heads=32, kv=8, dim=128,
             dtype="f16"),
        # A batch of prompts, packed, empty ones among them; q, k, v are slices of one merged projection.
        dict(name="prompts_24x0to1023", kind="packed", batch=24, low=0, high=1023, past=0, causal=True, heads=28, kv=4,
             dim=128, dtype="bf16"),
        # One long prompt with narrow heads.
        dict(name="prompt_8191_d64_f16", kind="packed", batch=1, low=8191, high=8191, past=0, causal=True, heads=16,
             kv=16, dim=64, dtype="f16"),
        # A piece of a prompt after what the cache holds already.
        dict(name="piece_509_after_16000", kind="packed", batch=1, low=509, high=509, past=16000, causal=True, heads=32,
             kv=8, dim=128, dtype="bf16"),
        # The denoiser's own: every token of a 21x30x52 latent sees every other, 40 heads.
        dict(name="full_32760", kind="packed", batch=1, low=32760, high=32760, past=0, causal=False, heads=40, kv=40,
             dim=128, dtype="bf16"),
        # One row (a token, a timestep's modulation) through a square projection.
        dict(name="w4_1x5120x5120", kind="w4", m=1, k=5120, n=5120, bias=False, dtype="bf16"),
        # One row through the wide input projection of the H3 FFN.
        dict(name="w4_1x5376x28672_f16", kind="w4", m=1, k=5376, n=28672, bias=True, dtype="f16"),
        # A few rows (a small decoding batch) through the H3 attention output.
        dict(name="w4_7x7168x5376", kind="w4", m=7, k=7168, n=5376, bias=True, dtype="bf16"),
        # A larger batch through a merged QKV projection.
        dict(name="w4_64x5120x15360", kind="w4", m=64, k=5120, n=15360, bias=False, dtype="bf16"),
        # A whole prompt through the FFN up-projection: the matrix cores count, not the weight's bytes.
        dict(name="w4_1021x5120x13824", kind="w4", m=1021, k=5120, n=13824, bias=True, dtype="bf16"),
    ]


def _log(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))) - 0.5)))


HEADS = ((32, 8, 128), (28, 4, 128), (40, 40, 128), (56, 56, 128), (16, 16, 64), (12, 2, 64), (24, 8, 96), (8, 1, 128),
         (20, 5, 80))


def draw(rng):
    kind = rng.choice(("step", "packed", "w4"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    if kind == "w4":
        m = _log(rng, 1, 1100)
        k, n = 64 * _log(rng, 4, 224), 128 * _log(rng, 2, 224)
        return dict(kind=kind, m=m, k=k, n=n, bias=rng.random() < 0.5, dtype=dtype)
    heads, kv, dim = rng.choice(HEADS)
    if kind == "step":
        batch = _log(rng, 1, 128)
        high = _log(rng, 1, min(131071, (1 << 28) // (batch * kv * dim)))
        return dict(kind=kind, batch=batch, low=_log(rng, 1, high), high=high, heads=heads, kv=kv, dim=dim, dtype=dtype)
    batch = _log(rng, 1, 48)
    high = _log(rng, 1, max(1, 24000 // batch))
    return dict(kind=kind, batch=batch, low=rng.choice((0, 1, high)), high=high,
                past=rng.choice((0, 0, _log(rng, 1, max(1, 16000 // batch)))), causal=rng.random() < 0.7, heads=heads,
                kv=kv, dim=dim, dtype=dtype)


def _lengths(case, seed=0):
    """The sequences' new lengths (those of the cache for ``step``), the longest among them.
    The case gives the lengths and the seed their order."""
    rng = random.Random("%d %d %d" % (case["batch"], case["low"], case["high"]))
    lengths = [case["high"]] + [rng.randint(case["low"], case["high"]) for _ in range(case["batch"] - 1)]
    random.Random(seed).shuffle(lengths)
    return lengths


def _offsets(lengths, device):
    total, out = 0, [0]
    for n in lengths:
        total += n
        out.append(total)
    return torch.tensor(out, dtype=torch.int64, device=device)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dtype):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=F32) * std).to(dtype)

    s = {"case": case}
    if case["kind"] == "w4":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = normal(m, k)
        s["bias"] = normal(n, std=0.02, dtype=torch.bfloat16) if case["bias"] else None
        s["packed"], s["scales"], s["alpha"] = _pack(normal(n, k, std=0.02, dtype=F32))
        if own:
            from vflash_amd.nvfp4_linear import NVFP4Execution, NVFP4Weight

            s["execution"] = NVFP4Execution(activations="unquantized")
            s["weight"] = NVFP4Weight(s["packed"], s["scales"], s["alpha"], torch.ones((), device="cuda"))
        return s
    lengths, heads, kv, dim = _lengths(case, seed), case["heads"], case["kv"], case["dim"]
    # Queries are wider than one so that the softmax prefers some keys, as a trained one does.
    if case["kind"] == "step":
        # The cache has room past every sequence; what lies there is left over from others.
        room = max(lengths) + 61
        s["q"] = normal(len(lengths), heads, dim, std=2.0)
        s["k"], s["v"] = (normal(len(lengths), room, kv, dim) for _ in range(2))
        s["nq"], s["nk"] = [1] * len(lengths), lengths
        s["k_first"] = [i * room for i in range(len(lengths))]
        s["k_offsets"] = torch.tensor(s["k_first"], dtype=torch.int64, device="cuda")
        s["k_lengths"] = torch.tensor(lengths, dtype=torch.int64, device="cuda")
        s["causal"] = True
    else:
        s["nq"], s["nk"] = lengths, [n + case["past"] for n in lengths]
        tokens, keys = sum(s["nq"]), sum(s["nk"])
        if case["past"]:
            s["q"] = normal(tokens, heads, dim, std=2.0)
            s["k"], s["v"] = (normal(keys, kv, dim) for _ in range(2))
        else:
            merged = normal(tokens, heads + 2 * kv, dim)
            merged[:, :heads] *= 2.0
            s["q"], s["k"], s["v"] = merged.split((heads, kv, kv), dim=1)
        s["k_first"] = [sum(s["nk"][:i]) for i in range(len(lengths))]
        s["k_offsets"], s["k_lengths"] = _offsets(s["nk"], "cuda"), None
        s["causal"] = case["causal"]
    s["q_offsets"] = _offsets(s["nq"], "cuda")
    return s


def _tiled(n, blocks, device):
    """Where the 128x4 order keeps the scale of (row, K block)."""
    row = torch.arange(n, device=device)[:, None]
    col = torch.arange(blocks, device=device)[None]
    return row // 128 * (128 * blocks) + col // 4 * 512 + row % 32 * 16 + row % 128 // 32 * 4 + col % 4


def _pack(w):
    """A weight in 4 bits: E2M1 codes, E4M3 scales of 16 values, one FP32 factor."""
    n, k = w.shape
    blocks = w.reshape(n, k // 16, 16)
    alpha = w.abs().amax() / 2688.0
    scale = (blocks.abs().amax(dim=-1) / (6.0 * alpha)).clamp(max=448.0).to(torch.float8_e4m3fn)
    step = (scale.float() * alpha).unsqueeze(-1)
    v = torch.where(step > 0, blocks / step, torch.zeros_like(blocks))
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
    code = (torch.bucketize(v.abs(), edges) + 8 * (v < 0)).to(torch.uint8).reshape(n, k // 2, 2)
    scales = torch.empty(n * (k // 16), dtype=torch.uint8, device=w.device)
    scales[_tiled(n, k // 16, w.device).reshape(-1)] = scale.view(torch.uint8).reshape(-1)
    return (code[..., 0] | code[..., 1] << 4).contiguous(), scales.reshape(n, k // 16), alpha.reshape(())


def run(s):
    if own:
        return _run_own(s)
    return _plain_w4(s) if s["case"]["kind"] == "w4" else _plain_attention(s)


def _run_own(s):
    case = s["case"]
    if case["kind"] == "w4":
        return s["execution"].linear(s["x"], s["weight"], s["bias"])
    from vflash_amd.attention import packed_attention

    k, v = s["k"], s["v"]
    if case["kind"] == "step":
        k, v = k.flatten(0, 1), v.flatten(0, 1)
    return packed_attention(s["q"], k, v, s["q_offsets"], s["k_offsets"], k_lengths=s["k_lengths"], causal=s["causal"])


def _plain_w4(s):
    packed, x = s["packed"], s["x"].float()
    n, k = packed.shape[0], 2 * packed.shape[1]
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                         device=x.device)
    w = table[torch.stack((packed & 15, packed >> 4), dim=-1).int()].reshape(n, k // 16, 16)
    scale = s["scales"].reshape(-1).view(torch.float8_e4m3fn).float()[_tiled(n, k // 16, x.device)]
    y = (x @ (w * scale.unsqueeze(-1)).reshape(n, k).T) * s["alpha"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(torch.bfloat16)


def _plain_attention(s):
    q, k, v = s["q"], s["k"], s["v"]
    tokens, heads, dim = q.shape
    k, v = k.reshape(-1, *k.shape[-2:]), v.reshape(-1, *v.shape[-2:])
    kv = k.shape[1]
    out = torch.zeros((tokens, heads, dim), dtype=q.dtype, device=q.device)
    first = 0
    for nq, nk, at in zip(s["nq"], s["nk"], s["k_first"]):
        if nq and nk:
            ks = k[at:at + nk].float().transpose(0, 1).contiguous()
            vs = v[at:at + nk].float().transpose(0, 1).contiguous()
            rows = max(1, BLOCK // (nk * heads))
            for a in range(0, nq, rows):
                b = min(nq, a + rows)
                qs = q[first + a:first + b].float().reshape(b - a, kv, heads // kv, dim).permute(1, 2, 0, 3)
                qs = qs.reshape(kv, heads // kv * (b - a), dim)
                p = torch.bmm(qs, ks.transpose(1, 2)).mul_(1.0 / math.sqrt(dim)).view(kv, heads // kv, b - a, nk)
                if s["causal"]:
                    i = torch.arange(a + nk - nq, b + nk - nq, device=q.device)[:, None]
                    p.masked_fill_(torch.arange(nk, device=q.device)[None] > i, -torch.inf)
                p.sub_(p.amax(dim=-1, keepdim=True)).exp_()
                p.div_(p.sum(dim=-1, keepdim=True))
                o = torch.bmm(p.view(kv, -1, nk), vs).view(kv, heads // kv, b - a, dim)
                out[first + a:first + b] = o.permute(2, 0, 1, 3).reshape(b - a, heads, dim).to(q.dtype)
        first += nq
    return out


def _pairs(case):
    """Query-key pairs that attend to each other, a head."""
    if case["kind"] == "step":
        return sum(_lengths(case))
    past = case["past"]
    if case["causal"]:
        return sum(n * past + n * (n + 1) // 2 for n in _lengths(case))
    return sum(n * (n + past) for n in _lengths(case))


def work(case):
    if case["kind"] == "w4":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * k + n * k // 2 + n * k // 16 + 2 * m * n + (2 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    lengths, row = _lengths(case), 2 * case["dim"]
    step = case["kind"] == "step"
    tokens = len(lengths) if step else sum(lengths)
    keys = sum(lengths) if step else sum(n + case["past"] for n in lengths)
    return {"bytes": row * (2 * tokens * case["heads"] + 2 * keys * case["kv"]),
            "flops": 4 * case["dim"] * case["heads"] * _pairs(case)}


def exact(case, seed):
    """What run() returns, from the definitions, in 64 bits."""
    s = prepare(case, seed)
    if case["kind"] == "w4":
        return _exact_w4(s)
    k, v = (t.flatten(0, 1) if t.ndim == 4 else t for t in (s["k"], s["v"]))
    tokens, heads, dim = s["q"].shape
    group = heads // k.shape[1]
    out = torch.zeros((tokens, heads, dim), dtype=F64, device=s["q"].device)
    first = 0
    for nq, nk, at in zip(s["nq"], s["nk"], s["k_first"]):
        for head in range(heads) if nq and nk else ():
            keys = k[at:at + nk, head // group].to(F64)
            values = v[at:at + nk, head // group].to(F64)
            for a in range(0, nq, 8192):
                b = min(nq, a + 8192)
                scores = s["q"][first + a:first + b, head].to(F64) @ keys.T / math.sqrt(dim)
                if s["causal"]:
                    # Query i of a sequence is its token nk - nq + i and sees the keys up to itself.
                    scores = torch.where(torch.ones_like(scores, dtype=torch.bool).tril_(a + nk - nq), scores,
                                         torch.full_like(scores, -torch.inf))
                out[first + a:first + b, head] = torch.softmax(scores, dim=-1) @ values
        first += nq
    return out


def _exact_w4(s):
    n, half = s["packed"].shape
    code = torch.stack((s["packed"] % 16, s["packed"] // 16), dim=-1).reshape(n, 2 * half).int()
    # E2M1: two bits of exponent (bias 1; 0 means the value is half the mantissa bit), one of mantissa.
    e, f = code % 8 // 2, (code % 2).to(F64)
    w = torch.where(e > 0, (1.0 + f / 2.0) * torch.exp2((e - 1).to(F64)), f / 2.0) * (1.0 - 2.0 * (code // 8).to(F64))
    # The 128x4 order as axes: 128-row tile, 4-column tile, row mod 32, row / 32, column mod 4.
    byte = s["scales"].reshape(n // 128, half // 32, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(n, half // 8).int()
    # E4M3: four bits of exponent (bias 7; 0 means multiples of 2^-9), three of mantissa.
    e, f = byte // 8 % 16, (byte % 8).to(F64)
    scale = torch.where(e > 0, (1.0 + f / 8.0) * torch.exp2((e - 7).to(F64)), f / 512.0)
    scale = scale * (1.0 - 2.0 * (byte // 128).to(F64))
    y = (s["x"].to(F64) @ (w.reshape(n, half // 8, 16) * scale.unsqueeze(-1)).reshape(n, 2 * half).T) * s["alpha"].to(F64)
    return y if s["bias"] is None else y + s["bias"].to(F64)
