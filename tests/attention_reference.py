"""Packed attention in 64 bits, and how far a kernel's output may be from it."""

import torch


def packed_attention(q, k, v, q_offsets, k_offsets, k_lengths=None, causal=False, scale=None):
    """The definition, on the CPU: the output and a bound on the error of a result whose
    probabilities and outputs are rounded to the operands' type and everything else to
    binary32."""
    q, k, v = (t.detach().cpu() for t in (q, k, v))
    dtype, (tokens, heads, dim) = q.dtype, q.shape
    group = heads // k.shape[1]
    scale = dim**-0.5 if scale is None else scale
    out = torch.zeros((tokens, heads, dim), dtype=torch.float64)
    bound = torch.zeros_like(out)
    half = torch.finfo(dtype).eps / 2
    starts = q_offsets.tolist()
    for b in range(len(starts) - 1):
        a, e = starts[b], starts[b + 1]
        first = int(k_offsets[b])
        nk = int(k_lengths[b]) if k_lengths is not None else int(k_offsets[b + 1]) - first
        nq = e - a
        if not nq or not nk:
            continue
        qs = q[a:e].double().permute(1, 0, 2)
        ks = k[first:first + nk].double().permute(1, 2, 0).repeat_interleave(group, 0)
        vs = v[first:first + nk].double().permute(1, 0, 2).repeat_interleave(group, 0)
        scores = qs @ ks * scale
        if causal:
            i = torch.arange(nq)[:, None] + nk - nq
            scores = scores.masked_fill(torch.arange(nk) > i, -torch.inf)
        top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float64).min)
        p = (scores - top).exp()
        total = p.sum(-1, keepdim=True)
        p = torch.where(total > 0, p / total, 0.0)
        o = p @ vs
        # A score is off by the roundings of its products' sum (dim of them at most) and of its
        # scaling, p by that and one rounding, each sum by a rounding per key.
        reach = (qs.abs() @ ks.abs()).amax(-1, keepdim=True) * scale
        off = half + 2.0**-24 * (2 * (dim + 8) * reach + 2 * nk + 64)
        mean = p @ vs.abs()
        # Binary16 probabilities carry 2^6 and round at 2^-25 where they are subnormal.
        floor = nk * 2.0**-31 * vs.abs().amax(1, keepdim=True) if dtype == torch.float16 else 0.0
        err = 2 * off * mean + floor + half * o.abs() + torch.finfo(dtype).smallest_normal * half * 2
        out[a:e] = o.permute(1, 0, 2)
        bound[a:e] = (torch.ones_like(o) * err).permute(1, 0, 2)
    return out, bound


def check(got, *args, **kwargs):
    want, bound = packed_attention(*args, **kwargs)
    assert got.shape == want.shape and got.dtype == args[0].dtype
    got = got.detach().cpu().double()
    assert bool(torch.isfinite(got).all())
    worst = ((got - want).abs() - bound).max().item() if got.numel() else 0.0
    assert worst <= 0, f"{worst} past the bound"
