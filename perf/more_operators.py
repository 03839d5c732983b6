"""The operators of a serving step of many requests, as cases that can be timed.

kind      entry point
rotate    ``rotary.rotate``: rotary positions of the query and key heads
append    ``paged.paged_append``: rotary positions, and the new keys and values into a paged cache
attend    ``paged.paged_attention``: one new token a sequence, or a few, over the paged cache
adapters  ``adapters.add_request_adapters``: the low-rank adapters of many requests beside a projection

``run`` computes them in elementary torch operations, or with ``own`` through the package.
"""

import math
import random

import torch

own = False

F32, F64, E4M3 = torch.float32, torch.float64, torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": E4M3}


def listed():
    return [
        # One new token, far into a long conversation, half of each head rotated.
        dict(name="rotate_1_far", kind="rotate", tokens=1, first=1000003, heads=32, kv=8, dim=128, part=64, layout="half",
             factor=8.0, axes=1, dtype="bf16"),
        # The denoiser's own: every token of a 21x30x52 latent, 40 heads, rotated along three axes.
        dict(name="rotate_32760_grid", kind="rotate", tokens=32760, first=0, heads=40, kv=40, dim=128, part=128,
             layout="interleaved", factor=1.0, axes=3, dtype="bf16"),
        # One new token of one sequence: the smallest append, latency alone.
        dict(name="append_1", kind="append", batch=1, low=1, high=1, past=76, heads=32, kv=8, dim=128, page=16, part=128,
             layout="half", factor=1.0, dtype="bf16", store="bf16"),
        # A decoding batch, the cache in 8 bits.
        dict(name="append_125_e4m3", kind="append", batch=125, low=1, high=1, past=501, heads=32, kv=8, dim=128, page=64,
             part=128, layout="half", factor=4.0, dtype="bf16", store="e4m3"),
        # A batch of prompts of different lengths.
        dict(name="append_9x1to2047_f16", kind="append", batch=9, low=1, high=2047, past=0, heads=28, kv=4, dim=128,
             page=32, part=128, layout="interleaved", factor=1.0, dtype="f16", store="f16"),
        # One new token of one sequence over a short prompt: latency alone.
        dict(name="attend_1x77", kind="attend", batch=1, low=77, high=77, new=1, heads=32, kv=8, dim=128, page=16,
             dtype="bf16", store="bf16"),
        # A decoding batch whose sequences are of very different lengths, the cache in 8 bits.
        dict(name="attend_61x1to8191_e4m3", kind="attend", batch=61, low=1, high=8191, new=1, heads=32, kv=8, dim=128,
             page=64, dtype="bf16", store="e4m3"),
        # One sequence with a long cache: the keys alone have to fill the card.
        dict(name="attend_1x131071", kind="attend", batch=1, low=131071, high=131071, new=1, heads=32, kv=8, dim=128,
             page=128, dtype="bf16", store="bf16"),
        # Drafted tokens that are checked together, four a sequence, narrow heads.
        dict(name="attend_15x4_d64_f16", kind="attend", batch=15, low=900, high=4099, new=4, heads=16, kv=4, dim=64,
             page=16, dtype="f16", store="f16"),
        # One request's adapter beside a square projection of one token.
        dict(name="adapters_1x5120x5120", kind="adapters", rows=1, k=5120, widths="5120", used=1, rank=16, order="mixed",
             dtype="bf16"),
        # A decoding batch in which most requests have adapters of their own, beside a merged QKV projection.
        dict(name="adapters_61x5376x10752", kind="adapters", rows=61, k=5376, widths="7168,1792,1792", used=23, rank=64,
             order="mixed", dtype="bf16"),
        # Prompts one after another, each with its request's adapter, beside the FFN up-projection.
        dict(name="adapters_4093x5120x13824_f16", kind="adapters", rows=4093, k=5120, widths="13824", used=9, rank=32,
             order="runs", dtype="f16"),
    ]


def _log(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))) - 0.5)))


HEADS = ((32, 8, 128), (28, 4, 128), (40, 40, 128), (56, 56, 128), (16, 16, 64), (12, 2, 64), (24, 8, 96), (8, 1, 128),
         (20, 5, 80))


def draw(rng):
    kind = rng.choice(("rotate", "append", "attend", "adapters"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    if kind == "adapters":
        rows, k = _log(rng, 1, 4093), 8 * _log(rng, 8, 896)
        widths = rng.choice(("%d" % (16 * _log(rng, 4, 864)), "%d,%d,%d" % ((64 * _log(rng, 1, 80),) * 3),
                             "%d,%d,%d" % ((128 * _log(rng, 1, 40),) + (32 * _log(rng, 1, 32),) * 2)))
        return dict(kind=kind, rows=rows, k=k, widths=widths, used=_log(rng, 1, min(rows, 24)),
                    rank=rng.choice((1, 8, 16, 24, 32, 64, 100, 128) if rows < 1000 else (4, 8, 16, 32)),
                    order=rng.choice(("mixed", "runs")), dtype=dtype)
    heads, kv, dim = rng.choice(HEADS)
    s = dict(kind=kind, heads=heads, kv=kv, dim=dim)
    if kind != "attend":
        s.update(layout=rng.choice(("half", "interleaved")), part=rng.choice((dim, dim, dim // 2, dim // 4 * 2 - 4)),
                 factor=rng.choice((1.0, 4.0, 32.0)), dtype=dtype)
    if kind == "rotate":
        s.update(tokens=_log(rng, 1, 32760 * 80 * 128 // ((heads + kv) * dim)), first=_log(rng, 1, 1 << 21),
                 axes=rng.choice((1, 1, 3)))
        s["tokens"] = min(s["tokens"], 32760)
        return s
    s.update(page=rng.choice((16, 32, 64, 128, 256)), dtype=dtype, store=rng.choice((dtype, "e4m3")))
    if kind == "append":
        batch = _log(rng, 1, 200)
        high = _log(rng, 1, max(1, 16000 * 36 * 128 // ((heads + 2 * kv) * dim) // batch))
        s.update(batch=batch, low=rng.choice((0, 1)), high=high, past=rng.choice((0, _log(rng, 1, 2000))))
        return s
    batch = _log(rng, 1, 128)
    high = _log(rng, 1, min(131071, (1 << 27) // (batch * kv * dim)))
    s.update(batch=batch, low=_log(rng, 1, high), high=high, new=rng.choice((1, 1, 1, 2, 5)))
    return s


def _lengths(case, seed=0):
    """The sequences' new lengths (those of the cache for ``attend``), the longest among them.
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


def _frequencies(case):
    """Radians a position, for each pair; the axis that it follows; and what sines and cosines are multiplied by."""
    pairs, axes = case["part"] // 2, case.get("axes", 1)
    each = [pairs // axes + (i < pairs % axes) for i in range(axes)]
    f = [10000.0 ** (-i / n) for n in each for i in range(n)]
    axis = [a for a, n in enumerate(each) for _ in range(n)]
    factor = case["factor"]
    if factor != 1.0:
        # Long contexts: pairs that turn less than once in 4096 positions are slowed by the factor, those that
        # turn 32 times are not, and those between are in proportion.
        keep = [min(1.0, max(0.0, (4096 * x / (2 * math.pi) - 1.0) / 31.0)) for x in f]
        f = [x * (g + (1.0 - g) / factor) for x, g in zip(f, keep)]
    return f, axis, 0.1 * math.log(factor) + 1.0


def _ranks(case):
    """The adapters' own ranks, the largest among them."""
    rng = random.Random("%d %d" % (case["used"], case["rank"]))
    return [case["rank"]] + [rng.randint((case["rank"] + 3) // 4, case["rank"]) for _ in range(case["used"] - 1)]


def _widths(case):
    return [int(w) for w in case["widths"].split(",")]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dtype):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=F32) * std).to(dtype)

    s = {"case": case}
    if case["kind"] == "adapters":
        rows, k, widths, ranks = case["rows"], case["k"], _widths(case), _ranks(case)
        n, width, count = sum(widths), -(-case["rank"] // 16) * 16, len(ranks)
        s["x"], s["base"] = normal(rows, k), normal(rows, n)
        # Each adapter's rows past its own rank are zeros.
        own_rank = torch.tensor(ranks, device="cuda")
        live = torch.arange(width, device="cuda") < own_rank[:, None]
        s["down"] = normal(count, len(widths), width, k, std=k**-0.5) * live[:, None, :, None].to(dtype)
        s["up"] = normal(count, n, width, std=0.3) * live[:, None, :].to(dtype)
        s["scaling"] = torch.rand(count, len(widths), generator=g, device="cuda") + 0.5
        s["ranks"] = own_rank.to(torch.int32)
        # Every adapter in use has a row; one request in eight has none.
        rng = random.Random(seed)
        index = list(range(count)) + [rng.choice([-1] + [rng.randrange(count)] * 7) for _ in range(rows - count)]
        rng.shuffle(index)
        s["index"] = torch.tensor(sorted(index) if case["order"] == "runs" else index, device="cuda")
        if own:
            from vflash_amd.adapters import RequestAdapters

            s["pack"] = RequestAdapters(s["down"].flatten(1, 2), s["up"], s["scaling"], s["ranks"], tuple(widths))
        return s
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    if case["kind"] != "attend":
        f, axis, s["magnitude"] = _frequencies(case)
        s["f"], s["axis"] = torch.tensor(f, dtype=F64, device="cuda"), torch.tensor(axis, device="cuda")
        if own:
            from vflash_amd.rotary import Rotary

            s["rotary"] = Rotary(f, layout=case["layout"], axes=axis, magnitude=s["magnitude"], device="cuda")
    if case["kind"] == "rotate":
        tokens = case["tokens"]
        at = torch.arange(tokens, device="cuda") + case["first"] + random.Random(seed).randrange(100)
        s["positions"] = at
        if case["axes"] == 3:
            s["positions"] = torch.stack((at // 1560, at % 1560 // 52, at % 52), dim=1)
        s["q"], s["k"], _ = normal(tokens, heads + 2 * kv, dim).split((heads, kv, kv), dim=1)
        return s
    lengths, page = _lengths(case, seed), case["page"]
    s["new"] = lengths if case["kind"] == "append" else [case["new"]] * len(lengths)
    s["all"] = [n + (case["past"] if case["kind"] == "append" else case["new"] - 1) for n in lengths]
    # Pages lie where the pool had room; a few are free.
    need = [-(-n // page) for n in s["all"]]
    pages, width = sum(need) + 3, max(max(need), 1)
    place = list(range(pages))
    random.Random(seed).shuffle(place)
    table, at = [], 0
    for n in need:
        table.append(place[at:at + n] + [0] * (width - n))
        at += n
    s["table"] = torch.tensor(table, device="cuda")
    s["lengths"] = torch.tensor(s["all"], device="cuda")
    s["q_offsets"] = None if s["new"] == [1] * len(lengths) else _offsets(s["new"], "cuda")
    tokens = sum(s["new"])
    shape = (pages, 2, kv, page, dim)
    s["scales"] = None
    if case["store"] == "e4m3":
        values = normal(*shape, dtype=F32)
        s["scales"] = values.abs().amax(dim=-1) / 448.0
        s["values"] = (values / s["scales"].unsqueeze(-1)).clamp(-448.0, 448.0).to(E4M3)
    else:
        s["values"] = normal(*shape)
    if case["kind"] == "append":
        s["q"], s["k"], s["v"] = normal(tokens, heads + 2 * kv, dim).split((heads, kv, kv), dim=1)
    else:
        # Queries are wider than one so that the softmax prefers some keys, as a trained one does.
        s["q"] = normal(tokens, heads, dim, std=2.0)
    if own:
        from vflash_amd.paged import PagedCache

        s["cache"] = PagedCache(s["values"], s["scales"])
    return s


def run(s):
    kind = s["case"]["kind"]
    if own:
        if kind == "rotate":
            from vflash_amd.rotary import rotate

            return rotate(s["q"], s["k"], s["positions"], s["rotary"])
        if kind == "adapters":
            from vflash_amd.adapters import add_request_adapters

            return add_request_adapters(s["base"], s["x"], s["pack"], s["index"])
        from vflash_amd.paged import paged_append, paged_attention

        if kind == "attend":
            return paged_attention(s["q"], s["cache"], s["table"], s["lengths"], q_offsets=s["q_offsets"])
        q = paged_append(s["cache"], s["k"], s["v"], s["table"], s["lengths"], q=s["q"], q_offsets=s["q_offsets"],
                         rotary=s["rotary"])
        return _written(s, q)
    if kind == "rotate":
        return _plain_rotate(s, s["q"], s["positions"]).to(s["q"].dtype), _plain_rotate(s, s["k"], s["positions"]).to(
            s["k"].dtype)
    return {"append": _plain_append, "attend": _plain_attend, "adapters": _plain_adapters}[kind](s)


def _written(s, q):
    return (q, s["values"]) if s["scales"] is None else (q, s["values"], s["scales"])


def _plain_rotate(s, x, positions):
    pairs = s["f"].numel()
    at = positions[:, None].expand(-1, pairs) if positions.ndim == 1 else positions[:, s["axis"]]
    angle = at.to(F64) * s["f"]
    cos, sin = ((t * s["magnitude"]).to(F32)[:, None] for t in (angle.cos(), angle.sin()))
    x = x.to(F32)
    turn, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if s["case"]["layout"] == "half":
        a, b = turn[..., :pairs], turn[..., pairs:]
        return torch.cat((a * cos - b * sin, a * sin + b * cos, rest), dim=-1)
    a, b = turn[..., 0::2], turn[..., 1::2]
    turn = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return torch.cat((turn.flatten(-2), rest), dim=-1)


def _rows(s):
    """Of each token: its position, its page and its place in that."""
    device, page = s["table"].device, s["case"]["page"]
    starts = s["q_offsets"] if s["q_offsets"] is not None else torch.arange(len(s["new"]) + 1, device=device)
    token = torch.arange(s["q"].shape[0], device=device)
    b = torch.searchsorted(starts, token, right=True) - 1
    at = s["lengths"][b] - (starts[b + 1] - token)
    return at, s["table"][b, at // page], at % page


def _plain_append(s):
    at, page, slot = _rows(s)
    dtype, store = s["q"].dtype, s["values"].dtype
    kv = torch.stack((_plain_rotate(s, s["k"], at), s["v"].to(F32)), dim=1)
    if s["scales"] is not None:
        top = kv.abs().amax(dim=-1)
        scale = torch.where(top > 0, top / 448.0, torch.ones_like(top))
        s["scales"][page, :, :, slot] = scale
        kv = (kv / scale.unsqueeze(-1)).clamp(-448.0, 448.0)
        s["values"].view(torch.uint8)[page, :, :, slot] = kv.to(store).view(torch.uint8)
    else:
        s["values"][page, :, :, slot] = kv.to(store)
    return _written(s, _plain_rotate(s, s["q"], at).to(dtype))


def _plain_attend(s):
    case, q = s["case"], s["q"]
    batch, new, heads, kv, dim = case["batch"], case["new"], case["heads"], case["kv"], case["dim"]
    # Every sequence's pages side by side: [batch, kv, width * page, dim].
    room = s["table"].shape[1] * case["page"]
    kvs = s["values"].view(torch.uint8)[s["table"]].view(s["values"].dtype).to(F32)
    if s["scales"] is not None:
        kvs = kvs * s["scales"][s["table"]].unsqueeze(-1)
    k, v = (kvs[:, :, i].transpose(1, 2).reshape(batch * kv, room, dim) for i in (0, 1))
    qs = q.to(F32).view(batch, new, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(batch * kv, -1, dim)
    p = torch.bmm(qs, k.transpose(1, 2).contiguous()).mul_(dim**-0.5).view(batch, kv, heads // kv, new, room)
    last = s["lengths"][:, None] - new + torch.arange(new, device=q.device)
    seen = torch.arange(room, device=q.device) <= last[..., None]
    p.masked_fill_(~seen[:, None, None], -torch.inf)
    p.sub_(p.amax(dim=-1, keepdim=True)).exp_()
    p.div_(p.sum(dim=-1, keepdim=True))
    o = torch.bmm(p.view(batch * kv, -1, room), v).view(batch, kv, heads // kv, new, dim)
    return o.permute(0, 3, 1, 2, 4).reshape(batch * new, heads, dim).to(q.dtype)


def _plain_adapters(s):
    x, down, up, index = s["x"].to(F32), s["down"].to(F32), s["up"].to(F32), s["index"]
    count, branches, width, k = down.shape
    # Every adapter for every row, and of these the row's own.
    t = (x @ down.view(-1, k).T).view(-1, count, branches, width) * s["scaling"][:, :, None]
    mine = index[:, None] == torch.arange(count, device=x.device)
    t = t * mine[:, :, None, None]
    ups = up.split(_widths(s["case"]), dim=1)
    delta = torch.cat([t[:, :, b].reshape(-1, count * width) @ u.transpose(1, 2).reshape(count * width, -1)
                       for b, u in enumerate(ups)], dim=1)
    return (s["base"].to(F32) + delta).to(s["base"].dtype)


def work(case):
    if case["kind"] == "adapters":
        widths, ranks, rows, k = _widths(case), _ranks(case), case["rows"], case["k"]
        n = sum(widths)
        return {"bytes": 2 * rows * (k + 2 * n) + 2 * sum(ranks) * (len(widths) * k + n),
                "flops": 2 * rows * sum(ranks) // len(ranks) * (len(widths) * k + n)}
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    if case["kind"] == "rotate":
        values = case["tokens"] * (heads + kv) * dim
        return {"bytes": 4 * values, "flops": 3 * values}
    lengths = _lengths(case)
    stored = dim + 4 if case["store"] == "e4m3" else 2 * dim
    if case["kind"] == "append":
        tokens = sum(lengths)
        return {"bytes": tokens * (4 * heads * dim + 2 * kv * (2 * dim + stored)), "flops": 3 * tokens * (heads + kv) * dim}
    keys, new = sum(lengths), case["new"]
    tokens = new * case["batch"]
    return {"bytes": 4 * tokens * heads * dim + 2 * (keys + case["batch"] * (new - 1)) * kv * stored,
            "flops": 4 * dim * heads * (new * keys + case["batch"] * new * (new - 1) // 2)}


def exact(case, seed):
    """What run() returns, from the definitions, in 64 bits."""
    s = prepare(case, seed)
    if case["kind"] == "adapters":
        out, first = s["base"].to(F64), 0
        for b, w in enumerate(_widths(case)):
            for a in range(case["used"]):
                rows = (s["index"] == a).nonzero()[:, 0]
                low = s["x"][rows].to(F64) @ s["down"][a, b].to(F64).T
                out[rows, first:first + w] += s["scaling"][a, b].to(F64) * (low @ s["up"][a, first:first + w].to(F64).T)
            first += w
        return out
    if case["kind"] == "rotate":
        return tuple(_exact_rotate(s, s[x], s["positions"]) for x in ("q", "k"))
    if case["kind"] == "append":
        starts = [0]
        for n in s["new"]:
            starts.append(starts[-1] + n)
        at = torch.tensor([n - m + i for n, m in zip(s["all"], s["new"]) for i in range(m)], device="cuda")
        b = torch.tensor([j for j, m in enumerate(s["new"]) for _ in range(m)], device="cuda")
        page, slot = s["table"][b, torch.div(at, case["page"], rounding_mode="floor")], at.remainder(case["page"])
        kv = torch.stack((_exact_rotate(s, s["k"], at), s["v"].to(F64)), dim=1)
        values = s["values"].to(F64)
        if s["scales"] is None:
            values[page, :, :, slot] = kv
            return _exact_rotate(s, s["q"], at), values
        scale = kv.abs().amax(dim=-1) / 448.0
        scale[scale == 0] = 1.0
        values[page, :, :, slot] = _nearest_e4m3(kv / scale.unsqueeze(-1))
        scales = s["scales"].to(F64)
        scales[page, :, :, slot] = scale
        return _exact_rotate(s, s["q"], at), values, scales
    heads, dim, new = case["heads"], case["dim"], case["new"]
    group = heads // case["kv"]
    out = torch.empty((len(s["all"]) * new, heads, dim), dtype=F64, device="cuda")
    for j, n in enumerate(s["all"]):
        pages = s["table"][j, :-(-n // case["page"])]
        kvs = torch.index_select(s["values"].view(torch.uint8), 0, pages).view(s["values"].dtype).to(F64)
        if s["scales"] is not None:
            kvs = kvs * s["scales"][pages].to(F64).unsqueeze(-1)
        k, v = (kvs[:, i].movedim(1, 0).reshape(case["kv"], -1, dim)[:, :n] for i in (0, 1))
        q = s["q"][j * new:(j + 1) * new].to(F64).unflatten(1, (case["kv"], group))
        scores = torch.einsum("ihgd,hkd->higk", q, k) / math.sqrt(dim)
        # Query i is token n - new + i and sees the keys up to itself.
        hidden = torch.ones((new, n), dtype=torch.bool, device="cuda").triu_(n - new + 1)
        scores = scores.masked_fill(hidden[None, :, None], -torch.inf)
        out[j * new:(j + 1) * new] = torch.einsum("higk,hkd->ihgd", torch.softmax(scores, dim=-1), v).flatten(1, 2)
    return out


def _exact_rotate(s, x, positions):
    """Each pair as a complex number, times magnitude e^(i position f)."""
    pairs = s["f"].numel()
    at = torch.stack([positions if positions.ndim == 1 else positions[:, a] for a in s["axis"].tolist()], dim=1)
    turn = torch.polar(torch.full_like(s["f"], s["magnitude"]).expand(at.shape), at.to(F64) * s["f"])[:, None]
    x = x.to(F64)
    head = x[..., :2 * pairs]
    if s["case"]["layout"] == "half":
        z = torch.view_as_real(torch.complex(head[..., :pairs], head[..., pairs:]) * turn).transpose(-1, -2)
    else:
        z = torch.view_as_real(torch.view_as_complex(head.unflatten(-1, (pairs, 2)).contiguous()) * turn)
    return torch.cat((z.flatten(-2), x[..., 2 * pairs:]), dim=-1)


def _nearest_e4m3(x):
    """x as the nearest E4M3 value, ties to even: three bits of mantissa down to 2^-6, steps of 2^-9 below."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0**-6))) - 3.0)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)
