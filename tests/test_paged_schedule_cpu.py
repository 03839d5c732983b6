"""Where the tokens of a paged append go, what the workgroups of paged attention take, and the sines of rotary
positions, on the CPU: nothing outside the operands is read, whatever offsets, lengths and tables hold."""

import math
import random
import subprocess

import pytest

from tests import attention_schedule
from tests.test_attention_schedule_cpu import LIMIT, bad, check

pytestmark = pytest.mark.skipif(not attention_schedule.COMPILER.exists(), reason="no clang++ for the host build")

PLACES = r"""
static RotateParams r;
static long wanted;
static void places() {
  for (long t = 0; t < wanted; ++t) {
    const TokenPlace place = token_place(r, t);
    if (threadIdx.x == 0) printf("place %lld %lld\n", (long long)place.position, (long long)place.page);
  }
}
int main() {
  long long batch, width, pages;
  int shift, given, at_end;
  while (scanf("%ld %lld %lld %lld %d %d %d", &wanted, &batch, &width, &pages, &shift, &given, &at_end) == 7) {
    r = RotateParams{};
    r.tokens = wanted, r.batch = batch;
    r.cache.width = width, r.cache.pages = pages, r.cache.page_shift = shift;
    if (given) r.q_offsets = vector(batch + 1, at_end);
    r.cache.lengths = vector(batch, at_end);
    r.cache.table = vector(batch * width, at_end);
    wave(places);
    printf("end\n");
  }
}
"""
SINES = r"""
int main() {
  unsigned long long phase;
  while (scanf("%llu", &phase) == 1) {
    const v2f cs = cos_sin((uint32_t)phase);
    printf("%.9g %.9g\n", cs[0], cs[1]);
  }
}
"""


def build(folder, program):
    """The harness of packed attention's schedule with another main."""
    (folder / "hip").mkdir()
    (folder / "hip" / "hip_runtime.h").write_text(attention_schedule.HIP)
    (folder / "program.cpp").write_text(program)
    for name in ("common.h", "attention.h", "attention_params.h", "attention_plan.h", "paged_params.h", "rotary.h"):
        (folder / name).write_text((attention_schedule.CSRC / name).read_text().replace(': "m0")', ': "memory")'))
    subprocess.run([str(attention_schedule.COMPILER), "-std=c++20", "-O2", "-w", "-U_FORTIFY_SOURCE", "-D_FORTIFY_SOURCE=0",
                    f"-I{folder}", str(folder / "program.cpp"), "-o", str(folder / "program")], check=True)
    return folder / "program"


def numbers(program, text):
    done = subprocess.run([str(program)], input=text, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, f"{done.returncode}: {done.stdout[-300:]}"
    return done.stdout.splitlines()


@pytest.fixture(scope="module")
def head():
    return attention_schedule.PROGRAM[:attention_schedule.PROGRAM.index("int main() {")]


def with_rotary(head):
    return head.replace('#include "attention.h"', '#include "attention.h"\n#include "rotary.h"')


def test_sines(tmp_path, head):
    rng = random.Random(1)
    phases = [k << 28 for k in range(16)] + [(k << 29) + d for k in range(8) for d in (-1, 1)] + [1, 2, (1 << 32) - 1]
    phases = [p % (1 << 32) for p in phases] + [rng.randrange(1 << 32) for _ in range(20000)]
    got = numbers(build(tmp_path, with_rotary(head) + SINES), "\n".join(map(str, phases)))
    for phase, line in zip(phases, got):
        c, s = map(float, line.split())
        a = 2 * math.pi * phase / 2**32
        # Two terms of a Taylor series left out (below 3e-8), and a few roundings of values up to 1.
        assert abs(c - math.cos(a)) <= 2.0**-22 and abs(s - math.sin(a)) <= 2.0**-22, phase


def test_places(tmp_path, head):
    program = build(tmp_path, with_rotary(head) + PLACES)
    rng = random.Random(5)
    calls, text = [], []
    for i, (batch, tokens) in enumerate([(1, 1), (1, 9), (5, 20), (63, 70), (64, 90), (65, 90), (300, 400), (4097, 60), (0, 5)] * 4):
        width, shift, pages = rng.choice((1, 3, 9)), rng.choice((4, 5, 7)), rng.choice((0, 4, 50))
        given = batch == 0 or tokens != batch or rng.random() < 0.5
        good = i < 18
        offsets = sorted(rng.randint(0, tokens) for _ in range(batch + 1)) if good else bad(rng, batch + 1, tokens)
        room = width << shift
        lengths = [rng.randint(0, room) if good else rng.choice((-LIMIT, -1, 0, room, room + 3, LIMIT - 1, rng.randint(0, room)))
                   for _ in range(batch)]
        table = [rng.randint(0, max(0, pages - 1)) if good else rng.choice((-LIMIT, -1, 0, pages, LIMIT - 1, rng.randint(0, 60)))
                 for _ in range(batch * width)]
        calls.append((tokens, batch, width, pages, shift, given, offsets, lengths, table, good))
        text.append(f"{tokens} {batch} {width} {pages} {shift} {int(given)} {i % 2}")
        text += [" ".join(map(str, v)) for v in (offsets if given else [], lengths, table)]
    lines = iter(numbers(program, "\n".join(text)))
    for tokens, batch, width, pages, shift, given, offsets, lengths, table, good in calls:
        for token in range(tokens):
            _, position, page = next(lines).split()
            position, page = int(position), int(page)
            assert position == -1 or (0 <= position < width << shift and 0 <= page < pages)
            if not good:
                continue
            owners = [b for b in range(batch) if offsets[b] <= token < offsets[b + 1]] if given else [token]
            want = (-1, None)
            if owners:
                b = owners[0]
                at = lengths[b] - (offsets[b + 1] - token if given else 1)
                if 0 <= at < width << shift and table[b * width + (at >> shift)] < pages:
                    want = at, table[b * width + (at >> shift)]
            assert position == want[0] and (want[1] is None or page == want[1]), (token, want, position, page)
        assert next(lines) == "end"


# tokens, room, sequences, heads, group, dim
SIZES = {
    "one a sequence": (90, 4096, 90, 8, 4, 128), "XCDs": (70, 2048, 70, 32, 2, 128), "not split": (40, 512, 40, 6, 3, 64),
    "many": (150, 131072, 150, 4, 4, 64), "very many": (4200, 4096, 4200, 2, 2, 64), "several": (90, 4096, 20, 8, 4, 64), "wide group": (3, 4096, 3, 40, 40, 64),
    "drafts, wide group": (9, 4096, 3, 40, 40, 64), "no sequence": (5, 4096, 0, 4, 2, 64), "a piece": (60, 512, 1, 32, 4, 128),
    "tiles, wide group": (300, 4096, 3, 40, 40, 64), "tiles, no sequence": (5000, 4096, 0, 4, 2, 64), "tiles": (900, 4096, 2, 8, 8, 128), "tiles, several": (700, 8192, 5, 8, 1, 64),
    "tiles, many": (4000, 2048, 100, 4, 2, 64), "tiles, not split": (6000, 512, 9, 7, 7, 64),
}


@pytest.mark.parametrize("size", SIZES.values(), ids=SIZES)
def test_paged_schedule(tmp_path, head, size):
    tokens, room, batch, heads, group, dim = size
    text = head.replace("attention_line(p,", "attention_line<true>(p,").replace("attention_segment(p,", "attention_segment<true>(p,")
    text = text.replace("      AttentionSegment seg = attention_segment<true>(p, line, (int)b, pos, stop);", """
      seg = pos == begin ? attention_segment<true>(p, line, (int)b, pos, stop)
                         : attention_following<true>(p, line, (int)b, seg, pos, stop);""")
    text = text.replace("    for (uint32_t pos = begin; pos < stop;) {", "    AttentionSegment seg{};\n    for (uint32_t pos = begin; pos < stop;) {")
    # What a workgroup leaves for the join is what the join of packed attention finds.
    text = text.replace("static void steps() {", "static AttentionBegun left[1 << 16];\nstatic void steps() {").replace("""      pos += seg.count;
    }
""", """      pos += seg.count;
    }
    const AttentionBegun own = attention_begun(p, line, (int)b, seg, stop);
    if (threadIdx.x == 0) left[b] = own;
""")
    text = text.replace("    if (begin >= stop) continue;", "    AttentionBegun own = left[b];\n    if (begin >= stop && own.segments) exit(13);\n    if (begin >= stop) continue;")
    text = text.replace("tile_end <= stop) continue;", "tile_end <= stop) { if (own.segments) exit(14); continue; }")
    text = text.replace("    for (int s = 0; s < segments && threadIdx.x == 0", """    const int row = seg.it.tile * p.tile_tokens;
    if (own.segments != segments || own.row != seg.it.seq.q0 + row || own.head_block != seg.it.head_block ||
        own.tokens != min(p.tile_tokens, seg.it.seq.nq - row)) exit(15);
    for (int s = 0; s < segments && threadIdx.x == 0""")
    assert all(text.count(part) == 1 for part in ("exit(13)", "exit(14)", "exit(15)", "left[b] = own"))
    text = text.replace("attention_item<false>(p,", "attention_item<false, true>(p,").replace("attention_item<true>(p,", "attention_item<true, true>(p,")
    text += r"""
int main() {
  int tokens, keys, heads, group, dim, given, at_end;
  long long batch;
  while (scanf("%d %d %lld %d %d %d %d %d", &tokens, &keys, &batch, &heads, &group, &dim, &given, &at_end) == 8) {
    p = AttentionParams{};
    p.tokens = tokens, p.keys = keys, p.batch = batch, p.heads = heads, p.group = group, p.dim = dim, p.causal = 1;
    if (given) p.q_offsets = vector(batch + 1, at_end);
    p.cache.lengths = vector(batch, at_end);
    plan = paged_attention_plan(p, at_end);
    printf("plan %d %d %d %d %d %lld %lld %d\n", plan.step, p.tile_tokens, p.heads_per_tile, p.parts, p.head_blocks,
           (long long)p.slots, (long long)plan.grid, plan.join != 0);
    blocks = (unsigned)plan.grid;
    wave(plan.step ? steps : tiles);
    if (plan.join) {
      blocks = (unsigned)(plan.step ? plan.grid : plan.join);
      wave(plan.step ? step_joins : joins);
    }
    printf("end\n");
  }
}
"""
    program = build(tmp_path, text)
    rng = random.Random(tokens)
    name = next(k for k, v in SIZES.items() if v == size)
    calls, lines = [], []
    for i in range(6):
        given = tokens != batch or i % 2 == 1
        offsets = sorted([0, tokens] + [rng.randint(0, tokens) for _ in range(batch - 1)])[:batch + 1] if i < 3 else bad(rng, batch + 1, tokens)
        lengths = [rng.choice((0, 1, room, rng.randint(0, room))) if i < 3 else
                   rng.choice((-LIMIT, -1, 0, room + 1, 1 << 31, LIMIT - 1, rng.randint(0, room))) for _ in range(batch)]
        if not given:
            offsets = list(range(batch + 1))
        calls.append((offsets, lengths))
        lines.append(f"{tokens} {room} {batch} {heads} {group} {dim} {int(given)} {i % 2}")
        lines += [" ".join(map(str, v)) for v in (offsets if given else [], lengths)]
    results = []
    for line in numbers(program, "\n".join(lines)):
        kind, *values = line.split()
        values = tuple(map(int, values))
        if kind == "plan":
            results.append((values, [], []))
        elif kind != "end":
            results[-1][1 if kind == "rows" else 2].append(values)
    assert len(results) == len(calls)
    for (offsets, lengths), (plan, rows, joins) in zip(calls, results):
        assert plan[0] == (not name.startswith("tiles"))
        # A sequence's number stands where packed attention has its first key; give it room after it.
        for row in rows:
            assert 0 <= row[8] < max(batch, 1) and 0 <= row[9] <= room
            assert row[9] == 0 or row[9] == min(max(lengths[row[8]], 0), room)
        check((tokens, room + max(batch, 1), batch, heads, group, dim), True, lengths, offsets, list(range(batch)), lengths,
              (plan, rows, joins))
