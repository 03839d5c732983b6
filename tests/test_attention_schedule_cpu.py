"""Which rows and keys the workgroups of packed attention take, on the CPU: every row of the output once and
nothing outside the operands, whatever the offsets hold."""

import random
from collections import defaultdict

import pytest

from tests import attention_schedule

pytestmark = pytest.mark.skipif(not attention_schedule.COMPILER.exists(), reason="no clang++ for the host build")

# tokens, keys, sequences, heads, group, dim: the step and the tile kernel, split and whole, head blocks that divide
# among the XCDs and that do not, groups wider than a tile, more sequences than a wave has lanes.
SIZES = {
    "step whole": (90, 300, 80, 4, 2, 64), "step split": (40, 5000, 5, 8, 2, 64), "step XCDs": (70, 3000, 5, 16, 2, 128),
    "step many": (150, 200000, 200, 6, 2, 64), "step wide group": (3, 900, 3, 40, 40, 64),
    "tiles whole": (900, 900, 2, 7, 7, 96), "tiles split": (300, 4000, 3, 4, 2, 128), "tiles XCDs": (700, 2000, 4, 8, 1, 64),
    "tiles many": (4000, 5000, 150, 4, 2, 64), "tiles many split": (2500, 9000, 70, 2, 2, 64),
    "tiles wide group": (130, 600, 2, 150, 150, 64), "no sequence": (90, 300, 0, 4, 2, 64),
}
LIMIT = 1 << 63


def split_at(rng, total, parts):
    return [0, *sorted(rng.randint(0, total) for _ in range(parts - 1)), total][: parts + 1] if parts else [0]


def bad(rng, n, hi):
    """Offsets that decrease, overlap, lie outside: whole runs of them, and single ones among good ones."""
    kind = rng.randrange(4)
    good = sorted(rng.randint(0, hi) for _ in range(n))
    if kind == 0:
        return [rng.choice((-LIMIT, -1, 0, hi, hi + 1, 1 << 31, (1 << 32) + 5, LIMIT - 1, rng.randint(-hi, 2 * hi))) for _ in range(n)]
    if kind == 1:
        return good[::-1]
    if kind == 2:  # falls back once, past the first 64 where there are that many
        at = min(n - 1, 70) if n > 1 else 0
        return good[:at] + [v // 2 for v in good[at:]]
    return [v if rng.random() < 0.8 else rng.choice((-5, 3 * hi, rng.randint(0, hi))) for v in good]


def check(size, causal, lengths, qo, ko, kl, result):
    tokens, keys, batch, heads, group, dim = size
    (step, tile_tokens, _, parts, head_blocks, slots, grid, join), rows, joins = result
    tiles = defaultdict(list)
    for q0, nq, tile, block, first, count, key_first, key_last, k0, nk, splits, slot in rows:
        assert 0 <= q0 and nq > 0 and q0 + nq <= tokens and 0 <= tile * tile_tokens < nq and 0 <= block < head_blocks
        assert k0 >= 0 and nk >= 0 and k0 + nk <= keys and 0 <= key_first and key_last <= nk
        tiles[block, q0, nq, k0, nk, tile].append((first, count, key_first, key_last, splits, slot))
    # Every row once.
    covered = defaultdict(list)
    for block, q0, nq, k0, nk, tile in tiles:
        covered[block].append((q0 + tile * tile_tokens, q0 + min(nq, (tile + 1) * tile_tokens)))
    assert len(covered) == head_blocks
    for spans in covered.values():
        end = 0
        for a, b in sorted(spans):
            assert a == end < b
            end = b
        assert end == tokens
    # Every key that a tile sees once, and its parts where the join looks for them.
    wanted, used = defaultdict(set), set()
    for (block, q0, nq, k0, nk, tile), found in tiles.items():
        last = min(nq, (tile + 1) * tile_tokens) - 1
        limit = max(0, min(nk, nk - nq + last + 1)) if causal else nk
        found.sort()
        end = unit = 0
        for first, count, key_first, key_last, splits, slot in found:
            assert first == unit
            unit += count
            if key_first < key_last:
                assert key_first == end
                end = key_last
            if step and count < splits:
                wanted[q0, nq, tile, block].add(slot)
                assert 0 <= slot < slots and slot not in used
                used.add(slot)
            elif not step and splits > 1:
                assert 0 <= slot + first < slots and slot + first not in used
                used.add(slot + first)
                if key_first < limit:
                    wanted[q0, nq, tile, block].add(slot + first)
        assert end == limit and unit == found[0][4]
        if not step and found[0][4] > 1:
            wanted[q0, nq, tile, block] |= set()
    assert join or not wanted
    read = defaultdict(list)
    for q0, nq, tile, block, n, slot in joins:
        read[q0, nq, tile, block] += [slot] if step else range(slot, slot + n)
    assert {key: sorted(v) for key, v in read.items()} == {key: sorted(v) for key, v in wanted.items()}
    return {(q0, nq, k0, nk) for _, q0, nq, k0, nk, _ in tiles}


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    return attention_schedule.build(tmp_path_factory.mktemp("schedule"))


@pytest.mark.parametrize("size", SIZES.values(), ids=SIZES)
def test_good_offsets(program, size):
    tokens, keys, batch, heads, group, dim = size
    rng = random.Random(str(size))
    calls = []
    for i in range(4):
        lengths = i % 2 == 1
        qo = split_at(rng, tokens, batch)
        ko = [rng.randint(0, keys) for _ in range(batch)] if lengths else split_at(rng, keys, batch)
        kl = [rng.randint(0, keys - k) for k in ko] if lengths else None
        calls.append((tokens, keys, heads, group, dim, i % 3 > 0, qo, ko, kl))
    for call, result in zip(calls, attention_schedule.run(program, calls)):
        causal, qo, ko, kl = call[5:]
        got = check(size, causal, kl is not None, qo, ko, kl, result)
        want = {(a, b - a, k, kl[i] if kl is not None else ko[i + 1] - k)
                for i, (a, b, k) in enumerate(zip(qo, qo[1:], ko)) if b > a}
        assert {(q0, nq, k0 if nk else 0, nk) for q0, nq, k0, nk in got} == (
            {(q0, nq, k0 if nk else 0, nk) for q0, nq, k0, nk in want} if batch else {(0, tokens, 0, 0)})


@pytest.mark.parametrize("size", SIZES.values(), ids=SIZES)
def test_bad_offsets(program, size):
    tokens, keys, batch, heads, group, dim = size
    rng = random.Random(str(size) + "bad")
    calls = []
    for i in range(6):
        kl = bad(rng, batch, keys) if i % 2 and batch else None
        calls.append((tokens, keys, heads, group, dim, i % 3 > 0, bad(rng, batch + 1, tokens),
                      bad(rng, batch if kl is not None else batch + 1, keys), kl))
    for call, result in zip(calls, attention_schedule.run(program, calls)):
        check(size, call[5], call[8] is not None, *call[6:], result)


def test_the_sizes_reach_every_plan(program):
    reached = set()
    for name, (tokens, keys, batch, heads, group, dim) in SIZES.items():
        rng = random.Random(1)
        call = (tokens, keys, heads, group, dim, True, split_at(rng, tokens, batch), split_at(rng, keys, batch), None)
        (step, *_, join), rows, joins = attention_schedule.run(program, [call])[0]
        assert name.startswith("step" if step else ("tiles", "no sequence")), name
        reached.add((step, join, batch > 62))
    assert reached == {(s, j, m) for s in (0, 1) for j in (0, 1) for m in (False, True)}
