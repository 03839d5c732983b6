"""The schedule of packed attention (csrc/attention.h, attention_plan.h), run on the CPU.

The device code is compiled for the host against a stand-in of the HIP header in which a wave is 64
fibers: each builtin that moves values between lanes stores the lane's value, lets the other lanes come
to the same builtin, and reads theirs.  Lanes that part ways are reported.  Offsets and lengths end
right before a page that cannot be read, and begin right after one.  The program takes calls on its
standard input and writes what their workgroups take, the kernels' loops over it (attention_tiles,
attention_join, attention_step, attention_step_join) included:

    rows q0 nq tile head_block first count key_first key_last k0 nk splits slot
    join q0 nq tile head_block splits slot
"""

import subprocess
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "vflash_amd" / "csrc"
COMPILER = Path("/opt/rocm/llvm/bin/clang++")

HIP = r"""
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <cstring>
#define __device__
#define __forceinline__ inline
using std::max;
using std::min;
struct dim3 { unsigned x, y, z; dim3(unsigned a = 1, unsigned b = 1, unsigned c = 1) : x(a), y(b), z(c) {} };
extern dim3 threadIdx, blockIdx, gridDim;
inline float __uint_as_float(uint32_t v) { float f; memcpy(&f, &v, 4); return f; }
inline uint32_t __float_as_uint(float v) { uint32_t u; memcpy(&u, &v, 4); return u; }
struct Rsrc {};
#define __amdgpu_buffer_rsrc_t Rsrc
template <class... A> inline Rsrc no_rsrc(A&&...) { abort(); }
template <class R, class... A> inline R none(A&&...) { abort(); }
struct Pair { uint32_t v[2]; uint32_t operator[](int i) const { return v[i]; } };
uint64_t exchange(int kind, uint32_t v, int lane);  // 0: lane's value, 1: the lanes whose value is not 0
inline int from_lane(int v, int lane) { return (int)exchange(0, (uint32_t)v, lane); }
inline int lane_shift(int old, int v, int control, bool zero) {
  if (control <= 0x110 || control > 0x11f || !zero) abort();
  const int lane = (int)threadIdx.x & 63, by = control - 0x110, other = from_lane(v, lane % 16 < by ? lane : lane - by);
  return lane % 16 < by ? 0 : other;
}
inline float __shfl_xor(float v, int o, int) { return __uint_as_float((uint32_t)exchange(0, __float_as_uint(v), ((int)threadIdx.x & 63) ^ o)); }
inline int __shfl_xor(int v, int o, int) { return from_lane(v, ((int)threadIdx.x & 63) ^ o); }
#define __builtin_amdgcn_update_dpp(old, v, c, r, b, z) lane_shift(old, v, c, z)
#define __builtin_amdgcn_readlane(v, l) from_lane(v, l)
#define __builtin_amdgcn_readfirstlane(v) from_lane(v, 0)
#define __builtin_amdgcn_ballot_w64(v) exchange(1, (v) ? 1u : 0u, 0)
#define __builtin_amdgcn_make_buffer_rsrc(...) no_rsrc()
#define __builtin_amdgcn_s_waitcnt(...) ((void)0)
#define __builtin_amdgcn_exp2f(v) exp2f(v)
#define __builtin_amdgcn_fdot2(...) none<float>()
#define __builtin_amdgcn_fdot2_f32_bf16(...) none<float>()
#define __builtin_amdgcn_ds_read_tr16_b64_v4i16(...) none<v4s16>()
#define __builtin_amdgcn_permlane32_swap(...) none<Pair>()
#define __builtin_amdgcn_permlane16_swap(...) none<Pair>()
#define __builtin_amdgcn_mfma_f32_32x32x16_f16(...) none<v16f>()
#define __builtin_amdgcn_mfma_f32_32x32x16_bf16(...) none<v16f>()
#define __builtin_amdgcn_mfma_f32_16x16x32_f16(...) none<v4f>()
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16(...) none<v4f>()
"""

PROGRAM = r"""
#include <setjmp.h>
#include <stdio.h>
#include <sys/mman.h>
#include <ucontext.h>
#include <hip/hip_runtime.h>
#include "attention.h"
#include "attention_plan.h"

dim3 threadIdx, blockIdx, gridDim;
namespace vfa { int compute_units() { return 256; } }
using namespace vfa;

static ucontext_t scheduler, start[64];
static jmp_buf back, lanes[64];
static bool started[64], ended[64];
static int kinds[2][64];
static uint32_t values[2][64];
static int turn[64];
static void (*body)();

uint64_t exchange(int kind, uint32_t v, int lane) {
  const int me = (int)threadIdx.x, t = turn[me];
  kinds[t][me] = kind;
  values[t][me] = v;
  if (!_setjmp(lanes[me])) _longjmp(back, 1);
  turn[me] = 1 - t;
  if (lane < 0 || lane > 63) { printf("a lane of %d\n", lane); exit(3); }
  if (kind == 0) return values[t][lane];
  uint64_t mask = 0;
  for (int i = 0; i < 64; ++i) mask |= uint64_t(values[t][i]) << i;
  return mask;
}
static void lane_main() {
  body();
  ended[threadIdx.x] = true;
  _longjmp(back, 1);
}
static void wave(void (*f)()) {
  static char stacks[64][1 << 16];
  body = f;
  for (int i = 0; i < 64; ++i) {
    started[i] = ended[i] = false;
    turn[i] = 0;
    getcontext(&start[i]);
    start[i].uc_stack.ss_sp = stacks[i];
    start[i].uc_stack.ss_size = sizeof stacks[i];
    start[i].uc_link = nullptr;
    makecontext(&start[i], lane_main, 0);
  }
  for (;;) {
    for (volatile int i = 0; i < 64; i = i + 1) {
      threadIdx.x = (unsigned)i;
      if (_setjmp(back)) continue;
      if (started[i]) _longjmp(lanes[i], 1);
      started[i] = true;
      setcontext(&start[i]);
    }
    for (int i = 1; i < 64; ++i)
      if (ended[i] != ended[0] || (!ended[0] && kinds[turn[i]][i] != kinds[turn[0]][0])) { printf("lanes part\n"); exit(3); }
    if (ended[0]) return;
  }
}

static AttentionParams p;
static AttentionPlan plan;
static unsigned blocks;

static void rows(const AttentionItem& it, uint32_t first, uint32_t count, int64_t key_first, int64_t key_last) {
  if (threadIdx.x == 0)
    printf("rows %d %d %d %d %u %u %lld %lld %d %d %d %lld\n", it.seq.q0, it.seq.nq, it.tile, it.head_block, first, count,
           (long long)key_first, (long long)key_last, it.seq.k0, it.seq.nk, it.splits, (long long)it.slot);
}
static int tile_limit_of(const AttentionItem& it) {
  return attention_limit(p, it.seq, min(it.seq.nq, (it.tile + 1) * p.tile_tokens) - 1);
}
static void tiles() {
  for (unsigned b = 0; b < blocks; ++b) {
    const AttentionItem it = attention_item<false>(p, b);
    if (!it.live) continue;
    const int limit = tile_limit_of(it), first = it.split * it.chunk;
    rows(it, (uint32_t)it.split, 1, first, min((int64_t)limit, (int64_t)first + it.chunk));
  }
}
static void joins() {
  for (unsigned b = 0; b < blocks; ++b) {
    const AttentionItem it = attention_item<true>(p, b);
    if (!it.live || it.splits == 1) continue;
    if (threadIdx.x == 0)
      printf("join %d %d %d %d %d %d\n", it.seq.q0, it.seq.nq, it.tile, it.head_block,
             (int)(((uint32_t)tile_limit_of(it) + (uint32_t)it.chunk - 1) / (uint32_t)it.chunk), it.slot);
  }
}
static void steps() {
  for (unsigned b = 0; b < blocks; ++b) {
    const AttentionLine line = attention_line(p, (int)blocks);
    const uint32_t begin = (b >> (line.xcds == 8 ? 3 : 0)) * line.quota, stop = min(begin + line.quota, line.end);
    for (uint32_t pos = begin; pos < stop;) {
      AttentionSegment seg = attention_segment(p, line, (int)b, pos, stop);
      if (!seg.it.live) break;
      seg.it.splits = (int)seg.of;
      seg.it.slot = (int)(seg.count == seg.of ? -1 : 2 * (int64_t)b + (seg.first == 0));
      const uint64_t first = min((uint64_t)seg.first << line.unit_shift, (uint64_t)INT32_MAX);
      rows(seg.it, seg.first, seg.count, (int64_t)first,
           (int64_t)min((uint64_t)tile_limit_of(seg.it), (uint64_t)(seg.first + seg.count) << line.unit_shift));
      pos += seg.count;
    }
  }
}
static void step_joins() {
  for (unsigned b = 0; b < blocks; ++b) {
    const AttentionLine line = attention_line(p, (int)blocks);
    const int part = (int)(b >> (line.xcds == 8 ? 3 : 0));
    const uint32_t begin = part * line.quota, stop = min(begin + line.quota, line.end);
    if (begin >= stop) continue;
    const AttentionSegment seg = attention_segment(p, line, (int)b, stop - 1, line.end);
    const uint32_t tile_begin = stop - 1 - seg.first, tile_end = tile_begin + seg.of;
    if (!seg.it.live || tile_begin < begin || tile_end <= stop) continue;
    const int segments = (int)((tile_end - 1) / line.quota) - part + 1;
    for (int s = 0; s < segments && threadIdx.x == 0; ++s)
      printf("join %d %d %d %d %d %lld\n", seg.it.seq.q0, seg.it.seq.nq, seg.it.tile, seg.it.head_block, segments,
             (long long)(2 * ((int64_t)b + line.xcds * s) + (s == 0)));
  }
}
// n int64, between two pages that cannot be read, at the end of the room or at its start.
static int64_t* fenced(long n, bool at_end) {
  const size_t page = 4096, bytes = n * 8, room = (bytes + page - 1) / page * page + page;
  char* m = (char*)mmap(nullptr, room + 2 * page, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
  mprotect(m + page, room, PROT_READ | PROT_WRITE);
  return (int64_t*)(at_end ? m + page + room - bytes : m + page);
}
static int64_t* vector(long n, bool at_end) {
  int64_t* v = fenced(n, at_end);
  for (long i = 0; i < n; ++i) {
    long long x;
    if (scanf("%lld", &x) != 1) exit(4);
    v[i] = x;
  }
  return v;
}
int main() {
  int tokens, keys, heads, group, dim, causal, lengths, at_end;
  long long batch;
  while (scanf("%d %d %lld %d %d %d %d %d %d", &tokens, &keys, &batch, &heads, &group, &dim, &causal, &lengths, &at_end) == 9) {
    p = AttentionParams{};
    p.tokens = tokens, p.keys = keys, p.batch = batch, p.heads = heads, p.group = group, p.dim = dim, p.causal = causal;
    p.q_offsets = vector(batch + 1, at_end);
    if (lengths || batch) p.k_offsets = vector(lengths ? batch : batch + 1, at_end);
    if (lengths) p.k_lengths = vector(batch, at_end);
    plan = attention_plan(p);
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


def build(folder):
    (folder / "hip").mkdir()
    (folder / "hip" / "hip_runtime.h").write_text(HIP)
    (folder / "schedule.cpp").write_text(PROGRAM)
    for name in ("common.h", "attention.h", "attention_params.h", "attention_plan.h"):
        # Inline assembly (which the schedule does not reach) without the register that the host lacks.
        (folder / name).write_text((CSRC / name).read_text().replace(': "m0")', ': "memory")'))
    program = folder / "schedule"
    subprocess.run([str(COMPILER), "-std=c++20", "-O2", "-w", "-U_FORTIFY_SOURCE", "-D_FORTIFY_SOURCE=0", f"-I{folder}",
                    str(folder / "schedule.cpp"), "-o", str(program)], check=True)
    return program


def run(program, calls):
    """``calls``: (tokens, keys, heads, group, dim, causal, q_offsets, k_offsets, k_lengths or None).  For each the
    plan, what its workgroups take, and what the join reads, as tuples of int."""
    text = []
    for i, (tokens, keys, heads, group, dim, causal, qo, ko, kl) in enumerate(calls):
        text.append(f"{tokens} {keys} {len(qo) - 1} {heads} {group} {dim} {int(causal)} {int(kl is not None)} {i % 2}")
        text += [" ".join(map(str, v)) for v in (qo, ko if kl is not None or len(qo) > 1 else [], kl or [])]
    done = subprocess.run([str(program)], input="\n".join(text), capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, f"{done.returncode}: {done.stdout[-300:]}"
    out = []
    for line in done.stdout.splitlines():
        kind, *values = line.split()
        values = tuple(map(int, values))
        if kind == "plan":
            out.append((values, [], []))
        elif kind != "end":
            out[-1][1 if kind == "rows" else 2].append(values)
    assert len(out) == len(calls)
    return out
