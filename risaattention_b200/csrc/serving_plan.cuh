// How the work of a step is divided among the CTAs of a launch.  Lengths live on the device, so every CTA
// computes the division itself: the units (sequence, key head, block of query rows) with their key steps,
// laid end to end, form one line, and worker c of n takes [W c / n, W (c + 1) / n) of it.  A unit that a
// border cuts is finished by several workers, each leaving a partial result in a slot of its own; a second
// launch joins them in order.  Equal shares whatever the lengths, at most two partial results per worker,
// and the same division (so the same bits) every time.
#pragma once
#include "serving.cuh"

namespace risa_b200 {
namespace serving {

struct LineArgs {
  StepView step;
  int kv_heads;
  Divisor group;           // query heads per key head
  Divisor rows;            // query rows of a block
  int min_rows, max_rows;  // sequences with fewer or more query rows per key head belong to another launch
  Divisor keys;            // keys of a step
  int causal, window;
};

// Steps [first, first + count) of a block.
struct StepRange {
  int first, count;
};
// How many blocks a sequence has per key head (0: nothing to do).  The functions of a line that know what its
// blocks and steps are: blocks_of and steps_of; here blocks of query rows and steps of keys.
__device__ __forceinline__ int blocks_of(const LineArgs& a, const Sequence& q) {
  const int rows = q.count * a.group;
  if (rows == 0 || rows < a.min_rows || rows > a.max_rows) return 0;
  return rows <= a.rows ? 1 : (rows + a.rows - 1) / a.rows;
}
// The key steps with a key that one of the block's rows sees, at least one.
__device__ __forceinline__ StepRange steps_of(const LineArgs& a, const Sequence& q, int block) {
  const int rows = q.count * a.group, row0 = block * a.rows;
  const int token0 = row0 / a.group, token1 = (row0 + min(a.rows.value, rows - row0) - 1) / a.group;
  const KeyRange oldest = visible(q.length - q.count + token0, q.length, a.causal, a.window);
  const KeyRange newest = visible(q.length - q.count + token1, q.length, a.causal, a.window);
  const int first = oldest.lo / a.keys, end = (newest.hi + a.keys - 1) / a.keys;
  return {first, max(end - first, 1)};
}

// Quotients of numbers that are rarely past 32 bits (a 64-bit division is some hundred instructions).
__device__ __forceinline__ int64_t quotient(int64_t n, int64_t d) {
  return ((n | d) >> 32) == 0 ? int64_t(uint32_t(n) / uint32_t(d)) : n / d;
}
// Border of worker c on a line of w steps, and the first worker whose border is not in front of step `at`.
__device__ __forceinline__ int64_t border(int64_t w, int c, int workers) { return quotient(w * c, workers); }
__device__ __forceinline__ int worker_from(int64_t w, int64_t at, int workers) { return int(quotient(at * workers + w - 1, w)); }
__device__ __forceinline__ int workers_of(int64_t w, int most, int min_steps) {
  return int(min(int64_t(most), quotient(w + min_steps - 1, min_steps)));
}

// Steps of one key head's blocks: one thread's sum, or a warp's (the same in every lane).
template <typename L>
__device__ __forceinline__ int64_t head_steps(const L& a, const Sequence& q) {
  const int blocks = blocks_of(a, q);
  int64_t sum = 0;
  for (int b = 0; b < blocks; ++b) sum += steps_of(a, q, b).count;
  return sum;
}
template <typename L>
__device__ __forceinline__ int64_t head_steps_of_warp(const L& a, const Sequence& q) {
  const int blocks = blocks_of(a, q);
  int64_t sum = 0;
  for (int b = threadIdx.x & 31; b < blocks; b += 32) sum += steps_of(a, q, b).count;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  return sum;
}

// Whole-block sums for blocks of NT threads (NT a multiple of 32, at most 1024).
template <int NT>
struct BlockScan {
  int64_t warp_sums[NT / 32];
};
template <int NT>
__device__ __forceinline__ int64_t block_inclusive_scan(int64_t v, BlockScan<NT>& s, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t below = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += below;
  }
  __syncthreads();  // an earlier scan's sums are read
  if (lane == 31) s.warp_sums[warp] = v;
  __syncthreads();
  total = 0;
  int64_t before = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    if (w == warp) before = total;
    total += s.warp_sums[w];
  }
  return v + before;
}

// A step of the line: its unit and how many of the unit's steps lie in front of it.
struct Place {
  int sequence, head, block, inside;
};
template <int NT>
struct LineShared {
  BlockScan<NT> scan;
  int64_t steps[NT / 32];
  int sequence;
  int64_t offset, per_head;
};

// Few sequences may have many blocks each: a warp adds up one of them.  Many sequences: a thread each.
template <int NT, typename L>
__device__ __forceinline__ int64_t line_total(const L& a, LineShared<NT>& s) {
  const int warp = threadIdx.x >> 5;
  int64_t sum = 0, total;
  if (a.step.batch <= NT / 32) {
    const int64_t steps = warp < a.step.batch ? head_steps_of_warp(a, sequence_of(a.step, warp)) : 0;
    if ((threadIdx.x & 31) == 0) {
      s.steps[warp] = steps;
      sum = steps * a.kv_heads;
    }
  } else {
    for (int i = threadIdx.x; i < a.step.batch; i += NT) sum += head_steps(a, sequence_of(a.step, i)) * a.kv_heads;
  }
  block_inclusive_scan<NT>(sum, s.scan, total);
  return total;
}

// Where step `at` (inside the line) lies; every thread of the block calls it, after line_total.
template <int NT, typename L>
__device__ __forceinline__ Place line_place(const L& a, int64_t at, LineShared<NT>& s) {
  int64_t base = 0;
  if (a.step.batch <= NT / 32) {
    int i = 0;
    for (; i + 1 < a.step.batch; ++i) {
      const int64_t w = s.steps[i] * a.kv_heads;
      if (at < base + w) break;
      base += w;
    }
    if (threadIdx.x == 0) {
      s.sequence = i;
      s.offset = at - base;
      s.per_head = s.steps[i];
    }
  } else {
    for (int i0 = 0; i0 < a.step.batch; i0 += NT) {
      const int i = i0 + threadIdx.x;
      const int64_t per_head = i < a.step.batch ? head_steps(a, sequence_of(a.step, i)) : 0;
      int64_t total;
      const int64_t w = per_head * a.kv_heads, through = base + block_inclusive_scan<NT>(w, s.scan, total);
      if (through - w <= at && at < through) {
        s.sequence = i;
        s.offset = at - (through - w);
        s.per_head = per_head;
      }
      base += total;
      if (base > at) break;
    }
  }
  __syncthreads();
  Place p{s.sequence, int(quotient(s.offset, s.per_head)), 0, 0};
  int64_t rest = s.offset - p.head * s.per_head;
  const Sequence q = sequence_of(a.step, p.sequence);
  const int blocks = blocks_of(a, q), lane = threadIdx.x & 31;
  for (;; p.block += 32) {  // 32 blocks at a time; every warp by itself
    const int b = p.block + lane, count = b < blocks ? steps_of(a, q, b).count : 0;
    int64_t through = count;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t below = __shfl_up_sync(0xffffffffu, through, off);
      if (lane >= off) through += below;
    }
    const unsigned int behind = __ballot_sync(0xffffffffu, rest < through);
    if (behind != 0) {
      const int first = __ffs(behind) - 1;
      p.block += first;
      p.inside = int(rest - __shfl_sync(0xffffffffu, through - count, first));
      break;
    }
    rest -= __shfl_sync(0xffffffffu, through, 31);
  }
  __syncthreads();  // the shared words may be written again
  return p;
}


// What a worker does next: steps [first, first + count) of one block; whole: all of the block's, opens: its
// first ones.
struct Piece {
  Sequence seq;
  int sequence, head, block;
  int first, count;
  bool whole, opens;
};
// Walks the pieces of one worker; every role of a CTA keeps a walk of its own.
struct Pieces {
  int64_t left;  // steps to go
  Place at;
  template <typename L>
  __device__ __forceinline__ bool next(const L& a, Piece& p) {
    if (left <= 0) return false;
    p.seq = sequence_of(a.step, at.sequence);
    int blocks = blocks_of(a, p.seq);
    while (at.block >= blocks) {
      at.block = 0;
      if (blocks == 0 || ++at.head == a.kv_heads) {
        at.head = 0;
        ++at.sequence;  // the line has steps left, so a sequence with work follows
        p.seq = sequence_of(a.step, at.sequence);
        blocks = blocks_of(a, p.seq);
      }
    }
    const StepRange range = steps_of(a, p.seq, at.block);
    p.sequence = at.sequence;
    p.head = at.head;
    p.block = at.block;
    p.first = range.first + at.inside;
    p.count = int(min(int64_t(range.count - at.inside), left));
    p.opens = at.inside == 0;
    p.whole = p.count == range.count;
    left -= p.count;
    at.inside += p.count;
    if (at.inside == range.count) {
      at.inside = 0;
      ++at.block;
    }
    return true;
  }
};

// ---- joining the parts of a cut unit ------------------------------------------------------------------------
// A slot holds a part's unnormalised output [rows][head_dim], its maxima [rows] (in units of log 2) and its sums
// [rows].  A worker's first slot takes a part of a unit that began before it, its second a unit's first part.
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Where a running maximum starts: below every score (in units of log 2) that 16-bit operands of use produce,
// and finite, so that a row that has seen nothing yet needs no case of its own.
constexpr float kNoMaximum = -1e30f;

__host__ __device__ __forceinline__ int64_t slot_floats(int rows, int head_dim) { return int64_t(rows) * (head_dim + 2); }
// What a worker leaves for the join: the unit whose first part it ended with, and over how many workers that unit goes
// (parts 0: it ended with a whole unit, or inside one that began before it).  Every CTA of a launch writes one.
struct JoinNote {
  int first_token, rows, head, block, parts, sequence;
};

struct JoinArgs {
  const float* parts;
  const JoinNote* notes;
  int unit_rows;
  Divisor group;
  int heads;
  void* out;
  int64_t on, oh;
  float* lse;
};

// Written once the walk over the pieces has come to its end (`at` behind the last step, `done` the last piece).
__device__ __forceinline__ JoinNote join_note(const LineArgs& a, const Piece& last, int64_t total, int64_t end, int worker, int workers) {
  if (!last.opens || last.whole) return {0, 0, 0, 0, 0, 0};
  const int64_t unit_end = end - last.count + steps_of(a, last.seq, last.block).count;
  return {last.seq.first, last.seq.count * a.group, last.head, last.block, min(worker_from(total, unit_end, workers), workers) - worker, last.sequence};
}

// Worker c's unit (grid x) is joined from the second slot of c and the first slots of those behind it, in the order of
// their keys, so that results do not depend on which worker ended first.  MANY: units of few rows and up to a hundred
// parts; a CTA joins one row (grid y), its warps a quarter of the parts each.  Else few parts: a warp joins four rows.
template <typename T, int D, bool MANY>
__global__ __launch_bounds__(128) void join_parts_kernel(const JoinArgs a) {
  __shared__ float tops[4], norms[4], sums[MANY ? 4 : 1][D];
  chain_wait();
  chain_release();
  const JoinNote note = a.notes[blockIdx.x];
  if (note.parts == 0) return;
  const int c = blockIdx.x, R = a.unit_rows, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t slot = slot_floats(R, D);
  auto slot_of = [&](int i) { return a.parts + (int64_t(c + i) * 2 + (i == 0 ? 1 : 0)) * slot; };
  constexpr int PER = D / 32;
  // this warp's share of one row's parts [from, to)
  auto add = [&](int r, int from, int to, float& top, float& norm, float (&sum)[PER]) {
    top = kNoMaximum;
    for (int i = from + lane; i < to; i += 32) top = fmaxf(top, slot_of(i)[R * D + r]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    norm = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) sum[e] = 0.f;
#pragma unroll(MANY ? 8 : 2)
    for (int i = from; i < to; ++i) {
      const float* s = slot_of(i);
      const float f = ex2_approx(s[R * D + r] - top);
      norm += f * s[R * D + R + r];
#pragma unroll
      for (int e = 0; e < PER / 2; ++e) {
        const float2 x = *reinterpret_cast<const float2*>(s + r * D + e * 64 + lane * 2);
        sum[2 * e] += f * x.x;
        sum[2 * e + 1] += f * x.y;
      }
    }
  };
  auto write = [&](int row, float top, float norm, const float (&sum)[PER]) {
    const float f = norm == 0.f ? 0.f : 1.0f / norm;
    const int token = row / a.group, h = note.head * a.group + row - token * a.group;
    T* out = static_cast<T*>(a.out) + int64_t(note.first_token + token) * a.on + int64_t(h) * a.oh;
#pragma unroll
    for (int e = 0; e < PER / 2; ++e)
      *reinterpret_cast<uint32_t*>(out + e * 64 + lane * 2) = Half2<T>::pack(sum[2 * e] * f, sum[2 * e + 1] * f);
    if (lane == 0 && a.lse != nullptr)
      a.lse[int64_t(note.first_token + token) * a.heads + h] = norm == 0.f ? -INFINITY : top * kLn2 + logf(norm);
  };
  float top, norm, sum[PER];
  if (MANY) {
    const int r = blockIdx.y, row = note.block * R + r;
    if (row >= note.rows) return;
    add(r, note.parts * warp / 4, note.parts * (warp + 1) / 4, top, norm, sum);
    if (lane == 0) {
      tops[warp] = top;
      norms[warp] = norm;
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) sums[warp][e * 32 + lane] = sum[e];
    __syncthreads();
    if (warp != 0) return;
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    norm = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) sum[e] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = ex2_approx(tops[w] - top);
      norm += f * norms[w];
#pragma unroll
      for (int e = 0; e < PER; ++e) sum[e] += f * sums[w][e * 32 + lane];
    }
    write(row, top, norm, sum);
  } else {
    for (int i = 0; i < 4; ++i) {
      const int r = (blockIdx.y * 4 + warp) * 4 + i, row = note.block * R + r;
      if (row >= note.rows) return;
      add(r, 0, note.parts, top, norm, sum);
      write(row, top, norm, sum);
    }
  }
}

}  // namespace serving
}  // namespace risa_b200
