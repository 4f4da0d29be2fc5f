// How the work of a step is divided among the CTAs of a launch.  Lengths live on the device, so every CTA
// computes the division itself from the lengths of all sequences: the units of a sequence (key head x
// block of query rows) hold equally many key steps, all steps of all units in their order form one line, and
// worker c of n takes [W c / n, W (c + 1) / n) of it.  A unit that a border cuts is finished by several
// workers, each leaving a partial result in a slot of its own; a second launch joins them in order.
#pragma once
#include "serving.cuh"

namespace risa_b200 {
namespace serving {

struct LineArgs {
  StepView step;
  int kv_heads, group;  // query heads per key head
  int rows;             // query rows of a unit
  int max_rows;         // sequences with more query rows per key head belong to another launch (0: none do)
  int keys;             // keys of a step
  int causal, window;
};

// One sequence's share of the line.
struct Share {
  int blocks;      // blocks of query rows per key head (0: nothing to do)
  int first_step;  // key step where its units start
  int steps;       // steps of each unit
};
__device__ __forceinline__ Share share_of(const LineArgs& a, const Sequence& q) {
  const int rows = q.count * a.group;
  if (rows == 0 || (a.max_rows > 0 && rows > a.max_rows)) return {0, 0, 0};
  // the first new token sees the oldest keys
  const int lo = a.window > 0 ? visible(q.length - q.count, q.length, true, a.window).lo : 0;
  const int first = lo / a.keys, end = (q.length + a.keys - 1) / a.keys;
  return {(rows + a.rows - 1) / a.rows, first, max(end - first, 1)};
}
__device__ __forceinline__ int64_t work_of(const LineArgs& a, const Share& h) {
  return int64_t(h.blocks) * a.kv_heads * h.steps;
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

template <int NT>
__device__ __forceinline__ int64_t line_total(const LineArgs& a, BlockScan<NT>& s) {
  int64_t sum = 0, total;
  for (int i = threadIdx.x; i < a.step.batch; i += NT) sum += work_of(a, share_of(a, sequence_of(a.step, i)));
  block_inclusive_scan<NT>(sum, s, total);
  return total;
}

// Where `at` (inside the line) lies: its sequence and the distance from where that sequence starts.
struct Place {
  int sequence;
  int64_t offset;
};
template <int NT>
__device__ __forceinline__ Place line_place(const LineArgs& a, int64_t at, BlockScan<NT>& s, Place& shared) {
  int64_t base = 0;
  for (int i0 = 0; i0 < a.step.batch; i0 += NT) {
    const int i = i0 + threadIdx.x;
    const int64_t w = i < a.step.batch ? work_of(a, share_of(a, sequence_of(a.step, i))) : 0;
    int64_t total;
    const int64_t through = base + block_inclusive_scan<NT>(w, s, total);
    if (through - w <= at && at < through) shared = {i, at - (through - w)};
    base += total;
    if (base > at) break;
  }
  __syncthreads();
  return shared;
}

// Border of worker c on a line of w steps.
__device__ __forceinline__ int64_t border(int64_t w, int c, int workers) { return w * c / workers; }

}  // namespace serving
}  // namespace risa_b200
