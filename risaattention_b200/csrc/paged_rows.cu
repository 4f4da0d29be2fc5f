// Attention of few query rows over a paged cache (single tokens, chunks of few tokens), the join of its partial
// results, and the attention weight that cached keys receive from few rows.
//
// What bounds it is reading the cache once: 2 * keys * head_dim values per key head for a handful of
// query rows.  So a warp works alone on steps of 16 keys: it fetches them with cp.async through a ring of
// its own (no barrier between warps, several KB in flight per warp), forms scores as K Q^T with the keys as
// the 16 rows of the matrix instruction and up to 8 query rows as its columns (no padding for groups of 8
// heads), keeps running maximum, sum and output in registers, and adds V^T P^T in the same orientation.
// Codes become fp16 in registers on the way to the matrix instruction (whole numbers up to 128 are exact, and fp16 takes
// half the instructions of bf16), so K's scale multiplies the score and V's the probability, both in 32 bits.  Queries
// in bf16 become fp16 too, their row multiplied by a power of two that brings its largest value to 2^14: nothing is lost
// but what is 2^-38 of that value.  Probability times scale fits fp16 because the running maximum is not that of the
// scores s but of s + log2(scale): what is rounded is at most 1, and exact relative to the largest contribution.
//
// Measured: 16 requests of up to 16K keys, 8 key heads of 128 bf16 channels, 110 us (6.1 TB/s, 95 % of a plain copy's rate);
// 32 requests of up to 32K keys as codes 244 us at full clocks (5.7 TB/s), 280 in long runs, where the conversion's
// instructions (schedulers 61 % busy) feel the lower clock.
#include "paged_tc.cuh"
#include "serving_plan.cuh"

#include <climits>
#include <type_traits>

namespace risa_b200 {
namespace serving {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
struct RowsArgs {
  LineArgs line;
  const void* q;
  int64_t qn, qh;
  void* out;
  int64_t on, oh;
  float* lse;
  const char* keys;
  const char* values;
  const float* key_scales;
  const float* value_scales;
  int pages;
  float scale_log2;
  int clear_rest;
  float* parts;   // two slots per worker: of a unit that began before it, of one that goes on after it
  JoinNote* notes;
  int min_steps;  // fewest steps that make a worker worth its share of the join
  unsigned int* status;
  // key weights only
  const float* row_lse;
  const float* previous;
  float* weights;
};

template <typename T_, bool INT8_, int D_, int NT_>
struct Tile {
  using T = T_;
  static constexpr bool INT8 = INT8_;
  static constexpr int D = D_, NT = NT_, R = 8 * NT_;
  using M = std::conditional_t<INT8_, __half, T_>;  // type of the matrix instructions' operands
  static constexpr int ROW = D * (INT8 ? 1 : 2);  // bytes of a key
  static constexpr int CHUNKS = ROW / 16;
  static constexpr int SIDE = 16 * ROW;  // the 16 keys (or values) of a step
  static constexpr int SCALES = INT8 ? 128 : 0;
  static constexpr int KS = D / 16;
  // CTAs of four warps that share an SM's shared memory: what hides the latency of HBM is bytes in flight, 96 KB or
  // more per SM.  Codes, whose conversion keeps the schedulers busy, gain from a third CTA (32 requests of up to 32K
  // keys: 280 us with two, 247 with three, 267 with four); 16-bit rows of 256 channels leave room for one.
  static constexpr int CTAS = D == 256 && !INT8 ? 1 : INT8 && D <= 128 && NT == 1 ? 3 : 2;
  static constexpr int BUDGET = 48 * 1024 / CTAS;  // per warp
  __host__ __device__ static constexpr int stages(int sides) {
    const int n = BUDGET / (sides * SIDE + SCALES);
    return n > 8 ? 8 : n;
  }
};

// 16-byte pieces of a row are permuted so that the reads below are free of bank conflicts.  16-bit rows:
// ldmatrix takes one piece of eight consecutive rows.  Codes: for K eight lanes read four pieces of two
// consecutive rows, for V two pieces of every other row.
template <typename C>
__device__ __forceinline__ int swizzled(int row, int piece) {
  if (!C::INT8) return piece ^ (row & 7);
  if (C::CHUNKS < 8) return piece;
  return piece ^ (((row & 1) << 2) ^ (((row >> 1) & 3) << 1));
}

__device__ __forceinline__ uint32_t shared_address(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldmatrix4(uint32_t* r, uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ void ldmatrix4_transposed(uint32_t* r, uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ uint32_t transposed8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint4 read16(uint32_t address) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(address) : "memory");
  return v;
}
__device__ __forceinline__ uint2 read8(uint32_t address) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(address) : "memory");
  return v;
}
__device__ __forceinline__ float read_float(uint32_t address) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(address) : "memory");
  return v;
}

// Codes as fp16: 0x6400 + u is 1024 + u, so (code + 128 as u) less 1152 is the code.  Bytes 2 i and 2 i + 1 of a word whose
// sign bits have been flipped; or two codes in the low bytes of the halves of a word (the high bytes are ignored).
__device__ __forceinline__ uint32_t less_1152(uint32_t u) {
  const uint32_t bias = 0x64806480u;
  const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&u), *reinterpret_cast<const __half2*>(&bias));
  return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ uint32_t pair_of_flipped(uint32_t word, int i) { return less_1152(__byte_perm(word, 0x64646464u, i ? 0x4342 : 0x4140)); }
__device__ __forceinline__ uint32_t pair_of_halves(uint32_t pair) { return less_1152((pair & 0x00ff00ffu) ^ 0x64806480u); }

// ---- a warp's walk over its steps -----------------------------------------------------------------------
// Steps first, first + kWarps, ... of one unit.  Page numbers are looked up 32 steps at a time, one set
// ahead; a page outside the pool is not read (its keys are hidden and the status word says so).
template <typename C, bool WITH_VALUES>
struct Walk {
  const RowsArgs& a;
  const int32_t* row;  // the sequence's row of the page table
  int head, first_key, low, length, count, sequence;
  int pages, pages_ahead;
  uint32_t base;
  unsigned int hidden;  // one bit per stage
  static constexpr int STAGES = C::stages(WITH_VALUES ? 2 : 1);
  static constexpr int STAGE = (WITH_VALUES ? 2 : 1) * C::SIDE + C::SCALES;
  static_assert(STAGES >= 2 && STAGES <= 32, "ring");

  __device__ __forceinline__ int key_of(int i) const { return first_key + i * (16 * kWarps); }
  __device__ __forceinline__ int look_up(int i) const {
    const int key = key_of(i);
    return i < count && key < length ? __ldg(row + (key >> a.line.step.page_shift)) : -1;
  }
  __device__ __forceinline__ void start() {
    const int lane = threadIdx.x & 31;
    pages = look_up(lane);
    pages_ahead = look_up(32 + lane);
    hidden = 0;
  }
  // Fetches step i into stage i % STAGES (its stage number is given) and closes a copy group either way.
  __device__ __forceinline__ void fetch(int i, int stage) {
    if (i < count) {
      if ((i & 31) == 0 && i > 0) {
        pages = pages_ahead;
        pages_ahead = look_up(i + 32 + (threadIdx.x & 31));
      }
      const int lane = threadIdx.x & 31, key = key_of(i);
      const int page = __shfl_sync(0xffffffffu, pages, i & 31);
      const bool good = key < length && page >= 0 && page < a.pages;
      if (key < length && !good && lane == 0) atomicCAS(a.status, 0u, unsigned(sequence) + 1u);
      hidden = good ? hidden & ~(1u << stage) : hidden | (1u << stage);
      const int64_t line = good ? (((int64_t(page) * a.line.kv_heads + head) << a.line.step.page_shift) +
                                   (key & ((1 << a.line.step.page_shift) - 1)))
                                : 0;
      const char* k = a.keys + line * C::ROW;
      const char* v = a.values + line * C::ROW;
      const uint32_t to = base + stage * STAGE;
#pragma unroll
      for (int j = 0; j < C::CHUNKS / 2; ++j) {
        const int index = j * 32 + lane, r = index / C::CHUNKS, piece = index % C::CHUNKS;
        const bool there = good && key + r < length && key + r >= low;
        const uint32_t at = to + r * C::ROW + swizzled<C>(r, piece) * 16;
        copy16(at, k + index * 16, there);
        if (WITH_VALUES) copy16(at + C::SIDE, v + index * 16, there);
      }
      if (C::INT8) {
        const float* s = lane < 16 ? a.key_scales : a.value_scales;
        const int r = lane & 15;
        copy4(to + (WITH_VALUES ? 2 : 1) * C::SIDE + lane * 4, s + line + r, good && key + r < length && key + r >= low);
      }
    }
    copies_commit();
  }
};

// Query rows as the B operand: [nt][ks][2].  With codes the channels of a 64-channel run are dealt so that
// a lane's 16 bytes of K serve four instructions: instruction 4 b + j takes channels 64 b + 16 t + 4 j ..
// + 3 from lane t; the sum over channels does not mind the order.
// factor: what multiplies the scores of rows 2 t and 2 t + 1 (the softmax scale in units of log 2, and the row's own).
template <typename C>
__device__ __forceinline__ void load_queries(const RowsArgs& a, const Sequence& seq, int head, int row0, int rows, uint32_t (&qf)[C::NT][C::KS][2],
                                             float (&factor)[C::NT][2]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < C::NT; ++nt) {
    const int r = row0 + nt * 8 + g;
    const bool there = r < rows;
    const int token = there ? r / a.line.group : 0, h = there ? r - token * a.line.group : 0;
    const typename C::T* q = static_cast<const typename C::T*>(a.q) + int64_t(seq.first + token) * a.qn +
                             int64_t(head * a.line.group + h) * a.qh;
#pragma unroll
    for (int ks = 0; ks < C::KS; ++ks) {
      const int c0 = C::INT8 ? (ks >> 2) * 64 + t * 16 + (ks & 3) * 4 : ks * 16 + t * 2;
      const int c1 = C::INT8 ? c0 + 2 : c0 + 8;
      qf[nt][ks][0] = there ? *reinterpret_cast<const uint32_t*>(q + c0) : 0u;
      qf[nt][ks][1] = there ? *reinterpret_cast<const uint32_t*>(q + c1) : 0u;
    }
    factor[nt][0] = factor[nt][1] = a.scale_log2;
    if constexpr (C::INT8 && std::is_same<typename C::T, __nv_bfloat16>::value) {
      uint32_t most = 0;  // bits of the largest magnitude
#pragma unroll
      for (int ks = 0; ks < C::KS; ++ks)
#pragma unroll
        for (int i = 0; i < 2; ++i) most = max(most, max((qf[nt][ks][i] & 0x7fffu) << 16, qf[nt][ks][i] & 0x7fff0000u));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // exponent e of the largest value: the row times 2^(14 - e), an infinity or a NaN stays one
      const int e = most == 0 ? 14 : min(max(int(most >> 23) - 127, -112), 126);
      const float up = __uint_as_float(uint32_t(127 + 14 - e) << 23), down = __uint_as_float(uint32_t(127 - 14 + e) << 23);
#pragma unroll
      for (int ks = 0; ks < C::KS; ++ks)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 x = Half2<__nv_bfloat16>::unpack(qf[nt][ks][i]);
          qf[nt][ks][i] = Half2<__half>::pack(x.x * up, x.y * up);
        }
      factor[nt][0] *= __shfl_sync(0xffffffffu, down, 8 * t);
      factor[nt][1] *= __shfl_sync(0xffffffffu, down, 8 * t + 4);
    }
  }
}

// acc[nt]: raw scores of keys g and g + 8 against query rows 2 t and 2 t + 1 (of column block nt).
template <typename C>
__device__ __forceinline__ void score_step(uint32_t keys, const uint32_t (&qf)[C::NT][C::KS][2], float (&acc)[C::NT][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[nt][i] = 0.f;
  if constexpr (C::INT8) {
#pragma unroll
    for (int b = 0; b < C::D / 64; ++b) {
      const uint4 lo = read16(keys + g * C::ROW + swizzled<C>(g, b * 4 + t) * 16);
      const uint4 hi = read16(keys + (g + 8) * C::ROW + swizzled<C>(g + 8, b * 4 + t) * 16);
      const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t l = wl[j] ^ 0x80808080u, h = wh[j] ^ 0x80808080u;
        const uint32_t af[4] = {pair_of_flipped(l, 0), pair_of_flipped(h, 0), pair_of_flipped(l, 1), pair_of_flipped(h, 1)};
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) mma16816<__half>(acc[nt], af, qf[nt][b * 4 + j]);
      }
    }
  } else {
    const int r = lane & 15;
#pragma unroll
    for (int ks = 0; ks < C::KS; ++ks) {
      uint32_t af[4];
      ldmatrix4(af, keys + r * C::ROW + swizzled<C>(r, 2 * ks + (lane >> 4)) * 16);
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt) mma16816<typename C::T>(acc[nt], af, qf[nt][ks]);
    }
  }
}

// out[nt][mt] += V^T P^T.  16-bit values: block mt holds channels 16 mt + g (and + 8).  Codes: a lane takes
// the channels of its own 16-byte pieces (8 bytes at 64 channels), two per instruction: see channel_of.
template <typename C>
__device__ __forceinline__ void value_step(uint32_t values, const uint32_t (&p)[C::NT][2], float (&out)[C::NT][C::D / 16][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if constexpr (C::INT8) {
    constexpr int RUNS = C::D == 256 ? 2 : 1, WORDS = C::D == 64 ? 2 : 4;
#pragma unroll
    for (int run = 0; run < RUNS; ++run) {
      uint32_t w[4][WORDS];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 2 * t + (i & 1) + (i >> 1) * 8;
        if constexpr (WORDS == 4) {
          const uint4 v = read16(values + key * C::ROW + swizzled<C>(key, g + 8 * run) * 16);
          w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
        } else {
          const uint2 v = read8(values + key * C::ROW + g * 8);
          w[i][0] = v.x; w[i][1] = v.y;
        }
      }
#pragma unroll
      for (int j = 0; j < WORDS; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // channels 4 j + 2 e and + 1 of the run
          const int lo = e ? 0x4642 : 0x4440, hi = e ? 0x4743 : 0x4541;
          const uint32_t af[4] = {pair_of_halves(__byte_perm(w[0][j], w[1][j], lo)), pair_of_halves(__byte_perm(w[0][j], w[1][j], hi)),
                                  pair_of_halves(__byte_perm(w[2][j], w[3][j], lo)), pair_of_halves(__byte_perm(w[2][j], w[3][j], hi))};
#pragma unroll
          for (int nt = 0; nt < C::NT; ++nt) mma16816<__half>(out[nt][run * 8 + j * 2 + e], af, p[nt]);
        }
    }
  } else {
    const int r = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
    for (int mt = 0; mt < C::D / 16; ++mt) {
      uint32_t af[4];
      ldmatrix4_transposed(af, values + r * C::ROW + swizzled<C>(r, 2 * mt + ((lane >> 3) & 1)) * 16);
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt) mma16816<typename C::T>(out[nt][mt], af, p[nt]);
    }
  }
}
template <typename C>
__device__ __forceinline__ int channel_of(int mt, int second) {
  const int g = (threadIdx.x & 31) >> 2;
  if (!C::INT8) return mt * 16 + g + second * 8;
  if (C::D == 64) return g * 8 + 2 * mt + second;
  return (g + 8 * (mt >> 3)) * 16 + 2 * (mt & 7) + second;
}

// ---- attention --------------------------------------------------------------------------------------------
template <typename C>
__global__ __launch_bounds__(kThreads, C::CTAS) void paged_rows_kernel(const RowsArgs a) {
  extern __shared__ __align__(128) char smem[];
  __shared__ LineShared<kThreads> shared;
  __shared__ float warp_max[kWarps][C::R], warp_sum[kWarps][C::R];
  using T = typename C::T;
  using W = Walk<C, true>;
  constexpr int D = C::D, NT = C::NT, R = C::R, MT = D / 16;
  constexpr int kRowStride = D + 4;  // of the output in shared memory: lanes t lie 8 banks apart
  static_assert(R * kRowStride * 4 <= W::STAGE * W::STAGES, "a warp's output fits its ring");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = shared_address(smem) + warp * (W::STAGE * W::STAGES);
  chain_wait();
  chain_release();
  if (a.clear_rest && a.line.step.offsets != nullptr) {
    const int heads = a.line.kv_heads * a.line.group, tokens = a.line.step.tokens;
    // tokens in front of the first sequence, then those behind the last
    const int front = min(max(__ldg(a.line.step.offsets), 0), tokens), back = max(__ldg(a.line.step.offsets + a.line.step.batch), front);
    for (int n = blockIdx.x; n < front || n - front < tokens - back; n += gridDim.x) {
      const int token = n < front ? n : n - front + back;
      if (a.clear_rest & 1) for (int i = threadIdx.x; i < heads * (D / 8); i += kThreads)
        *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + token * a.on + (i / (D / 8)) * a.oh + (i % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
      if ((a.clear_rest & 2) && a.lse != nullptr)
        for (int h = threadIdx.x; h < heads; h += kThreads) a.lse[int64_t(token) * heads + h] = -INFINITY;
    }
  }
  const int64_t total = line_total<kThreads>(a.line, shared);
  const int workers = workers_of(total, gridDim.x, a.min_steps);
  if (int(blockIdx.x) >= workers) {
    if (threadIdx.x == 0) a.notes[blockIdx.x] = JoinNote{};
    return;
  }
  const int64_t begin = border(total, blockIdx.x, workers), end = border(total, blockIdx.x + 1, workers);
  Pieces pieces{end - begin, line_place<kThreads>(a.line, begin, shared)};
  Piece piece;
  while (pieces.next(a.line, piece)) {
    const Sequence seq = piece.seq;
    const int s = piece.sequence, head = piece.head, row0 = piece.block * R, rows = seq.count * a.line.group, take = piece.count;

    uint32_t qf[NT][C::KS][2];
    float factor[NT][2];
    load_queries<C>(a, seq, head, row0, rows, qf, factor);
    int lo[NT][2], hi[NT][2];  // visible keys of rows 2 t and 2 t + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = row0 + nt * 8 + 2 * t + i;
        const KeyRange v = visible(seq.length - seq.count + r / a.line.group, seq.length, a.line.causal, a.line.window);
        lo[nt][i] = v.lo;
        hi[nt][i] = r < rows ? v.hi : 0;
      }
    // keys [all_lo, all_hi) are visible to every row of the unit
    const int last_row = min(row0 + R, rows) - 1;
    const int all_hi = visible(seq.length - seq.count + row0 / a.line.group, seq.length, a.line.causal, a.line.window).hi;
    const int all_lo = visible(seq.length - seq.count + last_row / a.line.group, seq.length, a.line.causal, a.line.window).lo;
    const int low = a.line.window > 0 ? visible(seq.length - seq.count, seq.length, true, a.line.window).lo : 0;

    W walk{a, a.line.step.table + int64_t(s) * a.line.step.width, head, (piece.first + warp) * 16, low, seq.length,
           take > warp ? (take - warp + kWarps - 1) / kWarps : 0, s};
    walk.base = ring;
    walk.start();
    float m[NT][2], l[NT][2], o[NT][MT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = kNoMaximum;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][mt][i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < W::STAGES - 1; ++i) walk.fetch(i, i);
    int stage = 0;
    for (int i = 0; i < walk.count; ++i) {
      {
        const int next = stage == 0 ? W::STAGES - 1 : stage - 1;  // the stage of step i + STAGES - 1
        copies_wait<W::STAGES - 2>();
        __syncwarp();
        walk.fetch(i + W::STAGES - 1, next);
      }
      const uint32_t data = ring + stage * W::STAGE;
      const int key = walk.key_of(i);
      const bool hidden = walk.hidden >> stage & 1;
      float acc[NT][4];
      score_step<C>(data, qf, acc);
      float ks0 = 1.f, ks1 = 1.f, vs0 = 1.f, vs1 = 1.f, lift0 = 0.f, lift1 = 0.f;
      if (C::INT8) {
        ks0 = read_float(data + 2 * C::SIDE + g * 4);
        ks1 = read_float(data + 2 * C::SIDE + (g + 8) * 4);
        vs0 = read_float(data + 2 * C::SIDE + 64 + g * 4);
        vs1 = read_float(data + 2 * C::SIDE + 64 + (g + 8) * 4);
        // a row of zeros must not let its own probability overflow, nor one that is not finite let the others vanish
        lift0 = vs0 < INFINITY ? lg2_approx(fmaxf(vs0, 0x1p-100f)) : 0.f;
        lift1 = vs1 < INFINITY ? lg2_approx(fmaxf(vs1, 0x1p-100f)) : 0.f;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][e] *= C::INT8 ? (e < 2 ? ks0 : ks1) * factor[nt][e & 1] : factor[nt][e & 1];
      if (hidden || key < all_lo || key + 16 > all_hi) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = key + g + (e >> 1) * 8;
            if (hidden || k < lo[nt][e & 1] || k >= hi[nt][e & 1]) acc[nt][e] = -INFINITY;
          }
      }
      uint32_t p[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float top[2], keep[2];
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
          float x = fmaxf(acc[nt][i2] + lift0, acc[nt][2 + i2] + lift1);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          top[i2] = fmaxf(m[nt][i2], x);
        }
        const bool moved = top[0] > m[nt][0] || top[1] > m[nt][1];
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int i2 = 0; i2 < 2; ++i2) {
            keep[i2] = ex2_approx(m[nt][i2] - top[i2]);
            m[nt][i2] = top[i2];
            l[nt][i2] *= keep[i2];
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            o[nt][mt][0] *= keep[0];
            o[nt][mt][1] *= keep[1];
            o[nt][mt][2] *= keep[0];
            o[nt][mt][3] *= keep[1];
          }
        }
        float e[4];
#pragma unroll
        for (int i2 = 0; i2 < 4; ++i2) e[i2] = ex2_approx(acc[nt][i2] - m[nt][i2 & 1]);
        l[nt][0] += e[0] + e[2];
        l[nt][1] += e[1] + e[3];
        // Probabilities (times scales) leave 32 bits here: half a step, 2^-8 of the value in bf16, 2^-11 in fp16.
        p[nt][0] = transposed8x8(Half2<typename C::M>::pack(C::INT8 ? e[0] * vs0 : e[0], C::INT8 ? e[1] * vs0 : e[1]));
        p[nt][1] = transposed8x8(Half2<typename C::M>::pack(C::INT8 ? e[2] * vs1 : e[2], C::INT8 ? e[3] * vs1 : e[3]));
      }
      value_step<C>(data + C::SIDE, p, o);
      stage = stage + 1 == W::STAGES ? 0 : stage + 1;
    }
    copies_wait<0>();
    __syncwarp();
    // join the four warps
    float* mine = reinterpret_cast<float*>(smem + warp * (W::STAGE * W::STAGES));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = l[nt][i];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (g == 0) {
          warp_max[warp][nt * 8 + 2 * t + i] = m[nt][i];
          warp_sum[warp][nt * 8 + 2 * t + i] = x;
        }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) mine[(nt * 8 + 2 * t + (i & 1)) * kRowStride + channel_of<C>(mt, i >> 1)] = o[nt][mt][i];
    }
    __syncthreads();
    const bool whole = piece.whole;
    float* slot = whole ? nullptr : a.parts + (int64_t(blockIdx.x) * 2 + (piece.opens ? 1 : 0)) * slot_floats(R, D);
    for (int i = threadIdx.x; i < R * (D / 4); i += kThreads) {
      const int r = i / (D / 4), c = (i % (D / 4)) * 4;
      if (row0 + r >= rows) continue;
      float top = warp_max[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, warp_max[w][r]);
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      float norm = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2_approx(warp_max[w][r] - top);
        const float4 x = *reinterpret_cast<const float4*>(smem + w * (W::STAGE * W::STAGES) + (r * kRowStride + c) * 4);
        sum.x += f * x.x;
        sum.y += f * x.y;
        sum.z += f * x.z;
        sum.w += f * x.w;
        norm += f * warp_sum[w][r];
      }
      if (!whole) {
        *reinterpret_cast<float4*>(slot + r * D + c) = sum;
        if (c == 0) {
          slot[R * D + r] = top;
          slot[R * D + R + r] = norm;
        }
      } else {
        const float f = norm == 0.f ? 0.f : 1.0f / norm;
        const int token = (row0 + r) / a.line.group, h = head * a.line.group + (row0 + r) % a.line.group;
        uint2 w2;
        w2.x = Half2<T>::pack(sum.x * f, sum.y * f);
        w2.y = Half2<T>::pack(sum.z * f, sum.w * f);
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + int64_t(seq.first + token) * a.on + int64_t(h) * a.oh + c) = w2;
        if (c == 0 && a.lse != nullptr)
          a.lse[int64_t(seq.first + token) * (a.line.kv_heads * a.line.group) + h] =
              norm == 0.f ? -INFINITY : top * kLn2 + logf(norm);
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) a.notes[blockIdx.x] = join_note(a.line, piece, total, end, blockIdx.x, workers);
}

// ---- key weights -------------------------------------------------------------------------------------------
// The same walk over K alone.  A key's weight is a sum over query rows, so a unit is (sequence, key head)
// with all its rows, a warp's 16 keys are its own and nothing is joined.
template <typename C>
__global__ __launch_bounds__(kThreads, C::CTAS) void weigh_rows_kernel(const RowsArgs a) {
  extern __shared__ __align__(128) char smem[];
  __shared__ LineShared<kThreads> shared;
  using W = Walk<C, false>;
  constexpr int NT = C::NT, R = C::R;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = shared_address(smem) + warp * (W::STAGE * W::STAGES);
  const int slots = a.line.step.width << a.line.step.page_shift, heads = a.line.kv_heads * a.line.group;
  chain_wait();
  chain_release();
  // what no step covers: in front of the window, behind the length
  for (int64_t u = blockIdx.x; u < int64_t(a.line.step.batch) * a.line.kv_heads; u += gridDim.x) {
    const Sequence seq = sequence_of(a.line.step, int(u / a.line.kv_heads));
    const int rows = seq.count * a.line.group;
    if (rows > a.line.max_rows) continue;
    const StepRange range = rows == 0 ? StepRange{0, 0} : steps_of(a.line, seq, 0);
    const int from = min(range.first * 16, slots), to = min((range.first + range.count) * 16, slots);
    for (int i = threadIdx.x; i < slots - (to - from); i += kThreads) {
      const int key = i < from ? i : i + (to - from);
      a.weights[u * slots + key] = a.previous != nullptr ? a.previous[u * slots + key] : 0.f;
    }
  }
  const int64_t total = line_total<kThreads>(a.line, shared);
  const int workers = workers_of(total, gridDim.x, a.min_steps);
  if (int(blockIdx.x) >= workers) return;
  const int64_t begin = border(total, blockIdx.x, workers);
  Pieces pieces{border(total, blockIdx.x + 1, workers) - begin, line_place<kThreads>(a.line, begin, shared)};
  Piece piece;
  while (pieces.next(a.line, piece)) {
    const Sequence seq = piece.seq;
    const int s = piece.sequence, head = piece.head, rows = seq.count * a.line.group, blocks = (rows + R - 1) / R, take = piece.count;
    const int low = a.line.window > 0 ? visible(seq.length - seq.count, seq.length, true, a.line.window).lo : 0;
    W walk{a, a.line.step.table + int64_t(s) * a.line.step.width, head, (piece.first + warp) * 16, low, seq.length,
           take > warp ? (take - warp + kWarps - 1) / kWarps : 0, s};
    walk.base = ring;
    walk.start();
#pragma unroll
    for (int i = 0; i < W::STAGES - 1; ++i) walk.fetch(i, i);
    uint32_t qf[NT][C::KS][2];
    int lo[NT][2], hi[NT][2];
    float lse2[NT][2], factor[NT][2];
    auto load_block = [&](int block) {
      load_queries<C>(a, seq, head, block * R, rows, qf, factor);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = block * R + nt * 8 + 2 * t + i;
          const bool there = r < rows;
          const int token = there ? r / a.line.group : 0;
          const float x = there ? __ldg(a.row_lse + int64_t(seq.first + token) * heads + head * a.line.group + r - token * a.line.group) : -INFINITY;
          const KeyRange v = visible(seq.length - seq.count + token, seq.length, a.line.causal, a.line.window);
          lo[nt][i] = v.lo;
          hi[nt][i] = x == -INFINITY ? 0 : v.hi;  // a row that saw nothing gives nothing
          lse2[nt][i] = x == -INFINITY ? 0.f : x * kLog2e;
        }
    };
    if (blocks == 1) load_block(0);
    int stage = 0;
    for (int i = 0; i < walk.count; ++i) {
      const int next = stage == 0 ? W::STAGES - 1 : stage - 1;
      copies_wait<W::STAGES - 2>();
      __syncwarp();
      walk.fetch(i + W::STAGES - 1, next);
      const uint32_t data = ring + stage * W::STAGE;
      const int key = walk.key_of(i);
      const bool hidden = walk.hidden >> stage & 1;
      float ks0 = 1.f, ks1 = 1.f;
      if (C::INT8) {
        ks0 = read_float(data + C::SIDE + g * 4);
        ks1 = read_float(data + C::SIDE + (g + 8) * 4);
      }
      float sum0 = 0.f, sum1 = 0.f;
      for (int block = 0; block < blocks; ++block) {
        if (blocks > 1) load_block(block);
        float acc[NT][4];
        score_step<C>(data, qf, acc);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = key + g + (e >> 1) * 8;
            const bool seen = !hidden && k >= lo[nt][e & 1] && k < hi[nt][e & 1];
            const float f = C::INT8 ? (e < 2 ? ks0 : ks1) * factor[nt][e & 1] : factor[nt][e & 1];
            const float w = seen ? ex2_approx(fmaf(acc[nt][e], f, -lse2[nt][e & 1])) : 0.f;
            if (e < 2) sum0 += w; else sum1 += w;
          }
      }
      sum0 += __shfl_xor_sync(0xffffffffu, sum0, 1);
      sum1 += __shfl_xor_sync(0xffffffffu, sum1, 1);
      sum0 += __shfl_xor_sync(0xffffffffu, sum0, 2);
      sum1 += __shfl_xor_sync(0xffffffffu, sum1, 2);
      if (t < 2) {
        const int k = key + g + t * 8;
        if (k < slots) {
          const int64_t index = (int64_t(s) * a.line.kv_heads + head) * slots + k;
          a.weights[index] = (t == 0 ? sum0 : sum1) + (a.previous != nullptr ? a.previous[index] : 0.f);
        }
      }
      stage = stage + 1 == W::STAGES ? 0 : stage + 1;
    }
    copies_wait<0>();
    __syncwarp();
  }
}

// ---- launches ------------------------------------------------------------------------------------------------
constexpr int kSms = 148, kMaxWorkers = kSms * 3;

template <typename F>
int with_tile(int dtype_code, bool codes, int head_dim, int column_blocks, F&& f) {
#define RISA_TILE(T, I8, D)                                              \
  return column_blocks == 1 ? f(Tile<T, I8, D, 1>{}) : f(Tile<T, I8, D, 2>{})
#define RISA_TILE_DIM(T, I8)                      \
  do {                                            \
    if (head_dim == 64) RISA_TILE(T, I8, 64);     \
    if (head_dim == 128) RISA_TILE(T, I8, 128);   \
    RISA_TILE(T, I8, 256);                        \
  } while (0)
  if (dtype_code == 1) {
    if (codes) RISA_TILE_DIM(__half, true);
    RISA_TILE_DIM(__half, false);
  }
  if (codes) RISA_TILE_DIM(__nv_bfloat16, true);
  RISA_TILE_DIM(__nv_bfloat16, false);
#undef RISA_TILE_DIM
#undef RISA_TILE
}

int column_blocks_of(const risa_b200_step& step, int group) { return step.query_offsets == nullptr && group <= 8 ? 1 : 2; }

int check_queries(const risa_b200_cache* cache, const risa_b200_step* step, const void* q, const int64_t qs[2], int q_heads,
                  int dtype_code, float scale, int is_causal, int window, const char* what) {
  if (const int bad = check_cache(cache, what)) return bad;
  if (const int bad = check_step(step, cache, what)) return bad;
  RISA_REQUIRE(q != nullptr, "%s: null tensor", what);
  RISA_REQUIRE(q_heads > 0 && q_heads % cache->kv_heads == 0, "%s: the query heads must be a multiple of the key heads", what);
  RISA_REQUIRE(dtype_code == 1 || dtype_code == 2, "%s: q must be float16 or bfloat16", what);
  RISA_REQUIRE(cache->dtype_code == kInt8 || cache->dtype_code == dtype_code, "%s: q must have the cache's type", what);
  RISA_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 && qs[0] % 8 == 0 && qs[1] % 8 == 0,
               "%s: query rows must start on 16-byte boundaries", what);
  RISA_REQUIRE(fabsf(scale * kLog2e) < INFINITY, "%s: the scale must be finite, also in units of log 2", what);
  RISA_REQUIRE(window >= 0 && (window == 0 || is_causal), "%s: a window needs the causal rule and at least one key", what);
  RISA_REQUIRE(int64_t(step->tokens) * (q_heads / cache->kv_heads) < (int64_t(1) << 31) - 1024, "%s: too many query rows", what);
  return RISA_B200_OK;
}

RowsArgs rows_args(const risa_b200_cache* cache, const risa_b200_step* step, const void* q, const int64_t qs[2], int q_heads,
                   float scale, int is_causal, int window, unsigned int* status) {
  RowsArgs a{};
  const int group = q_heads / cache->kv_heads;
  a.line = {view_of(*step, cache->page_size), cache->kv_heads, Divisor(group), Divisor(8 * column_blocks_of(*step, group)), 1, INT_MAX, Divisor(16),
            is_causal != 0, window};
  a.q = q;
  a.qn = qs[0];
  a.qh = qs[1];
  a.keys = static_cast<const char*>(cache->keys);
  a.values = static_cast<const char*>(cache->values);
  a.key_scales = cache->key_scales;
  a.value_scales = cache->value_scales;
  a.pages = cache->pages;
  a.scale_log2 = scale * kLog2e;
  a.min_steps = 16;  // one token over 8K keys: 16.8 us with 8 (256 workers), 15.5 with 16
  a.status = status;
  return a;
}

template <typename K>
int allow_shared(K kernel, int bytes, const char* what) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return fail(RISA_B200_CUDA, "%s: %s", what, cudaGetErrorString(cudaGetLastError()));
  return RISA_B200_OK;
}

}  // namespace
}  // namespace serving
}  // namespace risa_b200

using namespace risa_b200;
using namespace risa_b200::serving;

// Whether a step can hold sequences for the tensor-core kernel.
static bool takes_tensor_cores(const risa_b200_step& step, int group) {
  return (step.query_offsets == nullptr ? group : int64_t(step.tokens) * group) >= kTcFewestRows;
}
static size_t rows_scratch(const risa_b200_cache& cache, const risa_b200_step& step, int group) {
  return size_t(kMaxWorkers) * (2 * slot_floats(8 * column_blocks_of(step, group), cache.head_dim) * sizeof(float) + sizeof(JoinNote));
}

extern "C" size_t risa_b200_paged_attention_scratch_size(const risa_b200_cache* cache, const risa_b200_step* step, int q_heads) {
  if (cache == nullptr || step == nullptr || cache->kv_heads <= 0 || q_heads <= 0) return 0;
  const int group = q_heads / cache->kv_heads;
  size_t bytes = rows_scratch(*cache, *step, group);
  if (takes_tensor_cores(*step, group)) bytes += paged_tc_scratch(cache->head_dim);
  return bytes;
}

extern "C" int risa_b200_paged_attention(const risa_b200_cache* cache, const risa_b200_step* step, const void* q,
                                         const int64_t q_strides[2], int q_heads, int dtype_code, void* out,
                                         const int64_t out_strides[2], float* lse, float scale, int is_causal, int window,
                                         int clear_rest, void* scratch, size_t scratch_bytes, void* stream_ptr) {
  if (const int bad = check_queries(cache, step, q, q_strides, q_heads, dtype_code, scale, is_causal, window, "paged attention")) return bad;
  RISA_REQUIRE(out != nullptr && reinterpret_cast<uintptr_t>(out) % 16 == 0 && out_strides[0] % 8 == 0 && out_strides[1] % 8 == 0,
               "paged attention: output rows must start on 16-byte boundaries");
  RISA_REQUIRE(scratch != nullptr && reinterpret_cast<uintptr_t>(scratch) % 16 == 0 &&
                   scratch_bytes >= risa_b200_paged_attention_scratch_size(cache, step, q_heads),
               "paged attention: the scratch is too small");
  unsigned int* status = status_word();
  if (status == nullptr) return RISA_B200_CUDA;
  RowsArgs a = rows_args(cache, step, q, q_strides, q_heads, scale, is_causal, window, status);
  a.out = out;
  a.on = out_strides[0];
  a.oh = out_strides[1];
  a.lse = lse;
  a.clear_rest = clear_rest;
  a.parts = static_cast<float*>(scratch);
  a.notes = reinterpret_cast<JoinNote*>(a.parts + size_t(kMaxWorkers) * 2 * slot_floats(a.line.rows, cache->head_dim));
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  const bool tensor_cores = takes_tensor_cores(*step, a.line.group);
  if (tensor_cores) a.line.max_rows = kTcFewestRows - 1;
  const bool codes = cache->dtype_code == kInt8;
  int bad = with_tile(dtype_code, codes, cache->head_dim, a.line.rows / 8, [&](auto tile) {
    using C = decltype(tile);
    constexpr int bytes = kWarps * Walk<C, true>::STAGE * Walk<C, true>::STAGES;
    if (const int bad = allow_shared(paged_rows_kernel<C>, bytes, "paged attention")) return bad;
    return launched(launch_chained(paged_rows_kernel<C>, dim3(kSms * C::CTAS), dim3(kThreads), bytes, stream, a), "paged attention");
  });
  TcArgs t{};
  if (bad == RISA_B200_OK && tensor_cores) {
    t = paged_tc_args(TcArgs{a.line, q, a.qn, a.qh, out, a.on, a.oh, lse, a.keys, a.values, a.key_scales, a.value_scales, a.pages, a.scale_log2,
                             a.parts + rows_scratch(*cache, *step, a.line.group) / sizeof(float), nullptr, 2, status}, cache->head_dim);
    t.line.min_rows = kTcFewestRows;
    t.line.max_rows = INT_MAX;
    bad = paged_tc(t, dtype_code, codes, cache->head_dim, stream);
  }
  if (bad == RISA_B200_OK)
    bad = with_tile(dtype_code, codes, cache->head_dim, a.line.rows / 8, [&](auto tile) {
      using C = decltype(tile);
      const JoinArgs join{a.parts, a.notes, C::R, a.line.group, q_heads, out, a.on, a.oh, lse};
      return launched(launch_chained(join_parts_kernel<typename C::T, C::D, true>, dim3(kSms * C::CTAS - 1, C::R), dim3(128), 0, stream, join), "paged attention");
    });
  if (bad == RISA_B200_OK && tensor_cores) bad = paged_tc_join(t, dtype_code, cache->head_dim, stream);
  return bad;
}

extern "C" size_t risa_b200_key_weights_scratch_size(const risa_b200_cache* cache, const risa_b200_step* step, int q_heads) {
  if (cache == nullptr || step == nullptr || cache->kv_heads <= 0 || q_heads <= 0) return 0;
  return takes_tensor_cores(*step, q_heads / cache->kv_heads) ? weigh_tc_scratch() : 0;
}

extern "C" int risa_b200_key_weights(const risa_b200_cache* cache, const risa_b200_step* step, const void* q,
                                     const int64_t q_strides[2], int q_heads, int dtype_code, const float* lse, float scale,
                                     int is_causal, int window, const float* previous, float* weights, void* scratch,
                                     size_t scratch_bytes, void* stream_ptr) {
  if (const int bad = check_queries(cache, step, q, q_strides, q_heads, dtype_code, scale, is_causal, window, "key weights")) return bad;
  RISA_REQUIRE(lse != nullptr && weights != nullptr, "key weights: null tensor");
  unsigned int* status = status_word();
  if (status == nullptr) return RISA_B200_CUDA;
  RowsArgs a = rows_args(cache, step, q, q_strides, q_heads, scale, is_causal, window, status);
  const int column_blocks = a.line.rows / 8;
  a.line.rows = Divisor(1 << 30);  // all rows of a key head are one unit
  const bool tensor_cores = takes_tensor_cores(*step, a.line.group);
  RISA_REQUIRE(!tensor_cores || (scratch != nullptr && reinterpret_cast<uintptr_t>(scratch) % 16 == 0 && scratch_bytes >= weigh_tc_scratch()),
               "key weights: the scratch is too small");
  if (tensor_cores) a.line.max_rows = kTcFewestRows - 1;
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  a.row_lse = lse;
  a.previous = previous;
  a.weights = weights;
  int bad = with_tile(dtype_code, cache->dtype_code == kInt8, cache->head_dim, column_blocks, [&](auto tile) {
    using C = decltype(tile);
    constexpr int bytes = kWarps * Walk<C, false>::STAGE * Walk<C, false>::STAGES;
    if (const int bad = allow_shared(weigh_rows_kernel<C>, bytes, "key weights")) return bad;
    return launched(launch_chained(weigh_rows_kernel<C>, dim3(kSms * C::CTAS), dim3(kThreads), bytes, stream, a), "key weights");
  });
  if (bad == RISA_B200_OK && tensor_cores) {
    TcArgs t{};
    t.line = a.line;
    t.line.min_rows = kTcFewestRows;
    t.q = q;
    t.qn = a.qn;
    t.qh = a.qh;
    t.keys = a.keys;
    t.key_scales = a.key_scales;
    t.pages = a.pages;
    t.scale_log2 = a.scale_log2;
    t.parts = static_cast<float*>(scratch);
    t.min_steps = 2;
    t.status = status;
    bad = weigh_tc(t, lse, previous, weights, dtype_code, cache->dtype_code == kInt8, cache->head_dim, stream);
  }
  return bad;
}
