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
// 32 requests of up to 32K keys as codes 221 us in short runs (6.3 TB/s), 251 in long ones; in 4 bits 192 and 209 (3.7 TB/s): 360
// instructions a step, 160 of them conversion.  Neither HBM nor the issue slots (57 %) are full there: of the 2.8 warps that a
// scheduler has, 0.6 wait for a result of fixed latency, 0.3 for a math pipe, 0.4 for dispatch or instructions and 0.3 for
// memory, so that none is ready in four cycles of ten; a fourth CTA's warps have no registers.
#include "four_bits.cuh"
#include "paged_tc.cuh"
#include "serving_plan.cuh"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace risa_b200 {
namespace serving {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
struct RowsArgs {
  FrontLineArgs line;
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
// FRONT: first keys stay visible in front of the window (the walk over the keys then has a gap; all others are spared its
// instructions, which cost 32 requests of up to 32K codes 263 -> 302 us).
template <typename T_, int BITS_, int D_, int NT_, bool FRONT_>
struct Tile {
  using T = T_;
  static constexpr bool FRONT = FRONT_;
  using Line = std::conditional_t<FRONT, FrontLineArgs, LineArgs>;
  static constexpr int BITS = BITS_;
  static constexpr bool CODES = BITS < 16;
  static constexpr int D = D_, NT = NT_, R = 8 * NT_;
  using M = std::conditional_t<CODES, __half, T_>;  // type of the matrix instructions' operands
  static constexpr int ROW = D * BITS / 8;  // bytes of a key
  static constexpr int CHUNKS = ROW / 16;
  static constexpr int SIDE = 16 * ROW;  // the 16 keys (or values) of a step
  // bytes of the scales of a step's keys (or values)
  static constexpr int SCALES = BITS == 8 ? 16 * 4 : BITS == 4 ? 16 * token_scale_bytes<D>() : 0;
  static constexpr int KS = D / 16;
  // CTAs of four warps that share an SM's shared memory: what hides the latency of HBM is bytes in flight, 96 KB or
  // more per SM.  Codes, whose conversion keeps the schedulers busy, gain from a third CTA (32 requests of up to 32K
  // keys: 280 us with two, 247 with three, 267 with four); 16-bit rows of 256 channels leave room for one.
  static constexpr int CTAS = D == 256 && !CODES ? 1 : CODES && D <= 128 && NT == 1 ? 3 : 2;
  // Steps that share a maximum: with half of the bytes for the same instructions, 4-bit codes gain from halving the softmax's
  // (32 requests of up to 32K keys 264 -> 246 us when it was brought in, with 16 rows 311 -> 282); 16 rows of 256 channels have no registers for it.
  static constexpr int SUB = BITS == 4 && (NT == 1 || D <= 128) ? 2 : 1;
  static constexpr int BUDGET = 48 * 1024 / CTAS;  // per warp
  __host__ __device__ static constexpr int stages(int sides) {
    const int n = BUDGET / (sides * (SIDE + SCALES));
    return n > 8 ? 8 : n;
  }
};

// 16-byte pieces of a row are permuted so that the reads below are free of bank conflicts.  16-bit rows:
// ldmatrix takes one piece of eight consecutive rows.  Codes: for K eight lanes read four pieces of two
// consecutive rows, for V two pieces of every other row.  4-bit rows are read the same way, but several of them share 128 bytes
// (the width of the banks): there the pieces of a line are permuted by the line's number.
template <typename C>
__device__ __forceinline__ int offset_of(int row, int piece) {
  if (C::BITS == 16) return row * C::ROW + (piece ^ (row & 7)) * 16;
  if (C::ROW >= 128) return row * C::ROW + (piece ^ (((row & 1) << 2) ^ (((row >> 1) & 3) << 1))) * 16;
  if (C::BITS == 8) return row * C::ROW + piece * 16;
  constexpr int EACH = 128 / C::ROW;  // rows of a line: 2 or 4
  const int line = row / EACH, slot = row % EACH * C::CHUNKS + piece;
  return line * 128 + (slot ^ ((line & (EACH == 2 ? 3 : 1)) << 1)) * 16;
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
// A copy whose offsets are known to the compiler (as operands of their own they cost three instructions).
template <int TO, int FROM>
__device__ __forceinline__ void copy16_at(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(to), "l"(from), "n"(TO), "n"(FROM) : "memory");
}
template <int TO>
__device__ __forceinline__ void copy4_at(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0 + %2], [%1], 4;" ::"r"(to), "l"(from), "n"(TO) : "memory");
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
// Reads at an offset known to the compiler.
template <int AT>
__device__ __forceinline__ uint4 read16_at(uint32_t address) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4 + %5];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(address), "n"(AT) : "memory");
  return v;
}
template <int AT>
__device__ __forceinline__ uint2 read8_at(uint32_t address) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2 + %3];" : "=r"(v.x), "=r"(v.y) : "r"(address), "n"(AT) : "memory");
  return v;
}
template <int AT>
__device__ __forceinline__ uint32_t read4_at(uint32_t address) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(v) : "r"(address), "n"(AT) : "memory");
  return v;
}
template <int AT>
__device__ __forceinline__ uint32_t read2_at(uint32_t address) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1 + %2];" : "=h"(v) : "r"(address), "n"(AT) : "memory");
  return v;
}
template <int AT>
__device__ __forceinline__ uint32_t read1_at(uint32_t address) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1 + %2];" : "=r"(v) : "r"(address), "n"(AT) : "memory");
  return v;
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
__device__ __forceinline__ void write1(uint32_t address, uint32_t v) { asm volatile("st.shared.u8 [%0], %1;" ::"r"(address), "r"(v) : "memory"); }
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
__device__ __forceinline__ uint32_t pair_of_halves(uint32_t pair) {
  uint32_t u;  // (pair & 0x00ff00ff) ^ 0x64806480: one instruction, of which the compiler makes two
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(u) : "r"(pair), "r"(0x00ff00ffu), "r"(0x64806480u));
  return less_1152(u);
}

// Not in front of the window, or one of the first keys.
template <typename C>
__device__ __forceinline__ bool outside_gap(const FrontLineArgs& line, int key, int low) {
  if (C::FRONT) return uint32_t(key - line.sinks) >= uint32_t(max(low - line.sinks, 0));
  return key >= low;
}

// ---- a warp's walk over its steps -----------------------------------------------------------------------
// Steps first, first + kWarps, ... of one unit.  Page numbers are looked up 32 steps at a time, one set
// ahead; a page outside the pool is not read (its keys are hidden and the status word says so).
template <typename C, bool WITH_VALUES>
struct Walk {
  const RowsArgs& a;
  const int32_t* row;  // the sequence's row of the page table
  int head, first_key, low, length, count, sequence;
  int turn, skip;  // FRONT: from step `turn` on keys lie `skip` further, behind the first ones that stay visible
  int pages, pages_ahead;
  uint32_t base;
  // codes: this lane's pieces of the sequence's head in page 0, and bytes of a page
  const char *key_rows, *value_rows, *scales[2];
  int scale_each[2];
  std::conditional_t<C::BITS == 4, int, int64_t> page_rows, page_scales;
  unsigned int hidden;  // one bit per stage
  static constexpr int STAGES = C::stages(WITH_VALUES ? 2 : 1);
  static constexpr int SIDES = WITH_VALUES ? 2 : 1;
  static constexpr int STAGE = SIDES * (C::SIDE + C::SCALES);  // keys, values, scales of the keys, of the values
  static_assert(STAGES >= 2 && STAGES <= 32, "ring");

  __device__ __forceinline__ int key_of(int i) const { return first_key + i * (16 * kWarps) + (C::FRONT && i >= turn ? skip : 0); }
  __device__ __forceinline__ bool exists(int key) const { return key < length && (outside_gap<C>(a.line, key, low)); }
  __device__ __forceinline__ int look_up(int i) const {
    const int key = key_of(i);
    return i < count && key < length ? __ldg(row + (key >> a.line.step.page_shift)) : -1;
  }
  __device__ __forceinline__ void start() {
    const int lane = threadIdx.x & 31;
    pages = look_up(lane);
    pages_ahead = look_up(32 + lane);
    hidden = 0;
    if constexpr (C::CODES) {
      const int shift = a.line.step.page_shift, block = (C::BITS == 4 ? token_scale_bytes<C::D>() : 4) << shift;
      page_rows = (decltype(page_rows)(a.line.kv_heads) << shift) * C::ROW;
      page_scales = decltype(page_rows)(a.line.kv_heads) * block;
      const int64_t of_head = (int64_t(head) << shift) * C::ROW + lane * 16;
      key_rows = a.keys + of_head;
      value_rows = a.values + of_head;
#pragma unroll
      for (int j = 0; j < SCALE_ROUNDS; ++j) {  // of the keys, then of the values; 4 bits: exponents, then group scales
        const int index = j * 32 + lane, piece = index < SCALE_PIECES ? index : index - SCALE_PIECES;
        scales[j] = reinterpret_cast<const char*>(index < SCALE_PIECES ? a.key_scales : a.value_scales) + int64_t(head) * block +
                    (C::BITS == 8 ? piece * 4 : piece == 0 ? 0 : (1 << shift) + (piece - 1) * 16);
        scale_each[j] = C::BITS == 8 ? 4 : piece == 0 ? 1 : C::D / 16;
      }
    }
  }
  static constexpr int SCALE_BYTES = C::BITS == 8 ? 4 : 16, SCALE_PIECES = C::SCALES / SCALE_BYTES;  // of a copy, copies of a side
  static constexpr int SCALE_ROUNDS = (SIDES * SCALE_PIECES + 31) / 32;
  // What 512 bytes of a step further in the swizzle flip (offset_of's rows are 512 bytes apart by its lines).
  static constexpr int flip(int j) {
    return C::ROW == 128 ? (j & 1) * 64 : C::ROW == 256 ? (j & 3) * 32 : 0;
  }
  template <int J>
  __device__ __forceinline__ void copy_codes(uint32_t to, int first, const char* k, const char* v) {
    copy16_at<J * 512, J * 512>(to + (first ^ flip(J)), k);
    if constexpr (WITH_VALUES) copy16_at<C::SIDE + J * 512, J * 512>(to + (first ^ flip(J)), v);
    if constexpr (J + 1 < C::CHUNKS / 2) copy_codes<J + 1>(to, first, k, v);
  }
  // 16 keys that exist.
  __device__ __forceinline__ void fetch_codes(int key, int page, uint32_t to) {
    const int lane = threadIdx.x & 31, slot = key & ((1 << a.line.step.page_shift) - 1);
    const int64_t off = int64_t(page) * page_rows + slot * C::ROW;
    copy_codes<0>(to, offset_of<C>(lane / C::CHUNKS, lane % C::CHUNKS), key_rows + off, value_rows + off);
    const uint32_t scales_at = to + lane * SCALE_BYTES;
#pragma unroll
    for (int j = 0; j < SCALE_ROUNDS; ++j)
      if (SIDES * SCALE_PIECES >= (j + 1) * 32 || j * 32 + lane < SIDES * SCALE_PIECES) {
        const char* from = scales[j] + (int64_t(page) * page_scales + slot * scale_each[j]);
        if constexpr (C::BITS == 8) copy4_at<SIDES * C::SIDE>(scales_at, from);
        else if (j == 0) copy16_at<SIDES * C::SIDE, 0>(scales_at, from);
        else copy16_at<SIDES * C::SIDE + 512, 0>(scales_at, from);
      }
  }
  // Some of the 16 (or none: good false) exist; the others become zeros, their scales are cleared by who reads them.
  __device__ __forceinline__ void fetch_some_codes4(int key, int page, bool good, uint32_t to) {
    const int lane = threadIdx.x & 31, slot = key & ((1 << a.line.step.page_shift) - 1);
    const int64_t off = good ? int64_t(page) * page_rows + slot * C::ROW : 0;
    const char *k = key_rows + off, *v = value_rows + off;
#pragma unroll 1
    for (int j = 0; j < C::CHUNKS / 2; ++j) {
      const int r = (j * 32 + lane) / C::CHUNKS;
      const uint32_t at = to + offset_of<C>(r, lane % C::CHUNKS);
      const bool there = good && exists(key + r);
      copy16(at, k + j * 512, there);
      if (WITH_VALUES) copy16(at + C::SIDE, v + j * 512, there);
    }
#pragma unroll
    for (int j = 0; j < SCALE_ROUNDS; ++j)
      if (j * 32 + lane < SIDES * SCALE_PIECES)
        copy16(to + SIDES * C::SIDE + (j * 32 + lane) * 16, scales[j] + (good ? int64_t(page) * page_scales + slot * scale_each[j] : 0), good);
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
      if constexpr (C::CODES) {
        // nearly all steps are of 16 keys that exist
        if (uint32_t(page) < uint32_t(a.pages) && key >= low && key + 16 <= length) {
          fetch_codes(key, page, base + stage * STAGE);
          if (hidden != 0) hidden &= ~(1u << stage);
          copies_commit();
          return;
        }
      }
      const bool good = key < length && page >= 0 && page < a.pages;
      if (key < length && !good && lane == 0) atomicCAS(a.status, 0u, unsigned(sequence) + 1u);
      hidden = good ? hidden & ~(1u << stage) : hidden | (1u << stage);
      if constexpr (C::BITS == 4) {
        fetch_some_codes4(key, page, good, base + stage * STAGE);
        copies_commit();
        return;
      }
      const int64_t line = good ? (((int64_t(page) * a.line.kv_heads + head) << a.line.step.page_shift) +
                                   (key & ((1 << a.line.step.page_shift) - 1)))
                                : 0;
      const char* k = a.keys + line * C::ROW;
      const char* v = a.values + line * C::ROW;
      const uint32_t to = base + stage * STAGE;
      auto copy = [&](auto whole) {
#pragma unroll
        for (int j = 0; j < C::CHUNKS / 2; ++j) {
          const int index = j * 32 + lane, r = index / C::CHUNKS, piece = index % C::CHUNKS;
          const bool there = whole || (good && exists(key + r));
          const uint32_t at = to + offset_of<C>(r, piece);
          copy16(at, k + index * 16, there);
          if (WITH_VALUES) copy16(at + C::SIDE, v + index * 16, there);
        }
        if (C::BITS == 8 && (WITH_VALUES || lane < 16)) {
          const float* s = lane < 16 ? a.key_scales : a.value_scales;
          const int r = lane & 15;
          copy4(to + SIDES * C::SIDE + lane * 4, s + line + r, whole || (good && exists(key + r)));
        }
      };
      // nearly all steps are of 16 keys that exist
      if (good && key >= low && key + 16 <= length) copy(std::true_type{});
      else copy(std::false_type{});
    }
    copies_commit();
  }
  // Scales of 4-bit keys that do not exist (they lie beside those that do), or of a step that does not, become zeros.
  __device__ __forceinline__ void clear_missing(uint32_t data, int key, bool all) const {
    const int lane = threadIdx.x & 31;
    if (lane < 16 && (all || !exists(key + lane))) {
#pragma unroll
      for (int side = 0; side < SIDES; ++side) {
        const uint32_t scales = data + SIDES * C::SIDE + side * C::SCALES;
        write1(scales + lane, 0);
#pragma unroll
        for (int i = 0; i < C::D / 16; ++i) write1(scales + 16 + lane * (C::D / 16) + i, 0);
      }
    }
    __syncwarp();
  }
};

// The first of a warp's steps that lies behind the first keys that stay visible.
__device__ __forceinline__ int warp_turn(const Piece& piece) { return (piece.turn - int(threadIdx.x >> 5) + kWarps - 1) / kWarps; }

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
      constexpr int RUN = C::BITS == 4 && C::D >= 128 ? 32 : 16;  // channels that a lane takes at once
      const int c0 = C::CODES ? ks / (RUN / 4) * (4 * RUN) + t * RUN + ks % (RUN / 4) * 4 : ks * 16 + t * 2;
      const int c1 = C::CODES ? c0 + 2 : c0 + 8;
      qf[nt][ks][0] = there ? *reinterpret_cast<const uint32_t*>(q + c0) : 0u;
      qf[nt][ks][1] = there ? *reinterpret_cast<const uint32_t*>(q + c1) : 0u;
    }
    factor[nt][0] = factor[nt][1] = a.scale_log2;
    if constexpr (C::CODES && std::is_same<typename C::T, __nv_bfloat16>::value) {
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

// acc[nt]: raw scores of keys g and g + 8 against query rows 2 t and 2 t + 1 (of column block nt); scales: of 4-bit keys.
template <typename C>
__device__ __forceinline__ void score_step(uint32_t keys, uint32_t scales, const uint32_t (&qf)[C::NT][C::KS][2], float (&acc)[C::NT][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[nt][i] = 0.f;
  if constexpr (C::BITS == 4) {
    // a lane takes 16 channels (a group) of heads of 64, else 32 (two groups) at a time
    constexpr int RUNS = C::D == 256 ? 2 : 1, WORDS = C::D == 64 ? 2 : 4, GROUPS = WORDS / 2;
#pragma unroll
    for (int run = 0; run < RUNS; ++run) {
      // keys g and g + 8 lie alike in the swizzle
      constexpr int EIGHT = 8 * C::ROW, SCALE_EIGHT = 8 * (C::D / 16);
      uint32_t w[2][WORDS], scale[2];
      if constexpr (WORDS == 4) {
        const uint32_t at = keys + offset_of<C>(g, run * 4 + t), of = scales + g * (C::D / 16) + t * 2;
        const uint4 u = read16_at<0>(at), v = read16_at<EIGHT>(at);
        w[0][0] = u.x; w[0][1] = u.y; w[0][2] = u.z; w[0][3] = u.w;
        w[1][0] = v.x; w[1][1] = v.y; w[1][2] = v.z; w[1][3] = v.w;
        scale[0] = run ? read2_at<16 + 8>(of) : read2_at<16>(of);
        scale[1] = run ? read2_at<16 + 8 + SCALE_EIGHT>(of) : read2_at<16 + SCALE_EIGHT>(of);
      } else {
        const uint32_t at = keys + offset_of<C>(g, t >> 1) + (t & 1) * 8, of = scales + g * (C::D / 16) + t;
        const uint2 u = read8_at<0>(at), v = read8_at<EIGHT>(at);
        w[0][0] = u.x; w[0][1] = u.y;
        w[1][0] = v.x; w[1][1] = v.y;
        scale[0] = read1_at<16>(of);
        scale[1] = read1_at<16 + SCALE_EIGHT>(of);
      }
#pragma unroll
      for (int group = 0; group < GROUPS; ++group) {
        const GroupScale<__half> lo(__byte_perm(scale[0], 0, group ? 0x4141 : 0x4040)), hi(__byte_perm(scale[1], 0, group ? 0x4141 : 0x4040));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t l[4], h[4];
          scaled_codes(w[0][2 * group + j], lo, l);
          scaled_codes(w[1][2 * group + j], hi, h);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t af[4] = {l[2 * half], h[2 * half], l[2 * half + 1], h[2 * half + 1]};
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) mma16816<__half>(acc[nt], af, qf[nt][run * 8 + group * 4 + j * 2 + half]);
          }
        }
      }
    }
  } else if constexpr (C::BITS == 8) {
#pragma unroll
    for (int b = 0; b < C::D / 64; ++b) {
      const uint32_t at = keys + offset_of<C>(g, b * 4 + t);  // keys g and g + 8 lie alike in the swizzle
      const uint4 lo = read16_at<0>(at), hi = read16_at<8 * C::ROW>(at);
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
      ldmatrix4(af, keys + offset_of<C>(r, 2 * ks + (lane >> 4)));
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt) mma16816<typename C::T>(acc[nt], af, qf[nt][ks]);
    }
  }
}

// out[nt][mt] += V^T P^T.  16-bit values: block mt holds channels 16 mt + g (and + 8).  Codes: a lane takes
// the channels of its own 16-byte pieces (8 bytes at 64 channels; 4-bit codes half of that), two per instruction: see channel_of.
template <typename C>
__device__ __forceinline__ void value_step(uint32_t values, uint32_t scales, const uint32_t (&p)[C::NT][2], float (&out)[C::NT][C::D / 16][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if constexpr (C::BITS == 4) {
    constexpr int WORDS = C::D / 64;  // of a key: half a group, a group or two groups
    // keys 2 t and 2 t + 1, and those eight further, which lie alike in the swizzle
    constexpr int EIGHT = 8 * C::ROW, GROUP_BYTES = C::D / 16;
    uint32_t w[4][WORDS], scale[4];
    const uint32_t of = scales + 2 * t * GROUP_BYTES + (WORDS == 4 ? 2 * g : WORDS == 2 ? g : g >> 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t at = values + offset_of<C>(2 * t + i, WORDS == 4 ? g : WORDS == 2 ? g >> 1 : g >> 2) + (WORDS == 4 ? 0 : WORDS == 2 ? (g & 1) * 8 : (g & 3) * 4);
      if constexpr (WORDS == 4) {
        const uint4 u = read16_at<0>(at), v = read16_at<EIGHT>(at);
        w[i][0] = u.x; w[i][1] = u.y; w[i][2] = u.z; w[i][3] = u.w;
        w[i + 2][0] = v.x; w[i + 2][1] = v.y; w[i + 2][2] = v.z; w[i + 2][3] = v.w;
      } else if constexpr (WORDS == 2) {
        const uint2 u = read8_at<0>(at), v = read8_at<EIGHT>(at);
        w[i][0] = u.x; w[i][1] = u.y;
        w[i + 2][0] = v.x; w[i + 2][1] = v.y;
      } else {
        w[i][0] = read4_at<0>(at);
        w[i + 2][0] = read4_at<EIGHT>(at);
      }
    }
    if constexpr (WORDS == 4) {
      scale[0] = read2_at<16>(of);
      scale[1] = read2_at<16 + GROUP_BYTES>(of);
      scale[2] = read2_at<16 + 8 * GROUP_BYTES>(of);
      scale[3] = read2_at<16 + 9 * GROUP_BYTES>(of);
    } else {
      scale[0] = read1_at<16>(of);
      scale[1] = read1_at<16 + GROUP_BYTES>(of);
      scale[2] = read1_at<16 + 8 * GROUP_BYTES>(of);
      scale[3] = read1_at<16 + 9 * GROUP_BYTES>(of);
    }
#pragma unroll
    for (int group = 0; group < (WORDS + 1) / 2; ++group) {
      // the scales of keys 2 t and 2 t + 1, of 2 t + 8 and 2 t + 9
      const GroupScale<__half> near(__byte_perm(scale[0], scale[1], WORDS < 4 ? 0x7470 : group ? 0x3531 : 0x3430) & 0x00ff00ffu);
      const GroupScale<__half> far(__byte_perm(scale[2], scale[3], WORDS < 4 ? 0x7470 : group ? 0x3531 : 0x3430) & 0x00ff00ffu);
#pragma unroll
      for (int j = 2 * group; j < 2 * group + 2 && j < WORDS; ++j) {
        uint32_t x[4][4];  // even channels of near keys, odd ones; of far keys
        scaled_codes(__byte_perm(w[0][j], w[1][j], 0x5410), near, x[0]);
        scaled_codes(__byte_perm(w[0][j], w[1][j], 0x7632), near, x[1]);
        scaled_codes(__byte_perm(w[2][j], w[3][j], 0x5410), far, x[2]);
        scaled_codes(__byte_perm(w[2][j], w[3][j], 0x7632), far, x[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // channels 2 e and 2 e + 1 of the word
          const uint32_t af[4] = {x[0][e], x[1][e], x[2][e], x[3][e]};
#pragma unroll
          for (int nt = 0; nt < C::NT; ++nt) mma16816<__half>(out[nt][j * 4 + e], af, p[nt]);
        }
      }
    }
  } else if constexpr (C::BITS == 8) {
    constexpr int RUNS = C::D == 256 ? 2 : 1, WORDS = C::D == 64 ? 2 : 4;
#pragma unroll
    for (int run = 0; run < RUNS; ++run) {
      uint32_t w[4][WORDS];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 2 * t + (i & 1) + (i >> 1) * 8;
        if constexpr (WORDS == 4) {
          const uint4 v = read16(values + offset_of<C>(key, g + 8 * run));
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
      ldmatrix4_transposed(af, values + offset_of<C>(r, 2 * mt + ((lane >> 3) & 1)));
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt) mma16816<typename C::T>(out[nt][mt], af, p[nt]);
    }
  }
}
template <typename C>
__device__ __forceinline__ int channel_of(int mt, int second) {
  const int g = (threadIdx.x & 31) >> 2;
  if (!C::CODES) return mt * 16 + g + second * 8;
  if (C::D == 64) return g * 8 + 2 * mt + second;
  if (C::BITS == 4) return g * (C::D / 8) + 2 * mt + second;
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
  const typename C::Line& line = a.line;
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
  const int64_t total = line_total<kThreads>(line, shared);
  const int workers = workers_of(total, gridDim.x, a.min_steps);
  if (int(blockIdx.x) >= workers) {
    if (threadIdx.x == 0) a.notes[blockIdx.x] = JoinNote{};
    return;
  }
  const int64_t begin = border(total, blockIdx.x, workers), end = border(total, blockIdx.x + 1, workers);
  Pieces pieces{end - begin, line_place<kThreads>(line, begin, shared)};
  Piece piece;
  while (pieces.next(line, piece)) {
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
           take > warp ? (take - warp + kWarps - 1) / kWarps : 0, s, warp_turn(piece), piece.skip * 16};
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
    constexpr int SUB = C::SUB;
    static_assert(W::STAGES >= 2 * SUB, "ring");
#pragma unroll
    for (int i = 0; i < W::STAGES - SUB; ++i) walk.fetch(i, i);
    int stage = 0;
    for (int i = 0; i < walk.count; i += SUB) {
      int next = stage < SUB ? stage + W::STAGES - SUB : stage - SUB;  // the stages of the steps in front of i, free by now
      copies_wait<W::STAGES - 2 * SUB>();
      __syncwarp();
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        walk.fetch(i + W::STAGES - SUB + u, next);
        next = next + 1 == W::STAGES ? 0 : next + 1;
      }
      uint32_t data[SUB];
      int key[SUB];
      bool alone[SUB], hidden[SUB], masked = false, partial = false;
      float acc[SUB][NT][4], vs[SUB][2], lift[SUB][2];
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        data[u] = ring + stage * W::STAGE;
        key[u] = walk.key_of(i + u);
        alone[u] = SUB > 1 && i + u >= walk.count;  // the last step may stand alone
        hidden[u] = alone[u] || (walk.hidden >> stage & 1);
        masked = masked || hidden[u] || key[u] < all_lo || key[u] + 16 > all_hi;
        partial = partial || alone[u] || key[u] < low || key[u] + 16 > seq.length;
        stage = stage + 1 == W::STAGES ? 0 : stage + 1;
      }
      if (C::BITS == 4 && partial)
#pragma unroll
        for (int u = 0; u < SUB; ++u) walk.clear_missing(data[u], key[u], alone[u]);
      // no branch from here to the mask, so that the steps' chains of products run side by side
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        const uint32_t key_scales = data[u] + 2 * C::SIDE, value_scales = key_scales + C::SCALES;
        score_step<C>(data[u], key_scales, qf, acc[u]);
        float ks0 = 1.f, ks1 = 1.f;
        vs[u][0] = vs[u][1] = 1.f;
        lift[u][0] = lift[u][1] = 0.f;
        if (C::BITS == 4) {
          const uint32_t of = key_scales + g, e0 = read1_at<C::SCALES>(of), e1 = read1_at<C::SCALES + 8>(of);
          ks0 = power_of(read1_at<0>(of));
          ks1 = power_of(read1_at<8>(of));
          vs[u][0] = power_of(e0) * kGroupUnit;
          vs[u][1] = power_of(e1) * kGroupUnit;
          lift[u][0] = lift_of(e0);
          lift[u][1] = lift_of(e1);
        }
        if (C::BITS == 8) {
          ks0 = read_float(key_scales + g * 4);
          ks1 = read_float(key_scales + (g + 8) * 4);
          vs[u][0] = read_float(value_scales + g * 4);
          vs[u][1] = read_float(value_scales + (g + 8) * 4);
          // a row of zeros must not let its own probability overflow, nor one that is not finite let the others vanish
#pragma unroll
          for (int e = 0; e < 2; ++e) lift[u][e] = vs[u][e] < INFINITY ? lg2_approx(fmaxf(vs[u][e], 0x1p-100f)) : 0.f;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[u][nt][e] *= C::CODES ? (e < 2 ? ks0 : ks1) * factor[nt][e & 1] : factor[nt][e & 1];
      }
      if (masked) {
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int k = key[u] + g + (e >> 1) * 8;
              if (hidden[u] || !outside_gap<C>(a.line, k, lo[nt][e & 1]) || k >= hi[nt][e & 1]) acc[u][nt][e] = -INFINITY;
            }
      }
      uint32_t p[SUB][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float top[2], keep[2];
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
          float x = fmaxf(acc[0][nt][i2] + lift[0][0], acc[0][nt][2 + i2] + lift[0][1]);
#pragma unroll
          for (int u = 1; u < SUB; ++u) x = fmaxf(x, fmaxf(acc[u][nt][i2] + lift[u][0], acc[u][nt][2 + i2] + lift[u][1]));
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
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          float e[4];
#pragma unroll
          for (int i2 = 0; i2 < 4; ++i2) e[i2] = ex2_approx(acc[u][nt][i2] - m[nt][i2 & 1]);
          l[nt][0] += e[0] + e[2];
          l[nt][1] += e[1] + e[3];
          // Probabilities (times scales) leave 32 bits here: half a step, 2^-8 of the value in bf16, 2^-11 in fp16.
          p[u][nt][0] = transposed8x8(Half2<typename C::M>::pack(C::CODES ? e[0] * vs[u][0] : e[0], C::CODES ? e[1] * vs[u][0] : e[1]));
          p[u][nt][1] = transposed8x8(Half2<typename C::M>::pack(C::CODES ? e[2] * vs[u][1] : e[2], C::CODES ? e[3] * vs[u][1] : e[3]));
        }
      }
#pragma unroll
      for (int u = 0; u < SUB; ++u) value_step<C>(data[u] + C::SIDE, data[u] + 2 * C::SIDE + C::SCALES, p[u], o);
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
  if (threadIdx.x == 0) a.notes[blockIdx.x] = join_note(line, piece, total, end, blockIdx.x, workers);
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
  const typename C::Line& line = a.line;
  chain_wait();
  chain_release();
  // what no step covers: in front of the window (but for the first keys that stay visible), behind the length
  for (int64_t u = blockIdx.x; u < int64_t(a.line.step.batch) * a.line.kv_heads; u += gridDim.x) {
    const Sequence seq = sequence_of(a.line.step, int(u / a.line.kv_heads));
    const int rows = seq.count * a.line.group;
    if (rows > a.line.max_rows) continue;
    const StepRange range = rows == 0 ? StepRange{0, 0} : steps_of(line, seq, 0);
    const int front = range.front * 16, from = min(range.first * 16, slots), to = min((range.first + range.count - range.front) * 16, slots);
    for (int i = front + threadIdx.x; i < slots - (to - from); i += kThreads) {
      const int key = i < from ? i : i + (to - from);
      a.weights[u * slots + key] = a.previous != nullptr ? a.previous[u * slots + key] : 0.f;
    }
  }
  const int64_t total = line_total<kThreads>(line, shared);
  const int workers = workers_of(total, gridDim.x, a.min_steps);
  if (int(blockIdx.x) >= workers) return;
  const int64_t begin = border(total, blockIdx.x, workers);
  Pieces pieces{border(total, blockIdx.x + 1, workers) - begin, line_place<kThreads>(line, begin, shared)};
  Piece piece;
  while (pieces.next(line, piece)) {
    const Sequence seq = piece.seq;
    const int s = piece.sequence, head = piece.head, rows = seq.count * a.line.group, blocks = (rows + R - 1) / R, take = piece.count;
    const int low = a.line.window > 0 ? visible(seq.length - seq.count, seq.length, true, a.line.window).lo : 0;
    W walk{a, a.line.step.table + int64_t(s) * a.line.step.width, head, (piece.first + warp) * 16, low, seq.length,
           take > warp ? (take - warp + kWarps - 1) / kWarps : 0, s, warp_turn(piece), piece.skip * 16};
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
      if (C::BITS == 4) {
        if (key < low || key + 16 > seq.length) walk.clear_missing(data, key, false);
        ks0 = power_of(read1_at<C::SIDE>(data + g));
        ks1 = power_of(read1_at<C::SIDE + 8>(data + g));
      }
      if (C::BITS == 8) {
        ks0 = read_float(data + C::SIDE + g * 4);
        ks1 = read_float(data + C::SIDE + (g + 8) * 4);
      }
      float sum0 = 0.f, sum1 = 0.f;
      for (int block = 0; block < blocks; ++block) {
        if (blocks > 1) load_block(block);
        float acc[NT][4];
        score_step<C>(data, data + C::SIDE, qf, acc);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = key + g + (e >> 1) * 8;
            const bool seen = !hidden && outside_gap<C>(a.line, k, lo[nt][e & 1]) && k < hi[nt][e & 1];
            const float f = C::CODES ? (e < 2 ? ks0 : ks1) * factor[nt][e & 1] : factor[nt][e & 1];
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
int with_tile(int dtype_code, int bits, int head_dim, int column_blocks, bool front, F&& f) {
#define RISA_TILE(T, BITS, D)                                                                                   \
  return column_blocks == 1 ? (front ? f(Tile<T, BITS, D, 1, true>{}) : f(Tile<T, BITS, D, 1, false>{}))        \
                            : (front ? f(Tile<T, BITS, D, 2, true>{}) : f(Tile<T, BITS, D, 2, false>{}))
#define RISA_TILE_DIM(T, BITS)                      \
  do {                                              \
    if (head_dim == 64) RISA_TILE(T, BITS, 64);     \
    if (head_dim == 128) RISA_TILE(T, BITS, 128);   \
    RISA_TILE(T, BITS, 256);                        \
  } while (0)
#define RISA_TILE_BITS(T)                 \
  do {                                    \
    if (bits == 4) RISA_TILE_DIM(T, 4);   \
    if (bits == 8) RISA_TILE_DIM(T, 8);   \
    RISA_TILE_DIM(T, 16);                 \
  } while (0)
  if (dtype_code == 1) RISA_TILE_BITS(__half);
  RISA_TILE_BITS(__nv_bfloat16);
#undef RISA_TILE_BITS
#undef RISA_TILE_DIM
#undef RISA_TILE
}

int column_blocks_of(const risa_b200_step& step, int group) { return step.query_offsets == nullptr && group <= 8 ? 1 : 2; }

int check_queries(const risa_b200_cache* cache, const risa_b200_step* step, const void* q, const int64_t qs[2], int q_heads,
                  int dtype_code, float scale, int is_causal, int window, int sinks, const char* what) {
  if (const int bad = check_cache(cache, what)) return bad;
  if (const int bad = check_step(step, cache, what)) return bad;
  RISA_REQUIRE(q != nullptr, "%s: null tensor", what);
  RISA_REQUIRE(q_heads > 0 && q_heads % cache->kv_heads == 0, "%s: the query heads must be a multiple of the key heads", what);
  RISA_REQUIRE(dtype_code == 1 || dtype_code == 2, "%s: q must be float16 or bfloat16", what);
  RISA_REQUIRE(bits_of(*cache) < 16 || cache->dtype_code == dtype_code, "%s: q must have the cache's type", what);
  RISA_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 && qs[0] % 8 == 0 && qs[1] % 8 == 0,
               "%s: query rows must start on 16-byte boundaries", what);
  RISA_REQUIRE(fabsf(scale * kLog2e) < INFINITY, "%s: the scale must be finite, also in units of log 2", what);
  RISA_REQUIRE(bits_of(*cache) != 4 || fabsf(scale * kLog2e * kGroupUnit) < INFINITY, "%s: the scale is too large for 4-bit codes", what);
  RISA_REQUIRE(window >= 0 && (window == 0 || is_causal), "%s: a window needs the causal rule and at least one key", what);
  RISA_REQUIRE(sinks >= 0 && (sinks == 0 || window > 0), "%s: first keys stay visible in front of a window", what);
  RISA_REQUIRE(int64_t(step->tokens) * (q_heads / cache->kv_heads) < (int64_t(1) << 31) - 1024, "%s: too many query rows", what);
  return RISA_B200_OK;
}

RowsArgs rows_args(const risa_b200_cache* cache, const risa_b200_step* step, const void* q, const int64_t qs[2], int q_heads,
                   float scale, int is_causal, int window, int sinks, unsigned int* status) {
  RowsArgs a{};
  const int group = q_heads / cache->kv_heads;
  a.line = {{view_of(*step, cache->page_size), cache->kv_heads, Divisor(group), Divisor(8 * column_blocks_of(*step, group)), 1, INT_MAX, Divisor(16),
             is_causal != 0, window},
            std::min(sinks, int(RISA_B200_CACHE_MOST_SLOTS))};
  a.q = q;
  a.qn = qs[0];
  a.qh = qs[1];
  a.keys = static_cast<const char*>(cache->keys);
  a.values = static_cast<const char*>(cache->values);
  a.key_scales = cache->key_scales;
  a.value_scales = cache->value_scales;
  a.pages = cache->pages;
  a.scale_log2 = scale * kLog2e * (bits_of(*cache) == 4 ? kGroupUnit : 1.0f);
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
                                         int clear_rest, void* scratch, size_t scratch_bytes, void* stream) {
  return risa_b200_paged_attention_sinks(cache, step, q, q_strides, q_heads, dtype_code, out, out_strides, lse, scale, is_causal, window, 0,
                                         clear_rest, scratch, scratch_bytes, stream);
}

extern "C" int risa_b200_paged_attention_sinks(const risa_b200_cache* cache, const risa_b200_step* step, const void* q,
                                               const int64_t q_strides[2], int q_heads, int dtype_code, void* out,
                                               const int64_t out_strides[2], float* lse, float scale, int is_causal, int window,
                                               int sinks, int clear_rest, void* scratch, size_t scratch_bytes, void* stream_ptr) {
  if (const int bad = check_queries(cache, step, q, q_strides, q_heads, dtype_code, scale, is_causal, window, sinks, "paged attention")) return bad;
  RISA_REQUIRE(out != nullptr && reinterpret_cast<uintptr_t>(out) % 16 == 0 && out_strides[0] % 8 == 0 && out_strides[1] % 8 == 0,
               "paged attention: output rows must start on 16-byte boundaries");
  RISA_REQUIRE(scratch != nullptr && reinterpret_cast<uintptr_t>(scratch) % 16 == 0 &&
                   scratch_bytes >= risa_b200_paged_attention_scratch_size(cache, step, q_heads),
               "paged attention: the scratch is too small");
  unsigned int* status = status_word();
  if (status == nullptr) return RISA_B200_CUDA;
  RowsArgs a = rows_args(cache, step, q, q_strides, q_heads, scale, is_causal, window, sinks, status);
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
  const int bits = bits_of(*cache);
  int bad = with_tile(dtype_code, bits, cache->head_dim, a.line.rows / 8, sinks > 0, [&](auto tile) {
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
    bad = paged_tc(t, dtype_code, bits, cache->head_dim, stream);
  }
  if (bad == RISA_B200_OK)
    bad = with_tile(dtype_code, bits, cache->head_dim, a.line.rows / 8, false, [&](auto tile) {
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
                                     size_t scratch_bytes, void* stream) {
  return risa_b200_key_weights_sinks(cache, step, q, q_strides, q_heads, dtype_code, lse, scale, is_causal, window, 0, previous, weights,
                                     scratch, scratch_bytes, stream);
}

extern "C" int risa_b200_key_weights_sinks(const risa_b200_cache* cache, const risa_b200_step* step, const void* q,
                                           const int64_t q_strides[2], int q_heads, int dtype_code, const float* lse, float scale,
                                           int is_causal, int window, int sinks, const float* previous, float* weights, void* scratch,
                                           size_t scratch_bytes, void* stream_ptr) {
  if (const int bad = check_queries(cache, step, q, q_strides, q_heads, dtype_code, scale, is_causal, window, sinks, "key weights")) return bad;
  RISA_REQUIRE(lse != nullptr && weights != nullptr, "key weights: null tensor");
  unsigned int* status = status_word();
  if (status == nullptr) return RISA_B200_CUDA;
  RowsArgs a = rows_args(cache, step, q, q_strides, q_heads, scale, is_causal, window, sinks, status);
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
  int bad = with_tile(dtype_code, bits_of(*cache), cache->head_dim, column_blocks, sinks > 0, [&](auto tile) {
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
    bad = weigh_tc(t, lse, previous, weights, dtype_code, bits_of(*cache), cache->head_dim, stream);
  }
  return bad;
}
