// 16-bit tensor-core pieces shared by the kernels over a paged cache: operand descriptors, the matrix instructions with
// fp32 accumulators, tiles in shared memory and what fills them.
#pragma once
#include <type_traits>

#include "serving.cuh"
#include "tc_ptx.cuh"

namespace risa_b200 {
namespace serving {

// kind::f16 with fp32 accumulators, M = 128: types of A and B, B's major axis, N.
template <typename T> __host__ __device__ constexpr uint32_t idesc_f16(bool b_mn_major, int n) {
  const uint32_t type = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (type << 7) | (type << 10) | ((b_mn_major ? 1u : 0u) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}
// Operand descriptors as a constant upper half and a lower half to which offsets (in units of 16 bytes) are added.
// Rows of 64 channels are 128 bytes wide and swizzled, eight of them 1024 bytes; the next 64 channels are one block of
// the tile's rows further.  Q and K are read with the MMA's K axis along a row (the leading offset is unused), V with it across
// the rows (the leading offset leads to the next 64 channels).
constexpr uint32_t kDescHigh = (1024 >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint64_t descriptor(uint32_t low) { return uint64_t(kDescHigh) << 32 | low; }
__device__ __forceinline__ uint32_t along_row(uint32_t address) { return (address & 0x3ffffu) >> 4 | 1u << 16; }
template <int ROWS>
__device__ __forceinline__ uint32_t across_rows(uint32_t address) { return (address & 0x3ffffu) >> 4 | uint32_t(ROWS * 128 >> 4) << 16; }
// One thread issues.
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
// A from tensor memory: two 16-bit values along K per column.
__device__ __forceinline__ void mma_f16_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}

__device__ __forceinline__ void tmem_store16(uint32_t address, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(address),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
// The thread's arrival on a barrier once all its copies so far have landed; nothing waits for it here.  The copies are
// written through the generic proxy: whoever waits on the barrier fences before a matrix instruction reads them (or the
// thread itself waits, fences and arrives).
__device__ __forceinline__ void copies_arrive(uint32_t barrier) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(barrier) : "memory");
}
__device__ __forceinline__ void copies_drain() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void store16(uint32_t to, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// Byte offset of the 16-byte piece `piece` of row `row` in a tile of ROWS rows: blocks of 64 channels.
template <int ROWS = 128>
__device__ __forceinline__ uint32_t tile_offset(int row, int piece) {
  return uint32_t((piece >> 3) * (ROWS * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
}

// Codes are whole numbers of at most 128, exact in both 16-bit types.  Codes 2 i and 2 i + 1 of a word whose sign bits have
// been flipped (u = code + 128).  fp16: 0x6400 + u is 1024 + u, less 1152.  bf16, whose numbers from 128 to 256 are whole
// ones: 128 + the low seven bits, less 128 or 256 as the top bit says; two instructions more.
template <typename M> __device__ __forceinline__ uint32_t code_pair(uint32_t word, int i);
template <> __device__ __forceinline__ uint32_t code_pair<__half>(uint32_t word, int i) {
  const uint32_t u = __byte_perm(word, 0x64646464u, i ? 0x4342 : 0x4140), bias = 0x64806480u;
  const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&u), *reinterpret_cast<const __half2*>(&bias));
  return *reinterpret_cast<const uint32_t*>(&d);
}
template <> __device__ __forceinline__ uint32_t code_pair<__nv_bfloat16>(uint32_t word, int i) {
  const uint32_t u = __byte_perm(word, 0, i ? 0x4342 : 0x4140);
  const uint32_t low = (u & 0x007f007fu) | 0x43004300u, less = (u & 0x00800080u) ^ 0x43804380u;
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&low), *reinterpret_cast<const __nv_bfloat162*>(&less));
  return *reinterpret_cast<const uint32_t*>(&d);
}
// The 16 codes `w` of a row as numbers of type M: two pieces of its tile.
template <typename M, int ROWS>
__device__ __forceinline__ void store_codes(uint32_t tile, int row, int piece, uint4 w) {
  const uint32_t u[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
#pragma unroll
  for (int h = 0; h < 2; ++h)
    store16(tile + tile_offset<ROWS>(row, 2 * piece + h),
            make_uint4(code_pair<M>(u[2 * h], 0), code_pair<M>(u[2 * h], 1), code_pair<M>(u[2 * h + 1], 0), code_pair<M>(u[2 * h + 1], 1)));
}
// Queries in bf16 that meet codes become fp16: a row, held by LANES neighbouring threads as 16-byte pieces, is multiplied by
// the power of two that brings its largest value to 2^14 (what is lost is 2^-38 of that value; an infinity or a NaN stays
// one).  Returns the power's reciprocal.
template <int LANES>
__device__ __forceinline__ float row_to_half(uint4& v) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
  uint32_t most = 0;  // bits of the largest magnitude
#pragma unroll
  for (int i = 0; i < 4; ++i) most = max(most, max((w[i] & 0x7fffu) << 16, w[i] & 0x7fff0000u));
#pragma unroll
  for (int off = 1; off < LANES; off <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, off));
  const int e = most == 0 ? 14 : min(max(int(most >> 23) - 127, -112), 126);
  const float up = __uint_as_float(uint32_t(127 + 14 - e) << 23);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = Half2<__nv_bfloat16>::unpack(w[i]);
    w[i] = Half2<__half>::pack(x.x * up, x.y * up);
  }
  return __uint_as_float(uint32_t(127 - 14 + e) << 23);
}

// ---- keys of a paged sequence into tiles, by the 128 threads of a warpgroup ------------------------------------------------
// The code is short on purpose: what a CTA runs for the first time it first has to fetch, and unrolled copies were 10 us of
// instruction fetches in front of the first product.
struct PoolView {
  const char* rows;
  const float* scales;
  int kv_heads, page_shift;
  // Row of key `key` of a sequence in page `id`.
  __device__ __forceinline__ int64_t line(int id, int head, int key) const {
    return ((int64_t(id) * kv_heads + head) << page_shift) + (key & ((1 << page_shift) - 1));
  }
};
// Keys [low, length) of a sequence exist.  Lane i of every warp knows the page of the i-th run of 16 keys from key0 on, -1
// where there is none; `bad`: runs whose page is outside the pool although a key of theirs exists.
struct KeyRuns {
  int key0, low, length, id;
  uint32_t bad;
  __device__ __forceinline__ void look_up(const int32_t* row, int page_shift, int pages, int runs, int first_key, int first_existing, int sequence_length) {
    key0 = first_key;
    low = first_existing;
    length = sequence_length;
    const int lane = threadIdx.x & 31, key = key0 + 16 * lane;
    const bool exists = lane < runs && key < length && key + 16 > low;
    id = exists ? __ldg(row + (key >> page_shift)) : -1;
    bad = __ballot_sync(0xffffffffu, exists && (id < 0 || id >= pages));
    if (id >= pages) id = -1;
  }
};

// 16-bit rows: 16 bytes at a time straight into place, ROWS of them (tiles of 128 lie `tile_bytes` apart); rows that are not
// there become zeros (a stale NaN in V would spoil the product with a probability of 0).
template <int D, int ROWS>
__device__ __forceinline__ void copy_keys(const PoolView& pool, const KeyRuns& k, int head, uint32_t to, int tile_bytes, int thread) {
  constexpr int PIECES = D / 8, EACH = 128 / PIECES;  // rows that the warpgroup copies at a time
  const int piece = thread % PIECES;
#pragma unroll 4
  for (int r = thread / PIECES; r < ROWS; r += EACH) {
    const int key = k.key0 + r, page = __shfl_sync(0xffffffffu, k.id, r >> 4);
    const bool there = page >= 0 && key >= k.low && key < k.length;
    const int64_t line = there ? pool.line(page, head, key) : 0;
    copy16(to + (ROWS > 128 ? (r >> 7) * tile_bytes : 0) + tile_offset<(ROWS > 128 ? 128 : ROWS)>(r & 127, piece), pool.rows + line * (D * 2) + piece * 16, there);
  }
}
// Codes, 16 of them per load; a batch is what a thread has on its way at once, from row `from` of the tile on.
template <int D>
struct CodeBatch {
  static constexpr int PIECES = D / 16, EACH = 128 / PIECES, COUNT = 4, ROWS = COUNT * EACH;
  uint4 codes[COUNT];
  __device__ __forceinline__ void load(const PoolView& pool, const KeyRuns& k, int head, int from, int thread) {
    const int piece = thread % PIECES;
#pragma unroll
    for (int n = 0; n < COUNT; ++n) {
      const int r = from + thread / PIECES + n * EACH, key = k.key0 + r, page = __shfl_sync(0xffffffffu, k.id, r >> 4);
      const bool there = page >= 0 && key >= k.low && key < k.length;
      codes[n] = there ? *reinterpret_cast<const uint4*>(pool.rows + pool.line(page, head, key) * D + piece * 16) : make_uint4(0, 0, 0, 0);
    }
  }
  // As numbers of type M, into tiles of TILE rows that lie `tile_bytes` apart.
  template <typename M, int TILE>
  __device__ __forceinline__ void store(uint32_t to, int tile_bytes, int from, int thread) const {
    const int piece = thread % PIECES;
#pragma unroll
    for (int n = 0; n < COUNT; ++n) {
      const int r = from + thread / PIECES + n * EACH;
      store_codes<M, TILE>(to + r / TILE * tile_bytes, r % TILE, piece, codes[n]);
    }
  }
};

}  // namespace serving
}  // namespace risa_b200
