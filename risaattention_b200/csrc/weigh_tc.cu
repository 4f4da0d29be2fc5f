// The attention that cached keys receive from many query rows, on the tensor cores.
//
// With the rows' log-sum-exp known a weight needs no maximum and no order: w_j = sum over rows of 2^(s_rj - lse_r).  So
// the roles of the attention kernel turn around: 256 keys stay (the A operand, two groups of 128), query rows stream
// past them (128 at a time, the B operand), scores S = K Q^T arrive with a key per lane of tensor memory, and the
// thread that owns a key adds up its row of exponentials in a register.  K is read once, nothing is written but the
// weights.  What bounds it is the exponentials: one per (key, row) and 16 per clock and SM, 2048 clocks for 256 keys x
// 128 rows, against 1024 of the matrix instruction at 128 channels.  A tile takes 2550; 1024 tokens over 8K keys, 32 heads:
// 108 us in short runs (117 with the clock of long ones), of which ~10 are start-up; 16 tokens over 4 x 16K keys of 64
// channels: 48.  Exponentials by polynomial on the FP32 pipes for an eighth to three eighths of them cost as much issue time
// as they saved.
//
// Warps 0-15: the sums, four warpgroups: two for each group of keys, each with half of a tile's rows (four warps a
// scheduler hide the latencies of tensor memory and the exponential; two left a third of the time idle).  16-19: fetch
// query rows.  20-23: fetch keys.  24: issues the products.
#include "paged_tc.cuh"
#include "tc_f16.cuh"

#include <climits>

namespace risa_b200 {
namespace serving {

using namespace tc;

namespace {

constexpr int kThreads = 800;
constexpr int kBlockKeys = 256;
constexpr int kFetcher = 16, kKeyFetcher = 20, kIssuer = 24;
// Notes and log-sum-exps of the tiles in flight.  A slot is written again kDepth tiles later, by when the sums have
// left it: the fetchers are at most the query stages ahead of the issuer, the issuer two tiles ahead of the sums.
constexpr int kDepth = 8;
// Half sums on their way between the two warpgroups of a key group, each slot with a barrier of its own.  The scores of tile t
// are issued once all eight warps have freed those of tile t - 2, and a warp frees a tile before it hands over or takes the
// block that ends with it; so the giver is at most two blocks ahead of a warp that still has to take, three slots are in use,
// and the giver comes back to a slot only after every taker has passed it.  (One barrier waited for by parity would need the
// giver to be less than two phases ahead.)
constexpr int kHalves = 4;
// Bits of a note: first and last tile of a block, whether the block has more than 128 keys.
constexpr uint32_t kFirst = 1u, kLast = 2u, kTwoGroups = 4u;

// Blocks of 256 keys and steps of query rows (serving_plan.cuh's line the other way round).
struct WeighLine {
  StepView step;
  int kv_heads;
  Divisor group;
  int min_rows;
  Divisor tile_rows;  // query rows of a step
  int causal, window;
  int sinks;          // first keys that stay visible in front of a window
};
__device__ __forceinline__ int first_seen(const WeighLine& a, const Sequence& q) {
  return a.window > 0 ? visible(q.length - q.count, q.length, true, a.window).lo : 0;
}
// Blocks of the first keys that stay visible, as far as they lie in front of the window's.
__device__ __forceinline__ int front_blocks(const WeighLine& a, const Sequence& q) {
  return min((a.sinks + kBlockKeys - 1) / kBlockKeys, first_seen(a, q) / kBlockKeys);
}
__device__ __forceinline__ int blocks_of(const WeighLine& a, const Sequence& q) {
  if (q.count == 0 || q.count * a.group < a.min_rows || q.length == 0) return 0;
  return front_blocks(a, q) + (q.length + kBlockKeys - 1) / kBlockKeys - first_seen(a, q) / kBlockKeys;
}
__device__ __forceinline__ int first_key_of(const WeighLine& a, const Sequence& q, int block) {
  const int front = front_blocks(a, q);
  return (block < front ? block : first_seen(a, q) / kBlockKeys + block - front) * kBlockKeys;
}
// Rows [lo, hi) of the sequence that see a key; hi is INT_MAX where no window ends them.
struct RowRange {
  int lo, hi;
};
__device__ __forceinline__ RowRange rows_of(const WeighLine& a, const Sequence& q, int key) {
  if (!a.causal) return {0, INT_MAX};
  const int base = q.length - q.count;  // place of the first new token
  const int lo = min(max(key - base, 0), q.count) * a.group;
  if (a.window == 0 || key < a.sinks) return {lo, INT_MAX};
  const int64_t end = int64_t(key) + a.window - base;
  return {lo, end <= 0 ? 0 : end >= q.count ? INT_MAX : int(end) * a.group};
}
__device__ __forceinline__ StepRange steps_of(const WeighLine& a, const Sequence& q, int block) {
  const int key0 = first_key_of(a, q, block);
  const int rows = q.count * a.group, from = rows_of(a, q, key0).lo, to = min(rows_of(a, q, key0 < a.sinks ? key0 : key0 + kBlockKeys - 1).hi, rows);
  const int first = min(from, rows - 1) / a.tile_rows, end = (to + a.tile_rows - 1) / a.tile_rows;
  return {first, max(end - first, 1)};
}

struct WeighArgs {
  WeighLine line;
  const void* q;
  int64_t qn, qh;
  const float* row_lse;
  PoolView keys;
  int pages;
  float scale_log2;
  const float* previous;
  float* weights;
  float* parts;  // two slots of 256 floats per worker
  JoinNote* notes;  // as attention's, but for `rows`: the block's first key
  int min_steps;
  unsigned int* status;
};

template <typename T_, int BITS_, int D_>
struct Shape {
  using T = T_;
  static constexpr int BITS = BITS_;
  static constexpr bool CODES = BITS < 16;
  static constexpr int D = D_;
  static constexpr int ROWS = D == 256 ? 64 : 128;  // query rows of a tile
  static constexpr int GROUP = 128 * D * 2;         // 128 keys
  static constexpr int KEYS = 2 * GROUP, KEY_BUFFERS = D == 256 ? 1 : 2;
  static constexpr int TILE = ROWS * D * 2, STAGES = D == 64 ? 4 : 2;
  static constexpr int SMEM = KEY_BUFFERS * KEYS + STAGES * TILE + 1024;
  static_assert(STAGES + 2 < kDepth, "notes outlive their readers");
};

struct Barriers {
  uint64_t k_full[2], k_empty[2], q_full[4], q_empty[4], s_full[2][2], s_free[2][2], half_full[2][kHalves], drained;
};

// Byte offset of piece `piece` of row `row` in a tile of ROWS query rows.
template <int ROWS>
__device__ __forceinline__ uint32_t query_offset(int row, int piece) {
  return uint32_t((piece >> 3) * (ROWS * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
}

struct Notes {
  uint32_t tile[kDepth];
  uint32_t bad[kDepth];          // runs of 16 keys whose page is outside the pool, of the last blocks
  float minus_lse[kDepth][128];  // in units of log 2; -infinity for rows that give nothing
  float half[kHalves][2][128];   // what the second half of the rows adds to a key, of the last blocks
};

// A worker's key blocks.
template <typename C>
__device__ __forceinline__ void fetch_keys(const WeighArgs& a, Pieces pieces, Barriers* bars, volatile Notes* notes, uint32_t keys, uint32_t gave_up) {
  const int p = threadIdx.x - kKeyFetcher * 32;
  RingPos<C::KEY_BUFFERS> kb;
  uint32_t block = 0;
  Piece at;
  while (pieces.next(a.line, at)) {
    const int32_t* row = a.line.step.table + int64_t(at.sequence) * a.line.step.width;
    const int low = first_seen(a.line, at.seq), length = at.seq.length, key0 = first_key_of(a.line, at.seq, at.block);
    KeyRuns runs;
    runs.look_up(row, a.line.step.page_shift, a.pages, kBlockKeys / 16, key0, low, a.line.sinks, length);
    if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(bars->k_empty + kb.stage), kb.phase ^ 1, gave_up, 1101))) break;
    if (p == 0) {
      notes->bad[block % kDepth] = runs.bad;
      if (runs.bad) atomicCAS(a.status, 0u, unsigned(at.sequence) + 1u);
    }
    const uint32_t to = keys + kb.stage * C::KEYS;
    // codes as they are: a key's scale multiplies its scores in 32 bits.  (A batch ahead in registers, 4-bit ones too: a block of keys
    // stays for all query rows, and 1024 tokens over 8K keys, 32 heads of 128, take 111 us over 4 bits and INT8, 108 over bf16.)
    if constexpr (C::CODES) {
      using Batch = CodeBatch<C::D, C::BITS>;
      Batch batch, next;
      batch.load(a.keys, runs, at.head, 0, p);
#pragma unroll 1
      for (int from = 0; from < kBlockKeys; from += Batch::ROWS) {
        if (from + Batch::ROWS < kBlockKeys) next.load(a.keys, runs, at.head, from + Batch::ROWS, p);
        batch.template store<typename C::T, 128>(to, C::GROUP, from, p);
        batch = next;
      }
    } else {
      copy_keys<C::D, kBlockKeys>(a.keys, runs, at.head, to, C::GROUP, p);
    }
    if (C::CODES) {
      fence_async_smem();
      mbar_arrive(smem_u32(bars->k_full + kb.stage));
    } else {
      copies_arrive(smem_u32(bars->k_full + kb.stage));
    }
    mbar_arrive_warp(smem_u32(bars->k_full + kb.stage));  // the note is there
    kb.next();
    ++block;
  }
  copies_drain();
}

template <typename C>
__device__ __forceinline__ void fetch_queries(const WeighArgs& a, Pieces pieces, Barriers* bars, volatile Notes* notes, uint32_t queries,
                                      uint32_t gave_up) {
  const int p = threadIdx.x - kFetcher * 32;
  RingPos<C::STAGES> st;
  uint32_t tile = 0;
  Piece piece;
  auto lse_of = [&](const Piece& at, int tile) {  // this thread's row of a tile
    const int r = tile * C::ROWS + p, rows = at.seq.count * a.line.group;
    if (p >= C::ROWS || r >= rows) return -INFINITY;
    const int token = r / a.line.group;
    return __ldg(a.row_lse + int64_t(at.seq.first + token) * (a.line.kv_heads * a.line.group) + at.head * a.line.group + r - token * a.line.group);
  };
  bool more = pieces.next(a.line, piece);
  float lse = lse_of(piece, piece.first);
  while (more) {
    const Piece now = piece;
    const Sequence& seq = now.seq;
    const int key0 = first_key_of(a.line, seq, now.block), rows = seq.count * a.line.group;
    more = pieces.next(a.line, piece);
    constexpr int PIECES = C::D / 8, ROWS_EACH = 128 / PIECES;  // rows that the warpgroup copies at a time
    constexpr int COPIES = C::ROWS / ROWS_EACH;
    static_assert(ROWS_EACH == 4 || ROWS_EACH % 8 == 0, "a thread's rows lie alike in the swizzle");
    const int c = p % PIECES, r0 = p / PIECES;
    const int tokens_each = ROWS_EACH / a.line.group;
    const int64_t each = tokens_each * a.qn + (ROWS_EACH - tokens_each * a.line.group) * a.qh, wrap = a.qn - a.line.group * a.qh;
    for (int i = 0; i < now.count; ++i, ++tile) {
      const float x = lse;
      if (i + 1 < now.count) lse = lse_of(now, now.first + i + 1);
      else if (more) lse = lse_of(piece, piece.first);
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(bars->q_empty + st.stage), st.phase ^ 1, gave_up, 1102))) return copies_drain();
      int row = (now.first + i) * C::ROWS + r0;
      const int token = row / a.line.group;
      int h = row - token * a.line.group;
      const typename C::T* from = static_cast<const typename C::T*>(a.q) + int64_t(seq.first + token) * a.qn + int64_t(now.head * a.line.group + h) * a.qh + c * 8;
      const uint32_t to = queries + st.stage * C::TILE;
#pragma unroll
      for (int n = 0; n < COPIES; ++n) {
        // a row that does not exist is not read; the address then is the queries' own
        const bool there = row < rows;
        copy16(to + (ROWS_EACH % 8 == 0 ? query_offset<C::ROWS>(r0, c) + n * ROWS_EACH * 128 : query_offset<C::ROWS>(r0 + n * ROWS_EACH, c)),
               there ? from : static_cast<const typename C::T*>(a.q), there);
        row += ROWS_EACH;
        from += each;
        h += ROWS_EACH - tokens_each * a.line.group;
        if (h >= a.line.group) {
          h -= a.line.group;
          from += wrap;
        }
      }
      copies_arrive(smem_u32(bars->q_full + st.stage));
      if (p < C::ROWS) notes->minus_lse[tile % kDepth][p] = x == -INFINITY ? -INFINITY : -x * kLog2e;
      if (p == 0)
        notes->tile[tile % kDepth] = (i == 0 ? kFirst : 0u) | (i + 1 == now.count ? kLast : 0u) | (seq.length - key0 > 128 ? kTwoGroups : 0u);
      mbar_arrive_warp(smem_u32(bars->q_full + st.stage));  // the notes are there
      st.next();
    }
  }
  copies_drain();
}

template <typename C>
__device__ __forceinline__ void issue(int tiles, Barriers* bars, const volatile Notes* notes, uint32_t tmem, uint32_t keys, uint32_t queries,
                                      uint32_t gave_up) {
  constexpr uint32_t kScores = idesc_f16<typename C::T>(false, C::ROWS);
  RingPos<C::KEY_BUFFERS> kb;
  RingPos<C::STAGES> st;
  RingPos<2> buffer;
  const bool elected = elect_one();
  for (int tile = 0; tile < tiles; ++tile) {
    if (!mbar_wait(smem_u32(bars->q_full + st.stage), st.phase, gave_up, 1110)) return;
    const uint32_t note = notes->tile[tile % kDepth];
    if ((note & kFirst) && !mbar_wait(smem_u32(bars->k_full + kb.stage), kb.phase, gave_up, 1111)) return;
    fence_async_smem();  // the copies that the barriers have told of
    const int groups = note & kTwoGroups ? 2 : 1;
    for (int g = 0; g < 2; ++g) {
      // both groups' buffers take turns together, so a group that sits out hands its buffer on
      if (!mbar_wait(smem_u32(&bars->s_free[g][buffer.stage]), buffer.phase ^ 1, gave_up, 1112 + g)) return;
      tc_fence_after();
      if (!elected) continue;
      if (g < groups) {
        const uint32_t rows_k = along_row(keys + kb.stage * C::KEYS + g * C::GROUP), rows_q = along_row(queries + st.stage * C::TILE);
        const uint32_t to = tmem + (g * 2 + buffer.stage) * 128;
#pragma unroll 2
        for (int c = 0; c < C::D / 16; ++c)
          mma_f16(to, descriptor(rows_k + (c >> 2) * 1024 + (c & 3) * 2), descriptor(rows_q + (c >> 2) * (C::ROWS * 8) + (c & 3) * 2), kScores, c > 0);
      }
      mma_commit(smem_u32(&bars->s_full[g][buffer.stage]));
    }
    if (elected) {
      mma_commit(smem_u32(bars->q_empty + st.stage));
      if (note & kLast) mma_commit(smem_u32(bars->k_empty + kb.stage));
    }
    if (note & kLast) kb.next();
    st.next();
    buffer.next();
  }
}

// Adds the exponentials of ROWS query rows (from column `from` on) to a key's sum.  Every row sees the key, or (MASKED) rows
// [lo, hi) of the sequence do, the first column being row `row0`.
template <int ROWS, bool MASKED>
__device__ __forceinline__ void add_rows(uint32_t columns, const float* minus_lse, float factor, int row0, const RowRange& seen, float (&sum)[4],
                                         uint32_t freed) {
#pragma unroll
  for (int c = 0; c < ROWS; c += 32) {
    uint32_t x[32];
    tmem_load32(columns + c, x);
    tmem_load_wait();
    tmem_regs_ready<32>(x);
    if (c + 32 == ROWS) {
      tc_fence_before();
      mbar_arrive_warp(freed);
    }
    float u[32];
#pragma unroll
    for (int e = 0; e < 32; e += 4) {
      const float4 l = *reinterpret_cast<const float4*>(minus_lse + c + e);
      u[e] = fmaf(__uint_as_float(x[e]), factor, l.x);
      u[e + 1] = fmaf(__uint_as_float(x[e + 1]), factor, l.y);
      u[e + 2] = fmaf(__uint_as_float(x[e + 2]), factor, l.z);
      u[e + 3] = fmaf(__uint_as_float(x[e + 3]), factor, l.w);
    }
    if (MASKED) {
      const int lo = seen.lo - row0 - c, hi = seen.hi - row0 - c;
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (e < lo || e >= hi) u[e] = -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) u[e] = ex2_approx(u[e]);
#pragma unroll
    for (int e = 0; e < 32; ++e) sum[e & 3] += u[e];
  }
}

template <typename C>
__device__ __forceinline__ void add_up(const WeighArgs& a, Pieces pieces, Barriers* bars, uint32_t tmem, int g, int half, Notes* notes,
                                       uint32_t gave_up) {
  constexpr int ROWS = C::ROWS / 2;
  const int lane = threadIdx.x & 127;
  const uint32_t columns = tmem + (uint32_t(lane & ~31) << 16) + g * 256 + half * ROWS;
  const int slots = a.line.step.width << a.line.step.page_shift;
  RingPos<2> buffer;
  uint32_t tile = 0, block = 0;
  Piece piece;
  while (pieces.next(a.line, piece)) {
    const Sequence& seq = piece.seq;
    const int low = first_seen(a.line, seq), key0 = first_key_of(a.line, seq, piece.block) + g * 128, key = key0 + lane;
    const bool exists = (key >= low || key < a.line.sinks) && key < seq.length;
    const bool takes_part = g == 0 || seq.length - key0 > 0;
    RowRange mine = rows_of(a.line, seq, key);
    // the first to lose sight of a key of the group are those of its first key that is not always visible
    const int all_lo = rows_of(a.line, seq, key0 + 127).lo, all_hi = rows_of(a.line, seq, min(max(key0, a.line.sinks), key0 + 127)).hi;
    bool whole_group = (key0 >= low || key0 + 128 <= a.line.sinks) && key0 + 128 <= seq.length;
    if (!exists) mine.hi = 0;
    float factor = a.scale_log2;
    if (C::CODES && exists) {
      const int id = __ldg(a.line.step.table + int64_t(piece.sequence) * a.line.step.width + (key >> a.line.step.page_shift));
      if (id >= 0 && id < a.pages) {
        if (C::BITS == 4)
          factor *= power_of(__ldg(scales4<C::D>(a.keys.scales, id, a.keys.kv_heads, piece.head, a.keys.page_shift) + (key & ((1 << a.keys.page_shift) - 1))));
        else
          factor *= __ldg(a.keys.scales + a.keys.line(id, piece.head, key));
      }
    }
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < piece.count; ++i, ++tile) {
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&bars->s_full[g][buffer.stage]), buffer.phase, gave_up, 1120 + g))) return;
      tc_fence_after();
      if (i == 0) {
        const uint32_t bad = notes->bad[block % kDepth] >> (8 * g) & 0xff;
        if (bad != 0) whole_group = false;
        if (bad >> (lane >> 4) & 1) mine.hi = 0;
      }
      const uint32_t freed = smem_u32(&bars->s_free[g][buffer.stage]);
      if (takes_part) {
        const int row0 = (piece.first + i) * C::ROWS + half * ROWS;
        const float* lse = notes->minus_lse[tile % kDepth] + half * ROWS;
        if (whole_group && row0 >= all_lo && row0 <= all_hi - ROWS) {
          add_rows<ROWS, false>(columns + buffer.stage * 128, lse, factor, row0, mine, sum, freed);
        } else {
          add_rows<ROWS, true>(columns + buffer.stage * 128, lse, factor, row0, mine, sum, freed);
        }
      } else {
        mbar_arrive_warp(freed);
      }
      buffer.next();
    }
    float total = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    float* other = &notes->half[block % kHalves][g][lane];
    const uint32_t handed = smem_u32(&bars->half_full[g][block % kHalves]), parity = block / kHalves & 1;
    ++block;
    if (half == 1) {
      *other = total;
      mbar_arrive_warp(handed);
      continue;
    }
    if (!__all_sync(0xffffffffu, mbar_wait(handed, parity, gave_up, 1122 + g))) return;
    total += *other;
    if (!piece.whole) {
      a.parts[(int64_t(blockIdx.x) * 2 + (piece.opens ? 1 : 0)) * kBlockKeys + g * 128 + lane] = total;
    } else if (key < slots) {
      const int64_t index = (int64_t(piece.sequence) * a.line.kv_heads + piece.head) * slots + key;
      a.weights[index] = total + (a.previous != nullptr ? a.previous[index] : 0.f);
    }
  }
}

template <typename C>
__global__ __launch_bounds__(kThreads, 1) void weigh_tc_kernel(const WeighArgs a) {
  extern __shared__ char smem_raw[];
  __shared__ Barriers bars;
  __shared__ LineShared<kThreads> shared;
  __shared__ uint32_t tmem_base, gave_up_word;
  __shared__ __align__(16) Notes notes;
  const int warp = threadIdx.x >> 5;
  const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
  const uint32_t keys = smem, queries = keys + C::KEY_BUFFERS * C::KEYS, gave_up = smem_u32(&gave_up_word);
  if (threadIdx.x == 0) {
    gave_up_word = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(bars.k_full + i), 128 + 4);
      mbar_init(smem_u32(bars.k_empty + i), 1);
      for (int j = 0; j < kHalves; ++j) mbar_init(smem_u32(&bars.half_full[i][j]), 4);
      for (int g = 0; g < 2; ++g) {
        mbar_init(smem_u32(&bars.s_full[g][i]), 1);
        mbar_init(smem_u32(&bars.s_free[g][i]), 8);
      }
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(bars.q_full + i), 128 + 4);
      mbar_init(smem_u32(bars.q_empty + i), 1);
    }
    mbar_init(smem_u32(&bars.drained), 1);
    mbar_init_fence();
  }
  chain_release();  // and no wait: see paged_tc_kernel
  // what no block covers: in front of the window (but for the first keys that stay visible), behind the length
  const int slots = a.line.step.width << a.line.step.page_shift;
  for (int64_t u = blockIdx.x; u < int64_t(a.line.step.batch) * a.line.kv_heads; u += gridDim.x) {
    const Sequence seq = sequence_of(a.line.step, int(u / a.line.kv_heads));
    if (seq.count * a.line.group < a.line.min_rows) continue;
    const int blocks = blocks_of(a.line, seq), block0 = first_seen(a.line, seq) / kBlockKeys;
    const int front = blocks == 0 ? 0 : front_blocks(a.line, seq), from = blocks == 0 ? 0 : block0 * kBlockKeys;
    const int to = blocks == 0 ? 0 : min((block0 + blocks - front) * kBlockKeys, slots);
    for (int i = front * kBlockKeys + threadIdx.x; i < slots - (to - from); i += kThreads) {
      const int64_t index = u * slots + (i < from ? i : i + (to - from));
      a.weights[index] = a.previous != nullptr ? a.previous[index] : 0.f;
    }
  }
  const int64_t total = line_total<kThreads>(a.line, shared);
  const int workers = workers_of(total, gridDim.x, a.min_steps);
  if (int(blockIdx.x) >= workers) {
    if (threadIdx.x == 0) a.notes[blockIdx.x] = JoinNote{};
    chain_wait();
    return;
  }
  const int64_t begin = border(total, blockIdx.x, workers), finish = border(total, blockIdx.x + 1, workers);
  const Pieces pieces{finish - begin, line_place<kThreads>(a.line, begin, shared)};
  if (warp == kIssuer) tmem_alloc(smem_u32(&tmem_base), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  if (warp < kFetcher) {
    add_up<C>(a, pieces, &bars, tmem, warp >> 3, (warp >> 2) & 1, &notes, gave_up);
  } else if (warp < kKeyFetcher) {
    fetch_queries<C>(a, pieces, &bars, &notes, queries, gave_up);
  } else if (warp < kIssuer) {
    fetch_keys<C>(a, pieces, &bars, &notes, keys, gave_up);
  } else if (warp == kIssuer) {
    if ((threadIdx.x & 31) == 0) {
      Pieces all = pieces;
      Piece last;
      while (all.next(a.line, last)) {}
      JoinNote note{};
      if (last.opens && !last.whole) {
        const int64_t end = finish - last.count + steps_of(a.line, last.seq, last.block).count;
        note = {last.seq.first, first_key_of(a.line, last.seq, last.block), last.head, last.block,
                min(worker_from(total, end, workers), workers) - int(blockIdx.x), last.sequence};
      }
      a.notes[blockIdx.x] = note;
    }
    __syncwarp();
    issue<C>(int(pieces.left), &bars, &notes, tmem, keys, queries, gave_up);
    __syncwarp();
    // nothing of this CTA is in flight when tensor memory is handed back, also after a wait that ran out
    if (elect_one()) mma_commit(smem_u32(&bars.drained));
    __syncwarp();
    mbar_drain(smem_u32(&bars.drained), 0);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kIssuer) tmem_dealloc(tmem, 512);
  if (gave_up_word != 0 && threadIdx.x < kBlockKeys) {
    // a wait ran out: this worker's weights are marked
    Pieces all = pieces;
    Piece piece;
    while (all.next(a.line, piece)) {
      const int key = first_key_of(a.line, piece.seq, piece.block) + threadIdx.x;
      if (!piece.whole) a.parts[(int64_t(blockIdx.x) * 2 + (piece.opens ? 1 : 0)) * kBlockKeys + threadIdx.x] = NAN;
      else if (key < slots) a.weights[(int64_t(piece.sequence) * a.line.kv_heads + piece.head) * slots + key] = NAN;
    }
  }
  chain_wait();
}

// The parts of the block that worker blockIdx.x ended with, added up in order.
__global__ __launch_bounds__(kBlockKeys) void join_weights_kernel(const WeighArgs a) {
  chain_wait();
  chain_release();
  const JoinNote note = a.notes[blockIdx.x];
  if (note.parts == 0) return;
  float sum = a.parts[(int64_t(blockIdx.x) * 2 + 1) * kBlockKeys + threadIdx.x];
  for (int i = 1; i < note.parts; ++i) sum += a.parts[(int64_t(blockIdx.x) + i) * 2 * kBlockKeys + threadIdx.x];
  const int slots = a.line.step.width << a.line.step.page_shift, key = note.rows + threadIdx.x;
  if (key >= slots) return;
  const int64_t index = (int64_t(note.sequence) * a.line.kv_heads + note.head) * slots + key;
  a.weights[index] = sum + (a.previous != nullptr ? a.previous[index] : 0.f);
}

template <typename C>
int launch(WeighArgs a, cudaStream_t stream) {
  a.line.tile_rows = Divisor(C::ROWS);
  if (cudaFuncSetAttribute(weigh_tc_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
    return fail(RISA_B200_CUDA, "key weights: %s", cudaGetErrorString(cudaGetLastError()));
  if (const int bad = launched(launch_chained(weigh_tc_kernel<C>, dim3(kTcWorkers), dim3(kThreads), C::SMEM, stream, a), "key weights")) return bad;
  return launched(launch_chained(join_weights_kernel, dim3(kTcWorkers - 1), dim3(kBlockKeys), 0, stream, a), "key weights");
}
template <typename T, int BITS>
int launch_bits(const WeighArgs& a, int head_dim, cudaStream_t stream) {
  return head_dim == 64 ? launch<Shape<T, BITS, 64>>(a, stream) : head_dim == 128 ? launch<Shape<T, BITS, 128>>(a, stream) : launch<Shape<T, BITS, 256>>(a, stream);
}
template <typename T>
int launch_for(const WeighArgs& a, int bits, int head_dim, cudaStream_t stream) {
  return bits == 4 ? launch_bits<T, 4>(a, head_dim, stream) : bits == 8 ? launch_bits<T, 8>(a, head_dim, stream) : launch_bits<T, 16>(a, head_dim, stream);
}

}  // namespace

size_t weigh_tc_scratch() { return size_t(kTcWorkers) * (2 * kBlockKeys * sizeof(float) + sizeof(JoinNote)); }

int weigh_tc(const TcArgs& t, const float* row_lse, const float* previous, float* weights, int dtype_code, int bits, int head_dim,
             cudaStream_t stream) {
  const WeighArgs a{{t.line.step, t.line.kv_heads, t.line.group, t.line.min_rows, Divisor(), t.line.causal, t.line.window, t.line.sinks},
                    t.q, t.qn, t.qh, row_lse, {t.keys, t.key_scales, t.line.kv_heads, t.line.step.page_shift}, t.pages, t.scale_log2,
                    previous, weights, t.parts, reinterpret_cast<JoinNote*>(t.parts + size_t(kTcWorkers) * 2 * kBlockKeys), t.min_steps, t.status};
  return dtype_code == 1 ? launch_for<__half>(a, bits, head_dim, stream) : launch_for<__nv_bfloat16>(a, bits, head_dim, stream);
}

int weigh_tc_wait_status() {
  unsigned int status = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&status, g_wait_status, sizeof(status)) != cudaSuccess) return -1;
  if (status != 0) cudaMemcpyToSymbol(g_wait_status, &zero, sizeof(zero));
  return int(status);
}

}  // namespace serving
}  // namespace risa_b200
