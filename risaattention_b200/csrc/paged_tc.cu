// Attention of many query rows (chunks of prompts) over a paged cache on the tensor cores.
//
// A unit is 256 query rows of one key head, rows in the order (token, head of the group), so that all heads of a
// group share every key tile; two groups of 128 rows, each with accumulators of its own, take turns on the tensor pipe:
// while one group's scores become probabilities, the other's matrix products run.  Per 128-key tile and group:
// S = Q K^T (128 x 128 x head_dim, fp32 in tensor memory); two threads own a row, each reads 64 of its scores into
// registers, they exchange maxima (lanes of tensor memory are rows, so sums need no shuffle) and write P (16 bits) over
// the first half of S's columns; O += P V takes P from tensor memory and V from shared memory as it lies there (keys
// along K, channels contiguous).
//
// What bounds it: per tile and group the tensor pipe works 1024 clocks (head_dim 128) and the special-function unit 1024;
// the chain of a group's softmax (2100: load, maxima with an exchange, exponentials, store) and products (1450) is hidden
// by the other group's to about one half, so a tile of both takes 3850.  2048 tokens over 32K keys, 32 heads of 128 channels:
// 1.16 ms, 916 TFLOP/s, at the clock that the power limit leaves.  One thread for a row: the same; an issue warp per group let
// the groups fall into step (5500 clocks a tile); half of the next scores ahead of P V (N = 64 products) 4600; K and V by 128 copying threads
// instead of TMA 6300; exponentials from the maximum as it stood, redone where it had moved, ran out of registers (5600).
//
// Heads of 256 channels leave room for the outputs of 128 rows only.  There the two groups have the same rows and half of
// the channels of V each, over tiles of 64 keys; the scores are computed twice (3 products for 2) in exchange for the same
// taking of turns.
//
// Warps 0-15: softmax, query loads and epilogue, four for each half of the columns of each row group.  16-19: fetch K
// and V tiles from the pages (cp.async, or codes converted on the way) into the 128-byte-swizzled layout of the matrix
// instructions.  20: issues them (and owns tensor memory).  21-23 idle, so that registers can be dealt per warpgroup.
#include "serving_plan.cuh"
#include "paged_tc.cuh"
#include "tc_f16.cuh"

#include <algorithm>

namespace risa_b200 {
namespace serving {

using namespace tc;

namespace {

constexpr int kThreads = 768;
constexpr int kGroups = 2;
constexpr int kProducer = 16, kIssuer = 20;  // first warps of their roles
// 768 threads of at most 85 registers are launched with 80; the softmax warps hold 64 scores of a row.
constexpr int kRegsLaunch = 80, kRegsSoftmax = 96, kRegsProducer = 56, kRegsIssuer = 40;
static_assert(128 * (4 * kRegsSoftmax + kRegsProducer + kRegsIssuer) <= kThreads * kRegsLaunch, "register budget");
// A note for each tile in flight: runs of 16 keys that are hidden because their page is outside the pool, whether the
// tile is the first or the last of its unit, and whether the unit has more than 128 rows.
constexpr int kNotes = 16;
constexpr uint32_t kHiddenRuns = 0xff, kFirst = 1u << 8, kLast = 1u << 9, kTwoGroups = 1u << 10;
// A running maximum is followed only when the true one has run ahead of it by 2^8: until then probabilities grow to at
// most 256, which 16-bit types hold with the same relative precision, and the output in tensor memory stays as it is.
constexpr float kStale = 8.0f;

template <typename T_, bool INT8_, int D_>
struct Shape {
  using T = T_;
  using M = std::conditional_t<INT8_, __half, T_>;  // type of the matrix instructions' operands
  static constexpr bool INT8 = INT8_;
  static constexpr int D = D_;
  static constexpr bool SHARED = D == 256;             // both groups have the same rows
  static constexpr int KEYS = SHARED ? 64 : 128;       // of a tile
  static constexpr int ROWS = SHARED ? 128 : 256;      // of a unit
  static constexpr int OUT = SHARED ? D / 2 : D;       // channels of a group's output
  static constexpr int SIDE = KEYS * D * 2;            // a K or V tile as the matrix instructions read it
  static constexpr int BLOCK = KEYS * 128;             // 64 channels of it
  static constexpr int STAGES = D == 64 ? 4 : 2;
  static constexpr int QUERIES = 128 * D * 2, Q = (SHARED ? 1 : kGroups) * QUERIES;
  static constexpr int SMEM = Q + 2 * STAGES * SIDE + 1024;  // + alignment
};

struct Barriers {
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t q_full[kGroups], s_full[kGroups], p_full[kGroups], o_full[kGroups], o_free[kGroups], q_empty, drained;
};
// What the two threads of a row tell each other: maxima (of tiles in turn) and sums.
struct Exchange {
  float maximum[2][kGroups][2][128];
  float sum[kGroups][2][128];
};
// Over a cache of codes: scales of the tiles in flight (a slot is written again kScaleDepth tiles later, by when the softmax
// that read it has handed over its probabilities), those of values also in units of log 2, and what the queries' rows were
// divided by, of this unit and the one before.
constexpr int kScaleDepth = 8;
struct Scales {
  float key[kScaleDepth][128], value[kScaleDepth][128], lift[kScaleDepth][128];
  float row[2][kGroups][128];
};

// ---- the fetching warpgroup -----------------------------------------------------------------------------------
// Tiles of 16-bit rows that all exist come by TMA, a box of 64 channels x a page at a time: 128 threads that copy 16
// bytes each took 2800 clocks for a tile in a scheduler's company of four softmax warps.  The others (a sequence's end, the
// front of a window, pages outside the pool) are copied piece by piece with zeros in place of what is not there.
template <typename C>
__device__ __forceinline__ void fetch_tiles(const TcArgs& a, const CUtensorMap* key_map, const CUtensorMap* value_map, Pieces pieces, Barriers* bars,
                                            volatile uint32_t* notes, Scales* scales, uint32_t k_ring, uint32_t v_ring, uint32_t gave_up) {
  const int p = threadIdx.x - kProducer * 32;
  uint32_t issued = 0;
  RingPos<C::STAGES> stage;  // of both rings
  Piece piece;
  const PoolView keys{a.keys, a.key_scales, a.line.kv_heads, a.line.step.page_shift}, values{a.values, a.value_scales, a.line.kv_heads, a.line.step.page_shift};
  // What is under way lands before the CTA ends, also when the issuer gave up on it (a stage that was never filled passes
  // at once); `keys_ahead` is 1 where K's stage of this tile is filled and V's is not.
  auto land = [&](int keys_ahead) {
    copies_drain();
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_drain(smem_u32(bars->k_full + i), i < stage.stage + keys_ahead ? stage.phase : stage.phase ^ 1);
      mbar_drain(smem_u32(bars->v_full + i), i < stage.stage ? stage.phase : stage.phase ^ 1);
    }
  };
  while (pieces.next(a.line, piece)) {
    const int32_t* row = a.line.step.table + int64_t(piece.sequence) * a.line.step.width;
    const int length = piece.seq.length;
    const int low = a.line.window > 0 ? visible(piece.seq.length - piece.seq.count, length, true, a.line.window).lo : 0;
    const uint32_t two = C::SHARED || piece.seq.count * a.line.group - piece.block * C::ROWS > 128 ? kTwoGroups : 0u;
    KeyRuns ahead;
    ahead.look_up(row, a.line.step.page_shift, a.pages, C::KEYS / 16, piece.first * C::KEYS, low, length);
    // over codes: the next batch is on its way while one is converted
    CodeBatch<C::D> batch;
    if (C::INT8) batch.load(keys, ahead, piece.head, 0, p);
#pragma unroll 1
    for (int i = 0; i < piece.count; ++i) {
      const KeyRuns runs = ahead;
      if (i + 1 < piece.count) ahead.look_up(row, a.line.step.page_shift, a.pages, C::KEYS / 16, runs.key0 + C::KEYS, low, length);
#pragma unroll 1
      for (int side = 0; side < 2; ++side) {  // K, then V
        uint64_t* full = side ? bars->v_full : bars->k_full;
        uint64_t* empty = side ? bars->v_empty : bars->k_empty;
        const uint32_t to = (side ? v_ring : k_ring) + stage.stage * C::SIDE;
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(empty + stage.stage), stage.phase ^ 1, gave_up, 1001 + side))) {
          land(side);
          return;
        }
        if constexpr (C::INT8) {
          // codes as they are; the softmax multiplies scores and probabilities by their keys' scales, in 32 bits
          if (side == 0) {
            const int key = runs.key0 + p, page = __shfl_sync(0xffffffffu, runs.id, p >> 4), slot = issued % kScaleDepth;
            const bool there = page >= 0 && key >= low && key < length;
            const int64_t line = there ? keys.line(page, piece.head, key) : 0;
            const float v = there ? __ldg(values.scales + line) : 0.f;
            scales->key[slot][p] = there ? __ldg(keys.scales + line) : 0.f;
            scales->value[slot][p] = v;
            // a row of zeros must not let its own probability overflow, nor one that is not finite let the others vanish
            scales->lift[slot][p] = v < INFINITY ? lg2_approx(fmaxf(v, 0x1p-100f)) : 0.f;
          }
#pragma unroll 1
          for (int from = 0; from < C::KEYS; from += CodeBatch<C::D>::ROWS) {
            CodeBatch<C::D> next = batch;
            if (from + CodeBatch<C::D>::ROWS < C::KEYS) next.load(side ? values : keys, runs, piece.head, from + CodeBatch<C::D>::ROWS, p);
            else if (side == 0) next.load(values, runs, piece.head, 0, p);
            else if (i + 1 < piece.count) next.load(keys, ahead, piece.head, 0, p);
            batch.template store<__half, C::KEYS>(to, 0, from, p);
            batch = next;
          }
          fence_async_smem();
          mbar_arrive(smem_u32(full + stage.stage));
        } else if (runs.bad == 0 && runs.key0 >= low && runs.key0 + C::KEYS <= length) {
          const uint32_t bar = smem_u32(full + stage.stage);
          // boxes of a page's rows, or of the tile's where a page is larger
          const int shift = min(a.line.step.page_shift, C::KEYS == 64 ? 6 : 7), page = __shfl_sync(0xffffffffu, runs.id, (p << (shift - 4)) & 31);
          const int in_page = runs.key0 & ((1 << a.line.step.page_shift) - 1) & ~((1 << shift) - 1);
          if (p == 0) mbar_expect_tx(bar, C::SIDE);
          else mbar_arrive(bar);
          __syncwarp();
          if (p < C::KEYS >> shift) {
#pragma unroll
            for (int c = 0; c < C::D; c += 64)
              tma_load_3d(to + (c >> 6) * C::BLOCK + (p << shift) * 128, side ? value_map : key_map, bar, c, in_page, page * a.line.kv_heads + piece.head);
          }
        } else {
          copy_keys<C::D, C::KEYS>(side ? values : keys, runs, piece.head, to, 0, p);
          copies_drain();
          fence_async_smem();
          mbar_arrive(smem_u32(full + stage.stage));
        }
        if (side == 0 && p == 0) {
          notes[issued % kNotes] = runs.bad | (i == 0 ? kFirst : 0u) | (i + 1 == piece.count ? kLast : 0u) | two;
          if (runs.bad) atomicCAS(a.status, 0u, unsigned(piece.sequence) + 1u);
          mbar_arrive(smem_u32(bars->k_full + stage.stage));  // the note is there
        }
      }
      stage.next();
      ++issued;
    }
  }
  land(0);
}

// ---- the issuing warp ---------------------------------------------------------------------------------------------
// It goes by the tiles' notes alone (written before K is handed over): where a unit's tiles begin and end, and whether the
// second row group has rows.  One warp issues for both groups, in a fixed order, so that they take turns: with a warp each the
// pipe served both at half speed, the groups' softmaxes fell into step and fought for the special-function unit (tile period
// 5500 clocks).
template <typename C>
__device__ __forceinline__ void issue_products(int tiles, Barriers* bars, const volatile uint32_t* notes, uint32_t tmem, uint32_t q, uint32_t k_ring,
                                               uint32_t v_ring, uint32_t gave_up) {
  constexpr uint32_t kScores = idesc_f16<typename C::M>(false, C::KEYS), kOutput = idesc_f16<typename C::M>(true, C::OUT);
  RingPos<C::STAGES> k, v;
  uint32_t q_phase = 0, p_phase = 0, o_phase = 3;  // a bit per group
  const bool elected = elect_one();
  auto scores = [&](int g) {
    if (!elected) return;
    const uint32_t rows_q = along_row(q + (C::SHARED ? 0 : g * C::QUERIES)), rows_k = along_row(k_ring + k.stage * C::SIDE), to = tmem + g * C::KEYS;
#pragma unroll 2
    for (int c = 0; c < C::D / 16; ++c)
      mma_f16(to, descriptor(rows_q + (c >> 2) * 1024 + (c & 3) * 2), descriptor(rows_k + (c >> 2) * (C::BLOCK >> 4) + (c & 3) * 2), kScores, c > 0);
    mma_commit(smem_u32(bars->s_full + g));
  };
  for (int tile = 0; tile < tiles; ++tile) {
    if (tile == 0 && !mbar_wait(smem_u32(bars->k_full + k.stage), k.phase, gave_up, 1010)) return;
    const uint32_t note = notes[tile % kNotes];
    const bool first = note & kFirst, last = note & kLast;
    const int groups = note & kTwoGroups ? 2 : 1;
    if (first) {
      if (C::SHARED)
        for (int g = 0; g < 2; ++g)
          if (!mbar_wait(smem_u32(bars->q_full + g), q_phase >> g & 1, gave_up, 1011)) return;
      for (int g = 0; g < groups; ++g) {
        if (!C::SHARED && !mbar_wait(smem_u32(bars->q_full + g), q_phase >> g & 1, gave_up, 1011)) return;
        q_phase ^= 1u << g;
        tc_fence_after();
        scores(g);
      }
      if (elected) mma_commit(smem_u32(bars->k_empty + k.stage));
      k.next();
    }
    if (C::SHARED && last && elected) mma_commit(smem_u32(&bars->q_empty));  // both groups' last scores are issued
    for (int g = 0; g < groups; ++g) {
      if (g == 0 && !mbar_wait(smem_u32(bars->v_full + v.stage), v.phase, gave_up, 1012)) return;
      if (first) {  // the previous unit's output has been read
        if (!mbar_wait(smem_u32(bars->o_free + g), o_phase >> g & 1, gave_up, 1013)) return;
        o_phase ^= 1u << g;
      }
      if (!mbar_wait(smem_u32(bars->p_full + g), p_phase >> g & 1, gave_up, 1014)) return;
      p_phase ^= 1u << g;
      tc_fence_after();
      if (elected) {
        const uint32_t rows_v = across_rows<C::KEYS>(v_ring + v.stage * C::SIDE + (C::SHARED ? g * 2 * C::BLOCK : 0));
#pragma unroll 2
        for (int c = 0; c < C::KEYS / 16; ++c)
          mma_f16_tmem(tmem + kGroups * C::KEYS + g * C::OUT, tmem + g * C::KEYS + c * 8, descriptor(rows_v + c * 128), kOutput, c > 0 || !first);
        if (last) mma_commit(smem_u32(bars->o_full + g));
        if (g == groups - 1) mma_commit(smem_u32(bars->v_empty + v.stage));
      }
      if (!last) {
        if (g == 0 && !mbar_wait(smem_u32(bars->k_full + k.stage), k.phase, gave_up, 1015)) return;
        scores(g);  // behind the product that reads P from these columns
        if (g == groups - 1) {
          if (elected) mma_commit(smem_u32(bars->k_empty + k.stage));
          k.next();
        }
      }
    }
    v.next();
    if (last && tile + 1 < tiles && !mbar_wait(smem_u32(bars->k_full + k.stage), k.phase, gave_up, 1016)) return;
  }
}

// ---- the softmax warpgroups -------------------------------------------------------------------------------------------
// A meeting of the two warps that own the same 32 rows.  It has no limit of its own, so nobody may stay away: after a wait
// that ran out a warp does no more work, but comes to all the meetings that are left; its rows are marked at the end.
__device__ __forceinline__ void meet(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

// Query rows of group g (half of the rows that both groups share), by the 256 threads of its two warpgroups: 16-byte pieces,
// neighbouring threads along a row.  A
// negative scale flips their signs, so that the maximum of the scores is the maximum of the scaled ones.
template <typename C>
__device__ __forceinline__ void load_query_rows(const TcArgs& a, const Piece& piece, int g, uint32_t to, float* row_scale) {
  constexpr int PIECES = C::D / 8, EACH = 256 / PIECES;
  const int t = threadIdx.x & 255, rows = piece.seq.count * a.line.group, c = t % PIECES;
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  const int first = C::SHARED ? g * 64 : 0, end = C::SHARED ? first + 64 : 128;
#pragma unroll 4
  for (int r = first + t / PIECES; r < end; r += EACH) {
    const int row = piece.block * C::ROWS + (C::SHARED ? 0 : g * 128) + r;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < rows) {
      const int token = row / a.line.group, h = row - token * a.line.group;
      v = *reinterpret_cast<const uint4*>(static_cast<const typename C::T*>(a.q) + int64_t(piece.seq.first + token) * a.qn +
                                          int64_t(piece.head * a.line.group + h) * a.qh + c * 8);
    }
    if constexpr (C::INT8 && std::is_same<typename C::T, __nv_bfloat16>::value) {
      const float down = row_to_half<PIECES>(v);
      if (c == 0) row_scale[r] = down;
    }
    v.x ^= flip;
    v.y ^= flip;
    v.z ^= flip;
    v.w ^= flip;
    store16(to + tile_offset(r, c), v);
  }
  fence_async_smem();
}

template <typename C>
__device__ __forceinline__ void softmax_rows(const TcArgs& a, Pieces pieces, Barriers* bars, Exchange* exchange, Scales* scales, uint32_t tmem, uint32_t q, int g, int half,
                                             const volatile uint32_t* notes, uint32_t gave_up) {
  constexpr int D = C::D, KEYS = C::KEYS / 2, OUT = C::OUT;
  using T = typename C::T;
  const int r = threadIdx.x & 127, meeting = 1 + g * 4 + (r >> 5);
  const uint32_t lanes = tmem + (uint32_t(r & ~31) << 16);
  const uint32_t s_columns = lanes + g * C::KEYS, o_columns = lanes + kGroups * C::KEYS + g * OUT + half * (OUT / 2);
  const int group_row = C::SHARED ? 0 : g * 128;  // of the group's first row in the unit
  const float call_scale = fmaxf(fabsf(a.scale_log2), 1e-30f);  // a scale of 0 must leave hidden scores at -inf
  uint32_t s_phase = 0, o_phase = 0, q_phase = 0, tile = 0, turn = 0;
  Piece piece;
  bool more = pieces.next(a.line, piece);
  auto mine = [&](const Piece& p) { return p.seq.count * a.line.group - p.block * C::ROWS > group_row; };
  auto fetch = [&](const Piece& p) {
    turn ^= 1;
    load_query_rows<C>(a, p, g, q + (C::SHARED ? 0 : g * C::QUERIES), C::INT8 ? scales->row[turn][C::SHARED ? 0 : g] : nullptr);
    mbar_arrive_warp(smem_u32(bars->q_full + g));
  };
  auto wait = [&](uint32_t bar, uint32_t parity, unsigned int site) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, gave_up, site)); };
  auto meet_on = [&](int meetings) {  // of the present unit, then of all that follow
#pragma unroll 1
    while (more) {
#pragma unroll 1
      for (; meetings > 0; --meetings) meet(meeting);
      more = pieces.next(a.line, piece);
      meetings = more && mine(piece) ? piece.count + 1 : 0;
    }
  };
  if (more && mine(piece)) fetch(piece);
  while (more) {
    if (!mine(piece)) {
      tile += piece.count;
      more = pieces.next(a.line, piece);
      if (more && mine(piece)) fetch(piece);
      continue;
    }
    const int rows = piece.seq.count * a.line.group, row = piece.block * C::ROWS + group_row + r;
    KeyRange seen = visible(piece.seq.length - piece.seq.count + row / a.line.group, piece.seq.length, a.line.causal, a.line.window);
    if (row >= rows) seen = {0, 0};
    // keys that every row of the group sees need no test
    const int row0 = piece.block * C::ROWS + group_row, token0 = row0 / a.line.group, token1 = (min(row0 + 128, rows) - 1) / a.line.group;
    const int all_hi = visible(piece.seq.length - piece.seq.count + token0, piece.seq.length, a.line.causal, a.line.window).hi;
    const int all_lo = visible(piece.seq.length - piece.seq.count + token1, piece.seq.length, a.line.causal, a.line.window).lo;
    float m = kNoMaximum, l = 0.f, scale = call_scale;
    const uint32_t mine_turn = turn;
#pragma unroll 1
    for (int i = 0; i < piece.count; ++i, ++tile) {
      const int key0 = (piece.first + i) * C::KEYS + half * KEYS;
      if (!wait(smem_u32(bars->s_full + g), s_phase, 1020 + g)) return meet_on(piece.count - i + 1);
      s_phase ^= 1;
      tc_fence_after();
      uint32_t x[KEYS];
#pragma unroll
      for (int c = 0; c < KEYS; c += 32) tmem_load32(s_columns + half * KEYS + c, x + c);
      const uint32_t gone = notes[tile % kNotes] >> (half * (KEYS / 16)) & ((1u << (KEYS / 16)) - 1);
      tmem_load_wait();
      tmem_regs_ready<KEYS>(x);
      const int slot_of_tile = tile % kScaleDepth;
      if constexpr (C::INT8) {
        if (std::is_same<T, __nv_bfloat16>::value && i == 0) scale = call_scale * scales->row[mine_turn][C::SHARED ? 0 : g][r];
        const ulonglong2* k = reinterpret_cast<const ulonglong2*>(scales->key[slot_of_tile] + half * KEYS);
#pragma unroll
        for (int c = 0; c < KEYS; c += 4) {
          const ulonglong2 s = k[c / 4];
          float u[4];
          unpack_f32x2(mul_f32x2(pack_f32x2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), s.x), u[0], u[1]);
          unpack_f32x2(mul_f32x2(pack_f32x2(__uint_as_float(x[c + 2]), __uint_as_float(x[c + 3])), s.y), u[2], u[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[c + e] = __float_as_uint(u[e]);
        }
      }
      if (gone != 0 || key0 < all_lo || key0 + KEYS > all_hi) {
        asm volatile("" ::: "memory");  // a branch of its own: as selects in the common path it cost a quarter of the time
        const int lo = seen.lo - key0, hi = seen.hi - key0;
#pragma unroll
        for (int c = 0; c < KEYS; ++c)
          if (c < lo || c >= hi || (gone >> (c >> 4) & 1)) x[c] = 0xff800000u;
      }
      const uint64_t scale2 = pack_f32x2(scale, scale);
      float best;
      if constexpr (C::INT8) {
        // The maximum is that of the row's own probabilities times scales, hidden keys left out: what is rounded is at most 1
        // (2^8 where the running maximum lags), and neither the other keys of the tile nor other rows move it.  (Against the
        // largest scale of the tile, 1024 tokens over 8K codes, 32 heads: 271 us for 269 at 128 channels, 203 for 190 at 64.)
        const ulonglong2* lift = reinterpret_cast<const ulonglong2*>(scales->lift[slot_of_tile] + half * KEYS);
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < KEYS; c += 4) {
          const ulonglong2 of = lift[c / 4];
          float u[4];
          unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), scale2, of.x), u[0], u[1]);
          unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(x[c + 2]), __uint_as_float(x[c + 3])), scale2, of.y), u[2], u[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], u[e]);
        }
        best = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      } else {
        float top[4] = {__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]), __uint_as_float(x[3])};
#pragma unroll
        for (int c = 4; c < KEYS; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            top[e] = c + 4 + e < KEYS ? fmaxf(fmaxf(top[e], __uint_as_float(x[c + e])), __uint_as_float(x[c + 4 + e]))
                                      : fmaxf(top[e], __uint_as_float(x[c + e]));
        best = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
      }
      // also: from here on both halves of the scores are in registers, and P may be written over them
      exchange->maximum[tile & 1][g][half][r] = best;
      meet(meeting);
      best = fmaxf(best, exchange->maximum[tile & 1][g][half ^ 1][r]);
      const bool moves = best > m + kStale;
      if (__any_sync(0xffffffffu, moves)) {
        const float to = moves ? best : m, keep = ex2_approx(m - to);
        m = to;
        l *= keep;
        if (i > 0) {  // scores of this tile were issued behind the product with the last one, so that is complete
#pragma unroll 1
          for (int c = 0; c < OUT / 2; c += 16) {
            uint32_t o[16];
            tmem_load16(o_columns + c, o);
            tmem_load_wait();
            tmem_regs_ready<16>(o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
            tmem_store16(o_columns + c, o);
          }
        }
      }
      const uint64_t minus_m = pack_f32x2(-m, -m);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int part = 0; part < KEYS / 32; ++part) {
        uint32_t p[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const int at = part * 32 + 2 * c;
          float u, w;
          unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(x[at]), __uint_as_float(x[at + 1])), scale2, minus_m), u, w);
          u = ex2_approx(u);
          w = ex2_approx(w);
          sum[c & 1] = add_f32x2(sum[c & 1], pack_f32x2(u, w));
          if constexpr (C::INT8) {
            const float2 v = *reinterpret_cast<const float2*>(scales->value[slot_of_tile] + half * KEYS + at);
            u *= v.x;
            w *= v.y;
          }
          p[c] = Half2<typename C::M>::pack(u, w);
        }
        tmem_store16(s_columns + half * (KEYS / 2) + part * 16, p);
      }
      float s0, s1;
      unpack_f32x2(add_f32x2(sum[0], sum[1]), s0, s1);
      l += s0 + s1;
      tmem_store_wait();
      tc_fence_before();
      mbar_arrive_warp(smem_u32(bars->p_full + g));
    }
    // the last scores are here, so the queries have been read
    const Piece done = piece;
    more = pieces.next(a.line, piece);
    if (C::SHARED) {  // and by the other group
      if (!wait(smem_u32(&bars->q_empty), q_phase, 1024 + g)) {
        meet(meeting);
        return meet_on(more && mine(piece) ? piece.count + 1 : 0);
      }
      q_phase ^= 1;
    }
    if (more && mine(piece)) fetch(piece);
    exchange->sum[g][half][r] = l;
    meet(meeting);
    l += exchange->sum[g][half ^ 1][r];
    if (!wait(smem_u32(bars->o_full + g), o_phase, 1022 + g)) return meet_on(more && mine(piece) ? piece.count + 1 : 0);
    o_phase ^= 1;
    tc_fence_after();
    const bool there = row < rows;
    const int token = row / a.line.group, h = done.head * a.line.group + row - token * a.line.group;
    const float f = l == 0.f ? 0.f : 1.0f / l;
    const int channel0 = (C::SHARED ? g * OUT : 0) + half * (OUT / 2), in_block = group_row + r;
    T* out = static_cast<T*>(a.out) + int64_t(done.seq.first + token) * a.on + int64_t(h) * a.oh + channel0;
    float* slot = a.parts + (int64_t(blockIdx.x) * 2 + (done.opens ? 1 : 0)) * slot_floats(C::ROWS, D);
#pragma unroll 1
    for (int c = 0; c < OUT / 2; c += 16) {
      uint32_t o[16];
      tmem_load16(o_columns + c, o);
      tmem_load_wait();
      tmem_regs_ready<16>(o);
      if (!there) continue;
      if (done.whole) {
#pragma unroll
        for (int e = 0; e < 16; e += 8) {
          uint4 w;
          w.x = Half2<T>::pack(__uint_as_float(o[e]) * f, __uint_as_float(o[e + 1]) * f);
          w.y = Half2<T>::pack(__uint_as_float(o[e + 2]) * f, __uint_as_float(o[e + 3]) * f);
          w.z = Half2<T>::pack(__uint_as_float(o[e + 4]) * f, __uint_as_float(o[e + 5]) * f);
          w.w = Half2<T>::pack(__uint_as_float(o[e + 6]) * f, __uint_as_float(o[e + 7]) * f);
          *reinterpret_cast<uint4*>(out + c + e) = w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *reinterpret_cast<uint4*>(slot + int64_t(in_block) * D + channel0 + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
      }
    }
    if (half == 0 && there && (!C::SHARED || g == 0)) {
      if (!done.whole) {
        slot[C::ROWS * D + in_block] = m;
        slot[C::ROWS * D + C::ROWS + in_block] = l;
      } else if (a.lse != nullptr) {
        a.lse[int64_t(done.seq.first + token) * (a.line.kv_heads * a.line.group) + h] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
      }
    }
    tc_fence_before();
    mbar_arrive_warp(smem_u32(bars->o_free + g));
  }
}

template <typename C>
__global__ __launch_bounds__(kThreads, 1) void paged_tc_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map, const TcArgs a) {
  extern __shared__ char smem_raw[];
  __shared__ Barriers bars;
  __shared__ Exchange exchange;
  __shared__ __align__(16) typename std::conditional<C::INT8, Scales, char>::type scales_memory;
  Scales* scales = reinterpret_cast<Scales*>(&scales_memory);
  __shared__ LineShared<kThreads> shared;
  __shared__ uint32_t tmem_base, gave_up_word;
  __shared__ volatile uint32_t notes[kNotes];
  const int warp = threadIdx.x >> 5;
  const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
  const uint32_t q = smem, v_ring = q + C::Q, k_ring = v_ring + C::STAGES * C::SIDE, gave_up = smem_u32(&gave_up_word);
  if (threadIdx.x == 0) {
    gave_up_word = 0;
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(bars.k_full + i), 129);
      mbar_init(smem_u32(bars.v_full + i), 128);
      mbar_init(smem_u32(bars.k_empty + i), 1);
      mbar_init(smem_u32(bars.v_empty + i), 1);
    }
    for (int g = 0; g < kGroups; ++g) {
      mbar_init(smem_u32(bars.q_full + g), 8);
      mbar_init(smem_u32(bars.s_full + g), 1);
      mbar_init(smem_u32(bars.p_full + g), 8);
      mbar_init(smem_u32(bars.o_full + g), 1);
      mbar_init(smem_u32(bars.o_free + g), 8);
    }
    mbar_init(smem_u32(&bars.q_empty), 1);
    mbar_init(smem_u32(&bars.drained), 1);
    mbar_init_fence();
  }
  // The launch in front is this call's own, for the sequences of few rows, and its start waited for everything before
  // it; nothing it writes is read here.  So this one need not wait for it, only end behind it (the joins wait for this).
  chain_release();
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
  if (warp < kProducer) {
    regs_inc<kRegsSoftmax>();
    softmax_rows<C>(a, pieces, &bars, &exchange, scales, tmem, q, warp >> 3, (warp >> 2) & 1, notes, gave_up);
  } else if (warp < kIssuer) {
    regs_dec<kRegsProducer>();
    fetch_tiles<C>(a, &key_map, &value_map, pieces, &bars, notes, scales, k_ring, v_ring, gave_up);
  } else {
    regs_dec<kRegsIssuer>();
    if (warp == kIssuer + 1 && (threadIdx.x & 31) == 0) {
      Pieces all = pieces;
      Piece piece;
      while (all.next(a.line, piece)) {}
      a.notes[blockIdx.x] = join_note(a.line, piece, total, finish, blockIdx.x, workers);
    }
    if (warp == kIssuer) {
      issue_products<C>(int(pieces.left), &bars, notes, tmem, q, k_ring, v_ring, gave_up);
      __syncwarp();
      // nothing of this CTA is in flight when tensor memory is handed back, also after a wait that ran out
      if (elect_one()) mma_commit(smem_u32(&bars.drained));
      __syncwarp();
      mbar_drain(smem_u32(&bars.drained), 0);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kIssuer) tmem_dealloc(tmem, 512);
  if (gave_up_word != 0 && threadIdx.x < C::ROWS) {
    // a wait ran out: the rows of this worker's whole units are marked, parts poison their join
    Pieces all = pieces;
    Piece piece;
    while (all.next(a.line, piece)) {
      const int rows = piece.seq.count * a.line.group, row = piece.block * C::ROWS + threadIdx.x;
      if (piece.whole) {
        if (row >= rows) continue;
        const int token = row / a.line.group, h = piece.head * a.line.group + row % a.line.group;
        typename C::T* out = static_cast<typename C::T*>(a.out) + int64_t(piece.seq.first + token) * a.on + int64_t(h) * a.oh;
        for (int c = 0; c < C::D; ++c) out[c] = static_cast<typename C::T>(NAN);
      } else {
        float* slot = a.parts + (int64_t(blockIdx.x) * 2 + (piece.opens ? 1 : 0)) * slot_floats(C::ROWS, C::D);
        slot[C::ROWS * C::D + C::ROWS + threadIdx.x] = NAN;
      }
    }
  }
  chain_wait();
}

// The pool as {channels, a page's rows, pages x heads}, in boxes of 64 channels x a page with the 128-byte swizzle.
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult result;
    const bool good = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &result) == cudaSuccess && result == cudaDriverEntryPointSuccess;
    return good ? reinterpret_cast<EncodeFn>(ptr) : nullptr;
  }();
  return fn;
}
template <typename C>
bool pool_map(CUtensorMap* map, const char* pool, const TcArgs& a) {
  const cuuint64_t dims[3] = {cuuint64_t(C::D), cuuint64_t(1) << a.line.step.page_shift, cuuint64_t(a.pages) * a.line.kv_heads};
  const cuuint64_t strides[2] = {cuuint64_t(C::D) * 2, (cuuint64_t(C::D) * 2) << a.line.step.page_shift};
  const cuuint32_t box[3] = {64, std::min(1u << a.line.step.page_shift, cuuint32_t(C::KEYS)), 1}, ones[3] = {1, 1, 1};
  return encode_fn()(map, std::is_same<typename C::T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                     const_cast<char*>(pool), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
int join(const TcArgs& a, cudaStream_t stream) {
  constexpr int kRows = Shape<T, false, D>::ROWS;
  const JoinArgs join{a.parts, a.notes, kRows, a.line.group, a.line.kv_heads * a.line.group, a.out, a.on, a.oh, a.lse};
  return launched(launch_chained(join_parts_kernel<T, D, false>, dim3(kTcWorkers - 1, kRows / 16), dim3(128), 0, stream, join), "paged attention");
}

template <typename C>
int launch(const TcArgs& a, cudaStream_t stream) {
  CUtensorMap key_map{}, value_map{};
  RISA_REQUIRE(int64_t(a.pages) * a.line.kv_heads < (int64_t(1) << 31), "paged attention: the pool has too many pages");
  if (!C::INT8)
    if (encode_fn() == nullptr || !pool_map<C>(&key_map, a.keys, a) || !pool_map<C>(&value_map, a.values, a))
      return fail(RISA_B200_CUDA, "paged attention: no tensor map of the pool");
  if (cudaFuncSetAttribute(paged_tc_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
    return fail(RISA_B200_CUDA, "paged attention: %s", cudaGetErrorString(cudaGetLastError()));
  // setmaxnreg deals out what the CTA was launched with; a smaller launch count would block its waits for ever
  static const bool budget = [] {
    cudaFuncAttributes attributes;
    return cudaFuncGetAttributes(&attributes, paged_tc_kernel<C>) == cudaSuccess && attributes.numRegs == kRegsLaunch;
  }();
  RISA_REQUIRE(budget, "paged attention: the tensor-core kernel was not compiled for %d registers", kRegsLaunch);
  return launched(launch_chained(paged_tc_kernel<C>, dim3(kTcWorkers), dim3(kThreads), C::SMEM, stream, key_map, value_map, a), "paged attention");
}

}  // namespace

namespace {
int rows_of_unit(int head_dim) { return head_dim == 256 ? Shape<__half, false, 256>::ROWS : Shape<__half, false, 128>::ROWS; }
template <typename T>
int launch_for(const TcArgs& a, bool codes, int head_dim, cudaStream_t stream) {
  if (head_dim == 64) return codes ? launch<Shape<T, true, 64>>(a, stream) : launch<Shape<T, false, 64>>(a, stream);
  if (head_dim == 128) return codes ? launch<Shape<T, true, 128>>(a, stream) : launch<Shape<T, false, 128>>(a, stream);
  return codes ? launch<Shape<T, true, 256>>(a, stream) : launch<Shape<T, false, 256>>(a, stream);
}
template <typename T>
int join_for(const TcArgs& a, int head_dim, cudaStream_t stream) {
  return head_dim == 64 ? join<T, 64>(a, stream) : head_dim == 128 ? join<T, 128>(a, stream) : join<T, 256>(a, stream);
}
}  // namespace

size_t paged_tc_scratch(int head_dim) {
  return size_t(kTcWorkers) * (2 * slot_floats(rows_of_unit(head_dim), head_dim) * sizeof(float) + sizeof(JoinNote));
}
TcArgs paged_tc_args(TcArgs a, int head_dim) {
  a.line.rows = Divisor(rows_of_unit(head_dim));
  a.line.keys = Divisor(head_dim == 256 ? Shape<__half, false, 256>::KEYS : Shape<__half, false, 128>::KEYS);
  a.notes = reinterpret_cast<JoinNote*>(a.parts + size_t(kTcWorkers) * 2 * slot_floats(a.line.rows, head_dim));
  return a;
}
int paged_tc(const TcArgs& a, int dtype_code, bool codes, int head_dim, cudaStream_t stream) {
  return dtype_code == 1 ? launch_for<__half>(a, codes, head_dim, stream) : launch_for<__nv_bfloat16>(a, codes, head_dim, stream);
}
int paged_tc_join(const TcArgs& a, int dtype_code, int head_dim, cudaStream_t stream) {
  return dtype_code == 1 ? join_for<__half>(a, head_dim, stream) : join_for<__nv_bfloat16>(a, head_dim, stream);
}

// Site of the first wait of these kernels that ran out since the last call (0: none), or -1 on a CUDA error.
int paged_tc_wait_status() {
  unsigned int status = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&status, g_wait_status, sizeof(status)) != cudaSuccess) return -1;
  if (status != 0) cudaMemcpyToSymbol(g_wait_status, &zero, sizeof(zero));
  return int(status);
}

}  // namespace serving
}  // namespace risa_b200
