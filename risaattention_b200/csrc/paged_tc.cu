// Attention of many query rows (chunks of prompts) over a paged cache on the tensor cores.
//
// A unit is 256 query rows of one key head, rows in the order (token, head of the group), so that all heads of a
// group share every key tile; two groups of 128 rows (one softmax warpgroup and one accumulator each) take turns on
// the tensor pipe: while one group's scores become probabilities, the other's matrix products run.  Per 128-key tile
// and group: S = Q K^T (128 x 128 x head_dim, fp32 in tensor memory), the thread that owns a row reads it, keeps
// running maximum and sum without a shuffle, writes P (16 bits) over the columns of S, and O += P V takes P from
// tensor memory and V from shared memory as it lies there (keys along K, channels contiguous).
//
// Warps 0-3, 4-7: softmax, query loads, epilogue of their row group.  8-11: fetch K and V tiles from the pages
// (cp.async, or codes converted on the way) into the 128-byte-swizzled layout of the matrix instructions.  12: issues
// them (and owns tensor memory).  13-15 idle, so that registers can be dealt per warpgroup.
#include "serving_plan.cuh"
#include "paged_tc.cuh"
#include "tc_f16.cuh"

namespace risa_b200 {
namespace serving {

using namespace tc;

namespace {

constexpr int kThreads = 512;
constexpr int kTileKeys = 128, kGroups = 2, kRows = 128 * kGroups;
constexpr int kProducer = 8, kIssuer = 12;  // first warps of their roles
// The SM's 65,536 registers at 512 threads are 128 each; the softmax warps hold a row of 128 scores.
constexpr int kRegsLaunch = 128, kRegsSoftmax = 192, kRegsProducer = 88, kRegsIssuer = 40;
static_assert(128 * (2 * kRegsSoftmax + kRegsProducer + kRegsIssuer) <= kThreads * kRegsLaunch, "register budget");
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
  static constexpr bool INT8 = INT8_;
  static constexpr int D = D_;
  static constexpr int SIDE = kTileKeys * D * 2;  // a K or V tile as the matrix instructions read it
  static constexpr int HALVES = D / 64;           // blocks of 64 channels: 128 rows of 128 bytes
  static constexpr int STAGES = D == 128 ? 2 : 4;
  static constexpr int Q = kGroups * SIDE;
  static constexpr int SMEM = Q + 2 * STAGES * SIDE + 1024;  // + alignment
};

struct Barriers {
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t q_full[kGroups], s_full[kGroups], p_full[kGroups], o_full[kGroups], o_free[kGroups], drained;
};

// ---- the fetching warpgroup -----------------------------------------------------------------------------------
template <typename C>
struct Fetcher {
  const TcArgs& a;
  Barriers* bars;
  volatile uint32_t* notes;
  uint32_t v_ring, k_ring, gave_up;
  int p;            // thread of the group
  uint32_t issued;  // tiles so far
  RingPos<C::STAGES> k, v;

  __device__ __forceinline__ bool wait_stage(uint64_t* empty, int stage, uint32_t phase, unsigned site) const {
    return mbar_wait(smem_u32(empty + stage), phase ^ 1, gave_up, site);
  }
};

template <typename C>
__device__ __forceinline__ void fetch_tiles(Fetcher<C>& f, Pieces pieces) {
  const TcArgs& a = f.a;
  Piece piece;
  while (pieces.next(a.line, piece)) {
    const int32_t* row = a.line.step.table + int64_t(piece.sequence) * a.line.step.width;
    const int length = piece.seq.length;
    const int low = a.line.window > 0 ? visible(piece.seq.length - piece.seq.count, length, true, a.line.window).lo : 0;
    const PoolView keys{a.keys, a.key_scales, a.line.kv_heads, a.line.step.page_shift}, values{a.values, a.value_scales, a.line.kv_heads, a.line.step.page_shift};
    KeyRuns ahead;
    ahead.look_up(row, a.line.step.page_shift, piece.first * kTileKeys, low, length);
    for (int i = 0; i < piece.count; ++i) {
      const int key0 = (piece.first + i) * kTileKeys;
      const KeyRuns t = ahead;
      if (i + 1 < piece.count) ahead.look_up(row, a.line.step.page_shift, key0 + kTileKeys, low, length);
      const uint32_t bad = t.bad(a.pages);
      const uint32_t note = bad | (i == 0 ? kFirst : 0u) | (i + 1 == piece.count ? kLast : 0u) |
                            (piece.seq.count * a.line.group - piece.block * kRows > 128 ? kTwoGroups : 0u);
      const uint32_t k_to = f.k_ring + f.k.stage * C::SIDE, v_to = f.v_ring + f.v.stage * C::SIDE;
      if constexpr (C::INT8) {
        // scaled and rounded to the queries' type (half a step), as if the cache had held 16-bit values
        CodeTile<typename C::T, C::D> codes;
        codes.load(keys, t, bad, piece.head, f.p);
        if (!f.wait_stage(f.bars->k_empty, f.k.stage, f.k.phase, 1001)) return;
        codes.store(k_to, f.p);
        fence_async_smem();
        mbar_arrive(smem_u32(f.bars->k_full + f.k.stage));
        codes.load(values, t, bad, piece.head, f.p);
        if (!f.wait_stage(f.bars->v_empty, f.v.stage, f.v.phase, 1002)) return;
        codes.store(v_to, f.p);
        fence_async_smem();
        mbar_arrive(smem_u32(f.bars->v_full + f.v.stage));
      } else {
        if (!f.wait_stage(f.bars->k_empty, f.k.stage, f.k.phase, 1001)) return copies_drain();
        copy_keys<C::D>(keys, t, bad, piece.head, k_to, f.p);
        copies_arrive(smem_u32(f.bars->k_full + f.k.stage));
        if (!f.wait_stage(f.bars->v_empty, f.v.stage, f.v.phase, 1002)) return copies_drain();
        copy_keys<C::D>(values, t, bad, piece.head, v_to, f.p);
        copies_arrive(smem_u32(f.bars->v_full + f.v.stage));
      }
      if (f.p == 0) {
        f.notes[f.issued % kNotes] = note;
        if (bad) atomicCAS(a.status, 0u, unsigned(piece.sequence) + 1u);
        mbar_arrive(smem_u32(f.bars->k_full + f.k.stage));  // the note is there
      }
      f.k.next();
      f.v.next();
      ++f.issued;
    }
  }
  if (!C::INT8) copies_drain();
}

// ---- the issuing warp ---------------------------------------------------------------------------------------------
// Goes by the tiles' notes alone (written before K is handed over): where a unit's tiles begin and end, and whether its
// second row group has rows.
template <typename C>
__device__ __forceinline__ void issue_products(int tiles, Barriers* bars, const volatile uint32_t* notes, uint32_t tmem, uint32_t q,
                                               uint32_t k_ring, uint32_t v_ring, uint32_t gave_up) {
  constexpr uint32_t kScores = idesc_f16<typename C::T>(false, kTileKeys), kOutput = idesc_f16<typename C::T>(true, C::D);
  RingPos<C::STAGES> k, v;
  uint32_t q_phase = 0, p_phase = 0, o_phase = 3;  // a bit per group
  const bool elected = elect_one();
  auto scores = [&](int g) {
    fence_async_smem();  // K's copies, which the barrier has told of
    if (!elected) return;
    const uint32_t rows_q = along_row(q + g * C::SIDE), rows_k = along_row(k_ring + k.stage * C::SIDE);
#pragma unroll
    for (int c = 0; c < C::D / 16; ++c) {
      const uint32_t at = (c >> 2) * 1024 + (c & 3) * 2;
      mma_f16(tmem + g * kTileKeys, descriptor(rows_q + at), descriptor(rows_k + at), kScores, c > 0);
    }
    mma_commit(smem_u32(bars->s_full + g));
  };
  for (int tile = 0; tile < tiles; ++tile) {
    if (tile == 0 && !mbar_wait(smem_u32(bars->k_full + k.stage), k.phase, gave_up, 1010)) return;
    const uint32_t note = notes[tile % kNotes];
    const int groups = note & kTwoGroups ? 2 : 1;
    if (note & kFirst) {
      for (int g = 0; g < groups; ++g) {
        if (!mbar_wait(smem_u32(bars->q_full + g), q_phase >> g & 1, gave_up, 1011)) return;
        q_phase ^= 1u << g;
        tc_fence_after();
        scores(g);
      }
      if (elected) mma_commit(smem_u32(bars->k_empty + k.stage));
      k.next();
    }
    const bool last = note & kLast;
    for (int g = 0; g < groups; ++g) {
      if (g == 0 && !mbar_wait(smem_u32(bars->v_full + v.stage), v.phase, gave_up, 1012)) return;
      if (note & kFirst) {  // the previous unit's output has been read
        if (!mbar_wait(smem_u32(bars->o_free + g), o_phase >> g & 1, gave_up, 1013)) return;
        o_phase ^= 1u << g;
      }
      if (!mbar_wait(smem_u32(bars->p_full + g), p_phase >> g & 1, gave_up, 1014)) return;
      p_phase ^= 1u << g;
      tc_fence_after();
      fence_async_smem();  // V's copies
      if (elected) {
        const uint32_t rows_v = across_rows(v_ring + v.stage * C::SIDE);
#pragma unroll
        for (int c = 0; c < kTileKeys / 16; ++c)
          mma_f16_tmem(tmem + kGroups * kTileKeys + g * C::D, tmem + g * kTileKeys + c * 8, descriptor(rows_v + c * 128), kOutput,
                       c > 0 || !(note & kFirst));
        if (last) mma_commit(smem_u32(bars->o_full + g));
        if (g == groups - 1) mma_commit(smem_u32(bars->v_empty + v.stage));
      }
      if (!last) {
        if (g == 0 && !mbar_wait(smem_u32(bars->k_full + k.stage), k.phase, gave_up, 1015)) return;
        scores(g);
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

// ---- a softmax warpgroup ---------------------------------------------------------------------------------------------
// Query rows of group g: 16-byte pieces, neighbouring threads along a row.  A negative scale flips their signs, so that
// the maximum of the scores is the maximum of the scaled ones.
template <typename C>
__device__ __forceinline__ void load_query_rows(const TcArgs& a, const Piece& piece, int g, uint32_t to) {
  constexpr int PIECES = C::D / 8;
  const int t = threadIdx.x & 127, rows = piece.seq.count * a.line.group;
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
#pragma unroll 4
  for (int n = 0; n < PIECES; ++n) {
    const int index = n * 128 + t, r = index / PIECES, c = index % PIECES, row = piece.block * kRows + g * 128 + r;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < rows) {
      const int token = row / a.line.group, h = row - token * a.line.group;
      v = *reinterpret_cast<const uint4*>(static_cast<const typename C::T*>(a.q) + int64_t(piece.seq.first + token) * a.qn +
                                          int64_t(piece.head * a.line.group + h) * a.qh + c * 8);
      v.x ^= flip;
      v.y ^= flip;
      v.z ^= flip;
      v.w ^= flip;
    }
    store16(to + tile_offset(r, c), v);
  }
  fence_async_smem();
}

template <typename C>
__device__ __forceinline__ void softmax_rows(const TcArgs& a, Pieces pieces, Barriers* bars, uint32_t tmem, uint32_t q, int g,
                                             const volatile uint32_t* notes, uint32_t gave_up) {
  constexpr int D = C::D;
  using T = typename C::T;
  const int r = threadIdx.x & 127;
  const uint32_t lanes = tmem + (uint32_t(r & ~31) << 16);
  const uint32_t s_columns = lanes + g * kTileKeys, o_columns = lanes + kGroups * kTileKeys + g * D;
  const float scale = fmaxf(fabsf(a.scale_log2), 1e-30f);  // a scale of 0 must leave hidden scores at -inf
  uint32_t s_phase = 0, o_phase = 0, tile = 0;
  Piece piece;
  bool more = pieces.next(a.line, piece);
  auto mine = [&](const Piece& p) { return p.seq.count * a.line.group - p.block * kRows > g * 128; };
  auto fetch = [&](const Piece& p) {
    load_query_rows<C>(a, p, g, q + g * C::SIDE);
    mbar_arrive_warp(smem_u32(bars->q_full + g));
  };
  if (more && mine(piece)) fetch(piece);
  while (more) {
    if (!mine(piece)) {
      tile += piece.count;
      more = pieces.next(a.line, piece);
      if (more && mine(piece)) fetch(piece);
      continue;
    }
    const int rows = piece.seq.count * a.line.group, row = piece.block * kRows + g * 128 + r;
    const int token = row / a.line.group, h = piece.head * a.line.group + row - token * a.line.group;
    KeyRange seen = visible(piece.seq.length - piece.seq.count + token, piece.seq.length, a.line.causal, a.line.window);
    if (row >= rows) seen = {0, 0};
    // keys that every row of the group sees need no test
    const int token0 = (piece.block * kRows + g * 128) / a.line.group, token1 = (min(piece.block * kRows + g * 128 + 128, rows) - 1) / a.line.group;
    const int all_hi = visible(piece.seq.length - piece.seq.count + token0, piece.seq.length, a.line.causal, a.line.window).hi;
    const int all_lo = visible(piece.seq.length - piece.seq.count + token1, piece.seq.length, a.line.causal, a.line.window).lo;
    float m = kNoMaximum, l = 0.f;
    for (int i = 0; i < piece.count; ++i, ++tile) {
      const int key0 = (piece.first + i) * kTileKeys;
      if (!mbar_wait(smem_u32(bars->s_full + g), s_phase, gave_up, 1020 + g)) return;
      s_phase ^= 1;
      tc_fence_after();
      uint32_t x[kTileKeys];
#pragma unroll
      for (int c = 0; c < kTileKeys / 32; ++c) tmem_load32(s_columns + c * 32, x + c * 32);
      const uint32_t gone = notes[tile % kNotes] & kHiddenRuns;
      tmem_load_wait();
      tmem_regs_ready<kTileKeys>(x);
      if (gone != 0 || key0 < all_lo || key0 + kTileKeys > all_hi) {
        const int lo = seen.lo - key0, hi = seen.hi - key0;
#pragma unroll
        for (int c = 0; c < kTileKeys; ++c)
          if (c < lo || c >= hi || (gone >> (c >> 4) & 1)) x[c] = 0xff800000u;
      }
      float top[4] = {__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]), __uint_as_float(x[3])};
#pragma unroll
      for (int c = 4; c < kTileKeys; c += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          top[e] = c + 4 + e < kTileKeys ? fmaxf(fmaxf(top[e], __uint_as_float(x[c + e])), __uint_as_float(x[c + 4 + e]))
                                         : fmaxf(top[e], __uint_as_float(x[c + e]));
      const float best = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
      const bool moves = best > m + kStale;
      if (__any_sync(0xffffffffu, moves)) {
        const float to = moves ? best : m, keep = ex2_approx(m - to);
        m = to;
        l *= keep;
        if (i > 0) {  // scores of this tile were issued behind the product with the last one, so that is complete
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_load16(o_columns + c * 16, o);
            tmem_load_wait();
            tmem_regs_ready<16>(o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
            tmem_store16(o_columns + c * 16, o);
          }
        }
      }
      const uint64_t scale2 = pack_f32x2(scale, scale), minus_m = pack_f32x2(-m, -m);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int part = 0; part < 4; ++part) {
        uint32_t p[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const int at = part * 32 + 2 * c;
          float u, w;
          unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(x[at]), __uint_as_float(x[at + 1])), scale2, minus_m), u, w);
          u = ex2_approx(u);
          w = ex2_approx(w);
          sum[c & 1] = add_f32x2(sum[c & 1], pack_f32x2(u, w));
          p[c] = Half2<T>::pack(u, w);
        }
        tmem_store16(s_columns + part * 16, p);
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
    if (more && mine(piece)) fetch(piece);
    if (!mbar_wait(smem_u32(bars->o_full + g), o_phase, gave_up, 1022 + g)) return;
    o_phase ^= 1;
    tc_fence_after();
    const bool there = row < rows;
    if (done.whole) {
      const float f = l == 0.f ? 0.f : 1.0f / l;
      T* out = static_cast<T*>(a.out) + int64_t(done.seq.first + token) * a.on + int64_t(h) * a.oh;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_load32(o_columns + c * 32, o);
        tmem_load_wait();
        tmem_regs_ready<32>(o);
        if (there) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint4 w;
            w.x = Half2<T>::pack(__uint_as_float(o[8 * e]) * f, __uint_as_float(o[8 * e + 1]) * f);
            w.y = Half2<T>::pack(__uint_as_float(o[8 * e + 2]) * f, __uint_as_float(o[8 * e + 3]) * f);
            w.z = Half2<T>::pack(__uint_as_float(o[8 * e + 4]) * f, __uint_as_float(o[8 * e + 5]) * f);
            w.w = Half2<T>::pack(__uint_as_float(o[8 * e + 6]) * f, __uint_as_float(o[8 * e + 7]) * f);
            *reinterpret_cast<uint4*>(out + c * 32 + e * 8) = w;
          }
        }
      }
      if (there && a.lse != nullptr)
        a.lse[int64_t(done.seq.first + token) * (a.line.kv_heads * a.line.group) + h] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
    } else {
      float* slot = a.parts + (int64_t(blockIdx.x) * 2 + (done.opens ? 1 : 0)) * slot_floats(kRows, D);
      const int in_block = g * 128 + r;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_load32(o_columns + c * 32, o);
        tmem_load_wait();
        tmem_regs_ready<32>(o);
        if (there) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<uint4*>(slot + int64_t(in_block) * D + c * 32 + e * 4) = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
      }
      slot[kRows * D + in_block] = m;
      slot[kRows * D + kRows + in_block] = l;
    }
    tc_fence_before();
    mbar_arrive_warp(smem_u32(bars->o_free + g));
  }
}

template <typename C>
__global__ __launch_bounds__(kThreads, 1) void paged_tc_kernel(const TcArgs a) {
  extern __shared__ char smem_raw[];
  __shared__ Barriers bars;
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
      mbar_init(smem_u32(bars.q_full + g), 4);
      mbar_init(smem_u32(bars.s_full + g), 1);
      mbar_init(smem_u32(bars.p_full + g), 4);
      mbar_init(smem_u32(bars.o_full + g), 1);
      mbar_init(smem_u32(bars.o_free + g), 4);
    }
    mbar_init(smem_u32(&bars.drained), 1);
    mbar_init_fence();
  }
  chain_wait();
  chain_release();
  const int64_t total = line_total<kThreads>(a.line, shared);
  const int workers = workers_of(total, gridDim.x, a.min_steps);
  if (int(blockIdx.x) >= workers) return;
  const int64_t begin = border(total, blockIdx.x, workers);
  const Pieces pieces{border(total, blockIdx.x + 1, workers) - begin, line_place<kThreads>(a.line, begin, shared)};
  if (warp == kIssuer) tmem_alloc(smem_u32(&tmem_base), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  if (warp < kProducer) {
    regs_inc<kRegsSoftmax>();
    softmax_rows<C>(a, pieces, &bars, tmem, q, warp >> 2, notes, gave_up);
  } else if (warp < kIssuer) {
    regs_dec<kRegsProducer>();
    Fetcher<C> f{a, &bars, notes, v_ring, k_ring, gave_up, int(threadIdx.x) - kProducer * 32, 0};
    fetch_tiles<C>(f, pieces);
  } else {
    regs_dec<kRegsIssuer>();
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
  if (gave_up_word != 0 && threadIdx.x < 256) {
    // a wait ran out: the rows of this worker's whole units are marked, parts poison their join
    Pieces all = pieces;
    Piece piece;
    while (all.next(a.line, piece)) {
      const int rows = piece.seq.count * a.line.group, row = piece.block * kRows + threadIdx.x;
      if (piece.whole) {
        if (row >= rows) continue;
        const int token = row / a.line.group, h = piece.head * a.line.group + row % a.line.group;
        typename C::T* out = static_cast<typename C::T*>(a.out) + int64_t(piece.seq.first + token) * a.on + int64_t(h) * a.oh;
        for (int c = 0; c < C::D; ++c) out[c] = static_cast<typename C::T>(NAN);
      } else {
        float* slot = a.parts + (int64_t(blockIdx.x) * 2 + (piece.opens ? 1 : 0)) * slot_floats(kRows, C::D);
        slot[kRows * C::D + kRows + threadIdx.x] = NAN;
      }
    }
  }
}

template <typename C>
int launch(const TcArgs& a, cudaStream_t stream) {
  if (cudaFuncSetAttribute(paged_tc_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
    return fail(RISA_B200_CUDA, "paged attention: %s", cudaGetErrorString(cudaGetLastError()));
  // setmaxnreg deals out what the CTA was launched with; a smaller launch count would block its waits for ever
  static const bool budget = [] {
    cudaFuncAttributes attributes;
    return cudaFuncGetAttributes(&attributes, paged_tc_kernel<C>) == cudaSuccess && attributes.numRegs == kRegsLaunch;
  }();
  RISA_REQUIRE(budget, "paged attention: the tensor-core kernel was not compiled for %d registers", kRegsLaunch);
  launch_chained(paged_tc_kernel<C>, dim3(kTcWorkers), dim3(kThreads), C::SMEM, stream, a);
  const JoinArgs join{a.line, a.parts, kTcWorkers, a.min_steps, a.out, a.on, a.oh, a.lse};
  launch_chained(join_parts_kernel<typename C::T, C::D>, dim3(kTcWorkers - 1, kRows / 4), dim3(128), 0, stream, join);
  return RISA_B200_OK;
}

}  // namespace

int paged_tc_rows() { return kRows; }

int paged_tc(TcArgs a, int dtype_code, bool codes, int head_dim, cudaStream_t stream) {
  a.line.rows = Divisor(kRows);
  a.line.keys = Divisor(kTileKeys);
  if (dtype_code == 1)
    return head_dim == 64 ? (codes ? launch<Shape<__half, true, 64>>(a, stream) : launch<Shape<__half, false, 64>>(a, stream))
                          : (codes ? launch<Shape<__half, true, 128>>(a, stream) : launch<Shape<__half, false, 128>>(a, stream));
  return head_dim == 64 ? (codes ? launch<Shape<__nv_bfloat16, true, 64>>(a, stream) : launch<Shape<__nv_bfloat16, false, 64>>(a, stream))
                        : (codes ? launch<Shape<__nv_bfloat16, true, 128>>(a, stream) : launch<Shape<__nv_bfloat16, false, 128>>(a, stream));
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
