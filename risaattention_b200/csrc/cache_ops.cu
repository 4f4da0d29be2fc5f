// Rotary positions, the append that fills a paged key/value cache, and eviction from it: the serving
// operators that move data.  All are bounded by memory traffic (large) or by launch latency (steps).
#include "four_bits.cuh"
#include "paged_tc.cuh"
#include "serving.cuh"

namespace risa_b200 {
namespace serving {

__device__ unsigned int g_bad_page;

unsigned int* status_word() {
  void* address = nullptr;
  if (cudaGetSymbolAddress(&address, g_bad_page) != cudaSuccess) {
    fail(RISA_B200_CUDA, "cache status word: %s", cudaGetErrorString(cudaGetLastError()));
    return nullptr;
  }
  return static_cast<unsigned int*>(address);
}

// Reports (and clears) what the kernels recorded.
int device_status() {
  const int attention_site = paged_tc_wait_status(), weigh_site = weigh_tc_wait_status();
  const int site = attention_site != 0 ? attention_site : weigh_site;
  if (site < 0) return fail(RISA_B200_CUDA, "device status: %s", cudaGetErrorString(cudaGetLastError()));
  if (site > 0) return fail(RISA_B200_DEVICE, "kernel over a paged cache gave up waiting at site %d (bounded wait expired)", site);
  unsigned int status = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&status, g_bad_page, sizeof(status)) != cudaSuccess)
    return fail(RISA_B200_CUDA, "device status: %s", cudaGetErrorString(cudaGetLastError()));
  if (status == 0) return RISA_B200_OK;
  cudaMemcpyToSymbol(g_bad_page, &zero, sizeof(zero));
  return fail(RISA_B200_DEVICE, "a page table leads sequence %u to a page outside the pool, or ends before the sequence does",
              status - 1);
}

namespace {

// ---- angles --------------------------------------------------------------------------------------------
// Positions are whole numbers and an angle matters modulo one turn, so the angle is kept in units of
// 2^-64 turns: position * turns wraps modulo 2^64 exactly where the angle wraps, and a far position
// loses nothing (a 32-bit product of position 10^6 and a frequency near 1 is off by 0.03 radians).
// The top 32 bits as a signed number are the angle in (-1/2, 1/2] turns, which sincospi takes.
__device__ __forceinline__ void angle_of(int64_t position, uint64_t turns, float magnitude, float& c, float& s) {
  const uint64_t angle = uint64_t(position) * turns;
  sincospif(float(int32_t(angle >> 32)) * 0x1p-31f, &s, &c);
  c *= magnitude;
  s *= magnitude;
}

__device__ __forceinline__ int64_t position_at(const void* positions, int is64, int64_t index) {
  return is64 ? __ldg(static_cast<const long long*>(positions) + index)
              : int64_t(__ldg(static_cast<const int*>(positions) + index));
}

// ---- eight consecutive channels --------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Half2<T>::unpack(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float* x) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x) {
  uint4 raw;
  raw.x = Half2<T>::pack(x[0], x[1]);
  raw.y = Half2<T>::pack(x[2], x[3]);
  raw.z = Half2<T>::pack(x[4], x[5]);
  raw.w = Half2<T>::pack(x[6], x[7]);
  *reinterpret_cast<uint4*>(p) = raw;
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float* x) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// The same as it was loaded: as many of them as registers hold are on their way at once.
template <typename T>
struct Run {
  uint4 raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { raw = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void values(float* x) const { load8(reinterpret_cast<const T*>(&raw), x); }
};
template <>
struct Run<float> {
  float4 raw[2];
  __device__ __forceinline__ void load(const float* p) {
    raw[0] = reinterpret_cast<const float4*>(p)[0];
    raw[1] = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void values(float* x) const { load8(reinterpret_cast<const float*>(raw), x); }
};

// ---- rotation ----------------------------------------------------------------------------------------------
struct RotateArgs {
  const void* x;
  void* out;
  const void* positions;
  const uint64_t* turns;
  int64_t xb, xh, xn, ob, oh, on, pb, pn;
  int batch, heads, tokens, head_dim, rotary_dim, heads_each, chunks;
  int positions_64, interleaved, transposed;
  float magnitude;
  const uint8_t* axes;  // of the pairs, nullptr: all follow one axis
  int64_t pa;           // from one axis' positions to the next one's
  int last_axis;
};

// A thread owns eight pairs of one token (two runs of eight channels) in `heads_each` heads, so that
// its eight cosines and sines serve them all; behind the pairs come the threads that copy eight
// channels each.  Consecutive threads are consecutive runs of a row, then rows of consecutive tokens.  Bound by HBM: the
// loads of four heads are on their way at once (2 x 16 heads x 16K tokens of 128 bf16 channels, half of them rotated: 78 us
// with two, 57 with four, 4.7 TB/s).
// With positions of several axes each of the eight pairs looks up its own (the same few cache lines).  In FP32 the rows of four heads
// are 64 registers of the 64 that a thread has: 572 bytes of spill stores and 956 of loads, and 134 us for 2 x 16 heads x 16K rows of
// 128 channels (4.0 TB/s; 16-bit rows spill 48 and 100 bytes, 47 us, 5.7 TB/s).
constexpr int kHeadsAhead = 4;
template <typename T, bool AXES>
__global__ __launch_bounds__(256, 4) void rotate_kernel(const RotateArgs a) {
  chain_wait();
  chain_release();
  const int pairs = a.rotary_dim / 16, items = pairs + (a.head_dim - a.rotary_dim) / 8;
  const int64_t index = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (index >= int64_t(a.tokens) * items) return;
  const int token = int(index / items), item = int(index % items), b = blockIdx.z;
  const int h0 = blockIdx.y * a.heads_each, h1 = min(h0 + a.heads_each, a.heads);
  const T* x = static_cast<const T*>(a.x) + b * a.xb + token * a.xn;
  T* out = static_cast<T*>(a.out) + b * a.ob + token * a.on;
  if (item >= pairs) {
    if (a.out == a.x) return;
    const int c = a.rotary_dim + (item - pairs) * 8;
    for (int h = h0; h < h1; h += 8) {  // eight at a time on their way
      Run<T> v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (h + i < h1) v[i].load(x + (h + i) * a.xh + c);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (h + i < h1) *reinterpret_cast<Run<T>*>(out + (h + i) * a.oh + c) = v[i];
    }
    return;
  }
  const int64_t at = b * a.pb + token * a.pn;
  int64_t position = AXES ? 0 : position_at(a.positions, a.positions_64, at);
  uint2 axes = make_uint2(0, 0);
  if (AXES) axes = __ldg(reinterpret_cast<const uint2*>(a.axes) + item);
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (AXES) position = position_at(a.positions, a.positions_64, at + min(int((i < 4 ? axes.x : axes.y) >> (8 * (i & 3)) & 0xff), a.last_axis) * a.pa);
    angle_of(position, __ldg(reinterpret_cast<const unsigned long long*>(a.turns) + item * 8 + i), a.magnitude, cs[i], sn[i]);
    if (a.transposed) sn[i] = -sn[i];
  }
  const int c0 = a.interleaved ? item * 16 : item * 8;
  const int c1 = a.interleaved ? c0 + 8 : a.rotary_dim / 2 + item * 8;
  auto turn = [&](float (&u)[8], float (&v)[8]) {
    if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = u[2 * i], q = u[2 * i + 1];
        u[2 * i] = p * cs[i] - q * sn[i];
        u[2 * i + 1] = q * cs[i] + p * sn[i];
        const float r = v[2 * i], s = v[2 * i + 1];
        v[2 * i] = r * cs[4 + i] - s * sn[4 + i];
        v[2 * i + 1] = s * cs[4 + i] + r * sn[4 + i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = u[i], q = v[i];
        u[i] = p * cs[i] - q * sn[i];
        v[i] = q * cs[i] + p * sn[i];
      }
    }
  };
  int h = h0;
  for (; h + kHeadsAhead <= h1; h += kHeadsAhead) {
    Run<T> u[kHeadsAhead], v[kHeadsAhead];
#pragma unroll
    for (int i = 0; i < kHeadsAhead; ++i) {
      u[i].load(x + (h + i) * a.xh + c0);
      v[i].load(x + (h + i) * a.xh + c1);
    }
#pragma unroll
    for (int i = 0; i < kHeadsAhead; ++i) {
      float p[8], q[8];
      u[i].values(p);
      v[i].values(q);
      turn(p, q);
      store8(out + (h + i) * a.oh + c0, p);
      store8(out + (h + i) * a.oh + c1, q);
    }
  }
  for (; h < h1; ++h) {
    float u[8], v[8];
    load8(x + h * a.xh + c0, u);
    load8(x + h * a.xh + c1, v);
    turn(u, v);
    store8(out + h * a.oh + c0, u);
    store8(out + h * a.oh + c1, v);
  }
}

// Any even rotary width, any stride and alignment: one pair (or one copied channel) per thread.
template <typename T>
__global__ __launch_bounds__(256) void rotate_any_kernel(const RotateArgs a) {
  chain_wait();
  chain_release();
  const int pairs = a.rotary_dim / 2, items = pairs + a.head_dim - a.rotary_dim;
  const int64_t index = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (index >= int64_t(a.tokens) * items) return;
  const int token = int(index / items), item = int(index % items), b = blockIdx.z;
  const int h0 = blockIdx.y * a.heads_each, h1 = min(h0 + a.heads_each, a.heads);
  const T* x = static_cast<const T*>(a.x) + b * a.xb + token * a.xn;
  T* out = static_cast<T*>(a.out) + b * a.ob + token * a.on;
  if (item >= pairs) {
    const int c = a.rotary_dim + item - pairs;
    for (int h = h0; h < h1; ++h) out[h * a.oh + c] = x[h * a.xh + c];
    return;
  }
  const int64_t axis = a.axes != nullptr ? min(int(__ldg(a.axes + item)), a.last_axis) * a.pa : 0;
  const int64_t position = position_at(a.positions, a.positions_64, b * a.pb + token * a.pn + axis);
  float c, s;
  angle_of(position, __ldg(reinterpret_cast<const unsigned long long*>(a.turns) + item), a.magnitude, c, s);
  if (a.transposed) s = -s;
  const int c0 = a.interleaved ? item * 2 : item, c1 = a.interleaved ? c0 + 1 : pairs + item;
  for (int h = h0; h < h1; ++h) {
    const float p = static_cast<float>(x[h * a.xh + c0]), q = static_cast<float>(x[h * a.xh + c1]);
    out[h * a.oh + c0] = static_cast<T>(p * c - q * s);
    out[h * a.oh + c1] = static_cast<T>(q * c + p * s);
  }
}

// ---- append ------------------------------------------------------------------------------------------------
struct AppendArgs {
  StepView step;
  void* keys;
  void* values;
  float* key_scales;
  float* value_scales;
  const void *k, *v, *q;
  void* q_out;
  int64_t kn, kh, vn, vh, qn, qh, on, oh;
  int pages, kv_heads, q_heads, head_dim;
  const uint64_t* turns;  // nullptr: nothing turns
  const void* positions;
  int rotary_dim, interleaved, positions_64;
  float magnitude;
  const uint8_t* axes;  // of the pairs, nullptr: all follow one axis
  int64_t axis_stride;
  int last_axis;
  unsigned int* status;
};

// Largest |x| of a row held by `lanes` neighbouring threads; NaN wins, so that it shows in the scale.
__device__ __forceinline__ float row_absmax(const float* x, int lanes) {
  float m = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(x[i])));
  for (int off = lanes >> 1; off > 0; off >>= 1)
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(__shfl_xor_sync(0xffffffffu, m, off)));
  return m;
}

// A row in 4 bits (four_bits.cuh): this lane's eight channels, the scale of its group and the token's exponent.
struct Row4 {
  uint32_t word, group;
  int exponent;
};
// The token's scale is the smallest power of two, 2^-126 at least, of which the row's largest value is at most 3136 = 7 * 448.
constexpr uint32_t kAbove3136 = 0x7fffffu - 0x440000u;  // carries into the exponent where the mantissa is above that of 3136
__device__ __forceinline__ uint32_t e4m3_pair(float hi, float lo) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Channel 2 i + j in bits 16 j + 4 i.
__device__ __forceinline__ uint32_t code_bits(int code, int channel) { return uint32_t(min(max(code, -7), 7) + 8) << (16 * (channel & 1) + 4 * (channel >> 1)); }

// Group scale: the largest value of the group over 7 token scales, rounded to e4m3.  Code: the value over both scales, rounded
// to nearest even.  Values of 16 bits meet the borders between codes (and between scales) exactly or not nearly, so that
// for rows as they came this is decided in 32 bits: quotients corrected by their remainders are exact where they meet one.  Rotated
// values are off by 2^-20.9 of the row's largest value at most: the angle is rounded to 2^-25 of half a turn and sincospi gives two
// units in the last place, 2^-22.2 of a pair whose length is sqrt(2) times that value at most, and two roundings follow; the quotient
// adds 2^-22.8.  `doubtful` says that one of them lies within 1.5 x 2^-20, more than twice the sum, of a border: of its token's scale,
// and where this lane's channels were `turned` (a group is, or is not) of its group's scale, or between codes of a group that has any;
// or that the row is not finite, which a finite one of bf16 can become in 32 bits.  (Values below 2^-126 are whole multiples of 2^-149
// and so are the borders between their codes and scales: what is off by less than that meets a border or stays on its side.)
template <int LANES, bool ROTATED>
__device__ __forceinline__ Row4 row4_of(const float (&x)[8], bool turned, bool& doubtful) {
  float group = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(group) : "f"(fabsf(x[i])));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(group) : "f"(__shfl_xor_sync(0xffffffffu, group, 1)));
  float most = group;
#pragma unroll
  for (int off = LANES / 2; off > 1; off >>= 1)
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(__shfl_xor_sync(0xffffffffu, most, off)));
  const uint32_t bits = __float_as_uint(most) + kAbove3136;
  const bool usable = most > 0.f && most < INFINITY;
  Row4 r;
  r.exponent = usable ? max(int(bits >> 23) - 11, 1) : most == 0.f ? 0 : 255;
  const float to_units = __uint_as_float(uint32_t(254 - r.exponent) << 23), size = group * to_units, third = size * (1.0f / 7.0f);
  const float ratio = fmaf(fmaf(-third, 7.0f, size), 1.0f / 7.0f, third);  // exact where a border of scales is met
  r.group = e4m3_pair(0.f, ratio) & 0xffu;
  const float scale = __half2float(__ushort_as_half(uint16_t(r.group << 7))) * kGroupUnit;
  float inverse;
  asm("rcp.approx.f32 %0, %1;" : "=f"(inverse) : "f"(scale));
  float code[8], nearest = 1.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = x[i] * to_units, guess = y * inverse;
    const float quotient = fmaf(fmaf(-guess, scale, y), inverse, guess);  // exact where it is half of a whole number
    code[i] = (quotient + 12582912.0f) - 12582912.0f;
    if (ROTATED) nearest = fminf(nearest, fabsf(fabsf(quotient - code[i]) - 0.5f));
  }
  if (ROTATED) {
    const float slack = most * to_units * 0x1.8p-20f;
    const uint32_t around = e4m3_pair(fmaf(slack, 1.0f / 7.0f, ratio), fmaxf(fmaf(slack, -1.0f / 7.0f, ratio), 0.f));
    doubtful = !(most < INFINITY) || (usable && ((turned && ((r.group != 0 && nearest * scale < slack) || (around & 0xffu) != around >> 8)) ||
                                                 (bits - 24) >> 23 != (bits + 24) >> 23));
  }
  if (__any_sync(0xffffffffu, r.group < 8)) {  // scales below 2^-6 are rounded coarsely: quotients past 7
#pragma unroll
    for (int i = 0; i < 8; ++i) code[i] = fminf(fmaxf(code[i], -7.f), 7.f);
  }
  float half_words[2] = {8388608.0f + 0x8888, 8388608.0f + 0x8888};  // four codes + 8 in the low bits
#pragma unroll
  for (int i = 0; i < 8; ++i) half_words[i & 1] = fmaf(code[i], float(1 << (4 * (i >> 1))), half_words[i & 1]);
  r.word = usable && r.group != 0 ? __byte_perm(__float_as_uint(half_words[0]), __float_as_uint(half_words[1]), 0x5410) : 0x88888888u;
  r.group = usable ? r.group : 0;
  return r;
}
// The same for a rotated row that came too near a border, in 64 bits: from the channels as they came (`own`, and `other` of a
// lane half a rotated row away).  0.4 % of Gaussian rows of 128; nearly all rows with a turned group of 2^-18 to 2^-12 of the row's largest
// value, whose codes are hardly wider than the rotation's own error (8160 tokens of such keys 127 us, others 62).
template <typename T>
__device__ __noinline__ Row4 row4_of_rotated(const AppendArgs& a, Run<T> own, Run<T> other, int64_t token, int place, int lanes, int channel) {
  float u[8], v[8];
  own.values(u);
  other.values(v);
  auto larger = [](double m, double x) { return x > m || x != x ? x : m; };
  double x[8], most = 0.0;
  const int half = a.rotary_dim >> 1;
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    const int c = channel + i;
    x[i] = u[i];
    if (c < a.rotary_dim) {
      const bool second = a.interleaved ? c & 1 : c >= half;
      const int pair = a.interleaved ? c >> 1 : second ? c - half : c;
      const int64_t axis = a.axes != nullptr ? min(int(__ldg(a.axes + pair)), a.last_axis) * a.axis_stride : 0;
      const int64_t position = a.positions ? position_at(a.positions, a.positions_64, token + axis) : int64_t(place);
      const uint64_t angle = uint64_t(position) * __ldg(reinterpret_cast<const unsigned long long*>(a.turns) + pair);
      double sine, cosine;
      sincospi(double(int64_t(angle)) * 0x1p-63, &sine, &cosine);
      const double partner = a.interleaved ? u[i ^ 1] : v[i];
      x[i] = double(a.magnitude) * (u[i] * cosine + (second ? partner : -partner) * sine);
    }
    most = larger(most, fabs(x[i]));
  }
  const double group = larger(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = group;
  for (int off = lanes >> 1; off > 1; off >>= 1) most = larger(most, __shfl_xor_sync(0xffffffffu, most, off));
  Row4 r{0x88888888u, 0, 0};
  if (most == 0.0) return r;
  r.exponent = 255;  // not finite, or larger (by the table's magnitude) than any 7 * 448 token scales that readers take times 2^8
  if (!(most <= 3136.0 * 0x1p119)) return r;
  r.exponent = max(int((__double_as_longlong(most) + (0xfffffffffffffll - 0x8800000000000ll)) >> 52) - 1023 - 11 + 127, 1);
  const double to_units = __longlong_as_double(int64_t(1023 + 127 - r.exponent) << 52), ratio = group * to_units / 7.0;
  // steps of 2^-3 of the leading bit, 2^-9 at least
  const double step = __longlong_as_double(int64_t(max(int(__double_as_longlong(ratio) >> 52) - 3, 1023 - 9)) << 52);
  const double scale = rint(ratio / step) * step;
  r.group = e4m3_pair(0.f, float(scale)) & 0xffu;
  if (scale == 0.0) return r;
  r.word = 0;
#pragma unroll 1
  for (int i = 0; i < 8; ++i) r.word |= code_bits(int(rint(x[i] * to_units / scale)), i);
  return r;
}

// One CTA per new token.  head_dim / 8 lanes hold a row, eight channels each; the CTA's row slots walk
// the token's query heads, key heads and value heads with the cosines and sines of the lane's channels
// kept in registers.  A thread computes those of one pair for the whole token (8160 tokens below: 70 us where every lane
// computed its own).
// The second channel of a pair sits in the same lane (interleaved) or in the lane half a rotated row
// away, whose channels come by shuffle.  Codes: absolute maximum over 127, rounded to nearest even; a row of
// zeros has scale 0, a row with an infinity or a NaN reads back as NaN.  8160 tokens of 32 + 2 x 8 heads, bf16 to codes:
// 56 us (184 MB, 3.3 TB/s), bound by each CTA's chain of lookups and by the instructions of conversions; one token of 64
// requests, with the call: 11.5 to 12.4 us.
constexpr int kRowsAhead = 3;  // rows of a slot on their way at once: half of a token of 32 + 2 x 8 heads of 128
template <typename T, int BITS>
__global__ __launch_bounds__(128, 8) void append_kernel(const AppendArgs a) {
  __shared__ __align__(16) float cosines[128], sines[128];
  chain_wait();
  chain_release();
  const int token = blockIdx.x, lanes = a.head_dim >> 3;
  const int lane = threadIdx.x & (lanes - 1), slot = threadIdx.x / lanes, slots = 128 / lanes, channel = lane * 8;
  const int rows = a.q_heads + 2 * a.kv_heads;
  // Rows are on their way before their place is looked up: kRowsAhead of them from r0 on.
  Run<T> run[kRowsAhead];
  auto load_rows = [&](int r0) {
#pragma unroll
    for (int j = 0; j < kRowsAhead; ++j) {
      const int r = r0 + j * slots + slot;
      run[j].zero();
      if (r < rows)
        run[j].load((r < a.q_heads ? static_cast<const T*>(a.q) + token * a.qn + r * a.qh
                     : r < a.q_heads + a.kv_heads ? static_cast<const T*>(a.k) + token * a.kn + (r - a.q_heads) * a.kh
                                                  : static_cast<const T*>(a.v) + token * a.vn + (r - a.q_heads - a.kv_heads) * a.vh) +
                    channel);
    }
  };
  load_rows(0);
  // the sequence whose tokens include this one: as many as end in front of it, counted 128 at a time
  int s = token;
  if (a.step.offsets != nullptr) {
    s = 0;
    for (int i = 0; i < a.step.batch; i += 128)
      s += __syncthreads_count(i + int(threadIdx.x) < a.step.batch && __ldg(a.step.offsets + i + threadIdx.x + 1) <= token);
  }
  int place = -1;
  bool belongs = false;
  if (s < a.step.batch) {
    const int first = a.step.offsets ? __ldg(a.step.offsets + s) : s;
    const int end = a.step.offsets ? __ldg(a.step.offsets + s + 1) : s + 1;
    belongs = token >= first;
    place = __ldg(a.step.lengths + s) - (end - token);
  }
  if (!belongs) {  // a row behind the last sequence
    for (int h = slot; h < a.q_heads; h += slots)
      *reinterpret_cast<uint4*>(static_cast<T*>(a.q_out) + token * a.on + h * a.oh + lane * 8) = make_uint4(0, 0, 0, 0);
    return;
  }
  int64_t page = -1;
  if (place >= 0 && (place >> a.step.page_shift) < a.step.width) {
    page = __ldg(a.step.table + int64_t(s) * a.step.width + (place >> a.step.page_shift));
    if (page < 0 || page >= a.pages) {
      page = -1;
      if (threadIdx.x == 0) atomicCAS(a.status, 0u, unsigned(s) + 1u);
    }
  } else if (place >= 0 && threadIdx.x == 0) {
    atomicCAS(a.status, 0u, unsigned(s) + 1u);  // longer than its row of the table
  }
  const bool turned = a.turns != nullptr && channel < a.rotary_dim;
  float cs[8] = {}, sn[8] = {};
  int partner = threadIdx.x & 31;
  if (a.turns != nullptr) {  // one thread for each pair of the token, then every lane takes those of its channels
    const int half = a.rotary_dim >> 1;
    if (int(threadIdx.x) < half) {
      const int64_t axis = a.axes != nullptr ? min(int(__ldg(a.axes + threadIdx.x)), a.last_axis) * a.axis_stride : 0;
      const int64_t position = a.positions ? position_at(a.positions, a.positions_64, token + axis) : int64_t(place);
      angle_of(position, __ldg(reinterpret_cast<const unsigned long long*>(a.turns) + threadIdx.x), a.magnitude, cosines[threadIdx.x], sines[threadIdx.x]);
    }
    __syncthreads();
    if (turned) {
      const bool second = !a.interleaved && channel >= half;
      const int pair0 = a.interleaved ? channel >> 1 : second ? channel - half : channel;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        if (a.interleaved && i == 4) break;
        const float4 c = *reinterpret_cast<const float4*>(cosines + pair0 + i), d = *reinterpret_cast<const float4*>(sines + pair0 + i);
        cs[i] = c.x; cs[i + 1] = c.y; cs[i + 2] = c.z; cs[i + 3] = c.w;
        sn[i] = d.x; sn[i + 1] = d.y; sn[i + 2] = d.z; sn[i + 3] = d.w;
      }
      if (second)
#pragma unroll
        for (int i = 0; i < 8; ++i) sn[i] = -sn[i];  // b cos + a sin as b cos - a (-sin)
      if (!a.interleaved) partner = (threadIdx.x & 31) + (second ? -(half >> 3) : (half >> 3));
    }
  }
  const int slot_in_page = place & ((1 << a.step.page_shift) - 1);
  for (int r0 = 0; r0 < rows; r0 += slots * kRowsAhead) {
    if (r0 > 0) load_rows(r0);
#pragma unroll
    for (int j = 0; j < kRowsAhead; ++j) {
      if (r0 + j * slots >= rows) break;  // the same for the whole CTA
      const int r = r0 + j * slots + slot;
      const bool there = r < rows;
      const int kind = r < a.q_heads ? 0 : r < a.q_heads + a.kv_heads ? 1 : 2;
      const int h = kind == 0 ? r : kind == 1 ? r - a.q_heads : r - a.q_heads - a.kv_heads;
      float x[8];
      run[j].values(x);
      if (a.turns != nullptr && __any_sync(0xffffffffu, kind < 2)) {
        if (a.interleaved) {
          if (turned && kind < 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float p = x[2 * i], q = x[2 * i + 1];
              x[2 * i] = p * cs[i] - q * sn[i];
              x[2 * i + 1] = q * cs[i] + p * sn[i];
            }
          }
        } else {
          Run<T> other;
          other.raw.x = __shfl_sync(0xffffffffu, run[j].raw.x, partner);
          other.raw.y = __shfl_sync(0xffffffffu, run[j].raw.y, partner);
          other.raw.z = __shfl_sync(0xffffffffu, run[j].raw.z, partner);
          other.raw.w = __shfl_sync(0xffffffffu, run[j].raw.w, partner);
          if (turned && kind < 2) {
            float y[8];
            other.values(y);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * cs[i] - y[i] * sn[i];
          }
        }
      }
      const int64_t row = ((page * a.kv_heads + h) << a.step.page_shift) + slot_in_page;
      if (BITS == 8 && __any_sync(0xffffffffu, kind > 0)) {
        const float most = row_absmax(x, lanes), scale = most / 127.0f;
        if (there && kind > 0 && page >= 0) {
          // one reciprocal for the row; rows so small that it would overflow are divided
          const float inverse = 127.0f / most;
          float c[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) c[i] = most > 1e-35f ? x[i] * inverse : scale > 0.f ? x[i] / scale : 0.f;
          char* codes = static_cast<char*>(kind == 1 ? a.keys : a.values);
          *reinterpret_cast<uint2*>(codes + row * a.head_dim + channel) =
              make_uint2(pack4_s8(c[0], c[1], c[2], c[3]), pack4_s8(c[4], c[5], c[6], c[7]));
          if (lane == 0) (kind == 1 ? a.key_scales : a.value_scales)[row] = scale;
        }
      }
      if (BITS == 16 && there && kind > 0 && page >= 0) {
        store8(static_cast<T*>(kind == 1 ? a.keys : a.values) + row * a.head_dim + channel, x);
      }
      if (there && kind == 0) store8(static_cast<T*>(a.q_out) + token * a.on + h * a.oh + channel, x);
    }
  }
}

// In 4 bits: a kernel of its own, in which a CTA's row slots walk the token's query heads, then its keys, then its values (what is
// computed of a row in 4 bits is three times as much as of a rotated one).  8160 tokens of 32 + 2 x 8 heads of 128: 67 us with
// positions of three axes (184 MB, 2.7 TB/s), 62 with those of one; 87 in the kernel for all kinds of cache, whose every row paid for
// the registers of the call that decides doubtful ones.  Latency bounds it: of the 6.4 warps that a scheduler has, 1.1 wait for
// global memory (the look-ups in front of a token's rows, with nothing of another token on its way in that CTA), 1.4 for shared memory
// and shuffles, 1.0 for results of fixed latency and 0.6 at barriers; 56 % of the issue slots are used, HBM at 32 %.
constexpr int kQueriesAhead = 4;
template <typename T, int LANES>
__global__ __launch_bounds__(128, 7) void append4_kernel(const AppendArgs a) {
  __shared__ __align__(16) float cosines[128], sines[128];
  chain_wait();
  chain_release();
  constexpr int SLOTS = 128 / LANES, GROUPS = LANES / 2;
  const int token = blockIdx.x, lane = threadIdx.x % LANES, slot = threadIdx.x / LANES, channel = lane * 8;
  const T* const k0 = static_cast<const T*>(a.k) + token * a.kn + channel;
  const T* const v0 = static_cast<const T*>(a.v) + token * a.vn + channel;
  const T* const q0 = static_cast<const T*>(a.q) + token * a.qn + channel;
  T* const o0 = static_cast<T*>(a.q_out) + token * a.on + channel;
  // the first rows are on their way before their place is looked up
  Run<T> q[kQueriesAhead], k, v;
  auto load_queries = [&](int h0) {
#pragma unroll
    for (int j = 0; j < kQueriesAhead; ++j) {
      const int h = h0 + j * SLOTS + slot;
      q[j].zero();
      if (h < a.q_heads) q[j].load(q0 + h * a.qh);
    }
  };
  load_queries(0);
  k.zero();
  v.zero();
  if (slot < a.kv_heads) {
    k.load(k0 + slot * a.kh);
    v.load(v0 + slot * a.vh);
  }
  int s = token;
  if (a.step.offsets != nullptr) {
    s = 0;
    for (int i = 0; i < a.step.batch; i += 128)
      s += __syncthreads_count(i + int(threadIdx.x) < a.step.batch && __ldg(a.step.offsets + i + threadIdx.x + 1) <= token);
  }
  int place = -1;
  bool belongs = false;
  if (s < a.step.batch) {
    const int first = a.step.offsets ? __ldg(a.step.offsets + s) : s;
    const int end = a.step.offsets ? __ldg(a.step.offsets + s + 1) : s + 1;
    belongs = token >= first;
    place = __ldg(a.step.lengths + s) - (end - token);
  }
  if (!belongs) {  // a row behind the last sequence
    for (int h = slot; h < a.q_heads; h += SLOTS) *reinterpret_cast<uint4*>(o0 + h * a.oh) = make_uint4(0, 0, 0, 0);
    return;
  }
  int64_t page = -1;
  if (place >= 0) {
    if ((place >> a.step.page_shift) < a.step.width) page = __ldg(a.step.table + int64_t(s) * a.step.width + (place >> a.step.page_shift));
    if (page < 0 || page >= a.pages) {  // outside the pool, or the sequence is longer than its row of the table
      page = -1;
      if (threadIdx.x == 0) atomicCAS(a.status, 0u, unsigned(s) + 1u);
    }
  }
  const bool turns = a.turns != nullptr, turned = turns && channel < a.rotary_dim;
  float cs[8] = {}, sn[8] = {};
  int partner = threadIdx.x & 31;
  if (turns) {  // one thread for each pair of the token, then every lane takes those of its channels
    const int half = a.rotary_dim >> 1;
    if (int(threadIdx.x) < half) {
      const int64_t axis = a.axes != nullptr ? min(int(__ldg(a.axes + threadIdx.x)), a.last_axis) * a.axis_stride : 0;
      const int64_t position = a.positions ? position_at(a.positions, a.positions_64, token + axis) : int64_t(place);
      angle_of(position, __ldg(reinterpret_cast<const unsigned long long*>(a.turns) + threadIdx.x), a.magnitude, cosines[threadIdx.x], sines[threadIdx.x]);
    }
    __syncthreads();
    if (turned) {
      const bool second = !a.interleaved && channel >= half;
      const int pair0 = a.interleaved ? channel >> 1 : second ? channel - half : channel;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        if (a.interleaved && i == 4) break;
        const float4 c = *reinterpret_cast<const float4*>(cosines + pair0 + i), d = *reinterpret_cast<const float4*>(sines + pair0 + i);
        cs[i] = c.x; cs[i + 1] = c.y; cs[i + 2] = c.z; cs[i + 3] = c.w;
        sn[i] = d.x; sn[i + 1] = d.y; sn[i + 2] = d.z; sn[i + 3] = d.w;
      }
      if (second)
#pragma unroll
        for (int i = 0; i < 8; ++i) sn[i] = -sn[i];  // b cos + a sin as b cos - a (-sin)
      if (!a.interleaved) partner = (threadIdx.x & 31) + (second ? -(half >> 3) : (half >> 3));
    }
  }
  auto partner_of = [&](const Run<T>& run) {
    Run<T> other;
    other.raw.x = __shfl_sync(0xffffffffu, run.raw.x, partner);
    other.raw.y = __shfl_sync(0xffffffffu, run.raw.y, partner);
    other.raw.z = __shfl_sync(0xffffffffu, run.raw.z, partner);
    other.raw.w = __shfl_sync(0xffffffffu, run.raw.w, partner);
    return other;
  };
  auto turn = [&](const Run<T>& run, float (&x)[8]) {  // by the whole warp
    run.values(x);
    if (a.interleaved) {
      if (turned) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = x[2 * i], q = x[2 * i + 1];
          x[2 * i] = p * cs[i] - q * sn[i];
          x[2 * i + 1] = q * cs[i] + p * sn[i];
        }
      }
    } else {
      float y[8];
      partner_of(run).values(y);
      if (turned) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * cs[i] - y[i] * sn[i];
      }
    }
  };
  for (int h0 = 0; h0 < a.q_heads; h0 += SLOTS * kQueriesAhead) {
    if (h0 > 0) load_queries(h0);
#pragma unroll
    for (int j = 0; j < kQueriesAhead; ++j) {
      if (h0 + j * SLOTS >= a.q_heads) break;  // the same for the whole CTA
      float x[8];
      turn(q[j], x);
      const int h = h0 + j * SLOTS + slot;
      if (h < a.q_heads) store8(o0 + h * a.oh, x);
    }
  }
  if (page < 0) return;
  // where this lane's word of head 0 lies, and the scales of the token
  const int in_page = place & ((1 << a.step.page_shift) - 1);
  const int64_t of_page = page * a.kv_heads;
  const int64_t word0 = ((of_page << a.step.page_shift) + in_page) * LANES + lane, scales0 = (of_page * (1 + GROUPS)) << a.step.page_shift;
  auto store = [&](void* codes, float* scales, int h, const Row4& r) {
    static_cast<uint32_t*>(codes)[word0 + int64_t(h) * (LANES << a.step.page_shift)] = r.word;
    uint8_t* of = reinterpret_cast<uint8_t*>(scales) + scales0 + int64_t(h) * ((1 + GROUPS) << a.step.page_shift);
    if (lane == 0) of[in_page] = uint8_t(r.exponent);
    if ((lane & 1) == 0) of[(1 << a.step.page_shift) + in_page * GROUPS + (lane >> 1)] = uint8_t(r.group);
  };
  uint32_t again = 0;  // rounds (modulo 32) of this warp whose keys came too near a border
  for (int h0 = 0, round = 0; h0 < a.kv_heads; h0 += SLOTS, ++round) {
    const int h = h0 + slot;
    if (h0 > 0) {
      k.zero();
      v.zero();
      if (h < a.kv_heads) {
        k.load(k0 + h * a.kh);
        v.load(v0 + h * a.vh);
      }
    }
    float x[8];
    bool doubtful = false;
    if (turns) turn(k, x);
    else k.values(x);
    const Row4 of_key = row4_of<LANES, true>(x, turned, doubtful);
    if (turns && __any_sync(0xffffffffu, doubtful && h < a.kv_heads)) again |= 1u << (round & 31);
    v.values(x);
    const Row4 of_value = row4_of<LANES, false>(x, false, doubtful);
    if (h < a.kv_heads) {
      store(a.keys, a.key_scales, h, of_key);
      store(a.values, a.value_scales, h, of_value);
    }
  }
  // such rows once more, in 64 bits
#pragma unroll 1
  for (int h0 = 0, round = 0; again != 0 && h0 < a.kv_heads; h0 += SLOTS, ++round) {
    if (!(again >> (round & 31) & 1)) continue;
    const int h = h0 + slot;
    k.zero();
    if (h < a.kv_heads) k.load(k0 + h * a.kh);
    const Row4 r = row4_of_rotated<T>(a, k, partner_of(k), token, place, LANES, channel);
    if (h < a.kv_heads) store(a.keys, a.key_scales, h, r);
  }
}

// ---- reading back -----------------------------------------------------------------------------------------
struct ReadArgs {
  StepView step;
  const void* keys;
  const void* values;
  const float* key_scales;
  const float* value_scales;
  void *k, *v;
  int64_t kn, kh, vn, vh;
  int pages, kv_heads, head_dim;
  unsigned int* status;
};

// A warp per token of a step, tokens as append has them; head_dim / 8 lanes hold a row, and as many rows as fit the warp are
// taken at once, four times over before the first is stored.  (A CTA per token, 8160 tokens of 2 x 8 heads of 128 from 4 bits: 20 us,
// most of it the search for the sequence; so 13.)  Eight sequences of 8192 tokens: 84 us from bf16 (6.4 TB/s), 69 from INT8
// (5.9), 94 from 4 bits (3.7), whose copies are of 4 bytes a lane.
constexpr int kReadWarps = 4, kReadAhead = 4;
template <typename T, int BITS>
__global__ __launch_bounds__(kReadWarps * 32) void read_kernel(const ReadArgs a) {
  chain_wait();
  chain_release();
  const int token = blockIdx.x * kReadWarps + (threadIdx.x >> 5);
  if (token >= a.step.tokens) return;
  const int lanes = a.head_dim >> 3, lane = threadIdx.x & (lanes - 1), slot = (threadIdx.x & 31) / lanes, slots = 32 / lanes;
  int s = token;
  if (a.step.offsets != nullptr) {
    s = 0;
    for (int i = 0; i < a.step.batch; i += 32) {
      const int at = i + int(threadIdx.x & 31);
      const unsigned int in_front = __ballot_sync(0xffffffffu, at < a.step.batch && __ldg(a.step.offsets + at + 1) <= token);
      s += __popc(in_front);
      if (in_front != 0xffffffffu) break;
    }
  }
  int64_t page = -1;
  int place = -1;
  if (s < a.step.batch && (a.step.offsets == nullptr || token >= __ldg(a.step.offsets + s))) {
    place = __ldg(a.step.lengths + s) - ((a.step.offsets ? __ldg(a.step.offsets + s + 1) : s + 1) - token);
    if (place >= 0) {
      if ((place >> a.step.page_shift) < a.step.width) page = __ldg(a.step.table + int64_t(s) * a.step.width + (place >> a.step.page_shift));
      if (page < 0 || page >= a.pages) {
        page = -1;
        if ((threadIdx.x & 31) == 0) atomicCAS(a.status, 0u, unsigned(s) + 1u);
      }
    }
  }
  const int in_page = place & ((1 << a.step.page_shift) - 1), groups = lanes >> 1, rows = 2 * a.kv_heads;
  struct Row {
    uint4 raw;          // as stored
    uint32_t exponent;  // of a token in 4 bits
    float scale;        // of a token in 8; the group's bits in 4
  };
  for (int r0 = slot; r0 < rows; r0 += slots * kReadAhead) {
    Row row[kReadAhead];
#pragma unroll
    for (int j = 0; j < kReadAhead; ++j) {
      const int r = r0 + j * slots;
      row[j].raw = make_uint4(0, 0, 0, 0);
      row[j].exponent = 0;
      row[j].scale = 0.f;
      if (r >= rows || page < 0) continue;
      const bool is_key = r < a.kv_heads;
      const int64_t of_head = page * a.kv_heads + (is_key ? r : r - a.kv_heads), at = (of_head << a.step.page_shift) + in_page;
      const void* pool = is_key ? a.keys : a.values;
      const float* scales = is_key ? a.key_scales : a.value_scales;
      if (BITS == 16) {
        row[j].raw = __ldg(reinterpret_cast<const uint4*>(pool) + at * lanes + lane);
      } else if (BITS == 8) {
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(pool) + at * lanes + lane);
        row[j].raw.x = w.x;
        row[j].raw.y = w.y;
        row[j].scale = __ldg(scales + at);
      } else {
        row[j].raw.x = __ldg(reinterpret_cast<const uint32_t*>(pool) + at * lanes + lane);
        const uint8_t* of = reinterpret_cast<const uint8_t*>(scales) + ((of_head * (1 + groups)) << a.step.page_shift);
        row[j].exponent = __ldg(of + in_page);
        row[j].raw.y = __ldg(of + (1 << a.step.page_shift) + in_page * groups + (lane >> 1));
      }
    }
#pragma unroll
    for (int j = 0; j < kReadAhead; ++j) {
      const int r = r0 + j * slots;
      if (r >= rows) break;
      const bool is_key = r < a.kv_heads;
      const int h = is_key ? r : r - a.kv_heads;
      T* out = (is_key ? static_cast<T*>(a.k) + token * a.kn + h * a.kh : static_cast<T*>(a.v) + token * a.vn + h * a.vh) + lane * 8;
      uint4 raw = row[j].raw;
      if (BITS < 16) {
        float x[8];
        if (BITS == 8) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = float(int8_t((i < 4 ? raw.x : raw.y) >> (8 * (i & 3)))) * row[j].scale;
        } else {
          const float scale = power_of(row[j].exponent) * kGroupUnit;
          uint32_t pairs[4];
          scaled_codes(raw.x, GroupScale<__half>(twice(raw.y)), pairs);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = Half2<__half>::unpack(pairs[i]);
            x[2 * i] = f.x * scale;
            x[2 * i + 1] = f.y * scale;
          }
          if (page < 0)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 0.f;
        }
        store8(reinterpret_cast<T*>(&raw), x);
      }
      *reinterpret_cast<uint4*>(out) = raw;
    }
  }
}

// ---- eviction: which tokens stay ---------------------------------------------------------------------------
// Weights as whole numbers of the same order: NaN above everything, -0 equal to 0.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t bits = __float_as_uint(w + 0.0f);
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

struct SelectArgs {
  StepView step;
  const float* weights;
  int32_t* kept;
  float* new_weights;
  int kv_heads, budget, recent, target_slots;
};

constexpr int kSelectThreads = 1024;

// One CTA per (sequence, key head).  Warp w owns the tokens of one run, in rounds of 32; the first kHeld rounds' weights stay in
// registers between the passes over them, what is longer is read again.  The count-th largest of the unprotected weights is
// found digit by digit (11 + 11 + 10 bits) from histograms in shared memory; counters are whole numbers, so no order of the
// atomics shows in the result.  Then each warp goes over its run twice: counting what it keeps, and (after a scan over the
// warps) writing it, so that kept tokens stay in order and ties go to the lowest index.  128 CTAs of up to 16K tokens: 21 us
// (28 with the weights in shared memory instead), 8 of 4K: 13, most of it block-wide meetings.
constexpr int kHeld = 16;
__global__ __launch_bounds__(kSelectThreads) void select_kept_kernel(const SelectArgs a) {
  __shared__ unsigned int histogram[2048];
  __shared__ unsigned int warp_totals[2][32];
  __shared__ unsigned int found_digit, found_above;
  chain_wait();
  chain_release();
  const int head = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slots = a.step.width << a.step.page_shift;
  const int length = min(max(__ldg(a.step.lengths + s), 0), slots);
  const int64_t row = int64_t(s) * a.kv_heads + head;
  const float* weights = a.weights + row * slots;
  int32_t* kept = a.kept + row * a.budget;
  float* new_weights = a.new_weights + row * a.target_slots;
  const int count = min(length, a.budget), recent = min(a.recent, count);
  const int open = length - recent;         // tokens that compete
  const unsigned int wanted = count - recent;  // of which so many stay
  const int rounds = ((length + 31) / 32 + 31) / 32, begin = warp * rounds * 32;
  float held[kHeld];
#pragma unroll
  for (int n = 0; n < kHeld; ++n) {
    const int i = begin + n * 32 + lane;
    held[n] = n < rounds && i < length ? weights[i] : 0.f;
  }
  // f(token, weight) for every round of this warp, whole warps at a time
  auto each = [&](auto&& f) {
#pragma unroll
    for (int n = 0; n < kHeld; ++n)
      if (n < rounds) f(begin + n * 32 + lane, held[n]);
    for (int n = kHeld; n < rounds; ++n) {
      const int i = begin + n * 32 + lane;
      f(i, i < length ? weights[i] : 0.f);
    }
  };
  uint32_t threshold = 0;                    // larger ones stay,
  unsigned int equal_wanted = 0;             // and so many of those equal to it
  const bool all = int(wanted) >= open, none = wanted == 0;
  if (!all && !none) {
    unsigned int above = 0;  // tokens known to be larger than every one with the prefix
    uint32_t prefix = 0;
    int shift = 21;
#pragma unroll 1
    for (int digit = 0; digit < 3; ++digit) {
      const int bits = digit == 2 ? 10 : 11, bins = 1 << bits;
      for (int i = tid; i < bins; i += kSelectThreads) histogram[i] = 0;
      __syncthreads();
      each([&](int i, float w) {
        const uint32_t o = order_of(w);
        if (i < open && (digit == 0 || (o >> (shift + bits)) == prefix)) atomicAdd(&histogram[(o >> shift) & (bins - 1)], 1u);
      });
      __syncthreads();
      // suffix sums over the bins: the bin that holds the wanted-th largest.  A thread takes two bins, from the top down.
      const int top = bins - 1 - 2 * tid;
      const unsigned int h0 = top >= 0 ? histogram[top] : 0, h1 = top >= 1 ? histogram[top - 1] : 0;
      unsigned int sum = h0 + h1;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const unsigned int below = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += below;
      }
      if (lane == 31) warp_totals[0][warp] = sum;
      __syncthreads();
      const unsigned int before = above + __reduce_add_sync(0xffffffffu, lane < warp ? warp_totals[0][lane] : 0u);
      const unsigned int through = before + sum, until = through - h0 - h1;  // tokens above these two bins
      if (until < wanted && through >= wanted) {
        const bool first = until + h0 >= wanted;
        found_digit = first ? top : top - 1;
        found_above = first ? until : until + h0;
      }
      __syncthreads();
      prefix = (prefix << bits) | found_digit;
      above = found_above;
      shift -= digit == 1 ? 10 : 11;
      __syncthreads();
    }
    threshold = prefix;
    equal_wanted = wanted - above;
  }
  // stays for certain / ties with the threshold
  auto larger = [&](int i, float w) { return i < length && (i >= open || all || (!none && order_of(w) > threshold)); };
  auto equal = [&](int i, float w) { return i < open && !all && !none && order_of(w) == threshold; };
  unsigned int larger_count = 0, equal_count = 0;
  each([&](int i, float w) {
    larger_count += __popc(__ballot_sync(0xffffffffu, larger(i, w)));
    equal_count += __popc(__ballot_sync(0xffffffffu, equal(i, w)));
  });
  if (lane == 0) {
    warp_totals[0][warp] = larger_count;
    warp_totals[1][warp] = equal_count;
  }
  __syncthreads();
  unsigned int equal_before = __reduce_add_sync(0xffffffffu, lane < warp ? warp_totals[1][lane] : 0u);
  unsigned int at = __reduce_add_sync(0xffffffffu, lane < warp ? warp_totals[0][lane] : 0u) + min(equal_before, equal_wanted);
  each([&](int i, float w) {
    const bool ties = equal(i, w);
    const unsigned int tied = __ballot_sync(0xffffffffu, ties), below = (1u << lane) - 1;
    const bool stays = larger(i, w) || (ties && equal_before + __popc(tied & below) < equal_wanted);
    const unsigned int mask = __ballot_sync(0xffffffffu, stays);
    if (stays) {
      const unsigned int to = at + __popc(mask & below);
      kept[to] = i;
      new_weights[to] = w;
    }
    at += __popc(mask);
    equal_before += __popc(tied);
  });
  for (int i = count + tid; i < a.budget; i += kSelectThreads) kept[i] = -1;
  for (int i = count + tid; i < a.target_slots; i += kSelectThreads) new_weights[i] = 0.f;
}

// ---- eviction: their keys and values move --------------------------------------------------------------------
struct MoveArgs {
  StepView step;
  const int32_t* target;
  const int32_t* kept;
  int32_t* new_lengths;
  char* keys;
  char* values;
  float* key_scales;
  float* value_scales;
  int pages, kv_heads, budget, target_width, row_shift;  // a row is 16 << row_shift bytes
  int groups;                                            // 4-bit codes: of a row
  unsigned int* status;
};

constexpr int kMoveRows = 4;  // rows in flight per thread and pool

// Threads of 16 bytes; a row's threads are neighbours.  Four rows are looked up and loaded at a time,
// keys and values both, so that each thread has eight loads in flight (16 requests cut to 4K tokens of 8 heads of 128 bf16
// channels: 537 MB in 84 us, 6.4 TB/s, the rate of a plain copy).
__global__ __launch_bounds__(256) void move_kept_kernel(const MoveArgs a) {
  chain_wait();
  chain_release();
  const int s = blockIdx.z, head = blockIdx.y;
  const int slots = a.step.width << a.step.page_shift;
  // (the new length may lie over the old one: whichever a CTA reads, the count is the same)
  const int count = min(min(max(a.step.lengths[s], 0), slots), a.budget);
  if (blockIdx.x == 0 && head == 0 && threadIdx.x == 0) a.new_lengths[s] = count;
  const int per_pass = 256 >> a.row_shift, piece = threadIdx.x & ((1 << a.row_shift) - 1);
  const int j0 = blockIdx.x * per_pass * kMoveRows + (threadIdx.x >> a.row_shift);
  const int32_t* kept = a.kept + (int64_t(s) * a.kv_heads + head) * a.budget;
  const int in_page = (1 << a.step.page_shift) - 1;
  int64_t from[kMoveRows], to[kMoveRows];
  uint4 key[kMoveRows], value[kMoveRows];
  int32_t source[kMoveRows];
#pragma unroll
  for (int i = 0; i < kMoveRows; ++i) {
    const int j = j0 + i * per_pass;
    source[i] = j < count ? __ldg(kept + j) : -1;
  }
#pragma unroll
  for (int i = 0; i < kMoveRows; ++i) {
    from[i] = -1;
    const int j = j0 + i * per_pass;
    if (source[i] >= 0) {
      const int64_t p = __ldg(a.step.table + int64_t(s) * a.step.width + (source[i] >> a.step.page_shift));
      const int64_t t = __ldg(a.target + int64_t(s) * a.target_width + (j >> a.step.page_shift));
      if (p >= 0 && p < a.pages && t >= 0 && t < a.pages) {
        from[i] = ((p * a.kv_heads + head) << a.step.page_shift) + (source[i] & in_page);
        to[i] = ((t * a.kv_heads + head) << a.step.page_shift) + (j & in_page);
      } else {
        atomicCAS(a.status, 0u, unsigned(s) + 1u);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kMoveRows; ++i) {
    if (from[i] >= 0) {
      const int64_t byte = (from[i] << (a.row_shift + 4)) + piece * 16;
      key[i] = *reinterpret_cast<const uint4*>(a.keys + byte);
      value[i] = *reinterpret_cast<const uint4*>(a.values + byte);
    }
  }
#pragma unroll
  for (int i = 0; i < kMoveRows; ++i) {
    if (from[i] >= 0) {
      const int64_t byte = (to[i] << (a.row_shift + 4)) + piece * 16;
      *reinterpret_cast<uint4*>(a.keys + byte) = key[i];
      *reinterpret_cast<uint4*>(a.values + byte) = value[i];
      if (a.groups > 0 && piece < 2) {  // the first two threads of a row take the scales of a pool each
        auto scales = [&](int64_t row) {
          return reinterpret_cast<uint8_t*>(piece == 0 ? a.key_scales : a.value_scales) + (((row >> a.step.page_shift) * (1 + a.groups)) << a.step.page_shift);
        };
        uint8_t *f = scales(from[i]), *t = scales(to[i]);
        const int fs = int(from[i]) & in_page, ts = int(to[i]) & in_page;
        t[ts] = f[fs];
        f += (1 << a.step.page_shift) + fs * a.groups;
        t += (1 << a.step.page_shift) + ts * a.groups;
        for (int g = 0; g < a.groups; g += 4) *reinterpret_cast<uint32_t*>(t + g) = *reinterpret_cast<const uint32_t*>(f + g);
      } else if (a.key_scales != nullptr && a.groups == 0 && piece == 0) {
        a.key_scales[to[i]] = a.key_scales[from[i]];
        a.value_scales[to[i]] = a.value_scales[from[i]];
      }
    }
  }
}

template <typename T>
auto append4_for(int head_dim) { return head_dim == 64 ? append4_kernel<T, 8> : head_dim == 128 ? append4_kernel<T, 16> : append4_kernel<T, 32>; }

int check_rotary(const risa_b200_rotary* r, int head_dim, const char* what) {
  RISA_REQUIRE(r->turns != nullptr, "%s: null rotary table", what);
  RISA_REQUIRE(r->rotary_dim > 0 && r->rotary_dim % 2 == 0 && r->rotary_dim <= head_dim,
               "%s: rotary_dim must be even and at most head_dim", what);
  return RISA_B200_OK;
}
int check_axes(const risa_b200_rotary_axes* a, const char* what) {
  RISA_REQUIRE(a == nullptr || (a->axes != nullptr && a->count >= 1 && a->count <= RISA_B200_MOST_AXES),
               "%s: a rotary table follows 1 to 8 axes", what);
  return RISA_B200_OK;
}

}  // namespace
}  // namespace serving
}  // namespace risa_b200

using namespace risa_b200;
using namespace risa_b200::serving;

extern "C" int risa_b200_rotate(const void* x, void* out, int dtype_code, int batch, int heads,
                                int tokens, int head_dim, const int64_t xs[3], const int64_t os[3],
                                const void* positions, int positions_64, int64_t position_stride_b,
                                int64_t position_stride_n, const risa_b200_rotary* rotary,
                                int transposed, void* stream) {
  return risa_b200_rotate_axes(x, out, dtype_code, batch, heads, tokens, head_dim, xs, os, positions, positions_64, position_stride_b,
                               position_stride_n, rotary, nullptr, transposed, stream);
}

extern "C" int risa_b200_rotate_axes(const void* x, void* out, int dtype_code, int batch, int heads,
                                     int tokens, int head_dim, const int64_t xs[3], const int64_t os[3],
                                     const void* positions, int positions_64, int64_t position_stride_b,
                                     int64_t position_stride_n, const risa_b200_rotary* rotary,
                                     const risa_b200_rotary_axes* axes, int transposed, void* stream_ptr) {
  RISA_REQUIRE(x && out && positions && rotary, "rotate: null tensor");
  RISA_REQUIRE(dtype_code >= 0 && dtype_code <= 2, "rotate: dtype must be float32, float16 or bfloat16");
  RISA_REQUIRE(batch > 0 && batch <= 65535 && heads > 0 && heads <= 65535 && tokens > 0 && head_dim > 0,
               "rotate: sizes must be positive, batch and heads at most 65535");
  if (const int bad = check_rotary(rotary, head_dim, "rotate")) return bad;
  if (const int bad = check_axes(axes, "rotate")) return bad;
  RotateArgs a{x, out, positions, rotary->turns, xs[0], xs[1], xs[2], os[0], os[1], os[2],
               position_stride_b, position_stride_n, batch, heads, tokens, head_dim,
               rotary->rotary_dim, 1, 1, positions_64, rotary->interleaved, transposed,
               rotary->magnitude, axes ? axes->axes : nullptr, axes ? axes->position_stride : 0, axes ? axes->count - 1 : 0};
  // eight channels at a time where every run starts on a 16-byte boundary
  const int64_t size = dtype_code == 0 ? 4 : 2;
  bool wide = rotary->rotary_dim % 16 == 0 && head_dim % 8 == 0 &&
              (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) % 16 == 0;
  for (int i = 0; i < 3; ++i) wide = wide && xs[i] * size % 16 == 0 && os[i] * size % 16 == 0;
  wide = wide && reinterpret_cast<uintptr_t>(a.axes) % 8 == 0;
  const int items = wide ? rotary->rotary_dim / 16 + (head_dim - rotary->rotary_dim) / 8
                         : rotary->rotary_dim / 2 + head_dim - rotary->rotary_dim;
  const int64_t threads = int64_t(tokens) * items;
  RISA_REQUIRE((threads + 255) / 256 < (int64_t(1) << 31), "rotate: too many tokens");
  // up to eight heads share a thread's cosines while the launch still fills the SMs
  while (a.heads_each < 8 && a.heads_each < heads && threads * batch * heads / (2 * a.heads_each) >= 148 * 1024)
    a.heads_each *= 2;
  const dim3 grid(unsigned((threads + 255) / 256), unsigned((heads + a.heads_each - 1) / a.heads_each), unsigned(batch));
  RISA_DISPATCH_FLOAT(dtype_code, T, return launched(launch_chained(!wide ? rotate_any_kernel<T> : a.axes ? rotate_kernel<T, true> : rotate_kernel<T, false>, grid, dim3(256), 0,
                                                                    static_cast<cudaStream_t>(stream_ptr), a), "rotate"));
}

extern "C" int risa_b200_cache_append(const risa_b200_cache* cache, const risa_b200_step* step,
                                      const void* k, const int64_t ks[2], const void* v,
                                      const int64_t vs[2], const void* q, const int64_t qs[2],
                                      void* q_out, const int64_t os[2], int q_heads, int dtype_code,
                                      const risa_b200_rotary* rotary, const void* positions,
                                      int positions_64, void* stream) {
  return risa_b200_cache_append_axes(cache, step, k, ks, v, vs, q, qs, q_out, os, q_heads, dtype_code, rotary, nullptr, positions,
                                     positions_64, stream);
}

extern "C" int risa_b200_cache_append_axes(const risa_b200_cache* cache, const risa_b200_step* step,
                                           const void* k, const int64_t ks[2], const void* v,
                                           const int64_t vs[2], const void* q, const int64_t qs[2],
                                           void* q_out, const int64_t os[2], int q_heads, int dtype_code,
                                           const risa_b200_rotary* rotary, const risa_b200_rotary_axes* axes,
                                           const void* positions, int positions_64, void* stream_ptr) {
  if (const int bad = check_cache(cache, "append")) return bad;
  if (const int bad = check_step(step, cache, "append")) return bad;
  const int bits = bits_of(*cache);
  RISA_REQUIRE(k && v && (q == nullptr) == (q_out == nullptr), "append: null tensor");
  RISA_REQUIRE(dtype_code == 1 || dtype_code == 2, "append: q, k and v must be float16 or bfloat16");
  RISA_REQUIRE(bits < 16 || dtype_code == cache->dtype_code, "append: k and v must have the cache's type");
  RISA_REQUIRE(q == nullptr || rotary != nullptr, "append: q is only rotated, and there is no rotary table");
  RISA_REQUIRE(q == nullptr || q_heads > 0, "append: q needs heads");
  if (rotary != nullptr) {
    if (const int bad = check_rotary(rotary, cache->head_dim, "append")) return bad;
    RISA_REQUIRE(rotary->rotary_dim % 16 == 0, "append: rotary_dim must be a multiple of 16");
    if (const int bad = check_axes(axes, "append")) return bad;
  }
  const void* const pointers[] = {k, v, q, q_out};
  const int64_t* const strides[] = {ks, vs, qs, os};
  for (int i = 0; i < 4; ++i) {
    if (pointers[i] == nullptr) continue;
    RISA_REQUIRE(reinterpret_cast<uintptr_t>(pointers[i]) % 16 == 0 && strides[i][0] % 8 == 0 && strides[i][1] % 8 == 0,
                 "append: rows must start on 16-byte boundaries");
  }
  unsigned int* status = status_word();
  if (status == nullptr) return RISA_B200_CUDA;
  AppendArgs a{};
  a.step = view_of(*step, cache->page_size);
  a.keys = cache->keys;
  a.values = cache->values;
  a.key_scales = cache->key_scales;
  a.value_scales = cache->value_scales;
  a.k = k;
  a.v = v;
  a.q = q;
  a.q_out = q_out;
  a.kn = ks[0];
  a.kh = ks[1];
  a.vn = vs[0];
  a.vh = vs[1];
  if (q != nullptr) {
    a.qn = qs[0];
    a.qh = qs[1];
    a.on = os[0];
    a.oh = os[1];
  }
  a.pages = cache->pages;
  a.kv_heads = cache->kv_heads;
  a.q_heads = q == nullptr ? 0 : q_heads;
  a.head_dim = cache->head_dim;
  if (rotary != nullptr) {
    a.turns = rotary->turns;
    a.rotary_dim = rotary->rotary_dim;
    a.interleaved = rotary->interleaved;
    a.magnitude = rotary->magnitude;
    a.positions = positions;
    a.positions_64 = positions_64;
    if (axes != nullptr) {
      a.axes = axes->axes;
      a.axis_stride = axes->position_stride;
      a.last_axis = axes->count - 1;
    }
  }
  a.status = status;
  const auto kernel = dtype_code == 1 ? (bits == 4 ? append4_for<__half>(a.head_dim) : bits == 8 ? append_kernel<__half, 8> : append_kernel<__half, 16>)
                                      : (bits == 4 ? append4_for<__nv_bfloat16>(a.head_dim) : bits == 8 ? append_kernel<__nv_bfloat16, 8> : append_kernel<__nv_bfloat16, 16>);
  return launched(launch_chained(kernel, dim3(step->tokens), dim3(128), 0, static_cast<cudaStream_t>(stream_ptr), a), "append");
}

extern "C" int risa_b200_cache_read(const risa_b200_cache* cache, const risa_b200_step* step, void* k, const int64_t ks[2], void* v,
                                    const int64_t vs[2], int dtype_code, void* stream_ptr) {
  if (const int bad = check_cache(cache, "read")) return bad;
  if (const int bad = check_step(step, cache, "read")) return bad;
  const int bits = bits_of(*cache);
  RISA_REQUIRE(k && v, "read: null tensor");
  RISA_REQUIRE(dtype_code == 1 || dtype_code == 2, "read: keys and values are read as float16 or bfloat16");
  RISA_REQUIRE(bits < 16 || dtype_code == cache->dtype_code, "read: keys and values must have the cache's type");
  RISA_REQUIRE((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0 && (ks[0] | ks[1] | vs[0] | vs[1]) % 8 == 0,
               "read: rows must start on 16-byte boundaries");
  unsigned int* status = status_word();
  if (status == nullptr) return RISA_B200_CUDA;
  const ReadArgs a{view_of(*step, cache->page_size), cache->keys, cache->values, cache->key_scales, cache->value_scales, k, v,
                   ks[0], ks[1], vs[0], vs[1], cache->pages, cache->kv_heads, cache->head_dim, status};
  const auto kernel = dtype_code == 1 ? (bits == 4 ? read_kernel<__half, 4> : bits == 8 ? read_kernel<__half, 8> : read_kernel<__half, 16>)
                                      : (bits == 4 ? read_kernel<__nv_bfloat16, 4> : bits == 8 ? read_kernel<__nv_bfloat16, 8> : read_kernel<__nv_bfloat16, 16>);
  return launched(launch_chained(kernel, dim3((step->tokens + kReadWarps - 1) / kReadWarps), dim3(kReadWarps * 32), 0, static_cast<cudaStream_t>(stream_ptr), a), "read");
}

extern "C" int risa_b200_cache_evict(const risa_b200_cache* cache, const risa_b200_step* step,
                                     const float* weights, const int32_t* target_table,
                                     int target_width, int budget, int recent, int32_t* kept,
                                     int32_t* new_lengths, float* new_weights, void* stream_ptr) {
  if (const int bad = check_cache(cache, "evict")) return bad;
  RISA_REQUIRE(step && step->page_table && step->lengths && step->batch > 0 && step->batch <= 65535 && step->table_width > 0,
               "evict: null step, or batch not in 1..65535");
  RISA_REQUIRE(int64_t(step->table_width) * cache->page_size < RISA_B200_CACHE_MOST_SLOTS,
               "evict: a sequence may hold fewer than 2^31 - 8192 keys");
  RISA_REQUIRE(weights && target_table && kept && new_lengths && new_weights, "evict: null tensor");
  RISA_REQUIRE(cache->kv_heads <= 65535, "evict: too many heads");
  RISA_REQUIRE(budget > 0 && recent >= 0 && recent <= budget, "evict: budget must be positive and recent in 0..budget");
  RISA_REQUIRE(int64_t(target_width) * cache->page_size >= budget, "evict: the target pages do not hold the budget");
  RISA_REQUIRE(int64_t(target_width) * cache->page_size < RISA_B200_CACHE_MOST_SLOTS, "evict: the target table is too wide");
  RISA_REQUIRE(target_table != step->page_table, "evict: the target pages must not be the sequences' own");
  unsigned int* status = status_word();
  if (status == nullptr) return RISA_B200_CUDA;
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  const StepView view = view_of(*step, cache->page_size);
  const SelectArgs select{view, weights, kept, new_weights, cache->kv_heads, budget, recent,
                          target_width * cache->page_size};
  if (const int bad = launched(launch_chained(select_kept_kernel, dim3(cache->kv_heads, step->batch), dim3(kSelectThreads), 0, stream, select), "evict"))
    return bad;
  const int row_bytes = cache->head_dim * bits_of(*cache) / 8;
  int shift = 0;
  while ((16 << shift) < row_bytes) ++shift;
  const MoveArgs move{view, target_table, kept, new_lengths, static_cast<char*>(cache->keys), static_cast<char*>(cache->values),
                      cache->key_scales, cache->value_scales, cache->pages, cache->kv_heads, budget, target_width,
                      shift, cache->dtype_code == kInt4 ? cache->head_dim / 16 : 0, status};
  const int rows = (256 >> shift) * kMoveRows;
  return launched(launch_chained(move_kept_kernel, dim3((budget + rows - 1) / rows, cache->kv_heads, step->batch), dim3(256), 0, stream, move), "evict");
}
