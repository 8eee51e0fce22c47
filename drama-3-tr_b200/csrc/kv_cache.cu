// Rotary positions and the paged key-value cache (sm_100a): rope, kv_write, kv_read.
//
// Rotary positions turn each pair (a, b) of a head's first `rot` values by t = position * inv_freq:
//   a' = a cos t - b sin t,  b' = b cos t + a sin t        (times a factor)
// with pairs (2i, 2i + 1) in the interleaved layout and (i, i + rot / 2) in the half layout. t grows to
// 10^6 radians, where 32 bits keep no digit behind the comma, so t / pi is formed and reduced to
// [-1, 1] in 64 bits; the sine and cosine of the reduced angle are then taken in 32 bits. They are
// computed once a token and kept in shared memory for all of its heads.
//
// A cache is [pages][kv_heads][page_size][dim] (one page of one head is contiguous, so the attention
// kernel streams it), in bf16 or in e4m3 with one exponent a row (token, head): the row stands for
// code * 2^e with e the smallest integer that keeps amax <= 448 * 2^e. A power of two costs no
// precision against a free scale (e4m3 is a floating format), takes 1 byte a row, makes the
// cached values exact bf16 numbers, and joins the softmax's exponent in the attention kernel.
//
// All three kernels only move data: their bound is HBM bandwidth, or the launch when there are few tokens.
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>

#include "dm3.h"
#include "dm3_common.cuh"
#include "dm3_internal.h"
#include "dm3_kv.cuh"

namespace dm3 {
namespace kv {

constexpr int kThreads = 256;
constexpr int kMaxRot = 1024;
constexpr int kBlockTokens = 8;   // most tokens of one CTA
constexpr int kAngles = 1024;     // most (token, pair) angles of one CTA: 8 tokens of a 256-value head, or 2 of 1024

struct Heads {  // [tokens][heads][dim] bf16, unit stride in dim
  const __nv_bfloat16* p;
  int64_t ts, hs;  // strides in elements
  int n;           // heads
};

struct RopeParams {
  Heads x;
  __nv_bfloat16* y;  // [T][heads][dim]
  int T, dim, block;  // block: tokens of a CTA
  const int64_t* positions;
  const double* inv_freq;
  int rot, interleaved;
  double factor;
};

// Division by a fixed n < 2^16 of values below 2^16: (x * ceil(2^32 / n)) >> 32 is exact there.
struct Div {
  uint32_t n, m;
  explicit Div(int d) : n(d), m(d > 1 ? static_cast<uint32_t>(((uint64_t(1) << 32) + d - 1) / d) : 0) {}
  Div() : n(1), m(0) {}
  __device__ __forceinline__ int operator()(int x) const { return n > 1 ? static_cast<int>(__umulhi(static_cast<uint32_t>(x), m)) : x; }
};

struct Chunk {
  float v[8];
};
__device__ __forceinline__ Chunk unpack(uint4 r) {
  Chunk c;
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c.v[2 * i] = __uint_as_float(w[i] << 16);
    c.v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  return c;
}
__device__ __forceinline__ uint4 pack(const Chunk& c) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(c.v[2 * i], c.v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// (cos, sin) of position * inv_freq, times factor: reduced in 64 bits, then 32 (kLow false) or 64 bits as a
// pair of floats each, high and low part.
template <bool kLow>
__device__ __forceinline__ void angle(int64_t pos, double inv_freq, double factor, float2& high, float2& low) {
  double t = static_cast<double>(pos) * inv_freq * 0.31830988618379067154;  // 1 / pi
  t -= 2.0 * rint(t * 0.5);
  if (kLow) {
    double c, s;
    sincospi(t, &s, &c);
    c *= factor, s *= factor;
    high = make_float2(static_cast<float>(c), static_cast<float>(s));
    low = make_float2(static_cast<float>(c - high.x), static_cast<float>(s - high.y));
  } else {
    float c, s;
    sincospif(static_cast<float>(t), &s, &c);
    high = make_float2(c * static_cast<float>(factor), s * static_cast<float>(factor));
  }
}

// A thread works on 16 values of a row: pairs 8 * i .. 8 * i + 7. In the half layout they lie in the 8-value chunks i
// and i + rot / 16, in the interleaved one in 2i and 2i + 1, as do the values past rot in both.
struct Where {
  int a, b;
  bool turned;
};
template <bool kInter>
__device__ __forceinline__ Where where(int i, int rot) {
  const bool turned = i * 16 < rot;
  return turned && !kInter ? Where{i, i + rot / 16, true} : Where{2 * i, 2 * i + 1, turned};
}

// The angles of a CTA's tokens: cosines and sines of pairs 8i + 2k, 8i + 2k + 1 of token t as (c, c, s, s) at [t][k][i],
// so neighbouring threads read neighbouring 16 bytes.
template <bool kLow>
__device__ __forceinline__ void fill_angles(float2* high, float2* low, int tokens, const int64_t* positions,
                                            const double* inv_freq, int rot, double factor) {
  const int half = rot / 2, units = rot / 16;
  for (int x = threadIdx.x; x < tokens * half; x += blockDim.x) {
    const int t = x / half, f = x - t * half, at = t * rot + (((f & 7) >> 1) * units + (f >> 3)) * 4 + (f & 1);
    float2 h, l;
    angle<kLow>(positions[t], inv_freq[f], factor, h, l);
    reinterpret_cast<float*>(high)[at] = h.x, reinterpret_cast<float*>(high)[at + 2] = h.y;
    if (kLow) reinterpret_cast<float*>(low)[at] = l.x, reinterpret_cast<float*>(low)[at + 2] = l.y;
  }
}

// Two 32-bit values an instruction, each rounded as its scalar form.
struct Two {
  uint64_t v;
};
__device__ __forceinline__ Two two(float a, float b) {
  return {static_cast<uint64_t>(__float_as_uint(a)) | static_cast<uint64_t>(__float_as_uint(b)) << 32};
}
__device__ __forceinline__ float first(Two a) { return __uint_as_float(static_cast<uint32_t>(a.v)); }
__device__ __forceinline__ float second(Two a) { return __uint_as_float(static_cast<uint32_t>(a.v >> 32)); }
__device__ __forceinline__ Two operator-(Two a) { return two(-first(a), -second(a)); }
__device__ __forceinline__ Two mul(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two add(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Two sub(Two a, Two b) { return fma(b, two(-1.f, -1.f), a); }

// a c + b s to about 2^-46 of |a| + |b|: products and the sum with their rounding errors carried along. nc, ns: -c, -s;
// cl, sl: the low parts of c and s.
__device__ __forceinline__ Two exact_turn(Two a, Two b, Two c, Two nc, Two cl, Two s, Two ns, Two sl) {
  const Two p = mul(a, c), q = mul(b, s);
  const Two error = add(fma(a, nc, p), fma(b, ns, q));  // of both products, negated
  const Two d = add(p, q), z = sub(d, p);
  const Two de = add(sub(p, sub(d, z)), sub(q, z));
  return add(d, add(sub(de, error), fma(a, cl, mul(b, sl))));
}

// Turns the 16 values of unit i in place. high, low: the token's angles. The exact turn takes two values an instruction;
// the plain one, a few instructions, is slower so (rope of 2,643 tokens with 22 heads: 10.7 against 9.8 us).
template <bool kExact, bool kInter>
__device__ __forceinline__ void turn(Chunk& x, Chunk& y, int i, const float2* high, const float2* low, int rot) {
  const int units = rot / 16;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float4 h = *reinterpret_cast<const float4*>(high + (k * units + i) * 2);
    Chunk& z = k < 2 ? x : y;
    const int j = kInter ? 4 * (k % 2) : 2 * k;
    float &a0 = kInter ? z.v[j] : x.v[j], &b0 = kInter ? z.v[j + 1] : y.v[j];
    float &a1 = kInter ? z.v[j + 2] : x.v[j + 1], &b1 = kInter ? z.v[j + 3] : y.v[j + 1];
    if (kExact) {
      const float4 l = *reinterpret_cast<const float4*>(low + (k * units + i) * 2);
      const Two a = two(a0, a1), b = two(b0, b1), c = two(h.x, h.y), s = two(h.z, h.w), cl = two(l.x, l.y), sl = two(l.z, l.w);
      const Two ra = exact_turn(a, b, c, -c, cl, -s, s, -sl), rb = exact_turn(b, a, c, -c, cl, s, -s, sl);
      a0 = first(ra), a1 = second(ra), b0 = first(rb), b1 = second(rb);
    } else {
      auto plain = [](float& a, float& b, float c, float s) {
        const float a0 = a;
        a = a0 * c - b * s;
        b = b * c + a0 * s;
      };
      plain(a0, b0, h.x, h.z);
      plain(a1, b1, h.y, h.w);
    }
  }
}

// ------------------------------------------------------------------ rope
// A CTA takes a block of tokens (and a share of their rows, blockIdx.y, when there are few tokens), a thread 16
// values of a row at a time, the next row's loads in flight: 16,384 tokens x 20 heads of 128 take 29.1 us at five CTAs an
// SM (5.8 TB/s), against 31.7 with four that hold two rows at a time.
// A row belongs to 2^shift neighbouring lanes (dim / 16 of them at work), so a thread keeps its place in the row.
template <bool kInter>
__global__ void __launch_bounds__(kThreads, 5) rope_kernel(const __grid_constant__ RopeParams p, const int shift, const Div heads) {
  __shared__ __align__(16) float2 cs[kAngles];
  griddep_launch();
  griddep_wait();
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.block;
  const int tokens = p.T - t0 < p.block ? static_cast<int>(p.T - t0) : p.block;
  const int i = threadIdx.x & ((1 << shift) - 1), segs = kThreads >> shift, total = tokens * p.x.n;
  const Where w = where<kInter>(i, p.rot);
  const bool mine = i < p.dim / 16;
  struct Row {
    uint4 a, b;
    int t, row;
  };
  auto load = [&](Row& x, int base) {
    x.row = base + (threadIdx.x >> shift);
    if (x.row < total && mine) {
      x.t = heads(x.row);
      const __nv_bfloat16* src = p.x.p + (t0 + x.t) * p.x.ts + (x.row - x.t * p.x.n) * p.x.hs;
      x.a = __ldcs(reinterpret_cast<const uint4*>(src + w.a * 8));
      x.b = __ldcs(reinterpret_cast<const uint4*>(src + w.b * 8));
    }
  };
  Row now;
  load(now, blockIdx.y * segs);  // on its way while the angles are found
  fill_angles<false>(cs, nullptr, tokens, p.positions + t0, p.inv_freq, p.rot, p.factor);
  __syncthreads();
  for (int base = blockIdx.y * segs; base < total;) {
    base += gridDim.y * segs;
    Row next;
    load(next, base);
    if (now.row < total && mine) {
      Chunk x = unpack(now.a), y = unpack(now.b);
      if (w.turned) turn<false, kInter>(x, y, i, cs + now.t * (p.rot / 2), nullptr, p.rot);
      __nv_bfloat16* dst = p.y + (t0 * p.x.n + now.row) * p.dim;
      *reinterpret_cast<uint4*>(dst + w.a * 8) = pack(x);
      *reinterpret_cast<uint4*>(dst + w.b * 8) = pack(y);
    }
    now = next;
  }
}

// Any dim, rot, stride and alignment: one token a CTA, one value a thread at a time.
__global__ void __launch_bounds__(kThreads) rope_any_kernel(const __grid_constant__ RopeParams p) {
  __shared__ float2 cs[kMaxRot / 2];
  griddep_launch();
  griddep_wait();
  const int t = blockIdx.x;
  const int64_t pos = p.positions[t];
  float2 none;
  for (int i = threadIdx.x; i < p.rot / 2; i += blockDim.x) angle<false>(pos, p.inv_freq[i], p.factor, cs[i], none);
  __syncthreads();
  const int n = p.x.n * p.dim, half = p.rot / 2;
  for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < n; i += gridDim.y * blockDim.x) {
    const int h = i / p.dim, d = i - h * p.dim;
    const __nv_bfloat16* row = p.x.p + t * p.x.ts + h * p.x.hs;
    float y = __bfloat162float(row[d]);
    if (d < p.rot) {
      const bool second = p.interleaved ? (d & 1) : d >= half;
      const int j = p.interleaved ? d >> 1 : (second ? d - half : d);
      const float z = __bfloat162float(row[p.interleaved ? d ^ 1 : (second ? j : d + half)]);
      y = y * cs[j].x + z * (second ? cs[j].y : -cs[j].y);
    }
    p.y[(static_cast<int64_t>(t) * p.x.n + h) * p.dim + d] = __float2bfloat16_rn(y);
  }
}

// ------------------------------------------------------------------ kv_write
struct WriteParams {
  Heads q, k, v;     // q.n = 0: none
  __nv_bfloat16* y;  // the turned queries, [T][q.n][dim]
  int T, dim, block;
  const int64_t* rows;  // table row of each token; null: token i is row i
  const int64_t* positions;
  Cache c;
  const double* inv_freq;
  int rot;  // 0: no rotary positions
  double factor;
};

// 8 values as e4m3 codes of 1 / scale.
__device__ __forceinline__ uint2 encode(const Chunk& x, float scale) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = pack_e4m3x2(x.v[4 * i] * scale, x.v[4 * i + 1] * scale) |
           static_cast<uint32_t>(pack_e4m3x2(x.v[4 * i + 2] * scale, x.v[4 * i + 3] * scale)) << 16;
  return make_uint2(w[0], w[1]);
}

// The largest magnitude's bits of 16 bf16 values (magnitudes order as their bits do).
__device__ __forceinline__ uint32_t max_magnitude(uint4 a, uint4 b) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  return max(m & 0xffffu, m >> 16);
}

// The exponent of a row whose largest finite magnitude is amax: the smallest e with amax <= 448 * 2^e
// (448 = 1.75 * 2^8), kept where 2^e times every code is a finite, normal bf16 number.
__device__ __forceinline__ int row_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  if (b == 0) return 0;
  const int e = static_cast<int>(b >> 23) - ((b & 0x7fffffu) <= 0x600000u ? 135 : 134);
  return min(max(e, -110), 119);
}

// As rope_kernel, over the rows of q, then those of k, then those of v; each of the three starts with a warp, so a warp
// is at one of them at a time. A row belongs to kSeg neighbouring lanes, so the amax of a quantised row is a few
// shuffles. A quantised key is turned to 2^-46 by its angle, which is formed in 64 bits (2^-52 of its size): it is the code of
// the key turned by that, whichever call wrote it (in 32 bits about one value in 10^6 would fall on the other side of a
// code's border).
//
// Loads in flight: the next row's while a thread is at one, in four CTAs an SM; or (kMany) two rows' at a time in five.
// With a bf16 cache the second is faster for many tokens and slower for few (written and read back: 100,000 tokens with
// 32 + 4 + 4 heads of 64 213 against 235 us, 256 tokens with 16 + 2 + 2 of 256 3.7 against 3.1). An e4m3 cache is bound
// by its instructions and gains nothing (31,733 tokens with 32 + 8 + 8 of 128: 182 against 180).
// Alone, the first writes in 160 us (6.4 TB/s) and the last in 132 (5.4 TB/s).
template <int kSeg, bool kQuant, bool kInter, bool kMany>
__global__ void __launch_bounds__(kThreads, kMany ? 5 : 4) write_kernel(const __grid_constant__ WriteParams p, const Div by_q,
                                                                       const Div by_k) {
  __shared__ __align__(16) float2 high[kAngles], low[kQuant ? kAngles : 1];
  __shared__ int64_t s_at[kBlockTokens], s_exp[kBlockTokens];  // place of a token's row of head 0; -1: not cached
  __shared__ bool s_pad[kBlockTokens];
  griddep_launch();
  griddep_wait();
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.block;
  const int tokens = p.T - t0 < p.block ? static_cast<int>(p.T - t0) : p.block;
  constexpr int kSegs = kThreads / kSeg, kWarp = 32 / kSeg;
  const int i = threadIdx.x % kSeg;
  const int q_rows = (tokens * p.q.n + kWarp - 1) & -kWarp, k_rows = (tokens * p.k.n + kWarp - 1) & -kWarp;
  const int total = q_rows + 2 * k_rows;
  const Where w = where<kInter>(i, p.rot);
  const bool mine = i < p.dim / 16;
  struct Row {
    uint4 a, b;
    int side, t, head;  // side 0: query, 1: key, 2: value; head -1: no row
  };
  auto load = [&](Row& x, int base) {
    int r = base + threadIdx.x / kSeg;
    x.side = r < q_rows ? 0 : r < q_rows + k_rows ? 1 : 2;
    x.head = -1;
    x.a = x.b = make_uint4(0, 0, 0, 0);
    auto from = [&](const Heads& in, const Div& by) {
      x.t = by(r);
      if (x.t >= tokens || !mine) return;
      x.head = r - x.t * in.n;
      const __nv_bfloat16* row = in.p + t0 * in.ts + static_cast<uint32_t>(x.t) * in.ts + static_cast<uint32_t>(x.head) * in.hs;
      x.a = __ldcs(reinterpret_cast<const uint4*>(row + w.a * 8));
      x.b = __ldcs(reinterpret_cast<const uint4*>(row + w.b * 8));
    };
    if (x.side == 0) {
      from(p.q, by_q);
    } else if (x.side == 1) {
      r -= q_rows;
      from(p.k, by_k);
    } else {
      r -= q_rows + k_rows;
      from(p.v, by_k);
    }
  };
  constexpr int kBatch = kMany ? 2 : 1;
  Row now[kBatch];
#pragma unroll
  for (int b = 0; b < kBatch; ++b) load(now[b], (blockIdx.y * kBatch + b) * kSegs);  // while angles and places are found
  // a place is found by the last threads, while the first ones are at the angles
  bool padding = false;
  if (const int t = kThreads - 1 - threadIdx.x; t < tokens) {
    const int64_t pos = p.positions[t0 + t], r = p.rows ? p.rows[t0 + t] : t0 + t;
    padding = pos < 0 || r < 0;
    int64_t at = -1, x = 0;
    if (!padding) {
      const int64_t nth = pos / p.c.page_size, in = pos - nth * p.c.page_size;
      const int64_t page = r < p.c.rows && nth < p.c.per_row ? p.c.table[r * p.c.table_stride + nth] : -1;
      if (page >= 0 && page < p.c.pages)
        at = page * p.c.page_stride + in * p.dim, x = page * p.c.exp_stride + in;
      else
        set_status(p.c.status, STATUS_BAD_PAGE);
    }
    s_at[t] = at, s_exp[t] = x, s_pad[t] = padding;
  }
  if (p.rot) fill_angles<kQuant>(high, low, tokens, p.positions + t0, p.inv_freq, p.rot, p.factor);
  const bool padded = __syncthreads_or(padding);
  __nv_bfloat16* const queries = p.y + t0 * p.q.n * p.dim;
  // a row in the cache, once its values are final
  auto keep = [&](const Row& x, void* cache, int8_t* exps) {
    const int64_t place = x.head < 0 ? -1 : s_at[x.t];
    if (!kQuant) {
      if (place < 0) return;
      __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(cache) + place + static_cast<int64_t>(x.head * p.c.page_size) * p.dim;
      *reinterpret_cast<uint4*>(dst + w.a * 8) = x.a;
      *reinterpret_cast<uint4*>(dst + w.b * 8) = x.b;
      return;
    }
    uint32_t top = max_magnitude(x.a, x.b);
#pragma unroll
    for (int o = kSeg / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    Chunk a = unpack(x.a), b = unpack(x.b);  // a key as a bf16 cache would hold it
    if (__any_sync(0xffffffffu, top >= 0x7f80u)) {  // infinities and NaN: not counted, and NaN in the cache
      float amax = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        amax = fmaxf(amax, fmaxf(isfinite(a.v[j]) ? fabsf(a.v[j]) : 0.f, isfinite(b.v[j]) ? fabsf(b.v[j]) : 0.f));
        if (!isfinite(a.v[j])) a.v[j] = NAN;
        if (!isfinite(b.v[j])) b.v[j] = NAN;
      }
#pragma unroll
      for (int o = kSeg / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      top = __float_as_uint(amax) >> 16;
    }
    if (place < 0) return;
    const int e = row_exponent(__uint_as_float(top << 16)), row = x.head * p.c.page_size;
    uint8_t* dst = static_cast<uint8_t*>(cache) + place + static_cast<int64_t>(row) * p.dim;
    *reinterpret_cast<uint2*>(dst + w.a * 8) = encode(a, exp2i(-e));
    *reinterpret_cast<uint2*>(dst + w.b * 8) = encode(b, exp2i(-e));
    if (i == 0) exps[s_exp[x.t] + row] = static_cast<int8_t>(e);
  };
  auto finish = [&](Row& x) {
    if (x.side < 2 && w.turned && x.head >= 0) {
      Chunk a = unpack(x.a), b = unpack(x.b);
      const int at = x.t * (p.rot / 2);
      if (kQuant && x.side == 1)
        turn<kQuant, kInter>(a, b, i, high + at, low + at, p.rot);
      else
        turn<false, kInter>(a, b, i, high + at, nullptr, p.rot);
      x.a = pack(a), x.b = pack(b);
    }
    if (x.side == 0) {
      if (x.head < 0) return;
      if (padded && s_pad[x.t]) x.a = x.b = make_uint4(0, 0, 0, 0);
      __nv_bfloat16* dst = queries + (x.t * p.q.n + x.head) * p.dim;
      *reinterpret_cast<uint4*>(dst + w.a * 8) = x.a;
      *reinterpret_cast<uint4*>(dst + w.b * 8) = x.b;
    } else if (x.side == 1) {
      keep(x, p.c.k, p.c.k_exp);
    } else {
      keep(x, p.c.v, p.c.v_exp);
    }
  };
  for (int base = blockIdx.y * kBatch * kSegs; base < total;) {
    base += gridDim.y * kBatch * kSegs;
    if constexpr (kMany) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) finish(now[b]);
#pragma unroll
      for (int b = 0; b < kBatch; ++b) load(now[b], base + b * kSegs);
    } else {
      Row next;
      load(next, base);
      finish(now[0]);
      now[0] = next;
    }
  }
}

// ------------------------------------------------------------------ kv_read
struct ReadParams {
  Cache c;
  int heads;
  const int64_t* lengths;
  int64_t L;           // tokens a row of the outputs
  __nv_bfloat16* out[2];  // [rows][heads][L][dim]
};

// blockIdx = (kTokens tokens, head, row): where their tiles of 16 lie is looked up once, then a thread moves 16 output
// bytes at a time, kTokens * dim / 2048 of them in flight.
template <int kDim, bool kQuant, int kTokens>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int kTiles = kTokens / 16, kPer = kDim / 8, kRounds = (kTokens * kPer + kThreads - 1) / kThreads;
  __shared__ int64_t s_at[kTiles], s_exp[kQuant ? kTiles : 1];  // place of a tile's rows (-1: none) and exponents
  griddep_launch();
  griddep_wait();
  const int row = blockIdx.z, head = blockIdx.y, tid = threadIdx.x;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kTokens, span = static_cast<int64_t>(p.c.per_row) * p.c.page_size;
  int64_t n = p.lengths[row];
  if (n > span) {
    n = span;
    if (tid == 0) set_status(p.c.status, STATUS_BAD_PAGE);
  }
  if (n > p.L) n = p.L;
  if (tid < kTiles) {
    const int64_t tok = first + tid * 16;
    int64_t at = -1, x = 0;
    if (tok < n) {
      const int64_t nth = tok / p.c.page_size;
      const int64_t page = p.c.table[row * p.c.table_stride + nth];
      if (page < 0 || page >= p.c.pages) {
        set_status(p.c.status, STATUS_BAD_PAGE);
      } else {
        const int64_t r = static_cast<int64_t>(head) * p.c.page_size + (tok - nth * p.c.page_size);
        at = page * p.c.page_stride + r * kDim, x = page * p.c.exp_stride + r;
      }
    }
    s_at[tid] = at;
    if (kQuant) s_exp[tid] = x;
  }
  __syncthreads();
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    uint4 r[kRounds];
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int u = i * kThreads + tid, tok = u / kPer, c = u % kPer;
      const int64_t at = tok < kTokens ? s_at[tok / 16] : -1;
      r[i] = make_uint4(0, 0, 0, 0);
      if (at >= 0 && first + tok < n) {
        const int64_t x = at + tok % 16 * kDim + c * 8;
        if (kQuant) {
          const uint2 w = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(side ? p.c.v : p.c.k) + x));
          r[i] = make_uint4(w.x, w.y, static_cast<uint32_t>((side ? p.c.v_exp : p.c.k_exp)[s_exp[tok / 16] + tok % 16]), 0);
        } else {
          r[i] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(side ? p.c.v : p.c.k) + x));
        }
      }
    }
    __nv_bfloat16* const out = p.out[side] + ((static_cast<int64_t>(row) * p.heads + head) * p.L + first) * kDim;
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int u = i * kThreads + tid, tok = u / kPer;
      if (tok >= kTokens || first + tok >= p.L) break;
      if (kQuant) {
        const float s = exp2i(static_cast<int>(r[i].z));
        Chunk x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = unpack_e4m3x2(static_cast<uint16_t>((j < 2 ? r[i].x : r[i].y) >> (16 * (j & 1))));
          x.v[2 * j] = f.x * s;
          x.v[2 * j + 1] = f.y * s;
        }
        r[i] = pack(x);
      }
      *reinterpret_cast<uint4*>(out + u * 8) = r[i];
    }
  }
}

// ------------------------------------------------------------------ host side
template <typename... A>
static int launch(void (*kernel)(A...), dim3 grid, int threads, void* stream, const char* what, A... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (err != cudaSuccess) return set_error(std::string(what) + " launch: " + cudaGetErrorString(err)), DM3_ECUDA;
  note_launches(1);
  return DM3_OK;
}

static bool aligned(const Heads& h) {
  return reinterpret_cast<uintptr_t>(h.p) % 16 == 0 && h.ts % 8 == 0 && h.hs % 8 == 0;
}

// Tokens of a CTA: up to eight, so that their angles and places cost little beside their rows, but as few as fill the
// last wave of per_sm CTAs an SM. And CTAs that share a block's rows when there are few tokens.
struct Blocks {
  int tokens, shares;
};
static Blocks blocks(int64_t T, int rot, int64_t rounds_a_token, int per_sm) {
  int dev = 0;
  cudaGetDevice(&dev);
  const int64_t wave = per_sm * sm_count(dev), waves = (T + wave * kBlockTokens - 1) / (wave * kBlockTokens);
  Blocks b;
  b.tokens = static_cast<int>((T + wave * waves - 1) / (wave * waves));
  while (b.tokens * (rot / 2) > kAngles) --b.tokens;
  const int64_t want = (wave / 2 + T - 1) / T;
  b.shares = static_cast<int>(b.tokens > 1 ? 1 : want < rounds_a_token ? want : rounds_a_token);
  return b;
}

}  // namespace kv

bool kv_cache_ok(const kv::Cache& c, int kv_heads, int dim) {
  if (dim != 64 && dim != 128 && dim != 192 && dim != 256) return set_error("the cache's head size must be 64, 128, 192 or 256"), false;
  if (kv_heads < 1 || kv_heads > 65535) return set_error("the cache must have 1 to 65535 heads"), false;
  if (c.page_size < 16 || c.page_size % 16) return set_error("page_size must be a multiple of 16"), false;
  if (c.pages < 1 || !c.k || !c.v || !c.status) return set_error("cache: null pointer or no pages"), false;
  if (!c.k_exp != !c.v_exp) return set_error("cache: one of the exponent tables is missing"), false;
  if (c.rows < 0 || c.per_row < 0 || (c.rows > 0 && c.per_row > 0 && !c.table) || c.table_stride < 0 ||
      (c.table_stride < c.per_row && c.table_stride != 0))
    return set_error("bad page table"), false;
  if (static_cast<int64_t>(c.per_row) * c.page_size > INT32_MAX || static_cast<int64_t>(kv_heads) * c.page_size > INT32_MAX)
    return set_error("cache: a row's table, or a page, of 2^31 tokens and more"), false;
  const int64_t row = static_cast<int64_t>(kv_heads) * c.page_size;
  const int unit = c.k_exp ? 16 : 8;  // elements in 16 bytes
  if (c.page_stride < row * dim || c.page_stride % unit || (c.k_exp && (c.exp_stride < row || c.exp_stride % 16)))
    return set_error("cache: pages overlap, or do not start on 16 bytes"), false;
  if (reinterpret_cast<uintptr_t>(c.k) % 16 || reinterpret_cast<uintptr_t>(c.v) % 16 ||
      reinterpret_cast<uintptr_t>(c.k_exp) % 16 || reinterpret_cast<uintptr_t>(c.v_exp) % 16)
    return set_error("cache: the buffers must be 16-byte aligned"), false;
  return true;
}

}  // namespace dm3

// ------------------------------------------------------------------ C ABI
using namespace dm3;
using namespace dm3::kv;

extern "C" int dm3_rope(const void* x, int T, int heads, int dim, int64_t ts, int64_t hs, const int64_t* positions,
                        const double* inv_freq, int rot, int interleaved, double factor, void* y, void* stream) {
  note_launches(0);
  if (T < 0 || heads < 1 || dim < 1 || static_cast<int64_t>(heads) * dim > 1 << 24)
    return set_error("rope: bad token count, head count or head size"), DM3_EINVAL;
  if (rot < 2 || rot % 2 || rot > dim || rot > kMaxRot)
    return set_error("rope: the rotated part must be even, at most the head and at most 1024"), DM3_EINVAL;
  if (T == 0) return DM3_OK;
  if (!x || !positions || !inv_freq || !y) return set_error("rope: null pointer"), DM3_EINVAL;
  RopeParams p{{static_cast<const __nv_bfloat16*>(x), ts, hs, heads}, static_cast<__nv_bfloat16*>(y), T, dim, 1, positions,
               inv_freq, rot, interleaved, factor};
  // 16 bytes a thread at a time where rows and pairs fall on them, a row has at most a CTA's lanes, and a block's rows
  // are counted in 16 bits
  const bool wide = dim % 16 == 0 && rot % 16 == 0 && dim <= 16 * kThreads && heads <= 65535 / kBlockTokens && aligned(p.x) &&
                    reinterpret_cast<uintptr_t>(y) % 16 == 0;
  if (wide) {
    int shift = 0;
    while (16 << shift < dim) ++shift;
    const int round = kThreads >> shift;
    const Blocks b = blocks(T, rot, (heads + round - 1) / round, 5);
    p.block = b.tokens;
    return launch(interleaved ? rope_kernel<true> : rope_kernel<false>, dim3((T + b.tokens - 1) / b.tokens, b.shares), kThreads, stream, "rope", p, shift, Div(heads));
  }
  const Blocks b = blocks(T, 0, (heads * dim + kThreads - 1) / kThreads, 4);
  return launch(rope_any_kernel, dim3(T, b.shares), kThreads, stream, "rope", p);
}

extern "C" int dm3_kv_write(const void* q, int q_heads, int64_t q_ts, int64_t q_hs, const void* k, int64_t k_ts, int64_t k_hs,
                            const void* v, int64_t v_ts, int64_t v_hs, int T, int kv_heads, int dim, const int64_t* rows,
                            const int64_t* positions, const int32_t* table, int64_t table_stride, int table_rows, int per_row,
                            void* k_cache, void* v_cache, int64_t page_stride, int8_t* k_exp, int8_t* v_exp,
                            int64_t exp_stride, int pages, int page_size, const double* inv_freq, int rot, int interleaved,
                            double factor, void* q_out, uint32_t* status, void* stream) {
  note_launches(0);
  WriteParams p{};
  p.c = {k_cache, v_cache, k_exp, v_exp, page_stride, exp_stride, pages, page_size, table, table_stride, table_rows, per_row, status};
  if (!kv_cache_ok(p.c, kv_heads, dim)) return DM3_EINVAL;
  if (T < 0 || q_heads < 0 || q_heads > 65535) return set_error("kv_write: bad token or head count"), DM3_EINVAL;
  if (rot && (rot < 16 || rot % 16 || rot > dim || !inv_freq))
    return set_error("kv_write: the rotated part must be a multiple of 16, at most the head"), DM3_EINVAL;
  if (T == 0) return DM3_OK;
  if (!k || !v || !positions || (q_heads && (!q || !q_out))) return set_error("kv_write: null pointer"), DM3_EINVAL;
  p.q = {static_cast<const __nv_bfloat16*>(q), q_ts, q_hs, q_heads};
  p.k = {static_cast<const __nv_bfloat16*>(k), k_ts, k_hs, kv_heads};
  p.v = {static_cast<const __nv_bfloat16*>(v), v_ts, v_hs, kv_heads};
  if (!aligned(p.k) || !aligned(p.v) || (q_heads && (!aligned(p.q) || reinterpret_cast<uintptr_t>(q_out) % 16)))
    return set_error("kv_write: rows must start on 16 bytes"), DM3_EINVAL;
  p.y = static_cast<__nv_bfloat16*>(q_out);
  p.T = T, p.dim = dim, p.rows = rows, p.positions = positions;
  p.inv_freq = inv_freq, p.rot = rot, p.factor = factor;
  const int seg = dim == 64 ? 4 : dim == 128 ? 8 : 16, n = q_heads + 2 * kv_heads;
  if (n > 65535 / kBlockTokens) return set_error("kv_write: too many heads"), DM3_EINVAL;
  int dev = 0;
  cudaGetDevice(&dev);
  const bool many = !k_exp && T > 5 * kBlockTokens * sm_count(dev);  // more than one wave of full blocks
  const int round = (many ? 2 : 1) * kThreads / seg;
  const Blocks b = blocks(T, rot, (n + round - 1) / round, many ? 5 : 4);
  p.block = b.tokens;
  const dim3 grid((T + b.tokens - 1) / b.tokens, b.shares);
  auto go = [&](auto kernel) { return launch(kernel, grid, kThreads, stream, "kv_write", p, Div(q_heads), Div(kv_heads)); };
  auto pick = [&](auto lanes) {
    constexpr int kSeg = decltype(lanes)::value;
    if (k_exp) return interleaved ? go(write_kernel<kSeg, true, true, false>) : go(write_kernel<kSeg, true, false, false>);
    if (many) return interleaved ? go(write_kernel<kSeg, false, true, true>) : go(write_kernel<kSeg, false, false, true>);
    return interleaved ? go(write_kernel<kSeg, false, true, false>) : go(write_kernel<kSeg, false, false, false>);
  };
  return seg == 4   ? pick(std::integral_constant<int, 4>{})
         : seg == 8 ? pick(std::integral_constant<int, 8>{})
                    : pick(std::integral_constant<int, 16>{});
}

extern "C" int dm3_kv_read(const void* k_cache, const void* v_cache, int64_t page_stride, const int8_t* k_exp,
                           const int8_t* v_exp, int64_t exp_stride, int pages, int page_size, int kv_heads, int dim,
                           const int32_t* table, int64_t table_stride, int table_rows, int per_row, const int64_t* lengths,
                           int64_t max_length, void* k_out, void* v_out, uint32_t* status, void* stream) {
  note_launches(0);
  ReadParams p{};
  p.c = {const_cast<void*>(k_cache), const_cast<void*>(v_cache), const_cast<int8_t*>(k_exp), const_cast<int8_t*>(v_exp),
         page_stride, exp_stride, pages, page_size, table, table_stride, table_rows, per_row, status};
  if (!kv_cache_ok(p.c, kv_heads, dim)) return DM3_EINVAL;
  if (table_rows > 65535) return set_error("kv_read: at most 65535 rows"), DM3_EINVAL;
  if (max_length < 0 || max_length > (int64_t(1) << 31)) return set_error("kv_read: bad max_length"), DM3_EINVAL;
  if (table_rows == 0 || max_length == 0) return DM3_OK;
  if (!lengths || !k_out || !v_out || reinterpret_cast<uintptr_t>(k_out) % 16 || reinterpret_cast<uintptr_t>(v_out) % 16)
    return set_error("kv_read: null or misaligned pointer"), DM3_EINVAL;
  p.heads = kv_heads, p.lengths = lengths, p.L = max_length;
  p.out[0] = static_cast<__nv_bfloat16*>(k_out), p.out[1] = static_cast<__nv_bfloat16*>(v_out);
  // 64 tokens a CTA; 16 where that leaves SMs idle (5 rows of 1,237 tokens, 2 heads of 256: 5.9 and 4.7 us)
  int dev = 0;
  cudaGetDevice(&dev);
  const bool few = (max_length + 63) / 64 * kv_heads * table_rows < 2 * sm_count(dev);
  const dim3 grid(static_cast<unsigned>(few ? (max_length + 15) / 16 : (max_length + 63) / 64), kv_heads, table_rows);
  auto go = [&](auto kernel) { return launch(kernel, grid, kThreads, stream, "kv_read", p); };
  auto pick = [&](auto d) {
    constexpr int kDim = decltype(d)::value;
    if (k_exp) return few ? go(read_kernel<kDim, true, 16>) : go(read_kernel<kDim, true, 64>);
    return few ? go(read_kernel<kDim, false, 16>) : go(read_kernel<kDim, false, 64>);
  };
  switch (dim) {
    case 64: return pick(std::integral_constant<int, 64>{});
    case 128: return pick(std::integral_constant<int, 128>{});
    case 192: return pick(std::integral_constant<int, 192>{});
    default: return pick(std::integral_constant<int, 256>{});
  }
}
