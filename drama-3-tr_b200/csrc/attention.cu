// One new token's attention over the paged key-value cache (sm_100a).
//
//   s_t = scale * q . k_t,  p = softmax(s) over the tokens seen,  out = sum_t p_t v_t,
//   lse = log sum_t exp(s_t),  seen: max(0, n - window) <= t < n (window 0: all), n the row's length
//
// One pass with a running maximum M and sum l; a row that sees nothing gives zeros and lse = -inf.
//
// Bound: the bytes of the cache's rows, each used by the group of query heads that shares them
// (2 * group flops a byte and less), so the kernel is laid out to keep loads in flight, not for the tensor
// peak: the products run as warp-level m16n8k16 tiles whose operands come from global memory straight into
// registers, without shared memory, barriers between warps or a shuffle of the data. With tokens as the
// tile's 16 rows and the query heads as its 8 columns,
//   S^T = K Q^T:  a lane's 16-byte load of a key row holds the k-columns of 2 (bf16) or 4 (e4m3) tiles
//                 once the same permutation of dim is applied to Q;
//   O^T = V^T P^T: a lane loads 16 bytes of 4 tokens' value rows and interleaves pairs of tokens with byte
//                 permutes; P^T comes from S^T's accumulators by an 8x8 transpose (movmatrix).
// A group of up to 8 heads wastes nothing, where heads as rows would waste half of the tile and of the registers.
// Every warp walks its own 16-token tiles, the next keys loading while the softmax and the values' product
// run; the warps of a CTA join in shared memory at the end.
//
// Long rows are split: `splits` CTAs share a row's tiles evenly (the device reads the length, so one captured
// graph serves all lengths), each leaves (M, l, O) in fp32, and a second kernel joins them in order: no atomics,
// the same answer every time.
//
// An e4m3 row is code * 2^e. For keys 2^e joins the logit's scale. For values it joins the weight's exponent:
// w_t = 2^(s_t + e_t - M) with M the running maximum of s_t + e_t, so weights are in fp16's range whatever the rows'
// sizes, and l sums w_t * 2^-e_t. Codes are exact in fp16; queries are scaled by a power of two to
// [2^14, 2^15), where fp16 holds a bf16 row to 2^-40 of its largest value; a weight is rounded once to 11 bits.
// With a bf16 cache a weight goes to the tensor cores as a bf16 pair (high and low part, 16 bits).
#include <cmath>
#include <cstdint>
#include <string>

#include "dm3.h"
#include "dm3_common.cuh"
#include "dm3_internal.h"
#include "dm3_kv.cuh"

namespace dm3 {
namespace attn {

using kv::Cache;

constexpr int kWarps = 4;
constexpr int kTile = 16;  // tokens of one tile; pages hold whole tiles
// The maximum is raised only when a logit exceeds it by more than kSlack (log2): weights reach 2^kSlack. fp16
// weights carry 2^kLift besides, so that they stay normal down to 2^-(14 + kLift).
constexpr float kSlack = 8.f, kLift = 6.f;

struct Params {
  const __nv_bfloat16* q;  // [rows][q_heads][dim]
  int64_t q_rs, q_hs;
  int q_heads, kv_heads, group, head_tiles;
  Cache c;
  const int64_t* lengths;
  float scale_log2;  // scale * log2(e)
  int64_t window;
  int splits, min_tiles;
  __nv_bfloat16* out;  // [rows][q_heads][dim]
  float* lse;          // [rows][q_heads]
  float* part_o;       // [rows][q_heads][splits][dim]
  float2* part_ml;     // [rows][q_heads][splits]
};

// The tiles that a row sees, and how many of them each split takes.
struct Span {
  int64_t first, n;  // tokens seen: [first, n)
  int64_t tile0;     // tile of the first one
  int64_t tiles, chunk;
};
__device__ __forceinline__ Span row_span(const Params& p, int row) {
  Span s;
  const int64_t cap = static_cast<int64_t>(p.c.per_row) * p.c.page_size;
  s.n = p.lengths[row];
  if (s.n > cap) s.n = cap;
  if (s.n < 0) s.n = 0;
  s.first = p.window > 0 && s.n > p.window ? s.n - p.window : 0;
  s.tile0 = s.first / kTile;
  s.tiles = (s.n + kTile - 1) / kTile - s.tile0;
  s.chunk = (s.tiles + p.splits - 1) / p.splits;
  if (s.chunk < p.min_tiles) s.chunk = p.min_tiles;
  return s;
}

__device__ __forceinline__ uint4 ld16(const uint8_t* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ uint2 ld8(const uint8_t* p) {
  uint2 r;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}

// D[16x8] += A[16x16] B[16x8], fp32 accumulators; lane (g = lane / 4, q = lane % 4) holds A rows g, g + 8 at columns
// 2q, 2q + 1 (a0, a1) and 2q + 8, 2q + 9 (a2, a3), B column g at the same k, D rows g, g + 8 at columns 2q, 2q + 1.
template <bool kHalf>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (kHalf)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8x8 matrix of 16-bit values held as lane / 4 = row, 2 * (lane % 4) = column.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t half_pair(uint32_t codes) {  // 2 e4m3 codes in the low 16 bits -> fp16 pair
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
__device__ __forceinline__ uint32_t half_pair_hi(uint32_t codes) {  // the same for the high 16 bits
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// kNT: tiles of 8 query heads; kU: token tiles of one step of a warp.
template <int kDim, bool kQuant, int kNT, int kU>
struct Shape {
  static constexpr int kRow = kDim * (kQuant ? 1 : 2);                  // bytes of a cache row
  static constexpr int kKP = kRow / 64;                                 // 16-byte loads of a key row a lane
  static constexpr int kVB = kQuant && kDim % 128 ? 8 : 16;             // bytes of one value load a lane
  static constexpr int kVP = kRow / (8 * kVB), kVW = kVB / 4;           // loads a row, words a load
  static constexpr int kE = kQuant ? kVB : kVB / 2;                     // values a load
  static constexpr int kHeads = 8 * kNT;
  static constexpr bool kSharedQ = kRow == 512;  // the registers of keys and values leave none for the queries
  static constexpr int kPitch = 2 * kDim + 8;  // floats of a head pair in shared memory (8: no bank conflicts)
};

template <int kDim, bool kQuant, int kNT, int kU>
__global__ void __launch_bounds__(kWarps * 32) attend_kernel(const __grid_constant__ Params p) {
  using C = Shape<kDim, kQuant, kNT, kU>;
  __shared__ __align__(16) float s_o[kWarps][kNT * 4][C::kPitch];
  __shared__ uint4 s_q[C::kSharedQ ? kNT * C::kKP : 1][32];
  __shared__ float s_m[kWarps][C::kHeads], s_l[kWarps][C::kHeads];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lr = lane >> 2, lc = lane & 3;
  const int split = blockIdx.x, kvh = blockIdx.y / p.head_tiles, ht = blockIdx.y % p.head_tiles, row = blockIdx.z;
  const int h0 = ht * C::kHeads;  // first head of the group
  griddep_launch();
  griddep_wait();
  const Span sp = row_span(p, row);
  const int64_t begin = split * sp.chunk;  // tiles of this CTA, counted from sp.tile0
  const int64_t end = begin + sp.chunk < sp.tiles ? begin + sp.chunk : sp.tiles;
  const int64_t qrow = static_cast<int64_t>(row) * p.q_heads + kvh * p.group + h0;  // output row of head 0
  if (p.lengths[row] > sp.n && threadIdx.x == 0) kv::set_status(p.c.status, STATUS_BAD_PAGE);
  if (begin >= end) {
    if (split == 0) {  // a row that sees nothing
      for (int i = threadIdx.x; i < C::kHeads * kDim; i += blockDim.x)
        if (h0 + i / kDim < p.group) p.out[qrow * kDim + i] = __float2bfloat16_rn(0.f);
      if (threadIdx.x < C::kHeads && h0 + threadIdx.x < p.group) p.lse[qrow + threadIdx.x] = -INFINITY;
    }
    return;
  }

  // queries as B operands, the permutation of dim that 16-byte key loads give
  uint32_t qf[kNT][C::kSharedQ ? 1 : kDim / 8];
  float qs[kNT][2];  // logit scale of the lane's two heads of each tile
#pragma unroll
  for (int nt = 0; nt < kNT; ++nt) {
    const int h = h0 + nt * 8 + lr;
    const __nv_bfloat16* src = p.q + row * p.q_rs + static_cast<int64_t>(kvh * p.group + h) * p.q_hs;
    const bool on = h < p.group;
    if (C::kSharedQ) {
      for (int j = warp; j < C::kKP; j += kWarps)
        s_q[nt * C::kKP + j][lane] = on ? *reinterpret_cast<const uint4*>(src + j * 32 + lc * 8) : make_uint4(0, 0, 0, 0);
      qs[nt][0] = qs[nt][1] = p.scale_log2;
    } else if (!kQuant) {
#pragma unroll
      for (int j = 0; j < C::kKP; ++j) {
        const uint4 w = on ? *reinterpret_cast<const uint4*>(src + j * 32 + lc * 8) : make_uint4(0, 0, 0, 0);
        qf[nt][4 * j] = w.x, qf[nt][4 * j + 1] = w.y, qf[nt][4 * j + 2] = w.z, qf[nt][4 * j + 3] = w.w;
      }
      qs[nt][0] = qs[nt][1] = p.scale_log2;
    } else {
      uint32_t raw[kDim / 8];
      uint32_t top = 0;  // the largest magnitude's bits
#pragma unroll
      for (int j = 0; j < C::kKP; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 w = on ? *reinterpret_cast<const uint4*>(src + j * 64 + lc * 16 + i * 8) : make_uint4(0, 0, 0, 0);
          const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            raw[j * 8 + i * 4 + k] = x[k];
            top = max(top, max(x[k] << 16 & 0x7fffffffu, x[k] & 0x7fff0000u));
          }
        }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = min(max(static_cast<int>(top >> 23) - 127, -112), 126) - 14;  // 2^-e puts the largest in [2^14, 2^15)
      const float up = exp2i(-e);
#pragma unroll
      for (int i = 0; i < kDim / 8; ++i)
        qf[nt][i] = pack_half(__uint_as_float(raw[i] << 16) * up, __uint_as_float(raw[i] & 0xffff0000u) * up);
      const float down = p.scale_log2 * exp2i(e);  // of head lr; the accumulators' heads are 2 * lc and 2 * lc + 1
      qs[nt][0] = __shfl_sync(0xffffffffu, down, (2 * lc) * 4);
      qs[nt][1] = __shfl_sync(0xffffffffu, down, (2 * lc + 1) * 4);
    }
  }

  if (C::kSharedQ) __syncthreads();

  // a warp's steps: kU tiles each, warps in turn; lane i of a block of 32 knows the page of the block's tile i
  constexpr int kBlock = 32 / kU;  // steps a block
  const int steps = static_cast<int>((end - begin + kWarps * kU - 1) / (kWarps * kU));
  const int per_page = p.c.page_size / kTile;
  int pg, off;  // page (-1: not a tile of this CTA, or a bad page) and tile in the page
  auto find = [&](int step0, int& page, int& tile) {
    const int64_t t = begin + (static_cast<int64_t>(step0 + lane / kU) * kWarps + warp) * kU + lane % kU;
    page = -1, tile = 0;
    if (t < end) {
      const int64_t g = sp.tile0 + t;
      const int64_t nth = g / per_page;
      tile = static_cast<int>(g - nth * per_page);
      page = p.c.table[row * p.c.table_stride + nth];
      if (page < 0 || page >= p.c.pages) {
        page = -1;
        kv::set_status(p.c.status, STATUS_BAD_PAGE);
      }
    }
  };
  int next_pg, next_off;
  find(0, pg, off);
  find(kBlock, next_pg, next_off);

  const uint8_t* const kbase = static_cast<const uint8_t*>(p.c.k) + lr * C::kRow + lc * 16;
  const uint8_t* const vbase = static_cast<const uint8_t*>(p.c.v) + lc * 2 * C::kRow + lr * C::kVB;
  uint4 k[kU][2][C::kKP];
  uint32_t v[kU][4][C::kVP][C::kVW];
  int ek[kU][2], ev[kU][2];
  int64_t at[kU];  // byte offset of a tile's rows in either buffer
  int lo[kU], hi[kU];  // rows of the tile that are seen
  auto load_k = [&](int step) {
    if (step % kBlock == 0 && step > 0) {
      pg = next_pg, off = next_off;
      find(step + kBlock, next_pg, next_off);
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int from = (step % kBlock) * kU + u;
      const int page = __shfl_sync(0xffffffffu, pg, from), tile = __shfl_sync(0xffffffffu, off, from);
      const int64_t r = static_cast<int64_t>(kvh) * p.c.page_size + tile * kTile, pp = page < 0 ? 0 : page;
      at[u] = (pp * p.c.page_stride + r * kDim) * (kQuant ? 1 : 2);
      const int64_t t0 = (sp.tile0 + begin + (static_cast<int64_t>(step) * kWarps + warp) * kU + u) * kTile;
      lo[u] = sp.first > t0 ? static_cast<int>(sp.first - t0) : 0;
      hi[u] = page < 0 ? 0 : sp.n - t0 < kTile ? static_cast<int>(sp.n - t0) : kTile;
#pragma unroll
      for (int j = 0; j < C::kKP; ++j) {
        k[u][0][j] = ld16(kbase + at[u] + j * 64);
        k[u][1][j] = ld16(kbase + at[u] + j * 64 + 8 * C::kRow);
      }
      if (kQuant) {
        const int64_t x = pp * p.c.exp_stride + r + lr;
        ek[u][0] = p.c.k_exp[x], ek[u][1] = p.c.k_exp[x + 8];
        ev[u][0] = p.c.v_exp[x], ev[u][1] = p.c.v_exp[x + 8];
      }
    }
  };
  load_k(0);

  float o[kNT][kDim / 16][4];
  float m[kNT][2], l[kNT][2];  // of the lane's two heads a tile: m the same in all lanes of a head, l a lane's part
#pragma unroll
  for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
    for (int i = 0; i < kDim / 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[nt][i][j] = 0.f;
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
  }

  for (int step = 0; step < steps; ++step) {
    // this step's values start loading, then the keys' product
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < C::kVP; ++j) {
          const uint8_t* src = vbase + at[u] + ((i & 1) + (i >> 1) * 8) * C::kRow + j * 8 * C::kVB;
          if (C::kVB == 16) {
            const uint4 w = ld16(src);
            v[u][i][j][0] = w.x, v[u][i][j][1] = w.y, v[u][i][j][C::kVW - 2] = w.z, v[u][i][j][C::kVW - 1] = w.w;
          } else {
            const uint2 w = ld8(src);
            v[u][i][j][0] = w.x, v[u][i][j][1] = w.y;
          }
        }
    float s[kU][kNT][4];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[u][nt][j] = 0.f;
#pragma unroll
      for (int j = 0; j < C::kKP; ++j) {
        const uint32_t a[4] = {k[u][0][j].x, k[u][0][j].y, k[u][0][j].z, k[u][0][j].w};
        const uint32_t b[4] = {k[u][1][j].x, k[u][1][j].y, k[u][1][j].z, k[u][1][j].w};
        if (!kQuant) {
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) {
            const uint4 w = C::kSharedQ ? s_q[nt * C::kKP + j][lane]
                                        : make_uint4(qf[nt][4 * j], qf[nt][4 * j + 1], qf[nt][4 * j + 2], qf[nt][4 * j + 3]);
            mma<false>(s[u][nt], a[0], b[0], a[1], b[1], w.x, w.y);
            mma<false>(s[u][nt], a[2], b[2], a[3], b[3], w.z, w.w);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x0 = half_pair(a[i]), x1 = half_pair(b[i]), x2 = half_pair_hi(a[i]), x3 = half_pair_hi(b[i]);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) mma<true>(s[u][nt], x0, x1, x2, x3, qf[nt][8 * j + 2 * i], qf[nt][8 * j + 2 * i + 1]);
          }
        }
      }
    }
    // logits in log2 units (with the value rows' exponents), -inf where nothing is seen
    float kf[kU][2], vf[kU][2], back[kU][2];
    int low[kU], high[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      low[u] = lo[u], high[u] = hi[u];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        kf[u][r] = kQuant ? exp2i(ek[u][r]) : 1.f;
        vf[u][r] = kQuant ? static_cast<float>(ev[u][r]) : 0.f;
        back[u][r] = kQuant ? exp2i(-ev[u][r]) : 1.f;
      }
    }
    if (step + 1 < steps) load_k(step + 1);
    bool above = false;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float z = s[u][nt][j] * qs[nt][j & 1];
          if (kQuant) z = z * kf[u][j >> 1] + vf[u][j >> 1];
          s[u][nt][j] = z;
        }
      if (low[u] > 0 || high[u] < kTile)
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = lr + (j >> 1) * 8;
            if (r < low[u] || r >= high[u]) s[u][nt][j] = -INFINITY;
          }
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) above |= s[u][nt][j] > m[nt][j & 1] + kSlack;
    }
    if (__any_sync(0xffffffffu, above)) {
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x = m[nt][h];
#pragma unroll
          for (int u = 0; u < kU; ++u) x = fmaxf(x, fmaxf(s[u][nt][h], s[u][nt][2 + h]));
#pragma unroll
          for (int w = 4; w < 32; w *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
          const float f = m[nt][h] == -INFINITY ? 0.f : ex2(m[nt][h] - x);
          m[nt][h] = x;
          l[nt][h] *= f;
#pragma unroll
          for (int i = 0; i < kDim / 16; ++i) o[nt][i][h] *= f, o[nt][i][2 + h] *= f;
        }
    }
    // weights, as the second product's B operands
    uint32_t ph[kU][kNT][2], pl[kU][kNT][2];
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        float w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float mm = m[nt][j & 1] == -INFINITY ? 0.f : m[nt][j & 1];
          w[j] = ex2(s[u][nt][j] - mm + (kQuant ? kLift : 0.f));
          l[nt][j & 1] += kQuant ? (w[j] == 0.f ? 0.f : w[j] * back[u][j >> 1]) : w[j];
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (kQuant) {
            ph[u][nt][r] = transpose8(pack_half(w[2 * r], w[2 * r + 1]));
          } else {
            const uint32_t h = pack_bf16(w[2 * r], w[2 * r + 1]);
            ph[u][nt][r] = transpose8(h);
            pl[u][nt][r] = transpose8(pack_bf16(w[2 * r] - __uint_as_float(h << 16), w[2 * r + 1] - __uint_as_float(h & 0xffff0000u)));
          }
        }
      }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      // what lies in places not seen may be anything: no weight of zero makes a NaN harmless
      if (low[u] > 0 || high[u] < kTile)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = lc * 2 + (i & 1) + (i >> 1) * 8;
          if (r < low[u] || r >= high[u])
#pragma unroll
            for (int j = 0; j < C::kVP; ++j)
#pragma unroll
              for (int w = 0; w < C::kVW; ++w) v[u][i][j][w] = 0;
        }
#pragma unroll
      for (int j = 0; j < C::kVP; ++j)
#pragma unroll
        for (int w = 0; w < C::kVW; ++w) {
          const uint32_t t0 = v[u][0][j][w], t1 = v[u][1][j][w], t8 = v[u][2][j][w], t9 = v[u][3][j][w];
          if (!kQuant) {
            const int tile = j * 4 + w;
            const uint32_t a0 = __byte_perm(t0, t1, 0x5410), a1 = __byte_perm(t0, t1, 0x7632);
            const uint32_t a2 = __byte_perm(t8, t9, 0x5410), a3 = __byte_perm(t8, t9, 0x7632);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) {
              mma<false>(o[nt][tile], a0, a1, a2, a3, ph[u][nt][0], ph[u][nt][1]);
              mma<false>(o[nt][tile], a0, a1, a2, a3, pl[u][nt][0], pl[u][nt][1]);
            }
          } else {
            const int tile = (j * C::kVW + w) * 2;
            const uint32_t x0 = __byte_perm(t0, t1, 0x5140), x1 = __byte_perm(t0, t1, 0x7362);
            const uint32_t y0 = __byte_perm(t8, t9, 0x5140), y1 = __byte_perm(t8, t9, 0x7362);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) {
              mma<true>(o[nt][tile], half_pair(x0), half_pair_hi(x0), half_pair(y0), half_pair_hi(y0), ph[u][nt][0], ph[u][nt][1]);
              mma<true>(o[nt][tile + 1], half_pair(x1), half_pair_hi(x1), half_pair(y1), half_pair_hi(y1), ph[u][nt][0], ph[u][nt][1]);
            }
          }
        }
    }
  }

  // join the warps
#pragma unroll
  for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int w = 4; w < 32; w *= 2) l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], w);
      if (lr == 0) s_m[warp][nt * 8 + 2 * lc + h] = m[nt][h], s_l[warp][nt * 8 + 2 * lc + h] = l[nt][h];
    }
#pragma unroll
  for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
    for (int i = 0; i < kDim / 16; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r)  // (d, both heads) at [head pair][tile][r][lr]
        *reinterpret_cast<float2*>(&s_o[warp][nt * 4 + lc][(i * 16 + r * 8 + lr) * 2]) = make_float2(o[nt][i][2 * r], o[nt][i][2 * r + 1]);
  __syncthreads();
  const bool whole = sp.tiles <= sp.chunk;
  for (int i = threadIdx.x; i < C::kHeads * kDim; i += blockDim.x) {
    const int h = i / kDim, d = i % kDim;
    if (h0 + h >= p.group) break;
    float mm = -INFINITY, ll = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][h]);
    // d = pass * 8 * kE + lr * kE + 2 * (tile of the pass) + r
    const int in = d % (8 * C::kE), tile = d / (8 * C::kE) * (C::kE / 2) + in % C::kE / 2;
    const int at_ = (tile * 16 + (in & 1) * 8 + in / C::kE) * 2 + (h & 1);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = s_m[w][h] == -INFINITY ? 0.f : ex2(s_m[w][h] - mm);
      ll += s_l[w][h] * f;
      x += s_o[w][h >> 1][at_] * f;
    }
    if (whole) {
      p.out[(qrow + h) * kDim + d] = __float2bfloat16_rn(ll == 0.f ? 0.f : x / ll);
      if (d == 0) p.lse[qrow + h] = ll == 0.f ? -INFINITY : (mm - (kQuant ? kLift : 0.f) + log2f(ll)) * 0.69314718055994531f;
    } else {
      const int64_t to = (qrow + h) * p.splits + split;
      p.part_o[to * kDim + d] = x;
      if (d == 0) p.part_ml[to] = make_float2(mm, ll);
    }
  }
}

// Joins the splits of one query head: blockIdx = (head, row), a thread a value.
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Params p, int dim, float lift) {
  griddep_launch();
  griddep_wait();
  const int row = blockIdx.y;
  const Span sp = row_span(p, row);
  if (sp.tiles <= sp.chunk) return;  // written whole, or nothing to see
  const int n = static_cast<int>((sp.tiles + sp.chunk - 1) / sp.chunk);
  const int64_t head = static_cast<int64_t>(row) * p.q_heads + blockIdx.x;
  const float2* ml = p.part_ml + head * p.splits;
  const float* po = p.part_o + head * p.splits * dim + threadIdx.x;
  float mm = -INFINITY, ll = 0.f, x = 0.f;
  for (int i = 0; i < n; ++i) mm = fmaxf(mm, ml[i].x);
  for (int i = 0; i < n; ++i) {
    const float2 a = ml[i];
    const float f = a.x == -INFINITY ? 0.f : ex2(a.x - mm);
    ll += a.y * f;
    x += po[static_cast<int64_t>(i) * dim] * f;
  }
  p.out[head * dim + threadIdx.x] = __float2bfloat16_rn(ll == 0.f ? 0.f : x / ll);
  if (threadIdx.x == 0) p.lse[head] = ll == 0.f ? -INFINITY : (mm - lift + log2f(ll)) * 0.69314718055994531f;
}

// ------------------------------------------------------------------ host side
struct Plan {
  int head_tiles, splits, min_tiles;
};

static int sms() {
  int dev = 0;
  cudaGetDevice(&dev);
  return sm_count(dev);
}

static int tile_heads(int group, int dim) { return group > 8 && dim <= 128 ? 16 : 8; }

static Plan plan(int rows, int q_heads, int kv_heads, int dim, bool quant, int64_t tiles) {
  Plan r;
  const int group = q_heads / kv_heads, heads = tile_heads(group, dim);
  r.head_tiles = (group + heads - 1) / heads;
  const int64_t units = static_cast<int64_t>(rows) * kv_heads * r.head_tiles;
  r.min_tiles = 8;
  int64_t s = (static_cast<int64_t>(sms()) * 8 + units - 1) / units;
  const int64_t most = (tiles + r.min_tiles - 1) / r.min_tiles;
  if (s > most) s = most;
  r.splits = static_cast<int>(s < 1 ? 1 : s);
  return r;
}

template <typename... A>
static cudaError_t start(void (*kernel)(A...), dim3 grid, int threads, void* stream, A... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int kDim, bool kQuant>
static cudaError_t attend(const Params& p, dim3 grid, void* stream) {
  // token tiles a step: 32 registers of keys a lane (64 for 512-byte rows)
  constexpr int kRow = kDim * (kQuant ? 1 : 2), kU = kRow <= 64 ? 4 : kRow <= 128 ? 2 : 1;
  if constexpr (kDim <= 128) {
    if (tile_heads(p.group, kDim) == 16) return start(attend_kernel<kDim, kQuant, 2, kU>, grid, kWarps * 32, stream, p);
  }
  return start(attend_kernel<kDim, kQuant, 1, kU>, grid, kWarps * 32, stream, p);
}

}  // namespace attn
}  // namespace dm3

// ------------------------------------------------------------------ C ABI
extern "C" size_t dm3_paged_attention_workspace_bytes(int rows, int q_heads, int kv_heads, int dim, int page_size,
                                                      int per_row) {
  if (rows < 1 || q_heads < 1 || kv_heads < 1 || q_heads < kv_heads || dim < 1 || page_size < 16 || per_row < 0) return 0;
  const int64_t tiles = static_cast<int64_t>(per_row) * (page_size / dm3::attn::kTile);
  const int splits = dm3::attn::plan(rows, q_heads, kv_heads, dim, false, tiles).splits;
  return splits == 1 ? 0 : static_cast<size_t>(rows) * q_heads * splits * (dim * sizeof(float) + sizeof(float2));
}

extern "C" int dm3_paged_attention(const void* q, int64_t q_rs, int64_t q_hs, int q_heads, const void* k_cache,
                                   const void* v_cache, int64_t page_stride, const int8_t* k_exp, const int8_t* v_exp,
                                   int64_t exp_stride, int pages, int page_size, int kv_heads, int dim,
                                   const int32_t* table, int64_t table_stride, int rows, int per_row,
                                   const int64_t* lengths, float scale, int64_t window, void* out, float* lse,
                                   uint32_t* status, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace dm3;
  note_launches(0);
  attn::Params p{};
  p.c = {const_cast<void*>(k_cache), const_cast<void*>(v_cache), const_cast<int8_t*>(k_exp), const_cast<int8_t*>(v_exp),
         page_stride, exp_stride, pages, page_size, table, table_stride, rows, per_row, status};
  if (!kv_cache_ok(p.c, kv_heads, dim)) return DM3_EINVAL;
  if (q_heads < kv_heads || q_heads % kv_heads || q_heads > 65535)
    return set_error("paged_attention: the query heads must be a multiple of the cache's heads"), DM3_EINVAL;
  if (rows > 65535) return set_error("paged_attention: at most 65535 rows"), DM3_EINVAL;
  if (window < 0 || !std::isfinite(scale)) return set_error("paged_attention: bad window or scale"), DM3_EINVAL;
  if (rows == 0) return DM3_OK;
  if (!q || !lengths || !out || !lse) return set_error("paged_attention: null pointer"), DM3_EINVAL;
  if (reinterpret_cast<uintptr_t>(q) % 16 || q_rs % 8 || q_hs % 8 || reinterpret_cast<uintptr_t>(out) % 16)
    return set_error("paged_attention: rows must start on 16 bytes"), DM3_EINVAL;
  int64_t tiles = static_cast<int64_t>(per_row) * (page_size / attn::kTile);
  if (window > 0 && window / attn::kTile + 2 < tiles) tiles = window / attn::kTile + 2;  // the tiles that a window touches
  const attn::Plan plan = attn::plan(rows, q_heads, kv_heads, dim, k_exp != nullptr, tiles);
  p.q = static_cast<const __nv_bfloat16*>(q), p.q_rs = q_rs, p.q_hs = q_hs, p.q_heads = q_heads, p.kv_heads = kv_heads;
  p.group = q_heads / kv_heads, p.head_tiles = plan.head_tiles, p.splits = plan.splits, p.min_tiles = plan.min_tiles;
  p.lengths = lengths, p.scale_log2 = scale * 1.44269504088896341f, p.window = window;
  p.out = static_cast<__nv_bfloat16*>(out), p.lse = lse;
  const int64_t parts = static_cast<int64_t>(rows) * q_heads * plan.splits;
  if (plan.splits > 1) {
    if (workspace_bytes < parts * (dim * sizeof(float) + sizeof(float2))) return set_error("workspace too small"), DM3_ENOSPACE;
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256) return set_error("workspace must be 256-byte aligned"), DM3_EINVAL;
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + parts * dim);
  }
  const dim3 grid(plan.splits, kv_heads * plan.head_tiles, rows);
  cudaError_t err;
  switch (dim) {
    case 64: err = k_exp ? attn::attend<64, true>(p, grid, stream) : attn::attend<64, false>(p, grid, stream); break;
    case 128: err = k_exp ? attn::attend<128, true>(p, grid, stream) : attn::attend<128, false>(p, grid, stream); break;
    case 192: err = k_exp ? attn::attend<192, true>(p, grid, stream) : attn::attend<192, false>(p, grid, stream); break;
    default: err = k_exp ? attn::attend<256, true>(p, grid, stream) : attn::attend<256, false>(p, grid, stream); break;
  }
  if (err == cudaSuccess && plan.splits > 1)
    err = attn::start(attn::join_kernel, dim3(q_heads, rows), dim, stream, p, dim, k_exp ? attn::kLift : 0.f);
  if (err != cudaSuccess) return set_error(std::string("paged_attention launch: ") + cudaGetErrorString(err)), DM3_ECUDA;
  note_launches(plan.splits > 1 ? 2 : 1);
  return DM3_OK;
}
