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
#include <atomic>
#include <cmath>
#include <cstdint>
#include <string>

#include "dm3.h"
#include "dm3_common.cuh"
#include "dm3_internal.h"
#include "dm3_kv.cuh"
#include "dm3_tc.cuh"

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
  static constexpr int kRow = kDim * (kQuant ? 1 : 2);         // bytes of a cache row
  static constexpr int kKP = kRow / 64;                        // 16-byte copies of a key row a lane
  static constexpr int kVB = kQuant && kDim % 128 ? 8 : 16;    // bytes of one value copy a lane
  static constexpr int kVP = kRow / (8 * kVB), kVW = kVB / 4;  // copies a row, words a copy
  static constexpr int kE = kQuant ? kVB : kVB / 2;            // values a copy
  static constexpr int kHeads = 8 * kNT;
  // A tile arrives as boxes of kBox bytes x 16 tokens, swizzled: 16-byte chunk c of token t is at chunk
  // c ^ (t % 8) of its 128 bytes (c ^ (t / 2 % 4) of 64).
  static constexpr int kBox = kRow % 128 ? 64 : 128, kBoxes = kRow / kBox;
  static constexpr int kTileBytes = kTile * kRow;
  // Shared memory: a ring of kRing units a warp (a step's keys, its values, the next step's keys, ...), the
  // queries, the units' exponents, ranges and barriers, the join's maxima and sums. The join reuses the ring.
  static constexpr int kUnit = kU * kTileBytes;
  static constexpr int kQBytes = kNT * kDim * 16;  // 8 * kNT heads of kDim 16-bit values
  static constexpr int kSide = (kQuant ? kU * 32 : 0) + kU * 4 + 8 + 4;  // a unit's exponents, ranges and barrier
  static constexpr int kStats = (2 * kWarps + 1) * kHeads * 4;
  // Two CTAs an SM: few warps with much to do at once did better than more of them with smaller steps and fewer
  // registers (96 ragged rows, 16 heads a cache head, e4m3: 74.6 us; three CTAs and half the step 80.6, four 88.6)
  static constexpr int kRoom = 112 * 1024 - kQBytes - kStats - 1024;  // 1024: aligning the ring
  static constexpr int kFit = kRoom / kWarps / (kUnit + kSide), kRing = kFit < 6 ? kFit : 6;
  static constexpr int kPitch = 2 * kDim + 8;  // floats of a head pair in the join (8: no bank conflicts)
  static constexpr int kRingBytes = kWarps * kRing * kUnit;
  static constexpr int kShared = 1024 + kRingBytes + kQBytes + kWarps * kRing * kSide + kStats;
  static_assert(kRing >= 2 && kWarps * kNT * 4 * kPitch * 4 <= kRingBytes, "the ring holds two units and the join");
};
// The token that lane group lr's rows of a tile hold (and + 8): with it, the eight lanes of every 16-byte shared
// memory access, of keys (two lane groups, four chunks) as of values (two chunks, four tokens), fall on
// different chunks of 128-byte boxes.
template <int kBox>
__device__ __forceinline__ int token_of(int lr) {
  return kBox == 128 ? ((lr ^ lr >> 2) & 1) << 2 | (lr & 2) | lr >> 2 : lr;
}

template <int kDim, bool kQuant, int kNT, int kU>
__global__ void __launch_bounds__(kWarps * 32, 2)
    attend_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using C = Shape<kDim, kQuant, kNT, kU>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint4* const s_q = reinterpret_cast<uint4*>(smem + C::kRingBytes);  // [kNT][kDim / 32][32 lanes]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lr = lane >> 2, lc = lane & 3;
  uint8_t* side = smem + C::kRingBytes + C::kQBytes;
  uint8_t(*const s_exp)[kU][32] = reinterpret_cast<uint8_t(*)[kU][32]>(side) + (kQuant ? warp * C::kRing : 0);  // keys' 16, values' 16
  side += kQuant ? kWarps * C::kRing * kU * 32 : 0;
  uint64_t* const full = reinterpret_cast<uint64_t*>(side) + warp * C::kRing;
  side += kWarps * C::kRing * 8;
  int(*const s_range)[kU] = reinterpret_cast<int(*)[kU]>(side) + warp * C::kRing;  // rows of a tile that are seen: from | to << 8
  side += kWarps * C::kRing * kU * 4;
  float(*const s_m)[C::kHeads] = reinterpret_cast<float(*)[C::kHeads]>(side);
  float(*const s_l)[C::kHeads] = s_m + kWarps;
  float* const s_qs = s_m[2 * kWarps];
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < C::kRing; ++i) mbar_init(&full[i], kU);
    fence_mbar_init();
  }
  __syncwarp();

  const int split = blockIdx.x, kvh = blockIdx.y / p.head_tiles, ht = blockIdx.y % p.head_tiles, row = blockIdx.z;
  const int h0 = ht * C::kHeads;  // first head of the group
  griddep_launch();
  griddep_wait();
  fence_proxy_async();  // the cache's rows may have been written just before; the copies read them
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

  // A warp's steps: kU tiles each, warps in turn. Lane i of a block of 32 tiles knows where the block's tile i lies,
  // and asks for it.
  constexpr int kBlock = 32 / kU;  // steps a block
  int steps = static_cast<int>((end - begin - warp * kU + kWarps * kU - 1) / (kWarps * kU));  // 0 where fewer tiles than warps
  const int per_page = p.c.page_size / kTile;
  int page, y, range;  // y: first row of the tile in its page
  auto find = [&](int step0) {
    const int64_t t = begin + (static_cast<int64_t>(step0 + lane / kU) * kWarps + warp) * kU + lane % kU;
    int tile = 0;
    page = 0, range = 0;
    if (t < end) {
      const int64_t g = sp.tile0 + t, nth = g / per_page, t0 = g * kTile;
      tile = static_cast<int>(g - nth * per_page);
      page = p.c.table[row * p.c.table_stride + nth];
      if (page < 0 || page >= p.c.pages) {
        page = 0;
        kv::set_status(p.c.status, STATUS_BAD_PAGE);
      } else {
        range = (sp.first > t0 ? static_cast<int>(sp.first - t0) : 0) | (sp.n - t0 < kTile ? static_cast<int>(sp.n - t0) : kTile) << 8;
      }
    }
    y = kvh * p.c.page_size + tile * kTile;
  };
  find(0);

  uint8_t* const ring = smem + warp * C::kRing * C::kUnit;
  auto ask = [&](bool keys, int step, int slot) {
    if (step >= steps) return;
    if (keys && step % kBlock == 0 && step > 0) find(step);
    const int u = lane - (step % kBlock) * kU;
    if (u >= 0 && u < kU) {
      uint8_t* const to = ring + slot * C::kUnit + u * C::kTileBytes;
      s_range[slot][u] = range;
      mbar_arrive_expect_tx(&full[slot], C::kTileBytes + (kQuant && keys ? 32 : 0));
#pragma unroll
      for (int b = 0; b < C::kBoxes; ++b)
        tc::tma_load_3d(to + b * kTile * C::kBox, keys ? &kmap : &vmap, b * C::kBox, y, page, &full[slot]);
      if (kQuant && keys) {
        const int64_t x = page * p.c.exp_stride + y;
        bulk_g2s(s_exp[slot][u], p.c.k_exp + x, 16, &full[slot]);
        bulk_g2s(s_exp[slot][u] + 16, p.c.v_exp + x, 16, &full[slot]);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < C::kRing; ++i) ask(!(i & 1), i / 2, i);

  // Queries as B operands, in the permutation of dim that 16-byte key copies give; warp nt prepares tile nt.
  if (warp < kNT) {
    const int h = h0 + warp * 8 + lr;
    const __nv_bfloat16* src = p.q + row * p.q_rs + static_cast<int64_t>(kvh * p.group + h) * p.q_hs;
    uint4 w[kDim / 32];
#pragma unroll
    for (int j = 0; j < kDim / 32; ++j) {
      const int d = kQuant ? j / 2 * 64 + lc * 16 + j % 2 * 8 : j * 32 + lc * 8;
      w[j] = h < p.group ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0, 0, 0, 0);
    }
    float qs = p.scale_log2;  // logit scale of head h
    if (kQuant) {
      uint32_t top = 0;  // the largest magnitude's bits
      auto mag = [](uint32_t x) { return max(x << 16 & 0x7fffffffu, x & 0x7fff0000u); };
#pragma unroll
      for (int j = 0; j < kDim / 32; ++j) top = max(top, max(max(mag(w[j].x), mag(w[j].y)), max(mag(w[j].z), mag(w[j].w))));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = min(max(static_cast<int>(top >> 23) - 127, -112), 126) - 14;  // 2^-e puts the largest in [2^14, 2^15)
      const float up = exp2i(-e);
      auto half = [up](uint32_t x) { return pack_half(__uint_as_float(x << 16) * up, __uint_as_float(x & 0xffff0000u) * up); };
#pragma unroll
      for (int j = 0; j < kDim / 32; ++j) w[j] = make_uint4(half(w[j].x), half(w[j].y), half(w[j].z), half(w[j].w));
      qs *= exp2i(e);
    }
#pragma unroll
    for (int j = 0; j < kDim / 32; ++j) s_q[(warp * (kDim / 32) + j) * 32 + lane] = w[j];
    if (lc == 0) s_qs[warp * 8 + lr] = qs;
  }
  __syncthreads();

  float o[kNT][kDim / 16][4];
  // Of the lane's two heads a tile: the maximum m (the same in all lanes of a head), what is subtracted (m, or 0
  // before any logit was seen, less the lift), and a lane's part of l.
  float m[kNT][2], sub[kNT][2], l[kNT][2], qs[kNT][2];
#pragma unroll
  for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
    for (int i = 0; i < kDim / 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[nt][i][j] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) m[nt][h] = -INFINITY, sub[nt][h] = 0.f, l[nt][h] = 0.f, qs[nt][h] = s_qs[nt * 8 + 2 * lc + h];
  }

  const int tok = token_of<C::kBox>(lr), sw = C::kBox == 128 ? tok : tok >> 1;  // the lane's token of a key tile, its swizzle
  int vtok[2];                                                                    // its tokens of a value tile (and + 8)
#pragma unroll
  for (int i = 0; i < 2; ++i) vtok[i] = token_of<C::kBox>(2 * lc + i);
  int slot = 0;
  uint32_t parity = 0;
  // The unit in the current slot has landed; when the wait ran out, no more are asked for.
  auto landed = [&](int step) {
    if (__any_sync(0xffffffffu, !mbar_wait(&full[slot], parity))) {
      if (lane == 0) kv::set_status(p.c.status, STATUS_TIMEOUT);
      steps = min(steps, step + (C::kRing + 1) / 2);
    }
  };
  auto next_slot = [&] {
    if (++slot == C::kRing) slot = 0, parity ^= 1;
  };
  for (int step = 0; step < steps; ++step) {
    landed(step);
    const uint8_t* unit = ring + slot * C::kUnit;
    // a product takes the sum of the one before 25 cycles later: two sums side by side where a step has but one tile
    constexpr int kChains = kU * kNT == 1 ? 2 : 1;
    float s[kU][kNT][4], part[kChains][kU][kNT][4];
#pragma unroll
    for (int i = 0; i < kChains; ++i)
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[i][u][nt][j] = 0.f;
    auto key = [&](int u, int half, int j) {
      constexpr int kIn = C::kBox / 64;  // passes a box
      return *reinterpret_cast<const uint4*>(unit + u * C::kTileBytes + (j / kIn * kTile + tok + half * 8) * C::kBox +
                                             (((j % kIn) * 4 + lc) ^ (C::kBox == 128 ? sw : sw & 3)) * 16);
    };
#pragma unroll
    for (int j = 0; j < C::kKP; ++j) {
      if (!kQuant) {
        uint4 w[kNT];
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) w[nt] = s_q[(nt * (kDim / 32) + j) * 32 + lane];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const uint4 a = key(u, 0, j), b = key(u, 1, j);
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) {
            mma<false>(part[0][u][nt], a.x, b.x, a.y, b.y, w[nt].x, w[nt].y);
            mma<false>(part[kChains - 1][u][nt], a.z, b.z, a.w, b.w, w[nt].z, w[nt].w);
          }
        }
      } else {
        uint4 w[kNT][2];
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) w[nt][i] = s_q[(nt * (kDim / 32) + 2 * j + i) * 32 + lane];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const uint4 x = key(u, 0, j), y = key(u, 1, j);
          const uint32_t a[4] = {x.x, x.y, x.z, x.w}, b[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x0 = half_pair(a[i]), x1 = half_pair(b[i]), x2 = half_pair_hi(a[i]), x3 = half_pair_hi(b[i]);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
              mma<true>(part[i % kChains][u][nt], x0, x1, x2, x3, i & 1 ? w[nt][i / 2].z : w[nt][i / 2].x,
                        i & 1 ? w[nt][i / 2].w : w[nt][i / 2].y);
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[u][nt][j] = part[0][u][nt][j];
#pragma unroll
          for (int i = 1; i < kChains; ++i) s[u][nt][j] += part[i][u][nt][j];
        }
    // logits in log2 units (with the value rows' exponents), -inf where nothing is seen
    float back[kU][2];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      float kf[2], vf[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int8_t* x = reinterpret_cast<const int8_t*>(&s_exp[slot][u][r * 8 + tok]);
        kf[r] = kQuant ? exp2i(x[0]) : 1.f;
        vf[r] = kQuant ? __uint_as_float(0x4b400000u + x[16]) - 12582912.f : 0.f;  // the exponent as a float, off the conversion pipe
        back[u][r] = kQuant ? exp2i(-max(static_cast<int>(x[16]), -126)) : 1.f;  // finite in places not seen, too
      }
      const int seen = s_range[slot][u];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float z = s[u][nt][j] * qs[nt][j & 1];
          if (kQuant) z = z * kf[j >> 1] + vf[j >> 1];
          s[u][nt][j] = z;
        }
      if (seen != kTile << 8)
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = tok + (j >> 1) * 8;
            if (r < (seen & 255) || r >= seen >> 8) s[u][nt][j] = -INFINITY;
          }
    }
    __syncwarp();  // the unit is read
    ask(!(C::kRing & 1), step + C::kRing / 2, slot);
    next_slot();

    bool above = false;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x = fmaxf(s[0][nt][h], s[0][nt][2 + h]);
#pragma unroll
        for (int u = 1; u < kU; ++u) x = fmaxf(x, fmaxf(s[u][nt][h], s[u][nt][2 + h]));
        above |= x > m[nt][h] + kSlack;
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
          sub[nt][h] = (x == -INFINITY ? 0.f : x) - (kQuant ? kLift : 0.f);
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
          w[j] = ex2(s[u][nt][j] - sub[nt][j & 1]);
          l[nt][j & 1] += kQuant ? w[j] * back[u][j >> 1] : w[j];
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

    landed(step);
    unit = ring + slot * C::kUnit;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int seen = s_range[slot][u];
#pragma unroll
      for (int j = 0; j < C::kVP; ++j) {
        uint32_t v[4][C::kVW];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = vtok[i & 1], key = C::kBox == 128 ? t : t >> 1 & 3;
          const uint8_t* src = unit + u * C::kTileBytes + (j * kTile + t + (i >> 1) * 8) * C::kBox;
          if constexpr (C::kVB == 16) {
            const uint4 w = *reinterpret_cast<const uint4*>(src + (lr ^ key) * 16);
            v[i][0] = w.x, v[i][1] = w.y, v[i][2] = w.z, v[i][3] = w.w;
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(src + (lr * 8 ^ key * 16));
            v[i][0] = w.x, v[i][1] = w.y;
          }
        }
        // what lies in places not seen may be anything, and no weight of zero makes a NaN harmless
        if (seen != kTile << 8)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = vtok[i & 1] + (i >> 1) * 8;
            if (r < (seen & 255) || r >= seen >> 8)
#pragma unroll
              for (int w = 0; w < C::kVW; ++w) v[i][w] = 0;
          }
#pragma unroll
        for (int w = 0; w < C::kVW; ++w) {
          const uint32_t t0 = v[0][w], t1 = v[1][w], t8 = v[2][w], t9 = v[3][w];
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
            const uint32_t a0 = half_pair(x0), a1 = half_pair_hi(x0), a2 = half_pair(y0), a3 = half_pair_hi(y0);
            const uint32_t b0 = half_pair(x1), b1 = half_pair_hi(x1), b2 = half_pair(y1), b3 = half_pair_hi(y1);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) {
              mma<true>(o[nt][tile], a0, a1, a2, a3, ph[u][nt][0], ph[u][nt][1]);
              mma<true>(o[nt][tile + 1], b0, b1, b2, b3, ph[u][nt][0], ph[u][nt][1]);
            }
          }
        }
      }
    }
    __syncwarp();  // the unit is read
    ask(C::kRing & 1, step + (C::kRing + 1) / 2, slot);
    next_slot();
  }

  // join the warps; the ring's place is free once every warp is here (it has waited for all that it asked for)
  float(*s_o)[kNT * 4][C::kPitch] = reinterpret_cast<float(*)[kNT * 4][C::kPitch]>(smem);
#pragma unroll
  for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int w = 4; w < 32; w *= 2) l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], w);
      if (lr == 0) s_m[warp][nt * 8 + 2 * lc + h] = m[nt][h], s_l[warp][nt * 8 + 2 * lc + h] = l[nt][h];
    }
  __syncthreads();
  const bool whole = sp.tiles <= sp.chunk;
  if (threadIdx.x < C::kHeads) {  // each warp's factor into s_m, 1 / sum (or 1) into s_qs
    const int h = threadIdx.x;
    float mm = -INFINITY, ll = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][h]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = s_m[w][h] == -INFINITY ? 0.f : ex2(s_m[w][h] - mm);
      ll += s_l[w][h] * f;
      s_m[w][h] = f;
    }
    s_qs[h] = whole ? (ll == 0.f ? 0.f : 1.f / ll) : 1.f;
    if (h0 + h < p.group) {
      if (whole)
        p.lse[qrow + h] = ll == 0.f ? -INFINITY : (mm - (kQuant ? kLift : 0.f) + log2f(ll)) * 0.69314718055994531f;
      else
        p.part_ml[(qrow + h) * p.splits + split] = make_float2(mm, ll);
    }
  }
  // (value d of both heads of a pair) at d with its low bits turned by lr, so that neither these writes (lanes kE
  // values apart) nor the reads (neighbours) meet on a bank
#pragma unroll
  for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
    for (int i = 0; i < kDim / 16; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int d = i / (C::kE / 2) * 8 * C::kE + lr * C::kE + i % (C::kE / 2) * 2 + r;
        *reinterpret_cast<float2*>(&s_o[warp][nt * 4 + lc][(d ^ (lr & 3)) * 2]) = make_float2(o[nt][i][2 * r], o[nt][i][2 * r + 1]);
      }
  __syncthreads();
  for (int i = threadIdx.x; i < C::kHeads / 2 * kDim; i += blockDim.x) {
    const int hp = i / kDim, d = i % kDim, h = 2 * hp;
    if (h0 + h >= p.group) break;
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 v = *reinterpret_cast<const float2*>(&s_o[w][hp][(d ^ (d / C::kE & 3)) * 2]);
      const float2 f = *reinterpret_cast<const float2*>(&s_m[w][h]);
      x += v.x * f.x, y += v.y * f.y;
    }
    x *= s_qs[h], y *= s_qs[h + 1];
    const bool both = h0 + h + 1 < p.group;
    if (whole) {
      p.out[(qrow + h) * kDim + d] = __float2bfloat16_rn(x);
      if (both) p.out[(qrow + h + 1) * kDim + d] = __float2bfloat16_rn(y);
    } else {
      float* to = p.part_o + ((qrow + h) * p.splits + split) * kDim + d;
      to[0] = x;
      if (both) to[static_cast<int64_t>(p.splits) * kDim] = y;
    }
  }
}

// Joins the splits. 16 lanes hold 64 values of one query head (4 each); `groups` of them take its splits in turn,
// each with a running maximum of its own, and meet in shared memory: 16 / groups pieces of 64 values a CTA.
constexpr int kJoinThreads = 256, kJoinBatch = 4;
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ Params p, int dim, int groups, float lift) {
  __shared__ float s_m[kJoinThreads / 16], s_l[kJoinThreads / 16];
  __shared__ float4 s_x[kJoinThreads / 16][16];
  griddep_launch();
  griddep_wait();
  const int team = threadIdx.x / 16, c = threadIdx.x % 16, g = team % groups, pieces = dim / 64;
  const int64_t piece = static_cast<int64_t>(blockIdx.x) * (16 / groups) + team / groups, head = piece / pieces;
  const int64_t row = head / p.q_heads;
  bool on = row < p.c.rows;
  int n = 0;
  if (on) {
    const Span sp = row_span(p, static_cast<int>(row));
    on = sp.tiles > sp.chunk;  // else written whole, or nothing to see
    if (on) n = static_cast<int>((sp.tiles + sp.chunk - 1) / sp.chunk);
  }
  const int at = static_cast<int>(piece % pieces) * 16 + c;  // of the head's float4s
  const float2* ml = p.part_ml + head * p.splits;
  const float4* po = reinterpret_cast<const float4*>(p.part_o + head * p.splits * dim) + at;
  float m = -INFINITY, l = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = g; i0 < n; i0 += groups * kJoinBatch) {
    float2 a[kJoinBatch];
    float4 y[kJoinBatch];
#pragma unroll
    for (int b = 0; b < kJoinBatch; ++b) {
      const int i = i0 + b * groups;
      a[b] = i < n ? ml[i] : make_float2(-INFINITY, 0.f);
      y[b] = i < n ? po[static_cast<int64_t>(i) * (dim / 4)] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float mm = m;
#pragma unroll
    for (int b = 0; b < kJoinBatch; ++b) mm = fmaxf(mm, a[b].x);
    const float back = m == -INFINITY ? 0.f : ex2(m - mm);
    l *= back, x.x *= back, x.y *= back, x.z *= back, x.w *= back;
#pragma unroll
    for (int b = 0; b < kJoinBatch; ++b) {
      const float f = a[b].x == -INFINITY ? 0.f : ex2(a[b].x - mm);
      l += a[b].y * f;
      x.x += y[b].x * f, x.y += y[b].y * f, x.z += y[b].z * f, x.w += y[b].w * f;
    }
    m = mm;
  }
  if (groups > 1) {
    if (c == 0) s_m[team] = m, s_l[team] = l;
    s_x[team][c] = x;
    __syncthreads();
    if (g) return;
    float mm = m;
    for (int i = 1; i < groups; ++i) mm = fmaxf(mm, s_m[team + i]);
    const float f0 = m == -INFINITY ? 0.f : ex2(m - mm);
    l *= f0, x.x *= f0, x.y *= f0, x.z *= f0, x.w *= f0;
    for (int i = 1; i < groups; ++i) {
      const float f = s_m[team + i] == -INFINITY ? 0.f : ex2(s_m[team + i] - mm);
      const float4 y = s_x[team + i][c];
      l += s_l[team + i] * f;
      x.x += y.x * f, x.y += y.y * f, x.z += y.z * f, x.w += y.w * f;
    }
    m = mm;
  }
  if (!on) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(p.out + head * dim + at * 4) = make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
  if (at == 0) p.lse[head] = l == 0.f ? -INFINITY : (m - lift + log2f(l)) * 0.69314718055994531f;
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

static int tile_heads(int group) { return group > 8 ? 16 : 8; }

static Plan plan(int rows, int q_heads, int kv_heads, int dim, bool quant, int64_t tiles) {
  Plan r;
  const int group = q_heads / kv_heads, heads = tile_heads(group);
  r.head_tiles = (group + heads - 1) / heads;
  const int64_t units = static_cast<int64_t>(rows) * kv_heads * r.head_tiles;
  r.min_tiles = kWarps;
  int64_t s = (static_cast<int64_t>(sms()) * 4 + units - 1) / units;
  const int64_t most = (tiles + r.min_tiles - 1) / r.min_tiles;
  if (s > most) s = most;
  if (s > 65535) s = 65535;
  r.splits = static_cast<int>(s < 1 ? 1 : s);
  return r;
}

template <typename... A>
static cudaError_t start(void (*kernel)(A...), dim3 grid, int threads, int shared, void* stream, A... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int kDim, bool kQuant, int kNT, int kU>
static int attend(const Params& p, dim3 grid, void* stream) {
  using C = Shape<kDim, kQuant, kNT, kU>;
  CUtensorMap maps[2];
  for (int i = 0; i < 2; ++i)
    if (!tensor_map_boxes(&maps[i], i ? p.c.v : p.c.k, C::kRow, static_cast<uint64_t>(p.kv_heads) * p.c.page_size, p.c.pages,
                          static_cast<uint64_t>(p.c.page_stride) * (kQuant ? 1 : 2), C::kBox, kTile))
      return DM3_EINVAL;
  // once a device (a second thread setting it again does no harm)
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    const cudaError_t err = cudaFuncSetAttribute(attend_kernel<kDim, kQuant, kNT, kU>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kShared);
    if (err != cudaSuccess) return set_error(std::string("paged_attention: ") + cudaGetErrorString(err)), DM3_ECUDA;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  const cudaError_t err = start(attend_kernel<kDim, kQuant, kNT, kU>, grid, kWarps * 32, C::kShared, stream, p, maps[0], maps[1]);
  if (err != cudaSuccess) return set_error(std::string("paged_attention launch: ") + cudaGetErrorString(err)), DM3_ECUDA;
  return DM3_OK;
}

template <int kDim, bool kQuant>
static int attend(const Params& p, dim3 grid, void* stream) {
  // token tiles a step: 8 KB of keys, one unit of the ring (6 KB for 384-byte rows)
  constexpr int kRow = kDim * (kQuant ? 1 : 2), kU = kRow <= 64 ? 8 : kRow <= 128 ? 4 : kRow <= 256 ? 2 : 1;
  return tile_heads(p.group) == 16 ? attend<kDim, kQuant, 2, kU>(p, grid, stream) : attend<kDim, kQuant, 1, kU>(p, grid, stream);
}

}  // namespace attn
}  // namespace dm3

int dm3::wait_limit_attention(uint64_t ns) { return static_cast<int>(set_wait_limit_here(ns)); }

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
  int rc;
  switch (dim) {
    case 64: rc = k_exp ? attn::attend<64, true>(p, grid, stream) : attn::attend<64, false>(p, grid, stream); break;
    case 128: rc = k_exp ? attn::attend<128, true>(p, grid, stream) : attn::attend<128, false>(p, grid, stream); break;
    case 192: rc = k_exp ? attn::attend<192, true>(p, grid, stream) : attn::attend<192, false>(p, grid, stream); break;
    default: rc = k_exp ? attn::attend<256, true>(p, grid, stream) : attn::attend<256, false>(p, grid, stream); break;
  }
  if (rc) return rc;
  if (plan.splits > 1) {
    const int groups = plan.splits <= 4 ? 1 : plan.splits <= 24 ? 4 : 16;  // teams that share a head's splits
    const int64_t pieces = static_cast<int64_t>(rows) * q_heads * (dim / 64);
    const cudaError_t err = attn::start(attn::join_kernel, dim3(static_cast<unsigned>((pieces * groups + 15) / 16)), attn::kJoinThreads, 0,
                                        stream, p, dim, groups, k_exp ? attn::kLift : 0.f);
    if (err != cudaSuccess) return set_error(std::string("paged_attention launch: ") + cudaGetErrorString(err)), DM3_ECUDA;
  }
  note_launches(plan.splits > 1 ? 2 : 1);
  return DM3_OK;
}
