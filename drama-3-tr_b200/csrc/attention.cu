// One new token's attention over the paged key-value cache (sm_100a).
//
//   s_t = scale * q . k_t,  p = softmax(s) over the tokens seen,  out = sum_t p_t v_t,
//   lse = log sum_t exp(s_t),  seen: max(0, n - window) <= t < n (window 0: all), n the row's length
//
// One pass with a running maximum M and sum l; a row that sees nothing gives zeros and lse = -inf. A logit of -inf is a token
// that is not seen (its weight is 0); one of +inf or NaN makes l, and with it out and lse, NaN.
//
// Bound: the bytes of the cache's rows, each used by the group of query heads that shares them (2 * group flops a byte
// and less), so the kernel is laid out to keep copies in flight and to spend few instructions a row, not for the
// tensor peak: the products are warp-level m16n8k16 tiles with tokens as the 16 rows and query heads as the 8 columns
// (heads as rows would waste half of the tile and of the registers for groups of up to 8):
//   S^T = K Q^T:  a lane's 16 bytes of a key row hold the k-columns of 2 (bf16) or 4 (e4m3) tiles once the same
//                 permutation of dim is applied to Q;
//   O^T = V^T P^T: a lane takes 16 bytes of 4 tokens' value rows and interleaves pairs of tokens with byte permutes; P^T
//                 comes from S^T's accumulators by an 8x8 transpose (movmatrix).
// Every warp walks 16-token tiles of its own: TMA brings a step's keys and values, swizzled, into a ring of shared memory
// that belongs to the warp, so warps never wait for one another until the join at the end. (Loads straight into
// registers kept too little in flight, 82% of the copy bandwidth where this has all of it, 64 ragged rows of a bf16 cache;
// cp.async in their place doubled the traffic through L1 and was slower still. FP8 tensor instructions for the keys' product,
// with the queries as two e4m3 parts, took a quarter longer than converting the keys to fp16.)
//
// A unit is a row and up to 16 of the query heads that share a cache head. Units are split over CTAs by the lengths that the
// device reads, so one captured graph serves all lengths, in one of two ways (plan() says when); neither uses atomics,
// and the order of every sum is fixed by the lengths and sizes alone.
//   * Clusters: the `splits` CTAs of a cluster (1 to 8) share a unit's tiles and join over distributed shared memory: one
//     launch, for short rows.
//   * Stream: the tiles of all rows and heads are one sequence, cut into equal shares for two CTAs an SM whatever the
//     rows' lengths; a CTA leaves (M, l, R, O) in fp32 of a unit that it shares, and a second kernel joins them.
//
// An e4m3 row is code * 2^e. For keys 2^e joins the logit's scale. For values it joins the weight's exponent:
// w_t = 2^(s_t + e_t - M) with M the running maximum of s_t + e_t, so weights are in fp16's range whatever the rows'
// sizes, and l sums w_t * 2^-e_t. Codes are exact in fp16; queries are scaled by a power of two to
// [2^14, 2^15), where fp16 holds a bf16 row to 2^-39 of its largest value; a weight is rounded once to 11 bits, 2^-11 of
// it (1/8 of what rounding the output to bf16 costs), or, under 2^-20 of the row's largest weight, to 2^-31 of that one. With
// a bf16 cache a weight goes to the tensor cores as a bf16 pair, high and low part: 16 bits.
// s_t + e_t is held in 32 bits: where exponents lie over 64 lse is off by up to 2^-17 for it.
//
// l in terms of M can be anything from 2^-113 (one token at exponent 119) to 2^155 (2^31 tokens at -110, all just under the
// slack), more than 32 bits hold. So a warp sums w_t * 2^(e - e_t), e the exponent of the first row that it sees, while no other is
// more than 44 from it: then no term is over 2^58, and that of the largest logit not under 2^-38. From the first row that is,
// it sums 2^(s_t + e_t - M) * 2^-e_t, formed from the logit, in 64 bits in shared memory, at a price that only such rows pay.
// Warps, CTAs and parts are joined with a reference R of their sums beside M: sum exp = l 2^R, out = O 2^M / (l 2^R).
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
constexpr int kMaxCluster = 8;
constexpr int kTile = 16;  // tokens of one tile; pages hold whole tiles
// The maximum is raised only when a logit exceeds it by more than kSlack (log2): weights reach 2^kSlack. fp16
// weights carry 2^kLift besides, so that they stay normal down to 2^-(14 + kLift).
constexpr float kSlack = 8.f, kLift = 6.f;
// The exponents that a warp's 32-bit sum takes: within kNear of the first one's.
constexpr int kNear = 44;
struct Part {  // what a CTA leaves of a shared unit's head: maximum, sum and its reference
  float m, l, r, none;
};

struct Params {
  const __nv_bfloat16* q;  // [rows][q_heads][dim]
  int64_t q_rs, q_hs;
  int q_heads, kv_heads, group, head_tiles;
  Cache c;
  const int64_t* lengths;
  float scale_log2;  // scale * log2(e)
  int64_t window;
  int splits;          // CTAs of a cluster; 0: stream
  bool longest_first;  // one CTA a unit: blockIdx.z counts the rows by their tiles
  int hasty;           // the wait limit is below kHasty: what has not landed when it is needed has run out
  __nv_bfloat16* out;  // [rows][q_heads][dim]
  float* lse;          // [rows][q_heads]
  // stream: the first tile of each row in the sequence and their number ([rows + 1], a tile counted once a head unit),
  // and what a CTA leaves of the row that it starts in ([2 * cta]) and of the one that it ends in ([2 * cta + 1])
  int64_t* row_at;
  float* part_o;  // [2 * ctas][heads of a unit][dim]
  Part* part_ml;  // [2 * ctas][heads of a unit]
};

// The tokens and tiles that a row sees.
struct Span {
  int64_t first, n;  // tokens seen: [first, n)
  int64_t tile0;     // tile of the first one
  int64_t tiles;
  bool cut;  // the length lies behind the table
};
__device__ __forceinline__ Span row_span(const Params& p, int64_t row) {
  Span s;
  const int64_t cap = static_cast<int64_t>(p.c.per_row) * p.c.page_size;
  s.n = p.lengths[row];
  s.cut = s.n > cap;
  if (s.n > cap) s.n = cap;
  if (s.n < 0) s.n = 0;
  s.first = p.window > 0 && s.n > p.window ? s.n - p.window : 0;
  s.tile0 = s.first / kTile;
  s.tiles = (s.n + kTile - 1) / kTile - s.tile0;
  return s;
}
// Quotients of what hardly ever needs 64 bits
__device__ __forceinline__ int64_t div(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}
// Tiles of a CTA's share of the sequence: equal ones, but a tile for each warp, or a whole unit where units are shorter.
__device__ __forceinline__ int64_t share_of(int64_t tiles, int rows, int units, int ctas) {
  const int64_t q = div(tiles * units + ctas - 1, ctas), unit = div(tiles, rows), least = unit < 1 ? 1 : unit < kWarps ? unit : kWarps;
  return q < least ? least : q;
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
__device__ __forceinline__ float ex2_all(float x) {  // results below 2^-126 kept
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
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
  // queries, the units' exponents, ranges and barriers, the join's maxima, sums and factors. The join reuses the ring.
  static constexpr int kUnit = kU * kTileBytes;
  static constexpr int kQBytes = kNT * kDim * 16;  // 8 * kNT heads of kDim 16-bit values
  static constexpr int kSide = (kQuant ? kU * 32 : 0) + kU * 4 + 8 + 4;  // a unit's exponents, ranges and barrier
  static constexpr int kStats = (3 * kWarps + 1 + kMaxCluster) * kHeads * 4;
  // Two CTAs an SM: few warps with much to do at once did better than more of them with smaller steps and fewer
  // registers (96 ragged rows, 16 heads a cache head, e4m3: 74.6 us; three CTAs and half the step 80.6, four 88.6, all
  // three before sums held for every exponent; 77.0 now). The two CTAs' 255 registers are not enough for 16 heads of 256
  // (12 bytes spilled with a bf16 cache, 104 with an e4m3 one).
  static constexpr int kRoom = 112 * 1024 - kQBytes - kStats - 1024;  // 1024: aligning the ring
  static constexpr int kFit = kRoom / kWarps / (kUnit + kSide), kRing = kFit < 6 ? kFit : 6;
  static constexpr int kPitch = 2 * kDim + 8;  // floats of a head pair in the join (8: no bank conflicts)
  static constexpr int kRingBytes = kWarps * kRing * kUnit;
  static constexpr int kShared = 1024 + kRingBytes + kQBytes + kWarps * kRing * kSide + kStats;
  static_assert(kRing >= 2 && kWarps * kNT * 4 * kPitch * 4 <= kRingBytes, "the ring holds two units and the join");
  static_assert(kStats >= 129 * 4, "room for row_by_length");
};
// The token that lane group lr's rows of a tile hold (and + 8): with it, the eight lanes of every 16-byte shared
// memory access, of keys (two lane groups, four chunks) as of values (two chunks, four tokens), fall on
// different chunks of 128-byte boxes.
template <int kBox>
__device__ __forceinline__ int token_of(int lr) {
  return kBox == 128 ? ((lr ^ lr >> 2) & 1) << 2 | (lr & 2) | lr >> 2 : lr;
}

// l with its reference raised from `from` to `to`: l * 2^(from - to), where the power alone may vanish: those of e4m3 rows
// can lie 229 further apart than the logits. Before any logit l is 0, or NaN where all of them were.
__device__ __forceinline__ float raise_sum(float l, float from, float to) {
  const float h = from == -INFINITY ? 1.f : ex2(0.5f * (from - to));
  return l * h * h;
}
__device__ __forceinline__ double raise_sum(double l, float from, float to) {
  const float h = from == -INFINITY ? 1.f : ex2(0.25f * (from - to));
  const double hh = static_cast<double>(h) * h;
  return l * hh * hh;
}
__device__ __forceinline__ double exp2d(int e) { return __hiloint2double((1023 + e) << 20, 0); }
__device__ __forceinline__ float lse_of(float r, float l) {  // natural log of the sum, from log2 units
  return l == 0.f ? -INFINITY : (r + log2f(l)) * 0.69314718055994531f;
}
// What turns O into out, in two factors that stay in range where their product may not (2^-155 for 2^31 tokens at -110).
__device__ __forceinline__ float2 scale_of(float m, float r, float l, bool quant) {
  if (l == 0.f) return make_float2(0.f, 0.f);
  const float h = quant ? ex2(0.5f * (m - kLift - r)) : 1.f;
  return make_float2(1.f / l * h, h);
}

__device__ __forceinline__ bool elect_one() {  // true in one lane of the warp
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_cta(const void* p, int rank) {  // the place of p in another CTA of the cluster
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster(const float* p, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(in_cta(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(const void* p, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(in_cta(p, rank)) : "memory");
  return v;
}

template <typename T>
__device__ __forceinline__ T lane_sum(T x) {  // over the lanes of a head
#pragma unroll
  for (int w = 4; w < 32; w *= 2) x += __shfl_xor_sync(0xffffffffu, x, w);
  return x;
}
// The sums of a warp whose value rows' exponents lie far apart (kNear), a head's in its place of `sums`, referring to the
// maximum in its place of `refers`: begun with what the lanes hold, and a step's logits (with exponents, s) added. Out of the
// kernel's body, where the few calls that come here would cost every other one instructions to fetch (48 ragged e4m3 rows, 12
// heads of 192 a cache head: 46.9 us inlined, 45.9 so).
struct WideSums {
  double* sums;
  float* refers;
};
template <int kNT>
__device__ __noinline__ void begin_wide(WideSums to, const float (*l)[2], const float (*m)[2], int e) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 2 * kNT; ++i) {
    const float t = lane_sum(l[i / 2][i % 2]);
    const int head = i / 2 * 8 + 2 * (lane & 3) + i % 2;
    if (lane < 4) to.sums[head] = t * exp2d(-e), to.refers[head] = m[i / 2][i % 2];
  }
}
template <int kU, int kNT>
__device__ __noinline__ void add_wide(WideSums to, const float (*s)[kNT][4], const int (*ev)[2], const float (*m)[2], const float (*sub)[2]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 2 * kNT; ++i) {
    const int nt = i / 2, h = i % 2, head = nt * 8 + 2 * (lane & 3) + h;
    float t = 0.f;  // times 2^-4: up to 128 terms of 2^124; the largest logit's, 2^-113 at least, keeps 32 bits under it
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int r = 0; r < 2; ++r) t += ex2_all(s[u][nt][2 * r + h] - sub[nt][h] - static_cast<float>(ev[u][r] + 4));
    t = lane_sum(t);
    if (lane < 4) to.sums[head] = raise_sum(to.sums[head], to.refers[head], m[nt][h]) + 16. * t, to.refers[head] = m[nt][h];
  }
}

// The row with the nth most tiles, of 128 rows at most (the nth one where all are short). All threads call it; scratch: 129
// words, 16-byte aligned.
__device__ __forceinline__ int64_t row_by_length(const Params& p, int nth, int* scratch) {
  constexpr int kShort = 24;
  const int t = threadIdx.x, tiles = t < p.c.rows ? static_cast<int>(min(row_span(p, t).tiles, int64_t(1) << 23)) : 0;
  const int mine = t < p.c.rows ? tiles * (kWarps * 32) + kWarps * 32 - 1 - t : -1;  // tiles, then the lower row: no two alike
  scratch[t] = mine;
  if (!__syncthreads_or(tiles > kShort)) return nth;
  int before = 0;
  for (int j = 0; j < p.c.rows; j += 4) {
    const int4 x = *reinterpret_cast<const int4*>(scratch + j);
    before += (x.x > mine) + (x.y > mine) + (x.z > mine) + (x.w > mine);
  }
  if (t < p.c.rows && before == nth) scratch[kWarps * 32] = t;
  __syncthreads();
  const int64_t row = scratch[kWarps * 32];
  __syncthreads();  // the scratch is free
  return row;
}

// Stream: counts the rows' tiles and finds where this CTA's share of the sequence begins; CTA 0 leaves the rows' places for
// the join. All threads call it; scratch: 11 words. False when the CTA has no share.
__device__ __forceinline__ bool find_share(const Params& p, int units, int64_t* scratch, int64_t& row, int& unit, int64_t& begin,
                                           int64_t& left) {
  constexpr int kThreads = kWarps * 32;
  if (p.c.rows <= 32) {  // every warp by itself, a lane a row
    const int lane = threadIdx.x & 31;
    const int64_t mine = lane < p.c.rows ? row_span(p, lane).tiles : 0;
    int64_t upto = mine;
#pragma unroll
    for (int w = 1; w < 32; w *= 2) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, w);
      if (lane >= w) upto += x;
    }
    const int64_t total = __shfl_sync(0xffffffffu, upto, 31);
    if (blockIdx.x == 0 && threadIdx.x <= p.c.rows) p.row_at[threadIdx.x] = threadIdx.x < p.c.rows ? upto - mine : total;
    const int64_t share = share_of(total, p.c.rows, units, gridDim.x), from = blockIdx.x * share;
    if (from >= total * units) return false;
    left = min(share, total * units - from);
    const int hit = __ffs(__ballot_sync(0xffffffffu, mine > 0 && from < upto * units)) - 1;  // the first row that ends behind it
    const int64_t tiles = __shfl_sync(0xffffffffu, mine, hit), in = from - (__shfl_sync(0xffffffffu, upto, hit) - tiles) * units;
    row = hit;
    unit = static_cast<int>(div(in, tiles));
    begin = in - unit * tiles;
    return true;
  }
  int64_t *const s_sum = scratch, *const s_hit = scratch + kWarps;  // s_hit: the row found, its place, its tiles
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rows = p.c.rows;
  int64_t total = 0, mine = 0, upto = 0;  // this thread's row of a block of 128: its tiles, and the sum up to it
  if (threadIdx.x == 0) s_hit[0] = -1;
  auto scan = [&](int r0) {
    mine = r0 + static_cast<int>(threadIdx.x) < rows ? row_span(p, r0 + threadIdx.x).tiles : 0;
    upto = mine;
#pragma unroll
    for (int w = 1; w < 32; w *= 2) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, w);
      if (lane >= w) upto += x;
    }
    __syncthreads();
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    upto += total;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) upto += s_sum[w];
      total += s_sum[w];
    }
  };
  for (int r0 = 0; r0 < rows; r0 += kThreads) {
    scan(r0);
    if (blockIdx.x == 0 && r0 + threadIdx.x < rows) p.row_at[r0 + threadIdx.x] = upto - mine;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.row_at[rows] = total;
  const int64_t share = share_of(total, rows, units, gridDim.x), from = blockIdx.x * share;
  if (from >= total * units) return false;
  left = min(share, total * units - from);
  if (rows > kThreads) total = 0;  // block by block again, up to the one that holds `from`
  for (int r0 = 0; r0 < rows; r0 += kThreads) {
    if (rows > kThreads) scan(r0);
    const int64_t at = (upto - mine) * units;
    if (mine > 0 && from >= at && from < upto * units) s_hit[0] = r0 + threadIdx.x, s_hit[1] = at, s_hit[2] = mine;
    if (from < total * units) break;
  }
  __syncthreads();
  row = s_hit[0];
  if (row < 0) return false;
  const int64_t in = from - s_hit[1];
  unit = static_cast<int>(div(in, s_hit[2]));
  begin = in - unit * s_hit[2];
  __syncthreads();  // the scratch is free
  return true;
}

// Stream, once a CTA's share is done: CTAs take the rows in turn to write what one without tokens gives, and to report
// lengths behind the table.
template <int kDim>
__device__ __forceinline__ void tend_rows(const Params& p) {
  for (int64_t row = blockIdx.x; row < p.c.rows; row += gridDim.x) {
    const Span sp = row_span(p, row);
    if (sp.cut && threadIdx.x == 0) kv::set_status(p.c.status, STATUS_BAD_PAGE);
    if (sp.tiles) continue;
    const int64_t at = row * p.q_heads;
    for (int i = threadIdx.x; i < p.q_heads * kDim; i += blockDim.x) p.out[at * kDim + i] = __float2bfloat16_rn(0.f);
    for (int i = threadIdx.x; i < p.q_heads; i += blockDim.x) p.lse[at + i] = -INFINITY;
  }
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
  float2(*const s_l)[C::kHeads] = reinterpret_cast<float2(*)[C::kHeads]>(s_m + kWarps);    // sum and reference
  double(*const s_wide)[C::kHeads] = reinterpret_cast<double(*)[C::kHeads]>(s_m + kWarps);  // in their place until the join
  float(*const s_f)[C::kHeads] = reinterpret_cast<float(*)[C::kHeads]>(s_l + kWarps);       // [kMaxCluster]
  float* const s_qs = s_f[kMaxCluster];
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < C::kRing; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  __syncwarp();

  griddep_launch();
  griddep_wait();
  const int units = p.kv_heads * p.head_tiles;  // of a row
  // The segment at hand: tiles [begin, end) of a row and unit, counted from the row's first tile seen.
  int64_t row, begin, end;
  int unit;
  Span sp;
  int64_t left = 0;  // stream: tiles of this CTA's share from the segment on
  int part = 0;      // stream: segments done
  if (p.splits) {
    row = p.longest_first ? row_by_length(p, blockIdx.z, reinterpret_cast<int*>(s_m)) : blockIdx.z, unit = blockIdx.y;
    sp = row_span(p, row);
    const int64_t chunk = max((sp.tiles + p.splits - 1) / p.splits, static_cast<int64_t>(kWarps));
    begin = min(blockIdx.x * chunk, sp.tiles);
    end = min(begin + chunk, sp.tiles);
    if (sp.cut && threadIdx.x == 0) kv::set_status(p.c.status, STATUS_BAD_PAGE);
  } else {
    if (!find_share(p, units, reinterpret_cast<int64_t*>(s_m), row, unit, begin, left)) return tend_rows<kDim>(p);
    sp = row_span(p, row);
    end = min(begin + left, sp.tiles);
  }
  uint8_t* const ring = smem + warp * C::kRing * C::kUnit;
  int slot = 0;  // of the ring's next unit, and its barrier's parity
  uint32_t parity = 0;
  bool lost = false;  // a wait ran out
  const int tok = token_of<C::kBox>(lr), sw = C::kBox == 128 ? tok : tok >> 1;  // the lane's token of a key tile, its swizzle
  int vtok[2];                                                                    // its tokens of a value tile (and + 8)
#pragma unroll
  for (int i = 0; i < 2; ++i) vtok[i] = token_of<C::kBox>(2 * lc + i);
  const int per_page = p.c.page_size / kTile;

  for (;;) {
    const int kvh = unit / p.head_tiles, h0 = unit % p.head_tiles * C::kHeads;  // h0: first head of the group
    const int64_t qrow = row * p.q_heads + kvh * p.group + h0;                   // output row of head h0
    // A warp's steps: kU tiles each, tiles going to the warps in turn. Lane i of a block of 32 tiles knows where the
    // block's tile i lies, and asks for it.
    constexpr int kBlock = 32 / kU;  // steps a block
    const int mine = static_cast<int>((end - begin - warp + kWarps - 1) / kWarps);  // tiles of this warp
    const int steps = mine > 0 ? (mine + kU - 1) / kU : 0;
    int page, y, range;  // y: first row of the tile in its page
    auto find = [&](int step0) {
      const int64_t t = begin + (static_cast<int64_t>(step0) * kU + lane) * kWarps + warp;
      int tile = 0;
      page = 0, range = 0;
      if (t < end && lane < kBlock * kU) {
        const int64_t g = sp.tile0 + t, nth = div(g, per_page), t0 = g * kTile;
        tile = static_cast<int>(g - nth * per_page);
        page = p.c.table[row * p.c.table_stride + nth];
        if (page < 0 || page >= p.c.pages)
          kv::set_status(p.c.status, STATUS_BAD_PAGE);
        else
          range = (sp.first > t0 ? static_cast<int>(sp.first - t0) : 0) | (sp.n - t0 < kTile ? static_cast<int>(sp.n - t0) : kTile) << 8;
      }
      y = kvh * p.c.page_size + tile * kTile;
    };
    find(0);

    auto ask = [&](bool keys, int step, int to_slot) {
      if (step >= steps) return;
      if (keys && step % kBlock == 0 && step > 0) find(step);
      int pg[kU], yy[kU], rg[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int from = step % kBlock * kU + u;
        pg[u] = __shfl_sync(0xffffffffu, page, from), yy[u] = __shfl_sync(0xffffffffu, y, from), rg[u] = __shfl_sync(0xffffffffu, range, from);
      }
      if (elect_one()) {
        int tiles = 0;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          s_range[to_slot][u] = rg[u];
          tiles += rg[u] != 0;
        }
        mbar_arrive_expect_tx(&full[to_slot], tiles * (C::kTileBytes + (kQuant && keys ? 32 : 0)));
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          if (rg[u] == 0) continue;  // nothing there: no copy, the place keeps what it held, to be masked
          uint8_t* const to = ring + to_slot * C::kUnit + u * C::kTileBytes;
#pragma unroll
          for (int b = 0; b < C::kBoxes; ++b)
            tc::tma_load_3d(to + b * kTile * C::kBox, keys ? &kmap : &vmap, b * C::kBox, yy[u], pg[u], &full[to_slot]);
          if (kQuant && keys) {
            const int64_t x = pg[u] * p.c.exp_stride + yy[u];
            bulk_g2s(s_exp[to_slot][u], p.c.k_exp + x, 16, &full[to_slot]);
            bulk_g2s(s_exp[to_slot][u] + 16, p.c.v_exp + x, 16, &full[to_slot]);
          }
        }
      }
      __syncwarp();
    };
#pragma unroll
    for (int i = 0; i < C::kRing; ++i) ask(!(i & 1), i / 2, slot + i < C::kRing ? slot + i : slot + i - C::kRing);

    // Stream: the unit behind this one, its length on its way while this one is worked on (the share ends before the rows do)
    int64_t next_row = row;
    int next_unit = unit + 1;
    Span next_sp = sp;
    if (left > end - begin && next_unit == units) {
      next_unit = 0;
      while (++next_row < p.c.rows && (next_sp = row_span(p, next_row)).tiles == 0) {}
      if (next_row >= p.c.rows) left = end - begin;  // never, unless lengths change under the kernel
    }

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

    constexpr int kNone = 1 << 20;
    int ev0 = kNone;    // the exponent of the first value row seen
    bool wide = false;  // a later one is more than kNear away: from then on l is in s_wide

    auto next_slot = [&] {
      if (++slot == C::kRing) slot = 0, parity ^= 1;
    };
    // (a test before the wait: 96 ragged e4m3 rows, 16 heads a cache head, 77.0 against 78.3 us)
    auto landed = [&] { return __all_sync(0xffffffffu, mbar_test(&full[slot], parity) || (!p.hasty && mbar_wait(&full[slot], parity))); };
    int stuck = -1;  // the unit (a step's keys or its values) whose wait ran out: the segment ends there
    for (int step = 0; step < steps; ++step) {
      if (!landed()) {
        stuck = 2 * step;
        break;
      }
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
      int ev[kU][2];  // exponents of the value rows, ev0 in places not seen
      if (kQuant && ev0 == kNone)
#pragma unroll
        for (int u = kU - 1; u >= 0; --u)
          if (const int seen = s_range[slot][u]; seen != 0) ev0 = static_cast<int8_t>(s_exp[slot][u][16 + (seen & 255)]);
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        float kf[2], vf[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int8_t* x = reinterpret_cast<const int8_t*>(&s_exp[slot][u][r * 8 + tok]);
          kf[r] = kQuant ? exp2i(x[0]) : 1.f;
          vf[r] = kQuant ? __uint_as_float(0x4b400000u + x[16]) - 12582912.f : 0.f;  // the exponent as a float, off the conversion pipe
          ev[u][r] = kQuant ? x[16] : 0;
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
        if (seen != kTile << 8)  // places not seen hold anything, exponents among it: they count nowhere
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int t = tok + r * 8;
            if (t >= (seen & 255) && t < seen >> 8) continue;
            ev[u][r] = ev0;
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) s[u][nt][2 * r] = s[u][nt][2 * r + 1] = -INFINITY;
          }
      }
      __syncwarp();  // the unit is read
      ask(!(C::kRing & 1), step + C::kRing / 2, slot);
      next_slot();

      if constexpr (kQuant) {
        bool far = false;
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) far |= static_cast<uint32_t>(ev[u][r] - ev0 + kNear) > 2u * kNear;
        if (__builtin_expect(__any_sync(0xffffffffu, far && !wide), 0)) {
          wide = true;
          // before the maximum is raised, maybe by more than 32 bits hold
          float l_now[kNT][2], m_now[kNT][2];
#pragma unroll
          for (int i = 0; i < 2 * kNT; ++i) l_now[i / 2][i % 2] = l[i / 2][i % 2], m_now[i / 2][i % 2] = m[i / 2][i % 2];
          begin_wide<kNT>({s_wide[warp], s_m[warp]}, l_now, m_now, ev0);
        }
      }
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
            const float m_was = m[nt][h], f = m_was == -INFINITY ? 0.f : ex2(m_was - x);
            m[nt][h] = x;
            sub[nt][h] = (x == -INFINITY ? 0.f : x) - (kQuant ? kLift : 0.f);
            l[nt][h] = raise_sum(l[nt][h], m_was, x);
#pragma unroll
            for (int i = 0; i < kDim / 16; ++i) o[nt][i][h] *= f, o[nt][i][2 + h] *= f;
          }
      }
      if constexpr (kQuant)
        if (__builtin_expect(wide, 0)) {
          float s_now[kU][kNT][4], m_now[kNT][2], sub_now[kNT][2];
          int ev_now[kU][2];
#pragma unroll
          for (int u = 0; u < kU; ++u) {
#pragma unroll
            for (int i = 0; i < 4 * kNT; ++i) s_now[u][i / 4][i % 4] = s[u][i / 4][i % 4];
            ev_now[u][0] = ev[u][0], ev_now[u][1] = ev[u][1];
          }
#pragma unroll
          for (int i = 0; i < 2 * kNT; ++i) m_now[i / 2][i % 2] = m[i / 2][i % 2], sub_now[i / 2][i % 2] = sub[i / 2][i % 2];
          add_wide<kU, kNT>({s_wide[warp], s_m[warp]}, s_now, ev_now, m_now, sub_now);
        }
      // weights, as the second product's B operands
      uint32_t ph[kU][kNT][2], pl[kU][kNT][2];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        float back[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) back[r] = kQuant && !wide ? exp2i(ev0 - ev[u][r]) : 0.f;
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          float w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            w[j] = ex2(s[u][nt][j] - sub[nt][j & 1]);
            l[nt][j & 1] += kQuant ? w[j] * back[j >> 1] : w[j];
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if (kQuant) {
              ph[u][nt][r] = transpose8(pack_half(w[2 * r], w[2 * r + 1]));
            } else {
              // high part cut, so the low part has its sign and, kept from zero, an infinite value stays infinite
              const uint32_t x = __float_as_uint(w[2 * r]), y = __float_as_uint(w[2 * r + 1]);
              ph[u][nt][r] = transpose8(__byte_perm(x, y, 0x7632));
              pl[u][nt][r] = transpose8(pack_bf16(fmaxf(w[2 * r] - __uint_as_float(x & 0xffff0000u), 0x1p-120f),
                                                  fmaxf(w[2 * r + 1] - __uint_as_float(y & 0xffff0000u), 0x1p-120f)));
            }
          }
        }
      }

      if (!landed()) {
        stuck = 2 * step + 1;
        break;
      }
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

    // After a wait that ran out no more is asked for, and what was is waited for, that unit and those up to kRing behind it:
    // the join and, once this CTA has left, another one use their places.
    if (stuck >= 0) {
      if (lane == 0) kv::set_status(p.c.status, STATUS_TIMEOUT);
      lost = true;
      for (const int asked = min(2 * steps, stuck + C::kRing); stuck < asked; ++stuck) {
        mbar_drain(&full[slot], parity);
        next_slot();
      }
    }

    // join the warps; the ring's place is free once every warp is here (it has waited for all that it asked for)
    float(*s_o)[kNT * 4][C::kPitch] = reinterpret_cast<float(*)[kNT * 4][C::kPitch]>(smem);
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int w = 4; w < 32; w *= 2) l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], w);
        if (lr == 0) {
          const int head = nt * 8 + 2 * lc + h;
          s_m[warp][head] = m[nt][h];
          float2 sum = make_float2(l[nt][h], kQuant && ev0 != kNone ? m[nt][h] - kLift - ev0 : m[nt][h]);
          if (kQuant && wide) {  // the reference takes the 64 bits' exponent
            const double t = s_wide[warp][head];
            const int e = max((__double2hiint(t) >> 20) - 1023, -1000);
            sum = make_float2(static_cast<float>(t * exp2d(-e)), m[nt][h] - kLift + e);
          }
          s_l[warp][head] = sum;
        }
      }
    __syncthreads();
    const bool whole = p.splits ? p.splits == 1 : begin == 0 && end == sp.tiles;
    const int64_t to = 2 * static_cast<int64_t>(blockIdx.x) + (part ? 1 : 0);  // stream: where a shared row's part goes
    if (threadIdx.x < C::kHeads) {  // each warp's factor into s_m, the joined sum into s_l[0], maximum into [1], out's scale into [2]
      const int h = threadIdx.x;
      float mm = -INFINITY, rr = -INFINITY, ll = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][h]), rr = fmaxf(rr, s_l[w][h].y);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = s_m[w][h] == -INFINITY ? 0.f : ex2(s_m[w][h] - mm);
        ll += raise_sum(s_l[w][h].x, s_l[w][h].y, rr);
        s_m[w][h] = f;
      }
      s_l[0][h] = make_float2(ll, rr), s_l[1][h].x = mm;
      if (whole) {
        s_l[2][h] = scale_of(mm, rr, ll, kQuant);
        if (h0 + h < p.group) p.lse[qrow + h] = lse_of(rr, ll);
      } else if (!p.splits) {
        p.part_ml[to * C::kHeads + h] = {mm, ll, rr, 0.f};
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
    auto place = [&](int d) { return (d ^ (d / C::kE & 3)) * 2; };
    auto put = [&](int h, int d, float x, float y) {
      const float4 by = *reinterpret_cast<const float4*>(&s_l[2][h]);
      x *= by.x, y *= by.z;
      if (kQuant) x *= by.y, y *= by.w;
      if (h0 + h < p.group) p.out[(qrow + h) * kDim + d] = __float2bfloat16_rn(x);
      if (h0 + h + 1 < p.group) p.out[(qrow + h + 1) * kDim + d] = __float2bfloat16_rn(y);
    };
    for (int i = threadIdx.x; i < C::kHeads / 2 * kDim; i += blockDim.x) {
      const int hp = i / kDim, d = i % kDim, h = 2 * hp;
      float x = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 v = *reinterpret_cast<const float2*>(&s_o[w][hp][place(d)]);
        const float2 f = *reinterpret_cast<const float2*>(&s_m[w][h]);
        x += v.x * f.x, y += v.y * f.y;
      }
      if (whole) {
        put(h, d, x, y);
      } else if (p.splits) {
        *reinterpret_cast<float2*>(&s_o[0][hp][place(d)]) = make_float2(x, y);  // read by this thread alone so far
      } else {
        float* dst = p.part_o + (to * C::kHeads + h) * kDim + d;
        dst[0] = x, dst[kDim] = y;
      }
    }
    if (p.splits) {
      if (p.splits == 1) return;
      // every CTA of the cluster joins its part of the values
      const int rank = blockIdx.x;
      cluster_sync();
      // (maximum, sum, reference) of every CTA's heads, fetched at once, one a thread, into a place of the ring that is free now
      float4(*const s_all)[C::kHeads] = reinterpret_cast<float4(*)[C::kHeads]>(s_o[1]);
      static_assert(kMaxCluster * C::kHeads <= kWarps * 32 && kMaxCluster * C::kHeads * 16 <= sizeof(s_o[1]));
      if (const int i = threadIdx.x; i < p.splits * C::kHeads) {
        const int r = i / C::kHeads, h = i % C::kHeads;
        const float2 sum = ld_cluster2(&s_l[0][h], r);
        s_all[r][h] = make_float4(ld_cluster(&s_l[1][h].x, r), sum.x, sum.y, 0.f);
      }
      __syncthreads();
      if (threadIdx.x < C::kHeads) {
        const int h = threadIdx.x;
        float mm = -INFINITY, rr = -INFINITY, ll = 0.f;
        for (int r = 0; r < p.splits; ++r) mm = fmaxf(mm, s_all[r][h].x), rr = fmaxf(rr, s_all[r][h].z);
        for (int r = 0; r < p.splits; ++r) {
          const float4 part = s_all[r][h];
          ll += raise_sum(part.y, part.z, rr);
          s_f[r][h] = part.x == -INFINITY ? 0.f : ex2(part.x - mm);
        }
        s_l[2][h] = scale_of(mm, rr, ll, kQuant);
        if (rank == 0 && h0 + h < p.group) p.lse[qrow + h] = lse_of(rr, ll);
      }
      __syncthreads();
      for (int i = rank * blockDim.x + threadIdx.x; i < C::kHeads / 2 * kDim; i += p.splits * blockDim.x) {
        const int hp = i / kDim, d = i % kDim, h = 2 * hp;
        float x = 0.f, y = 0.f;
#pragma unroll 4
        for (int r = 0; r < p.splits; ++r) {
          const float2 v = ld_cluster2(&s_o[0][hp][place(d)], r);
          x += v.x * s_f[r][h], y += v.y * s_f[r][h + 1];
        }
        put(h, d, x, y);
      }
      cluster_sync();  // no CTA leaves while another reads its shared memory
      return;
    }
    left -= end - begin;
    if (left <= 0) return tend_rows<kDim>(p);
    ++part;
    row = next_row, unit = next_unit, sp = next_sp;
    begin = 0, end = min(left, sp.tiles);
    tc::fence_proxy_async_smem();  // the join's reads and writes of the ring come before the next copies into it
    if (__syncthreads_or(lost)) return tend_rows<kDim>(p);
  }
}

// Joins the parts of a shared row's unit: blockIdx = (row and unit, slice of its heads' values). A thread holds 4 values;
// `groups` threads take their parts in turn, each with a running maximum of its own, and meet in shared memory.
constexpr int kJoinThreads = 256, kJoinBatch = 4;
__global__ void __launch_bounds__(kJoinThreads, 4) join_kernel(const __grid_constant__ Params p, int dim, int ctas, int heads, int groups, bool quant) {
  __shared__ float s_m[kJoinThreads], s_l[kJoinThreads], s_r[kJoinThreads];
  __shared__ float4 s_x[kJoinThreads];
  griddep_launch();
  griddep_wait();
  const int units = p.kv_heads * p.head_tiles, row = blockIdx.x / units, unit = blockIdx.x % units;
  const int64_t at = p.row_at[row], tiles = p.row_at[row + 1] - at, share = share_of(p.row_at[p.c.rows], p.c.rows, units, ctas);
  const int64_t from = at * units + unit * tiles, first = div(from, share), last = div(from + tiles - 1, share);
  if (tiles == 0 || last == first) return;  // nothing to see, or written whole
  const int n = static_cast<int>(last - first + 1), skip = from > first * share;  // skip: the row is not its first CTA's first
  const int per = kJoinThreads / groups, g = threadIdx.x / per, i4 = blockIdx.y * per + threadIdx.x % per;
  const int h = i4 * 4 / dim, in_group = unit % p.head_tiles * heads + h;
  const bool on = h < heads && in_group < p.group;
  const float4* const ml = reinterpret_cast<const float4*>(p.part_ml + 2 * first * heads + h);
  const float4* const po = reinterpret_cast<const float4*>(p.part_o + 2 * first * heads * dim) + i4;
  float m = -INFINITY, l = 0.f, r = -INFINITY;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = g; i0 < n && on; i0 += groups * kJoinBatch) {
    float4 a[kJoinBatch];  // parts
    float4 y[kJoinBatch];
#pragma unroll
    for (int b = 0; b < kJoinBatch; ++b) {
      const int i = i0 + b * groups, slot = 2 * i + (i == 0 ? skip : 0);
      a[b] = i < n ? ml[slot * heads] : make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
      y[b] = i < n ? po[slot * (heads * dim / 4)] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float mm = m, rr = r;
#pragma unroll
    for (int b = 0; b < kJoinBatch; ++b) mm = fmaxf(mm, a[b].x), rr = fmaxf(rr, a[b].z);
    const float back = m == -INFINITY ? 0.f : ex2(m - mm);
    l = raise_sum(l, r, rr);
    x.x *= back, x.y *= back, x.z *= back, x.w *= back;
#pragma unroll
    for (int b = 0; b < kJoinBatch; ++b) {
      const float f = a[b].x == -INFINITY ? 0.f : ex2(a[b].x - mm);
      l += raise_sum(a[b].y, a[b].z, rr);
      x.x += y[b].x * f, x.y += y[b].y * f, x.z += y[b].z * f, x.w += y[b].w * f;
    }
    m = mm, r = rr;
  }
  if (groups > 1) {
    s_m[threadIdx.x] = m, s_l[threadIdx.x] = l, s_r[threadIdx.x] = r, s_x[threadIdx.x] = x;
    __syncthreads();
    if (g) return;
    float mm = m, rr = r;
    for (int i = 1; i < groups; ++i) mm = fmaxf(mm, s_m[i * per + threadIdx.x]), rr = fmaxf(rr, s_r[i * per + threadIdx.x]);
    const float f0 = m == -INFINITY ? 0.f : ex2(m - mm);
    l = raise_sum(l, r, rr);
    x.x *= f0, x.y *= f0, x.z *= f0, x.w *= f0;
    for (int i = 1; i < groups; ++i) {
      const float mi = s_m[i * per + threadIdx.x], f = mi == -INFINITY ? 0.f : ex2(mi - mm);
      const float4 y = s_x[i * per + threadIdx.x];
      l += raise_sum(s_l[i * per + threadIdx.x], s_r[i * per + threadIdx.x], rr);
      x.x += y.x * f, x.y += y.y * f, x.z += y.z * f, x.w += y.w * f;
    }
    m = mm, r = rr;
  }
  if (!on) return;
  const int64_t head = static_cast<int64_t>(row) * p.q_heads + unit / p.head_tiles * p.group + in_group;
  const float2 scale = scale_of(m, r, l, quant);
  auto value = [scale](float v) { return v * scale.x * scale.y; };
  const int d = i4 * 4 - h * dim;
  *reinterpret_cast<uint2*>(p.out + head * dim + d) = make_uint2(pack_bf16(value(x.x), value(x.y)), pack_bf16(value(x.z), value(x.w)));
  if (d == 0) p.lse[head] = lse_of(r, l);
}

// ------------------------------------------------------------------ host side
// A wait on an mbarrier sleeps in hardware for longer than any copy takes before its time is looked at, so limits below
// this many nanoseconds would have no effect; they are kept for each device, and the kernel then does not wait at all.
constexpr uint64_t kHasty = 1000;
static std::atomic<uint64_t> g_hasty{0};  // a bit a device

static int sms() {
  int dev = 0;
  cudaGetDevice(&dev);
  return sm_count(dev);
}

static int tile_heads(int group) { return group > 8 ? 16 : 8; }

// How a call is laid out, from its sizes and the table's width (`tiles` of 16 tokens a row at most): the quickest by a model
// of the time in microseconds, in which the longest row fills the table and the rows are 0.7 of it on average.
//   A CTA reads about 56 KB a microsecond (35 KB of e4m3), the machine 6.2 MB (4.5 MB). A launch with its first copies and
//   last sums takes 4.5 (one CTA a unit) or 7.5 (a cluster a unit). One CTA a unit leaves the machine idle at the end, 5%,
//   unless the units are more than run at once and the longest start first, which takes 1.5 (row_by_length). The
//   stream takes 12 (the count of the rows, and the join's launch).
// Measured at 1 / 2 / 32 / 128 units (one row, 2 x 1, 8 x 4, 16 x 8) of up to 1,000 tokens: one CTA a unit 20.5 / 20.6 /
// 12.8 / 15.9 us, clusters 8.2 / 8.4 / 8.6 / -, stream 10.3 / 14.0 / 14.3 / 23.1; of up to 8,000: 133 / 133 / 76 / 84,
// 22.7 / 22.9 / 26.5 / -, 13.5 / 18.0 / 24.7 / 68 (256-value heads for the first two, else 128; bf16). 512 units (64 x 8) of up
// to 8,192: one CTA a unit 195, longest first 171, stream 192; of up to 2,000 50.7 and 44.5; of up to 600 21.5 and 22.1.
// What the rule does not know is lengths: of those 512 units, one row of 8,192 tokens among rows of 200 to 400 takes 82 us by
// it, where the stream would take 36.
struct Plan {
  int head_tiles, splits, ctas;  // splits: CTAs of a cluster, 0: stream over `ctas`
  bool longest_first;            // more CTAs than run at once: the long rows' start first
};
static Plan plan(int rows, int q_heads, int kv_heads, int dim, int page_size, int per_row, bool quant, int64_t window) {
  Plan r{};
  int64_t tiles = static_cast<int64_t>(per_row) * (page_size / kTile);
  if (window > 0 && window / kTile + 2 < tiles) tiles = window / kTile + 2;  // the tiles that a window touches
  const int group = q_heads / kv_heads, heads = tile_heads(group), ctas = 2 * sms();
  r.head_tiles = (group + heads - 1) / heads;
  const double units = static_cast<double>(rows) * kv_heads * r.head_tiles, unit = static_cast<double>(tiles) * dim * (quant ? 32 : 64);
  const double all = 0.7 * units * unit / (quant ? 4.5e6 : 6.2e6);
  const bool sorted = units > ctas && tiles >= 48 && rows > 1 && rows <= kWarps * 32;
  double best = 12 + all;
  r.ctas = ctas;
  for (int s = 1; s <= kMaxCluster && (s == 1 || units * s <= sms()); s *= 2) {
    const double one = unit / s / (quant ? 35e3 : 56e3), end = s == 1 && !sorted ? 1.05 * all : all;
    const double t = (s > 1 ? 7.5 : sorted ? 6 : 4.5) + (one > end ? one : end);
    if (t < best) best = t, r.splits = s;
  }
  r.longest_first = r.splits == 1 && sorted;
  return r;
}
static size_t part_bytes(const Plan& r, int rows, int q_heads, int kv_heads, int dim) {
  if (r.splits) return 0;
  const size_t heads = tile_heads(q_heads / kv_heads);
  return 2 * static_cast<size_t>(r.ctas) * heads * (dim * sizeof(float) + sizeof(Part)) + (static_cast<size_t>(rows) + 1) * sizeof(int64_t);
}

template <typename... A>
static cudaError_t start(void (*kernel)(A...), dim3 grid, int threads, int shared, int cluster, void* stream, A... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
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
    cudaError_t err = cudaFuncSetAttribute(attend_kernel<kDim, kQuant, kNT, kU>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kShared);
    if (err == cudaSuccess) err = cudaFuncSetAttribute(attend_kernel<kDim, kQuant, kNT, kU>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (err != cudaSuccess) return set_error(std::string("paged_attention: ") + cudaGetErrorString(err)), DM3_ECUDA;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  const cudaError_t err = start(attend_kernel<kDim, kQuant, kNT, kU>, grid, kWarps * 32, C::kShared, p.splits, stream, p, maps[0], maps[1]);
  if (err != cudaSuccess) return set_error(std::string("paged_attention launch: ") + cudaGetErrorString(err)), DM3_ECUDA;
  return DM3_OK;
}

template <int kDim, bool kQuant>
static int attend(const Params& p, dim3 grid, void* stream) {
  // token tiles a step: 8 KB of keys, one unit of the ring (6 KB for 384-byte rows)
  constexpr int kRow = kDim * (kQuant ? 1 : 2), kU = kRow <= 64 ? 8 : kRow <= 128 ? 4 : kRow <= 256 ? 2 : 1;
  return tile_heads(p.group) == 16 ? attend<kDim, kQuant, 2, (kU > 2 ? 3 : kU)>(p, grid, stream) : attend<kDim, kQuant, 1, kU>(p, grid, stream);
}

}  // namespace attn
}  // namespace dm3

int dm3::wait_limit_attention(uint64_t ns) {
  const cudaError_t err = set_wait_limit_here(ns);
  if (err != cudaSuccess) return static_cast<int>(err);
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  ns < attn::kHasty ? attn::g_hasty.fetch_or(bit) : attn::g_hasty.fetch_and(~bit);
  return 0;
}

// ------------------------------------------------------------------ C ABI
extern "C" size_t dm3_paged_attention_workspace_bytes(int rows, int q_heads, int kv_heads, int dim, int page_size,
                                                      int per_row, int quantised, int64_t window) {
  if (rows < 1 || kv_heads < 1 || q_heads < kv_heads || dim < 1 || page_size < dm3::attn::kTile || per_row < 0) return 0;
  return dm3::attn::part_bytes(dm3::attn::plan(rows, q_heads, kv_heads, dim, page_size, per_row, quantised != 0, window), rows, q_heads,
                               kv_heads, dim);
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
  if (static_cast<int64_t>(rows) * q_heads > INT32_MAX) return set_error("paged_attention: too many rows and heads"), DM3_EINVAL;
  if (window < 0 || !std::isfinite(scale)) return set_error("paged_attention: bad window or scale"), DM3_EINVAL;
  if (rows == 0) return DM3_OK;
  if (!q || !lengths || !out || !lse) return set_error("paged_attention: null pointer"), DM3_EINVAL;
  if (reinterpret_cast<uintptr_t>(q) % 16 || q_rs % 8 || q_hs % 8 || reinterpret_cast<uintptr_t>(out) % 16)
    return set_error("paged_attention: rows must start on 16 bytes"), DM3_EINVAL;
  const attn::Plan plan = attn::plan(rows, q_heads, kv_heads, dim, page_size, per_row, k_exp != nullptr, window);
  p.q = static_cast<const __nv_bfloat16*>(q), p.q_rs = q_rs, p.q_hs = q_hs, p.q_heads = q_heads, p.kv_heads = kv_heads;
  p.group = q_heads / kv_heads, p.head_tiles = plan.head_tiles, p.splits = plan.splits, p.longest_first = plan.longest_first;
  int dev = 0;
  cudaGetDevice(&dev);
  p.hasty = attn::g_hasty.load(std::memory_order_relaxed) >> (dev & 63) & 1;
  p.lengths = lengths, p.scale_log2 = scale * 1.44269504088896341f, p.window = window;
  p.out = static_cast<__nv_bfloat16*>(out), p.lse = lse;
  const int heads = attn::tile_heads(p.group);
  if (!plan.splits) {
    if (workspace_bytes < attn::part_bytes(plan, rows, q_heads, kv_heads, dim)) return set_error("workspace too small"), DM3_ENOSPACE;
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256) return set_error("workspace must be 256-byte aligned"), DM3_EINVAL;
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<attn::Part*>(p.part_o + 2 * static_cast<int64_t>(plan.ctas) * heads * dim);
    p.row_at = reinterpret_cast<int64_t*>(p.part_ml + 2 * static_cast<int64_t>(plan.ctas) * heads);
  }
  const dim3 grid = plan.splits ? dim3(plan.splits, kv_heads * plan.head_tiles, rows) : dim3(plan.ctas);
  int rc;
  switch (dim) {
    case 64: rc = k_exp ? attn::attend<64, true>(p, grid, stream) : attn::attend<64, false>(p, grid, stream); break;
    case 128: rc = k_exp ? attn::attend<128, true>(p, grid, stream) : attn::attend<128, false>(p, grid, stream); break;
    case 192: rc = k_exp ? attn::attend<192, true>(p, grid, stream) : attn::attend<192, false>(p, grid, stream); break;
    default: rc = k_exp ? attn::attend<256, true>(p, grid, stream) : attn::attend<256, false>(p, grid, stream); break;
  }
  if (rc) return rc;
  if (!plan.splits) {
    // threads that share a unit's parts: few where there are many units, which have two or three parts each
    const int64_t units = static_cast<int64_t>(rows) * kv_heads * plan.head_tiles;
    const int groups = units * 4 >= plan.ctas ? 2 : 16;
    const dim3 joins(static_cast<unsigned>(units), (heads * (dim / 4) * groups + attn::kJoinThreads - 1) / attn::kJoinThreads);
    const cudaError_t err = attn::start(attn::join_kernel, joins, attn::kJoinThreads, 0, 1, stream, p, dim, plan.ctas, heads, groups, k_exp != nullptr);
    if (err != cudaSuccess) return set_error(std::string("paged_attention launch: ") + cudaGetErrorString(err)), DM3_ECUDA;
  }
  note_launches(plan.splits ? 1 : 2);
  return DM3_OK;
}
