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

#include "dm3.h"
#include "dm3_common.cuh"
#include "dm3_internal.h"
#include "dm3_kv.cuh"

namespace dm3 {
namespace kv {

constexpr int kThreads = 256;
constexpr int kMaxRot = 1024;  // angles of one token in shared memory

struct Heads {  // [tokens][heads][dim] bf16, unit stride in dim
  const __nv_bfloat16* p;
  int64_t ts, hs;  // strides in elements
  int n;           // heads
};

struct RopeParams {
  Heads x;
  __nv_bfloat16* y;  // [T][heads][dim]
  int T, dim;
  const int64_t* positions;
  const double* inv_freq;
  int rot, interleaved;
  double factor;
};

// (cos, sin) of position * inv_freq, times factor. In 64 bits up to the reduced angle; `T` is the type
// of what follows: double where a rotated key is quantised next.
template <typename T>
__device__ __forceinline__ void angle(int64_t pos, double inv_freq, double factor, T& c, T& s) {
  double t = static_cast<double>(pos) * inv_freq * 0.31830988618379067154;  // 1 / pi
  t -= 2.0 * rint(t * 0.5);
  if (sizeof(T) == 8) {
    double cd, sd;
    sincospi(t, &sd, &cd);
    c = static_cast<T>(cd * factor);
    s = static_cast<T>(sd * factor);
  } else {
    float cf, sf;
    sincospif(static_cast<float>(t), &sf, &cf);
    c = static_cast<T>(cf * static_cast<float>(factor));
    s = static_cast<T>(sf * static_cast<float>(factor));
  }
}

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

// Turns the 8 values of chunk `at` (of dim / 8) of the row at `row`; `own` is that chunk. cs holds the
// token's (cos, sin). rot is a multiple of 16, so a chunk's partners are one chunk.
template <typename T>
__device__ __forceinline__ Chunk turn(const __nv_bfloat16* row, uint4 own, int at, const T* cosv, const T* sinv, int rot,
                                      int interleaved) {
  Chunk x = unpack(own);
  if (at * 8 >= rot) return x;
  Chunk y;
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T c = cosv[at * 4 + i], s = sinv[at * 4 + i], a = x.v[2 * i], b = x.v[2 * i + 1];
      y.v[2 * i] = static_cast<float>(a * c - b * s);
      y.v[2 * i + 1] = static_cast<float>(b * c + a * s);
    }
  } else {
    const int half = rot / 16;
    const bool second = at >= half;
    const int j = second ? at - half : at;
    const Chunk z = unpack(*reinterpret_cast<const uint4*>(row + (second ? j : at + half) * 8));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T c = cosv[j * 8 + i], s = second ? sinv[j * 8 + i] : -sinv[j * 8 + i];
      y.v[i] = static_cast<float>(static_cast<T>(x.v[i]) * c + static_cast<T>(z.v[i]) * s);
    }
  }
  return y;
}

// ------------------------------------------------------------------ rope
// One CTA a token (and a share of its heads, blockIdx.y, when there are few tokens).
__global__ void __launch_bounds__(kThreads) rope_kernel(const __grid_constant__ RopeParams p) {
  __shared__ float cosv[kMaxRot / 2], sinv[kMaxRot / 2];
  griddep_launch();
  griddep_wait();
  const int t = blockIdx.x;
  const int64_t pos = p.positions[t];
  for (int i = threadIdx.x; i < p.rot / 2; i += blockDim.x) angle(pos, p.inv_freq[i], p.factor, cosv[i], sinv[i]);
  __syncthreads();
  const int per = p.dim / 8, n = p.x.n * per;
  for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < n; i += gridDim.y * blockDim.x) {
    const int h = i / per, c = i - h * per;
    const __nv_bfloat16* row = p.x.p + t * p.x.ts + h * p.x.hs;
    const uint4 own = *reinterpret_cast<const uint4*>(row + c * 8);
    *reinterpret_cast<uint4*>(p.y + (static_cast<int64_t>(t) * p.x.n + h) * p.dim + c * 8) =
        pack(turn(row, own, c, cosv, sinv, p.rot, p.interleaved));
  }
}

// Any dim, rot, stride and alignment: one value at a time.
__global__ void __launch_bounds__(kThreads) rope_any_kernel(const __grid_constant__ RopeParams p) {
  __shared__ float cosv[kMaxRot / 2], sinv[kMaxRot / 2];
  griddep_launch();
  griddep_wait();
  const int t = blockIdx.x;
  const int64_t pos = p.positions[t];
  for (int i = threadIdx.x; i < p.rot / 2; i += blockDim.x) angle(pos, p.inv_freq[i], p.factor, cosv[i], sinv[i]);
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
      y = y * cosv[j] + z * (second ? sinv[j] : -sinv[j]);
    }
    p.y[(static_cast<int64_t>(t) * p.x.n + h) * p.dim + d] = __float2bfloat16_rn(y);
  }
}

// ------------------------------------------------------------------ kv_write
struct WriteParams {
  Heads q, k, v;     // q.n = 0: none
  __nv_bfloat16* y;  // the turned queries, [T][q.n][dim]
  int T, dim;
  const int64_t* rows;  // table row of each token; null: token i is row i
  const int64_t* positions;
  Cache c;
  const double* inv_freq;
  int rot, interleaved;  // rot = 0: no rotary positions
  double factor;
};

// The 8 values as e4m3 codes of 2^-e; what is not finite becomes NaN.
__device__ __forceinline__ uint2 encode(const Chunk& x, int e) {
  const float s = exp2i(-e);
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = x.v[4 * i + j];
      f[j] = isfinite(a) ? a * s : NAN;
    }
    w[i] = pack_e4m3x2(f[0], f[1]) | static_cast<uint32_t>(pack_e4m3x2(f[2], f[3])) << 16;
  }
  return make_uint2(w[0], w[1]);
}

// The exponent of a row whose largest finite magnitude is amax: the smallest e with amax <= 448 * 2^e
// (448 = 1.75 * 2^8), kept where 2^e times every code is a finite, normal bf16 number.
__device__ __forceinline__ int row_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  if (b == 0) return 0;
  const int e = static_cast<int>(b >> 23) - ((b & 0x7fffffu) <= 0x600000u ? 135 : 134);
  return min(max(e, -110), 119);
}

// One CTA a token (and a share of its rows, blockIdx.y). A row (one head of q, k or v) belongs to
// kSeg neighbouring lanes, 8 values each, so the amax of a quantised row is a few shuffles.
template <int kSeg, bool kQuant>
__global__ void __launch_bounds__(kThreads) write_kernel(const __grid_constant__ WriteParams p) {
  using T = typename std::conditional<kQuant, double, float>::type;
  __shared__ T cosv[kMaxDim / 2], sinv[kMaxDim / 2];
  griddep_launch();
  griddep_wait();
  const int t = blockIdx.x;
  const int64_t pos = p.positions[t];
  const int64_t r = p.rows ? p.rows[t] : t;
  const bool padding = pos < 0 || r < 0;
  for (int i = threadIdx.x; i < p.rot / 2; i += blockDim.x) angle(pos, p.inv_freq[i], p.factor, cosv[i], sinv[i]);
  __syncthreads();
  int64_t page = -1;
  int in_page = 0;
  if (!padding) {
    const int64_t nth = pos / p.c.page_size;
    if (r < p.c.rows && nth < p.c.per_row) page = p.c.table[r * p.c.table_stride + nth];
    in_page = static_cast<int>(pos - nth * p.c.page_size);
    if (page < 0 || page >= p.c.pages) {
      page = -1;
      if (threadIdx.x == 0) set_status(p.c.status, STATUS_BAD_PAGE);
    }
  }
  const int seg = threadIdx.x / kSeg, c = threadIdx.x % kSeg, segs = blockDim.x / kSeg, per = p.dim / 8;
  const int n = p.q.n + 2 * p.k.n;
  // all lanes of a warp make the same number of rounds: the shuffles need them
  for (int h0 = blockIdx.y * segs; h0 < n; h0 += gridDim.y * segs) {
    const int h = h0 + seg;
    const bool on = h < n && c < per;
    Chunk x{};
    int side = 0, head = h;  // 0: query, 1: key, 2: value
    if (on) {
      if (head >= p.q.n) head -= p.q.n, side = 1;
      if (side == 1 && head >= p.k.n) head -= p.k.n, side = 2;
      const Heads& in = side == 0 ? p.q : side == 1 ? p.k : p.v;
      const __nv_bfloat16* row = in.p + t * in.ts + head * in.hs;
      const uint4 own = *reinterpret_cast<const uint4*>(row + c * 8);
      if (side == 2 || p.rot == 0)
        x = unpack(own);
      else
        x = turn(row, own, c, cosv, sinv, p.rot, p.interleaved);
    }
    if (on && side == 0)
      *reinterpret_cast<uint4*>(p.y + (static_cast<int64_t>(t) * p.q.n + head) * p.dim + c * 8) =
          padding ? make_uint4(0, 0, 0, 0) : pack(x);
    if (!kQuant) {
      if (on && side != 0 && page >= 0)
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(side == 1 ? p.c.k : p.c.v) + page * p.c.page_stride +
                                  (static_cast<int64_t>(head) * p.c.page_size + in_page) * p.dim + c * 8) = pack(x);
      continue;
    }
    if (side == 1) x = unpack(pack(x));  // the key as a bf16 cache would hold it
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, isfinite(x.v[i]) ? fabsf(x.v[i]) : 0.f);
#pragma unroll
    for (int o = kSeg / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (on && side != 0 && page >= 0) {
      const int e = row_exponent(amax);
      const int64_t at = static_cast<int64_t>(head) * p.c.page_size + in_page;
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(side == 1 ? p.c.k : p.c.v) + page * p.c.page_stride + at * p.dim +
                                c * 8) = encode(x, e);
      if (c == 0) (side == 1 ? p.c.k_exp : p.c.v_exp)[page * p.c.exp_stride + at] = static_cast<int8_t>(e);
    }
  }
}

// ------------------------------------------------------------------ kv_read
struct ReadParams {
  Cache c;
  int heads, dim;
  const int64_t* lengths;
  int64_t L;           // tokens a row of the outputs
  __nv_bfloat16* out[2];  // [rows][heads][L][dim]
};

// blockIdx = (tile of a row's 16-byte output chunks, head, 2 * row + side).
template <bool kQuant>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ ReadParams p) {
  griddep_launch();
  griddep_wait();
  const int row = blockIdx.z >> 1, side = blockIdx.z & 1, head = blockIdx.y, per = p.dim / 8;
  int64_t n = p.lengths[row];
  const int64_t span = static_cast<int64_t>(p.c.per_row) * p.c.page_size;
  if (n > span) {
    n = span;
    if (threadIdx.x == 0) set_status(p.c.status, STATUS_BAD_PAGE);
  }
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t tok = i / per;
  const int c = static_cast<int>(i - tok * per);
  if (tok >= p.L) return;
  uint4 r = make_uint4(0, 0, 0, 0);
  if (tok < n) {
    const int64_t nth = tok / p.c.page_size;
    const int in_page = static_cast<int>(tok - nth * p.c.page_size);
    const int64_t page = p.c.table[row * p.c.table_stride + nth];
    if (page < 0 || page >= p.c.pages) {
      set_status(p.c.status, STATUS_BAD_PAGE);
    } else {
      const int64_t at = static_cast<int64_t>(head) * p.c.page_size + in_page;
      const void* base = side == 0 ? p.c.k : p.c.v;
      if (kQuant) {
        const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(base) + page * p.c.page_stride + at * p.dim + c * 8);
        const float s = exp2i((side == 0 ? p.c.k_exp : p.c.v_exp)[page * p.c.exp_stride + at]);
        Chunk x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = unpack_e4m3x2(static_cast<uint16_t>((j < 2 ? w.x : w.y) >> (16 * (j & 1))));
          x.v[2 * j] = f.x * s;
          x.v[2 * j + 1] = f.y * s;
        }
        r = pack(x);
      } else {
        r = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(base) + page * p.c.page_stride + at * p.dim + c * 8);
      }
    }
  }
  *reinterpret_cast<uint4*>(p.out[side] + ((static_cast<int64_t>(row) * p.heads + head) * p.L + tok) * p.dim + c * 8) = r;
}

// ------------------------------------------------------------------ host side
template <typename K, typename P>
static int launch(K kernel, dim3 grid, int threads, const P& p, void* stream, const char* what) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, p);
  if (err != cudaSuccess) return set_error(std::string(what) + " launch: " + cudaGetErrorString(err)), DM3_ECUDA;
  note_launches(1);
  return DM3_OK;
}

static bool aligned(const Heads& h) {
  return reinterpret_cast<uintptr_t>(h.p) % 16 == 0 && h.ts % 8 == 0 && h.hs % 8 == 0;
}

// CTAs a token: enough that few tokens still spread over the machine, at most one a round of rows.
static int shares(int64_t tokens, int rounds) {
  int dev = 0;
  cudaGetDevice(&dev);
  const int64_t want = (2 * sm_count(dev) + tokens - 1) / tokens;
  return static_cast<int>(want < rounds ? want : rounds);
}

}  // namespace kv

bool kv_cache_ok(const kv::Cache& c, int kv_heads, int dim) {
  if (dim != 64 && dim != 128 && dim != 192 && dim != 256) return set_error("the cache's head size must be 64, 128, 192 or 256"), false;
  if (kv_heads < 1 || kv_heads > 65535) return set_error("the cache must have 1 to 65535 heads"), false;
  if (c.page_size < 16 || c.page_size % 16) return set_error("page_size must be a multiple of 16"), false;
  if (c.pages < 1 || !c.k || !c.v || !c.status) return set_error("cache: null pointer or no pages"), false;
  if (!c.k_exp != !c.v_exp) return set_error("cache: one of the exponent tables is missing"), false;
  if (c.rows < 0 || c.per_row < 0 || (c.rows > 0 && c.per_row > 0 && !c.table) || c.table_stride < c.per_row)
    return set_error("bad page table"), false;
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
  RopeParams p{{static_cast<const __nv_bfloat16*>(x), ts, hs, heads}, static_cast<__nv_bfloat16*>(y), T, dim, positions,
               inv_freq, rot, interleaved, factor};
  // 16 bytes a thread where rows and pairs fall on them
  const bool wide = dim % 8 == 0 && rot % 16 == 0 && aligned(p.x) && reinterpret_cast<uintptr_t>(y) % 16 == 0;
  const int units = wide ? heads * (dim / 8) : heads * dim;
  const int threads = units < kThreads ? (units + 31) / 32 * 32 : kThreads;
  const dim3 grid(T, shares(T, (units + threads - 1) / threads));
  return wide ? launch(rope_kernel, grid, threads, p, stream, "rope") : launch(rope_any_kernel, grid, threads, p, stream, "rope");
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
  p.inv_freq = inv_freq, p.rot = rot, p.interleaved = interleaved, p.factor = factor;
  const int seg = dim == 64 ? 8 : dim == 128 ? 16 : 32, per_round = kThreads / seg, n = q_heads + 2 * kv_heads;
  const dim3 grid(T, shares(T, (n + per_round - 1) / per_round));
  auto go = [&](auto kernel) { return launch(kernel, grid, kThreads, p, stream, "kv_write"); };
  if (k_exp) return seg == 8 ? go(write_kernel<8, true>) : seg == 16 ? go(write_kernel<16, true>) : go(write_kernel<32, true>);
  return seg == 8 ? go(write_kernel<8, false>) : seg == 16 ? go(write_kernel<16, false>) : go(write_kernel<32, false>);
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
  if (table_rows > 32767) return set_error("kv_read: at most 32767 rows"), DM3_EINVAL;
  if (max_length < 0 || max_length > (int64_t(1) << 31)) return set_error("kv_read: bad max_length"), DM3_EINVAL;
  if (table_rows == 0 || max_length == 0) return DM3_OK;
  if (!lengths || !k_out || !v_out || reinterpret_cast<uintptr_t>(k_out) % 16 || reinterpret_cast<uintptr_t>(v_out) % 16)
    return set_error("kv_read: null or misaligned pointer"), DM3_EINVAL;
  p.heads = kv_heads, p.dim = dim, p.lengths = lengths, p.L = max_length;
  p.out[0] = static_cast<__nv_bfloat16*>(k_out), p.out[1] = static_cast<__nv_bfloat16*>(v_out);
  const int64_t chunks = max_length * (dim / 8);
  const dim3 grid(static_cast<unsigned>((chunks + kThreads - 1) / kThreads), kv_heads, 2 * table_rows);
  return k_exp ? launch(read_kernel<true>, grid, kThreads, p, stream, "kv_read")
               : launch(read_kernel<false>, grid, kThreads, p, stream, "kv_read");
}
