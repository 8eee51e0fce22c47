// One new token's attention over the paged key-value cache (sm_100a).
//
//   s_t = scale * q . k_t,  p = softmax(s) over the tokens seen,  out = sum_t p_t v_t,
//   lse = log sum_t exp(s_t),  seen: max(0, n - window) <= t < n (window 0: all), n the row's length
//
// in one pass with the running maximum and sum; a row that sees nothing gives zeros and lse = -inf.
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

constexpr int kWarps = 8;

struct Params {
  const __nv_bfloat16* q;  // [rows][q_heads][dim]
  int64_t q_rs, q_hs;
  int q_heads, kv_heads;
  Cache c;
  const int64_t* lengths;
  float scale_log2;  // scale * log2(e)
  int64_t window;
  __nv_bfloat16* out;  // [rows][q_heads][dim]
  float* lse;          // [rows][q_heads]
};

// One CTA a query head and row; each warp takes every kWarps-th token, a lane dim / 32 values.
template <int kDim, bool kQuant>
__global__ void __launch_bounds__(kWarps * 32) attend_kernel(const __grid_constant__ Params p) {
  constexpr int kPer = kDim / 32;
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][kDim];
  griddep_launch();
  griddep_wait();
  const int head = blockIdx.x, row = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = head / (p.q_heads / p.kv_heads);
  int64_t n = p.lengths[row];
  const int64_t span = static_cast<int64_t>(p.c.per_row) * p.c.page_size;
  if (n > span) {
    n = span;
    if (threadIdx.x == 0) kv::set_status(p.c.status, STATUS_BAD_PAGE);
  }
  const int64_t first = p.window > 0 && n > p.window ? n - p.window : 0;
  float q[kPer], o[kPer], m = -INFINITY, l = 0.f;
  const __nv_bfloat16* qr = p.q + row * p.q_rs + head * p.q_hs + lane * kPer;
#pragma unroll
  for (int i = 0; i < kPer; ++i) q[i] = __bfloat162float(qr[i]), o[i] = 0.f;
  auto load = [&](const void* base, int64_t at, float e, float (&x)[kPer]) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (kQuant)
        x[i] = unpack_e4m3x2(static_cast<const uint8_t*>(base)[at + lane * kPer + i]).x * e;
      else
        x[i] = __bfloat162float(static_cast<const __nv_bfloat16*>(base)[at + lane * kPer + i]);
    }
  };
  for (int64_t t = first + warp; t < n; t += kWarps) {
    const int64_t nth = t / p.c.page_size;
    const int64_t page = p.c.table[row * p.c.table_stride + nth];
    if (page < 0 || page >= p.c.pages) {
      if (lane == 0) kv::set_status(p.c.status, STATUS_BAD_PAGE);
      continue;
    }
    const int64_t r = static_cast<int64_t>(kvh) * p.c.page_size + (t - nth * p.c.page_size);
    float x[kPer], s = 0.f;
    load(p.c.k, page * p.c.page_stride + r * kDim, kQuant ? exp2i(p.c.k_exp[page * p.c.exp_stride + r]) : 1.f, x);
#pragma unroll
    for (int i = 0; i < kPer; ++i) s += q[i] * x[i];
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    s *= p.scale_log2;
    const float mm = fmaxf(m, s);
    const float a = m == -INFINITY ? 0.f : exp2f(m - mm), w = mm == -INFINITY ? 0.f : exp2f(s - mm);
    load(p.c.v, page * p.c.page_stride + r * kDim, kQuant ? exp2i(p.c.v_exp[page * p.c.exp_stride + r]) : 1.f, x);
    l = l * a + w;
    m = mm;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = o[i] * a + w * x[i];
  }
  if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
  for (int i = 0; i < kPer; ++i) so[warp][lane * kPer + i] = o[i];
  __syncthreads();
  float mm = -INFINITY, ll = 0.f;
  for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm[w]);
  for (int w = 0; w < kWarps; ++w) ll += sm[w] == -INFINITY ? 0.f : sl[w] * exp2f(sm[w] - mm);
  const int64_t at = static_cast<int64_t>(row) * p.q_heads + head;
  for (int d = threadIdx.x; d < kDim; d += blockDim.x) {
    float x = 0.f;
    for (int w = 0; w < kWarps; ++w) x += sm[w] == -INFINITY ? 0.f : so[w][d] * exp2f(sm[w] - mm);
    p.out[at * kDim + d] = __float2bfloat16_rn(ll > 0.f ? x / ll : 0.f);
  }
  if (threadIdx.x == 0) p.lse[at] = ll > 0.f ? (mm + log2f(ll)) * 0.69314718055994531f : -INFINITY;
}

template <int kDim>
static int launch(const Params& p, void* stream) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.q_heads, p.c.rows);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = p.c.k_exp ? cudaLaunchKernelEx(&cfg, attend_kernel<kDim, true>, p)
                                    : cudaLaunchKernelEx(&cfg, attend_kernel<kDim, false>, p);
  if (err != cudaSuccess) return set_error(std::string("paged_attention launch: ") + cudaGetErrorString(err)), DM3_ECUDA;
  note_launches(1);
  return DM3_OK;
}

}  // namespace attn
}  // namespace dm3

// ------------------------------------------------------------------ C ABI
extern "C" size_t dm3_paged_attention_workspace_bytes(int rows, int q_heads, int kv_heads, int dim, int page_size,
                                                      int per_row) {
  return 0;
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
  if (workspace_bytes < dm3_paged_attention_workspace_bytes(rows, q_heads, kv_heads, dim, page_size, per_row))
    return set_error("workspace too small"), DM3_ENOSPACE;
  p.q = static_cast<const __nv_bfloat16*>(q), p.q_rs = q_rs, p.q_hs = q_hs, p.q_heads = q_heads, p.kv_heads = kv_heads;
  p.lengths = lengths, p.scale_log2 = scale * 1.44269504088896341f, p.window = window;
  p.out = static_cast<__nv_bfloat16*>(out), p.lse = lse;
  switch (dim) {
    case 64: return attn::launch<64>(p, stream);
    case 128: return attn::launch<128>(p, stream);
    case 192: return attn::launch<192>(p, stream);
    default: return attn::launch<256>(p, stream);
  }
}
