// Attention over the pages of a cache: every row of a step (a decode token, a
// few, a whole prompt) against the positions that its window and the first
// `sinks` positions leave visible.
//   s_j = scale q . k_j,  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m)
// with the running maximum m and sum of the online softmax in fp32.
#include <cmath>
#include "paged.cuh"
#include "stage.cuh"

namespace fmoe {
namespace pa {

struct AttnArgs {
  const bf16* q;  // [tokens][Hq][D], rows qs values apart
  bf16* out;      // [tokens][Hq][D]
  int64_t qs;
  int Hq, layer, window, sinks;
  float scale;
};

// Lane l's values l * P .. of row `slot` of a block.
template <int P>
__device__ __forceinline__ void load_page_row(const PagedDev& c, const uint8_t* blk, int slot, int lane, float (&v)[P]) {
  constexpr int D = 32 * P, LG = 64 / P, NG = P / 2;
  if (c.bits == 16) {
    const bf16* r = reinterpret_cast<const bf16*>(blk) + (int64_t)slot * D + lane * P;
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = bf2f(r[i]);
    return;
  }
  const uint32_t* words = reinterpret_cast<const uint32_t*>(blk + slot * (D / 2));
  const uint32_t pair = reinterpret_cast<const uint32_t*>(blk + c.ps * (D / 2) + slot * (D / 16))[lane / LG];
  const float s = bf16lo(pair), b = bf16hi(pair);
#pragma unroll
  for (int o = 0; o < P / 8; ++o) {
    const uint32_t w = words[((lane % LG) * (P / 8) + o) * NG + lane / LG];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[8 * o + i] = fmaf(s, (float)((w >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15u), b);
  }
}

// One CTA per (row, query head); a warp takes every 8th visible position.
template <int P>
__global__ void __launch_bounds__(256) paged_attn_rows_kernel(PagedDev c, BatchDev b, AttnArgs a) {
  constexpr int D = 32 * P;
  __shared__ float sm[8], sl[8], so[8][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, g = h / (a.Hq / c.Hkv);
  int i = 0;
  for (int k = 0; k < b.n; k += blockDim.x)
    i += __syncthreads_count(k + (int)threadIdx.x < b.n && b.q_start[k + threadIdx.x + 1] <= t);
  if (i >= b.n) return;
  const int pos = b.kv_len[i] - b.q_start[i + 1] + (int)t;
  const int low = a.window ? max(0, pos - a.window + 1) : 0;
  const int first = a.window ? min(a.sinks, low) : 0;  // positions [0, first) and [low, pos]
  float q[P], o[P], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < P; ++e) {
    q[e] = bf2f(a.q[t * a.qs + (int64_t)h * D + lane * P + e]) * a.scale;
    o[e] = 0.f;
  }
  for (int n = warp; n < first + pos - low + 1; n += 8) {
    const int j = n < first ? n : low + n - first;
    const int page = page_of(c, b.seqs[i], j >> c.log_ps);
    if (page < 0) continue;
    float x[P], s = 0.f;
    load_page_row<P>(c, page_block(c, a.layer, page, g, 0), j & (c.ps - 1), lane, x);
#pragma unroll
    for (int e = 0; e < P; ++e) s = fmaf(q[e], x[e], s);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    const float mn = fmaxf(m, s), f = expf(m - mn), w = expf(s - mn);
    load_page_row<P>(c, page_block(c, a.layer, page, g, 1), j & (c.ps - 1), lane, x);
    l = l * f + w;
#pragma unroll
    for (int e = 0; e < P; ++e) o[e] = o[e] * f + w * x[e];
    m = mn;
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < P; ++e) so[warp][lane * P + e] = o[e];
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < 8; ++w) M = fmaxf(M, sm[w]);
  for (int w = 0; w < 8; ++w) L += sm[w] > -INFINITY ? sl[w] * expf(sm[w] - M) : 0.f;
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float x = 0.f;
    for (int w = 0; w < 8; ++w) x += sm[w] > -INFINITY ? so[w][d] * expf(sm[w] - M) : 0.f;
    a.out[(t * a.Hq + h) * D + d] = __float2bfloat16_rn(L > 0.f ? x / L : 0.f);
  }
}

}  // namespace pa
}  // namespace fmoe

using namespace fmoe;

extern "C" {

size_t fmoe_paged_attend_workspace_bytes(const fmoe_paged_kv_t* cache, int q_heads, int32_t n, int64_t tokens,
                                         int32_t max_new) {
  PagedDev c;
  if (paged_to_dev(cache, &c, false) || q_heads < 1 || q_heads % c.Hkv || q_heads / c.Hkv > 8 || n < 0 || tokens < 0)
    return 0;
  return 256;
}

int fmoe_paged_attend(const fmoe_paged_kv_t* cache, int layer, const void* q, int64_t q_stride, int q_heads,
                      const fmoe_paged_batch_t* batch, int window, int sinks, float scale, void* out,
                      void* workspace, size_t workspace_bytes, void* stream) {
  PagedDev c;
  BatchDev b;
  int rc;
  if ((rc = paged_to_dev(cache, &c, true)) || (rc = batch_to_dev(batch, &b))) return rc;
  if (layer < 0 || layer >= c.layers) return set_error(FMOE_ERR_INVALID, "paged_attend: layer %d of %d", layer, c.layers);
  if (q_heads < 1 || q_heads % c.Hkv || q_heads / c.Hkv > 8)
    return set_error(FMOE_ERR_UNSUPPORTED, "paged_attend: %d query heads over %d kv heads (1..8 per kv head)", q_heads,
                     c.Hkv);
  if (window < 0 || sinks < 0) return set_error(FMOE_ERR_INVALID, "paged_attend: window %d sinks %d", window, sinks);
  if (!std::isfinite(scale)) return set_error(FMOE_ERR_INVALID, "paged_attend: scale %g", (double)scale);
  if (b.tokens == 0 || b.n == 0) return FMOE_OK;
  if (!q || !out || !aligned(q, 16) || !aligned(out, 16))
    return set_error(FMOE_ERR_ALIGN, "paged_attend: q/out null or not 16-byte aligned");
  if (q_stride % 8 || q_stride < (int64_t)q_heads * c.D)
    return set_error(FMOE_ERR_ALIGN, "paged_attend: q rows %lld values apart (a multiple of 8, at least %lld)",
                     (long long)q_stride, (long long)q_heads * c.D);
  const size_t need = fmoe_paged_attend_workspace_bytes(cache, q_heads, b.n, b.tokens, b.max_new);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
    return set_error(FMOE_ERR_WORKSPACE, "paged_attend: workspace of %zu bytes, %zu needed (16-byte aligned)",
                     workspace_bytes, need);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  pa::AttnArgs a = {static_cast<const bf16*>(q), static_cast<bf16*>(out), q_stride, q_heads, layer, window, sinks, scale};
  ProfScope prof_("paged_attn_rows_kernel", st);
  const dim3 grid((unsigned)b.tokens, (unsigned)q_heads);
  if (c.D == 256)
    pa::paged_attn_rows_kernel<8><<<grid, 256, 0, st>>>(c, b, a);
  else
    pa::paged_attn_rows_kernel<16><<<grid, 256, 0, st>>>(c, b, a);
  return check_launch("paged_attn_rows_kernel");
}

}  // extern "C"
