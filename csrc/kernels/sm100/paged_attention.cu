// Attention over a paged key-value cache.
//
// o_i = sum_j p_ij v_j over the keys that query i sees, p_ij = exp(scale q_i k_j - m_i) / l_i.  One pass over the keys with
// the running maximum m_i and sum l_i of the exponentials, in fp32; o_i is rescaled when m_i grows.
#include "paged.cuh"

#include <math_constants.h>

namespace incin {

// One warp per query row and head; a lane keeps D / 32 neighbouring elements of q and o.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_attention_kernel(const PagedView c, const uint16_t* x, long long x_row, long long x_head, uint16_t* out,
                                                              float scale_log2) {
  constexpr int PER = D / 64;   // packed pairs a lane
  pdl_launch_dependents();
  pdl_wait();
  const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= (long long)c.rows * c.Hq) return;
  const int t = (int)(item / c.Hq), h = (int)(item % c.Hq), hk = h / (c.Hq / c.Hkv);
  const int s = paged_sequence(c, t);
  const int keys = s < 0 ? 0 : c.offsets ? paged_length(c, s) - c.offsets[s + 1] + t + 1 : paged_length(c, s);
  float2 q[PER], o[PER];
  float m = -CUDART_INF_F, l = 0.f;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    q[e] = T::unpack(reinterpret_cast<const uint32_t*>(x + t * x_row + h * x_head)[lane * PER + e]);
    o[e] = make_float2(0.f, 0.f);
  }
  int page = -1;
  for (int j = 0; j < keys; ++j) {
    const int slot = j & ((1 << c.page_shift) - 1);
    if (slot == 0) page = paged_page(c, s, j >> c.page_shift);
    uint32_t k[PER] = {}, v[PER] = {};
    if (page >= 0) {
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        k[e] = reinterpret_cast<const uint32_t*>(c.k + page * c.k_page + hk * c.k_head + slot * c.k_token)[lane * PER + e];
        v[e] = reinterpret_cast<const uint32_t*>(c.v + page * c.v_page + hk * c.v_head + slot * c.v_token)[lane * PER + e];
      }
    }
    float z = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const float2 kk = T::unpack(k[e]);
      z = fmaf(q[e].x, kk.x, fmaf(q[e].y, kk.y, z));
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) z += __shfl_xor_sync(0xffffffffu, z, w);
    z *= scale_log2;
    if (z > m) {
      const float alpha = exp2f(m - z);
      m = z;
      l *= alpha;
#pragma unroll
      for (int e = 0; e < PER; ++e) o[e] = make_float2(o[e].x * alpha, o[e].y * alpha);
    }
    const float p = exp2f(z - (m == -CUDART_INF_F ? 0.f : m));
    l += p;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const float2 vv = T::unpack(v[e]);
      o[e] = make_float2(fmaf(p, vv.x, o[e].x), fmaf(p, vv.y, o[e].y));
    }
  }
  const float inv = keys > 0 ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < PER; ++e)
    reinterpret_cast<uint32_t*>(out + item * D)[lane * PER + e] = T::pack(o[e].x * inv, o[e].y * inv);
}

template <typename T, int D>
static cudaError_t launch_paged(const incin_paged_desc* d, cudaStream_t stream) {
  PagedView c = paged_view(d);
  const long long warps = (long long)d->rows * d->Hq;
  return launch_pdl<true>(paged_attention_kernel<T, D>, dim3((unsigned)((warps + 7) / 8)), dim3(256), 0, stream, c, (const uint16_t*)d->x,
                          d->x_stride_row, d->x_stride_head, (uint16_t*)d->out, d->scale * 1.4426950408889634f);
}

static int attend(const incin_paged_desc* d, void* stream) {
  const int rc = check_paged(d);
  if (rc) return rc;
  if ((long long)d->rows * d->Hq > (1ll << 33)) return INCIN_ERR_TOO_LARGE;
  const cudaStream_t s = (cudaStream_t)stream;
  const bool half = d->dtype == INCIN_GEMM_IN_FP16;
  cudaError_t e;
  if (d->D == 64) e = half ? launch_paged<Fp16, 64>(d, s) : launch_paged<Bf16, 64>(d, s);
  else e = half ? launch_paged<Fp16, 128>(d, s) : launch_paged<Bf16, 128>(d, s);
  return e == cudaSuccess ? INCIN_OK : INCIN_ERR_LAUNCH;
}

}  // namespace incin

extern "C" long long incin_prompt_attention_workspace(const incin_paged_desc*) { return 0; }
extern "C" int incin_prompt_attention(const incin_paged_desc* d, void* stream) {
  if (!d || !d->offsets) return INCIN_ERR_ARGUMENT;
  return incin::attend(d, stream);
}
