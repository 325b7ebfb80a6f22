// What the kernels over a paged key-value cache share: the cache as a launch sees it, and how a position finds its slot.
#pragma once
#include <cuda_fp16.h>

#include "../../include/incin_b200.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace incin {

int device_sm_count();

struct PagedView {
  const uint16_t *k, *v;
  long long k_page, k_head, k_token, v_page, v_head, v_token;
  const int32_t* table;
  long long table_stride;
  const int32_t *lengths, *offsets;
  int table_width, seqs, rows, pages, page_shift, Hq, Hkv;
  int* status;
};

inline PagedView paged_view(const incin_paged_desc* d) {
  int shift = 0;
  while ((1 << shift) < d->page_size) ++shift;
  return {(const uint16_t*)d->k_pages, (const uint16_t*)d->v_pages, d->k_stride_page, d->k_stride_head, d->k_stride_token,
          d->v_stride_page, d->v_stride_head, d->v_stride_token, d->table, d->table_stride, d->lengths, d->offsets,
          d->table_width, d->seqs, d->rows, d->pages, shift, d->Hq, d->Hkv, (int*)d->status};
}

// What every entry point over a cache refuses.
inline int check_paged(const incin_paged_desc* d) {
  if (!d || !d->k_pages || !d->v_pages || !d->table || !d->lengths || !d->x || !d->out || d->seqs <= 0 || d->rows <= 0 ||
      d->pages <= 0 || d->table_width <= 0 || d->Hq <= 0 || d->Hkv <= 0 || d->Hq % d->Hkv || d->Hq / d->Hkv > 128 || d->Hq > 32768)
    return INCIN_ERR_ARGUMENT;
  if (d->page_size != 16 && d->page_size != 32 && d->page_size != 64 && d->page_size != 128) return INCIN_ERR_UNSUPPORTED;
  if (d->D != 64 && d->D != 128) return INCIN_ERR_UNSUPPORTED;
  if (d->dtype != INCIN_GEMM_IN_BF16 && d->dtype != INCIN_GEMM_IN_FP16) return INCIN_ERR_UNSUPPORTED;
  if (((uintptr_t)d->k_pages | (uintptr_t)d->v_pages | (uintptr_t)d->x | (uintptr_t)d->out) & 15 || ((uintptr_t)d->workspace & 31))
    return INCIN_ERR_ALIGNMENT;
  if ((long long)d->table_width * d->page_size > (1ll << 30)) return INCIN_ERR_TOO_LARGE;   // positions are counted in 32 bits
  const long long strides[] = {d->k_stride_page, d->k_stride_head, d->k_stride_token, d->v_stride_page, d->v_stride_head,
                               d->v_stride_token, d->x_stride_row, d->x_stride_head};
  for (long long s : strides)
    if (s % 8) return INCIN_ERR_ALIGNMENT;
  return INCIN_OK;
}
// ... and attention besides.
inline int check_paged_attention(const incin_paged_desc* d) {
  const int rc = check_paged(d);
  return rc || (d->scale >= 0.f && d->scale <= 1e38f) ? rc : INCIN_ERR_ARGUMENT;   // times log2(e) in 32 bits
}

__device__ __forceinline__ void flag_bad_index(int* status) {
  if (status) atomicCAS(status, 0, kStatusBadArgument);
}
// Tokens of sequence s that its table can hold; a length outside that range is reported.
__device__ __forceinline__ int paged_length(const PagedView& c, int s) {
  const int n = c.lengths[s];
  const long long room = (long long)c.table_width << c.page_shift;
  if (n < 0 || n > room) {
    flag_bad_index(c.status);
    return n < 0 ? 0 : (int)room;
  }
  return n;
}
// Whether the rows [a, b) of a sequence fall or lie outside the rows there are.
__device__ __forceinline__ bool bad_offsets(const PagedView& c, int a, int b) { return a < 0 || b < a || b > c.rows; }
// Page of entry i of sequence s, or -1 (and a report) when the entry names none.
__device__ __forceinline__ int paged_page(const PagedView& c, int s, int i) {
  const int page = c.table[s * c.table_stride + i];
  if ((unsigned)page < (unsigned)c.pages) return page;
  flag_bad_index(c.status);
  return -1;
}
// WEIGHT_LOG2: attention's weights are held as 2^WEIGHT_LOG2 at a row's reference, which the largest score may pass by 2^8.  fp16
// has 2^16 above 1 and loses what is below 2^-25, which a long cache has much of, so the range above is used, too.
struct Bf16 {
  static constexpr float WEIGHT_LOG2 = 0.f;
  static __device__ __forceinline__ float2 unpack(uint32_t u) { return unpack_bf16x2(u); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
struct Fp16 {
  static constexpr float WEIGHT_LOG2 = 7.f;
  static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
};

}  // namespace incin
