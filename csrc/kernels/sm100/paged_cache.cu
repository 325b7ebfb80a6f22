// Writing a paged key-value cache and moving its pages.
#include "paged.cuh"

#include <cmath>

namespace incin {

// ----------------------------------------------------------------------------- append
// Rotary pairs (i, i + D/2) turn by position * theta^(-2i/D).  The turn is kept as a 64-bit fraction of a full circle:
// position * frequency modulo 2^64 is an exact integer product, so a far position costs no accuracy (position *
// frequency in fp32 is off by 0.004 at position 100000, as much as a bf16 rounding).  The remainder, rounded to fp32 half
// turns, is within 2^-24 of a turn.
struct RopeTurns {
  uint64_t per_token[64];   // theta^(-2i/D) / (2 pi), in units of 2^-64 turns
};

// A block takes up to eight rows.  A thread asks for its first 32 bytes before anything is known about their place: which
// sequence, which position and page and the angles are a chain of four loads that the data need not wait for.  (More than
// 32 bytes ahead cost occupancy: 8190 rows of 40 heads of 128, 33.2 us, 64 bytes 35.1, 128 bytes 36.6.)  Bound by memory.
constexpr int APPEND_ROWS = 8, APPEND_BLOCK_BYTES = 40 << 10;

template <typename T, int D>
__global__ void __launch_bounds__(256) kv_append_kernel(const PagedView c, const uint16_t* x, long long x_row, long long x_head, uint16_t* q,
                                                        const __grid_constant__ RopeTurns turns, int rotate, int tokens) {
  constexpr int HALF = D / 2, VECS = HALF / 8;
  __shared__ float2 angle[APPEND_ROWS * HALF];
  __shared__ int pos_of[APPEND_ROWS], page_of[APPEND_ROWS];   // -1 where there is none
  pdl_launch_dependents();
  pdl_wait();
  const int first = blockIdx.x * tokens, n = min(tokens, c.rows - first), per = (c.Hq + 2 * c.Hkv) * VECS, total = n * per;
  uint4 lo, hi;
  auto load = [&](int i) {
    if (i < total) {
      const int r = i / per, k = i - r * per;
      const uint16_t* src = x + (first + r) * x_row + k / VECS * x_head + k % VECS * 8;
      lo = *reinterpret_cast<const uint4*>(src);
      hi = *reinterpret_cast<const uint4*>(src + HALF);
    }
  };
  load(threadIdx.x);
  if (threadIdx.x < 32) {
    const int t = first + threadIdx.x;
    int s = -1, pos = -1, page = -1;
    if (!c.offsets) {
      if (threadIdx.x < n && t < c.seqs) s = t;
    } else {   // sequences that end in front of the block's first row; a row's own lies there or a little behind
      int ended = 0;
      for (int i = threadIdx.x; i - (int)threadIdx.x < c.seqs; i += 32) ended += __popc(__ballot_sync(0xffffffffu, i < c.seqs && c.offsets[i + 1] <= first));
      if (threadIdx.x < n) {
        s = ended;
        while (s < c.seqs && c.offsets[s + 1] <= t) ++s;
        if (s >= c.seqs || c.offsets[s] > t) s = -1;
      }
    }
    if (s >= 0) {
      const int len = paged_length(c, s);
      pos = c.offsets ? len - c.offsets[s + 1] + t : len - 1;
      if (pos >= 0) page = paged_page(c, s, pos >> c.page_shift);
      else if (c.offsets) flag_bad_index(c.status);   // more new rows than tokens; without offsets an idle sequence
    }
    if (threadIdx.x < n) {
      pos_of[threadIdx.x] = pos;
      page_of[threadIdx.x] = page;
    }
  } else if (blockIdx.x == 0 && c.offsets) {   // once a launch, beside the chain above
    for (int s = threadIdx.x - 32; s < c.seqs; s += 256 - 32)
      if (bad_offsets(c, c.offsets[s], c.offsets[s + 1])) flag_bad_index(c.status);
  }
  __syncthreads();
  if (rotate) {
    for (int i = threadIdx.x; i < n * HALF; i += 256) {
      const uint64_t turn = (uint64_t)max(pos_of[i / HALF], 0) * turns.per_token[i % HALF];
      float sn, cs;
      sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &sn, &cs);
      angle[i] = make_float2(cs, sn);
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < total; i += 256) {
    if (i >= 256) load(i);
    const int r = i / per, k = i - r * per, h = k / VECS, v = k % VECS * 8, pos = pos_of[r];
    uint16_t* dst;
    if (h < c.Hq) {
      dst = q + ((long long)(first + r) * c.Hq + h) * D;
      if (pos < 0) lo = hi = make_uint4(0, 0, 0, 0);
    } else {
      const int page = page_of[r];
      if (page < 0) continue;
      const int slot = pos & ((1 << c.page_shift) - 1), hk = h - c.Hq;
      dst = hk < c.Hkv ? const_cast<uint16_t*>(c.k) + page * c.k_page + hk * c.k_head + slot * c.k_token
                       : const_cast<uint16_t*>(c.v) + page * c.v_page + (hk - c.Hkv) * c.v_head + slot * c.v_token;
    }
    if (rotate && h < c.Hq + c.Hkv && pos >= 0) {
      uint32_t *a = &lo.x, *b = &hi.x;
      const float2* cs = angle + r * HALF + v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 p = T::unpack(a[e]), o = T::unpack(b[e]), t0 = cs[2 * e], t1 = cs[2 * e + 1];
        a[e] = T::pack(p.x * t0.x - o.x * t0.y, p.y * t1.x - o.y * t1.y);
        b[e] = T::pack(o.x * t0.x + p.x * t0.y, o.y * t1.x + p.y * t1.y);
      }
    }
    *reinterpret_cast<uint4*>(dst + v) = lo;
    *reinterpret_cast<uint4*>(dst + HALF + v) = hi;
  }
}

// ----------------------------------------------------------------------------- page copies
constexpr int COPY_THREADS = 256, COPY_UNROLL = 8;

// Block (x, y): slices x, x + gridDim.x, ... of pairs y, y + gridDim.y, ...; a slice is 32 KB of a page in one run.  A block
// looks at all pairs once for each of its own (a conflict is a matter of two pairs), so it takes many slices of few pairs.
// Bound by memory: 777 pages of 26 layers, 2.65 GB read and written, 429 us, 6.2 TB/s (gathering and scattering them 6040 us);
// one page of 22 layers 2.8 us.
__global__ void __launch_bounds__(COPY_THREADS) copy_pages_kernel(uint4* storage, const int32_t* src, const int32_t* dst, int pairs,
                                                                  long long outer, int pages, long long page_vecs, int* status) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int SLICE = COPY_THREADS * COPY_UNROLL;
  const long long per_page = (page_vecs + SLICE - 1) / SLICE, slices = outer * per_page;
  for (int i = blockIdx.y; i < pairs; i += gridDim.y) {
    const int from = src[i], to = dst[i];
    bool bad = (unsigned)from >= (unsigned)pages || (unsigned)to >= (unsigned)pages;
    for (int j = threadIdx.x; j < pairs; j += COPY_THREADS) {
      if (j == i || !((src[j] == to && from != to) || (j < i && dst[j] == to))) continue;
      bad |= (unsigned)src[j] < (unsigned)pages && (unsigned)dst[j] < (unsigned)pages;   // a pair that names no page excludes none
    }
    if (__syncthreads_or(bad)) {
      if (threadIdx.x == 0) flag_bad_index(status);
      continue;
    }
    if (from == to) continue;
    for (long long s = blockIdx.x; s < slices; s += gridDim.x) {
      const long long run = s / per_page, at = (s - run * per_page) * SLICE;
      const uint4* a = storage + (run * pages + from) * page_vecs + at;
      uint4* b = storage + (run * pages + to) * page_vecs + at;
      const int n = (int)min((long long)SLICE, page_vecs - at);
      uint4 r[COPY_UNROLL];
#pragma unroll
      for (int u = 0; u < COPY_UNROLL; ++u)
        if (u * COPY_THREADS + threadIdx.x < n) r[u] = a[u * COPY_THREADS + threadIdx.x];
#pragma unroll
      for (int u = 0; u < COPY_UNROLL; ++u)
        if (u * COPY_THREADS + threadIdx.x < n) b[u * COPY_THREADS + threadIdx.x] = r[u];
    }
  }
}

template <typename T, int D>
static cudaError_t launch_append(const incin_paged_desc* d, const RopeTurns& turns, int rotate, cudaStream_t stream) {
  // rows of about 40 KB a block: 8190 rows of 40 heads of 128, 8 a block 34.1 us, 4 33.2; 8000 of 40 heads of 64, 8 17.1, 4 17.9, 2
  // 19.2; but at least two blocks an SM
  const long long row_bytes = (d->Hq + 2ll * d->Hkv) * D * 2;
  int tokens = APPEND_ROWS;
  while (tokens > 1 && (d->rows < 2 * device_sm_count() * tokens || tokens * row_bytes > APPEND_BLOCK_BYTES * 5 / 4)) tokens /= 2;
  return launch_pdl(kv_append_kernel<T, D>, dim3((d->rows + tokens - 1) / tokens), dim3(256), 0, stream, paged_view(d), (const uint16_t*)d->x,
                    d->x_stride_row, d->x_stride_head, (uint16_t*)d->out, turns, rotate, tokens);
}

}  // namespace incin

extern "C" int incin_kv_append(const incin_paged_desc* d, double theta, void* stream) {
  using namespace incin;
  const int rc = check_paged(d);
  if (rc) return rc;
  if (!(theta == 0.0 || (theta >= 1.0 && theta < 1e300)) || (!d->offsets && d->rows != d->seqs)) return INCIN_ERR_ARGUMENT;
  static thread_local RopeTurns turns;   // of the last theta and head_dim: a model's layers share them
  static thread_local double of_theta = 0.0;
  static thread_local int of_dim = 0;
  if (theta != 0.0 && (theta != of_theta || d->D != of_dim)) {
    for (int i = 0; i < d->D / 2; ++i)   // at most 1 / (2 pi) of a turn
      turns.per_token[i] = (uint64_t)std::ldexp(std::pow(theta, -2.0 * i / d->D) / 6.283185307179586476925, 64);
    of_theta = theta, of_dim = d->D;
  }
  const cudaStream_t s = (cudaStream_t)stream;
  const int rotate = theta != 0.0;
  const bool half = d->dtype == INCIN_GEMM_IN_FP16;
  cudaError_t e;
  if (d->D == 64) e = half ? launch_append<Fp16, 64>(d, turns, rotate, s) : launch_append<Bf16, 64>(d, turns, rotate, s);
  else e = half ? launch_append<Fp16, 128>(d, turns, rotate, s) : launch_append<Bf16, 128>(d, turns, rotate, s);
  return e == cudaSuccess ? INCIN_OK : INCIN_ERR_LAUNCH;
}

extern "C" int incin_copy_pages(void* storage, const int32_t* src, const int32_t* dst, int pairs, long long outer, int pages,
                                long long page_bytes, void* status, void* stream) {
  using namespace incin;
  if (!storage || !src || !dst || pairs <= 0 || outer <= 0 || pages <= 0 || page_bytes <= 0) return INCIN_ERR_ARGUMENT;
  if ((page_bytes & 15) || ((uintptr_t)storage & 15)) return INCIN_ERR_ALIGNMENT;
  const long long vecs = page_bytes / 16, slice = COPY_THREADS * COPY_UNROLL, slices = outer * ((vecs + slice - 1) / slice);
  const int blocks = device_sm_count() * 8;
  const unsigned y = (unsigned)(pairs < blocks ? pairs : blocks);
  long long x = (blocks + y - 1) / y;
  if (x > slices) x = slices;
  const cudaError_t e = launch_pdl(copy_pages_kernel, dim3((unsigned)x, y), dim3(COPY_THREADS), 0, (cudaStream_t)stream, (uint4*)storage, src, dst,
                                   pairs, outer, pages, vecs, (int*)status);
  return e == cudaSuccess ? INCIN_OK : INCIN_ERR_LAUNCH;
}
