// Attention of one new token per sequence over a paged key-value cache.
//
//   o_h = sum_j p_hj v_j,  p_hj = 2^(c (z_hj - m_h)) / l_h,  z = q_h k_j,  c = scale log2(e),  j < lengths[b]
//
// Every cached key and value is read once for up to 16 query heads of its key head, so the bytes of the cache bound it.  (More
// heads are dealt out in blocks of 16, each of which reads it again: 64 sequences of up to 8192, one key head of 128: 8 query
// heads 31 us, 16 33, 32 56, 64 100, 128 187.)  The query heads of a key head are the columns of one product: S^T [16 keys x 8
// heads] = K Q^T and O^T [D x 8 heads] += V^T P^T with m16n8k16 matrix instructions (tcgen05.mma wants 128 rows; here a row of
// its operand would be a key that is used for 8 columns, and the tiles would have to pass through shared memory).  Both
// operands go from global memory straight into the registers that the instructions read, 16 bytes a load: the order in which a
// product runs over D, and in which its rows of V^T are numbered, is free, so it is chosen to be the order in which the bytes
// arrive.  K: lane (r, c) = (lane / 4, lane % 4) loads key rows r and r + 8 at element 32 j + 8 c: its four 32-bit words are
// the k indices of two instructions, and the queries are held in the same order. V: it loads keys 2c, 2c + 1, 2c + 8, 2c + 9 at
// element 64 j + 8 r; a pair of keys and a word make two rows of V^T by two byte permutes.  P^T comes out of S^T by transposing
// 8 x 8 blocks between the lanes (movmatrix).  No shared memory, no barrier in the loop: a warp asks for its next keys as soon
// as the present ones are used, and values likewise.
//
// Work is dealt out by the tokens that are really there: unit = 64 tokens of one (sequence, key head), a CTA takes an equal run
// of all units, each warp 16 tokens of every one.  Where CTAs get several units, a pair of sequence and head has one more
// than its tokens fill, since to begin and end one costs about as much (64 sequences of up to 4096, 32 / 4 heads of 64: CTAs
// with short sequences took 27 us, the others 20; 31.2 -> 28.0 us in all when it was added).  A pair that crosses CTAs leaves fp32 parts (O, m, l),
// which a second kernel joins in a fixed order.  So the lengths are needed on the device only, one long sequence uses all SMs,
// and a captured launch stays balanced whatever its lengths become.
//
// Bytes of the cache a second, of a measured copy's 6.47 TB/s: 128 sequences of up to 8192 tokens, 24 / 8 heads of 128, 334 us,
// 6.7 TB/s; one of 131071, 88.7 us, 6.1; 256 of up to 4096, 32 / 4 heads of 64, 87.9 us, 6.1; 64 of them 26.4 us, 4.6.  What is left
// is a chain at both ends: lengths, page numbers, first keys (4 us from the launch to the first product), and 3 us for the join.
#include "paged.cuh"

#include <math_constants.h>

namespace incin {

constexpr int DEC_WARPS = 4, DEC_STEP = 16 * DEC_WARPS;   // keys a CTA takes at a time, 16 a warp
constexpr int DEC_SEQS = 512;   // sequences a launch

template <int D, int NT>
struct DecCfg {   // NT: blocks of 8 query heads
  static constexpr int HEADS = 8 * NT;
  static constexpr int CTAS_PER_SM = (D == 64 ? 4 : 3) - (NT - 1);
  static constexpr int SLOT = HEADS * (D + 2);   // floats of a part: O [HEADS][D], m [HEADS], l [HEADS]
  static constexpr int ROW = D + 4;              // of O in shared memory
  // of an SM's CTAs: O, m and l of the warps, the sequences' lengths and units, 1 KB each for the system
  static constexpr int SHARED = CTAS_PER_SM * (DEC_WARPS * HEADS * (ROW + 2) * 4 + 8 * DEC_SEQS + 64 + 1024);
};

struct DecParams {
  PagedView c;
  const uint16_t* x;
  long long x_row, x_head;
  uint16_t* out;
  float scale_log2;
  int unit;            // tokens of a unit of work, a multiple of DEC_STEP
  int group, chunks;   // query heads of a key head, and the blocks of HEADS they are dealt in
  int4* open;          // per CTA: {sequence, head block, last CTA} of the pair that it begins and others continue, or -1; NULL where none can
  float* parts;        // per CTA two slots: the continuation of a pair, the beginning of one
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<Bf16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<Fp16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// transpose of an 8 x 8 block of 16-bit elements held in the accumulator's order
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// 16 bytes that no other load wants again; zeros where `there` is false (nothing is read then)
__device__ __forceinline__ void load16(uint32_t (&w)[4], const uint16_t* p, bool there) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %5, 0;\n"
      "mov.b32 %0, 0; mov.b32 %1, 0; mov.b32 %2, 0; mov.b32 %3, 0;\n"
      "@p ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];\n"
      "}\n"
      : "=&r"(w[0]), "=&r"(w[1]), "=&r"(w[2]), "=&r"(w[3])
      : "l"(p), "r"((int)there));
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(DEC_WARPS * 32, DecCfg<D, NT>::CTAS_PER_SM) decode_attention_kernel(const DecParams p) {
  using Cfg = DecCfg<D, NT>;
  constexpr int KJ = D / 32, VJ = D / 64;
  __shared__ int before[DEC_SEQS + 1];   // units of one head in front of each sequence
  __shared__ int length[DEC_SEQS];
  __shared__ int warp_sum[DEC_WARPS];
  __shared__ __align__(16) int next_run[DEC_WARPS][8];
  __shared__ float sm_m[DEC_WARPS][Cfg::HEADS], sm_l[DEC_WARPS][Cfg::HEADS];
  __shared__ __align__(16) float sm_o[DEC_WARPS][Cfg::HEADS][Cfg::ROW];
  const PagedView& c = p.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, q4 = lane & 3;
  pdl_launch_dependents();
  pdl_wait();

  const int head_blocks = c.Hkv * p.chunks;
  int extra;   // units of a pair without tokens
  {   // units in front of each sequence; one without tokens has one of them too, which writes its zeros
    const int per = (c.seqs + DEC_WARPS * 32 - 1) / (DEC_WARPS * 32), s0 = threadIdx.x * per, s1 = min(s0 + per, c.seqs);
    int sum = 0;
    for (int s = s0; s < s1; ++s) {
      length[s] = paged_length(c, s);
      sum += max(1, (length[s] + p.unit - 1) / p.unit);
    }
    int incl = sum;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, incl, w);
      if (lane >= w) incl += other;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int at = incl - sum, all = 0;
#pragma unroll
    for (int w = 0; w < DEC_WARPS; ++w) {
      if (w < warp) at += warp_sum[w];
      all += warp_sum[w];
    }
    extra = all * head_blocks > (int)gridDim.x ? 1 : 0;   // where a CTA has a unit at most, all cost the same
    for (int s = s0; s < s1; ++s) {
      before[s] = at + s * extra;
      at += max(1, (length[s] + p.unit - 1) / p.unit);
    }
    if (threadIdx.x == 0) before[c.seqs] = all + c.seqs * extra;
    __syncthreads();
  }
  const int units = before[c.seqs] * head_blocks;   // (the host has seen to it that they fit)
  const int ctas = min((int)gridDim.x, units);
  if ((int)blockIdx.x >= ctas) {
    if (threadIdx.x == 0 && p.open) p.open[blockIdx.x] = make_int4(-1, 0, 0, 0);
    return;
  }
  const unsigned each = (unsigned)units / ctas, left_over = units - each * ctas;
  auto start = [&](int i) { return (int)(each * i + left_over * i / (unsigned)ctas); };   // first unit of CTA i: units i / ctas
  int u = start(blockIdx.x);
  const int u_end = start(blockIdx.x + 1);
  int4 opened = make_int4(-1, 0, 0, 0);
  int b;   // the sequence of unit u
  {
    int lo = 0, hi = c.seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (before[mid] * head_blocks <= u) lo = mid; else hi = mid - 1;
    }
    b = lo;
  }

  // A run of units of one pair of sequence and key head; the extra unit comes first.  Nothing is done for a run of that
  // unit alone, the pair then begins in the next CTA (t0 is 1 there).
  int n_units, hb, t0, t1, key_from, key_end;
  auto enter = [&](int& seq, int unit) -> bool {
    while (before[seq + 1] * head_blocks <= unit) ++seq;
    n_units = before[seq + 1] - before[seq];
    const unsigned rest = unit - before[seq] * head_blocks;
    hb = rest / (unsigned)n_units;
    t0 = rest - hb * n_units;
    t1 = min(n_units, t0 + (u_end - unit));
    key_from = max(t0 - extra, 0) * p.unit;
    key_end = min(length[seq], (t1 - extra) * p.unit);
    return t1 > extra;
  };
  auto key_head = [&](int block) { return p.chunks == 1 ? block : block / p.chunks; };
  auto first_of = [&](int block) { return p.chunks == 1 ? 0 : block % p.chunks * Cfg::HEADS; };   // query head of the group
  // 16 keys from a multiple of 16 on lie in one page.  A lane holds the page of one of the next 32 steps of its warp.
  auto pages_from = [&](int seq, int key) {
    const int mine = key + lane * DEC_STEP;
    return mine < key_end ? paged_page(c, seq, mine >> c.page_shift) : -1;
  };
  // what a lane's rows and elements add to the first key's address; 16 rows of a page are less than 2^31 elements apart
  const int k_token = (int)c.k_token, v_token = (int)c.v_token, k_lane = r * k_token + q4 * 8, v_lane = q4 * 2 * v_token + r * 8;
  const int page_mask = (1 << c.page_shift) - 1;
  uint32_t q[NT][KJ][4], kr[2][KJ][4], vr[4][VJ][4];
  auto load_q = [&]() {
    const int h0 = first_of(hb), heads = p.group - h0;
    const uint16_t* base = p.x + b * p.x_row + (key_head(hb) * p.group + h0 + r) * p.x_head + q4 * 8;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < KJ; ++j) load16(q[t][j], base + t * 8 * p.x_head + j * 32, t * 8 + r < heads);
  };
  int pages;   // -1 where there is none
  auto load_k = [&](int key, int step) {
    const int page = __shfl_sync(0xffffffffu, pages, step), left = page < 0 ? 0 : key_end - key;
    const uint16_t* base = c.k + key_head(hb) * c.k_head + page * c.k_page + ((key & page_mask) * k_token + k_lane);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < KJ; ++j) load16(kr[i][j], base + (i * 8 * k_token + j * 32), r + i * 8 < left);
  };
  auto load_v = [&](int key, int step) {
    const int page = __shfl_sync(0xffffffffu, pages, step), left = page < 0 ? 0 : key_end - key;
    const uint16_t* base = c.v + key_head(hb) * c.v_head + page * c.v_page + ((key & page_mask) * v_token + v_lane);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = (i & 1) + (i >> 1) * 8;
#pragma unroll
      for (int j = 0; j < VJ; ++j) load16(vr[i][j], base + (row * v_token + j * 64), q4 * 2 + row < left);
    }
  };
  if (!enter(b, u)) {
    if (threadIdx.x == 0 && p.open) p.open[blockIdx.x] = opened;
    return;
  }
  pages = pages_from(b, key_from + warp * 16);
  float o[NT][VJ][4][4], m[NT][2], l[NT][2];
  int done_b = 0, done_hb = 0, done_t0 = 0, done_t1 = 0, done_units = 0, done_end = 0;
  bool done = false;   // a run whose warps have to be joined

  while (true) {
    // The queries and first keys and values of a run are on their way while the warps of the last one are joined.
    const bool live = u < u_end;
    if (live) {
      load_q();
      load_k(key_from + warp * 16, 0);
      load_v(key_from + warp * 16, 0);
    }
    if (done) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], w);
          if (r == 0) {
            sm_m[warp][t * 8 + q4 * 2 + e] = m[t][e];
            sm_l[warp][t * 8 + q4 * 2 + e] = l[t][e];
          }
#pragma unroll
          for (int j = 0; j < VJ; ++j) {
            float4* row = reinterpret_cast<float4*>(&sm_o[warp][t * 8 + q4 * 2 + e][j * 64 + r * 8]);
            row[0] = make_float4(o[t][j][0][e], o[t][j][0][e + 2], o[t][j][1][e], o[t][j][1][e + 2]);
            row[1] = make_float4(o[t][j][2][e], o[t][j][2][e + 2], o[t][j][3][e], o[t][j][3][e + 2]);
          }
        }
      __syncthreads();
      const int h0 = first_of(done_hb), first_head = key_head(done_hb) * p.group + h0, heads = min(Cfg::HEADS, p.group - h0);
      const bool whole = done_t0 <= extra && done_t1 == done_units;
      float* slot = p.parts + (2ll * blockIdx.x + (done_t0 <= extra)) * Cfg::SLOT;
      for (int i = threadIdx.x; i < Cfg::HEADS * (D / 8); i += DEC_WARPS * 32) {
        const int h = i / (D / 8), d = i % (D / 8) * 8;
        if (h >= heads) continue;
        float top = -CUDART_INF_F, sum = 0.f, acc[8] = {};
#pragma unroll
        for (int w = 0; w < DEC_WARPS; ++w) top = fmaxf(top, sm_m[w][h]);
#pragma unroll
        for (int w = 0; w < DEC_WARPS; ++w) {
          // a warp without keys has m = -inf, l = 0 and O = 0
          const float f = sm_m[w][h] == top ? 1.f : exp2f((sm_m[w][h] - top) * p.scale_log2);
          sum += f * sm_l[w][h];
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] += f * sm_o[w][h][d + e];
        }
        if (whole) {
          const float inv = done_end > 0 ? 1.f / sum : 0.f;
          *reinterpret_cast<uint4*>(p.out + ((long long)done_b * c.Hq + first_head + h) * D + d) =
              make_uint4(T::pack(acc[0] * inv, acc[1] * inv), T::pack(acc[2] * inv, acc[3] * inv), T::pack(acc[4] * inv, acc[5] * inv),
                         T::pack(acc[6] * inv, acc[7] * inv));
        } else {
          float4* dst = reinterpret_cast<float4*>(slot + h * D + d);
          dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
          dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
          if (d == 0) {
            slot[Cfg::HEADS * D + h] = top;
            slot[Cfg::HEADS * (D + 1) + h] = sum;
          }
        }
      }
      if (done_t0 <= extra && !whole) {
        const int last = before[done_b] * head_blocks + (done_hb + 1) * done_units - 1;   // unit of the pair
        int cta = (int)((float)last * ctas / units);
        while (start(cta) > last) --cta;
        while (start(cta + 1) <= last) ++cta;
        opened = make_int4(done_b, done_hb, cta, 0);
      }
      if (!live) break;
      __syncthreads();
    }
    const int first = key_from + warp * 16;
    int next_u = u + (t1 - t0);
    int next_pages = -1;
    if (next_u < u_end) {   // asked for now, needed when this run ends; kept in shared memory: working it out again cost 3 % of 256 short pairs
      const int keep[6] = {n_units, hb, t0, t1, key_from, key_end};
      int next_b = b;
      if (enter(next_b, next_u)) next_pages = pages_from(next_b, key_from + warp * 16);
      else next_u = u_end;
      if (lane == 0) {   // worked out once
        *reinterpret_cast<int4*>(next_run[warp]) = make_int4(n_units, hb, t0, t1);
        *reinterpret_cast<int4*>(next_run[warp] + 4) = make_int4(key_from, key_end, next_b, 0);
      }
      n_units = keep[0], hb = keep[1], t0 = keep[2], t1 = keep[3], key_from = keep[4], key_end = keep[5];
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t][0] = m[t][1] = -CUDART_INF_F;
      l[t][0] = l[t][1] = 0.f;
#pragma unroll
      for (int j = 0; j < VJ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[t][j][i][e] = 0.f;
    }

    int step = 0;   // of the steps whose pages the lanes hold
    for (int key = first; key < key_end; key += DEC_STEP) {
      const int next = key + DEC_STEP;
      if (++step == 32) {
        step = 0;
        pages = pages_from(b, next);
      }
      float s[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float even[4] = {0.f, 0.f, 0.f, 0.f}, odd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          mma16816<T>(even, kr[0][j][0], kr[1][j][0], kr[0][j][1], kr[1][j][1], q[t][j][0], q[t][j][1]);
          mma16816<T>(odd, kr[0][j][2], kr[1][j][2], kr[0][j][3], kr[1][j][3], q[t][j][2], q[t][j][3]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = even[e] + odd[e];
      }
      if (next < key_end) load_k(next, step);
      // element e of s: key r (+ 8 from e = 2 on), head 2 q4 + (e & 1)
      if (key + 16 > key_end) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key + r + (e >> 1) * 8 >= key_end) s[t][e] = -CUDART_INF_F;
      }
      // The reference m of the exponentials moves only when the maximum has grown by more than 2^8; O and l are divided by
      // each other in the end.  m is a score before its scale: the difference is exactly 0 at the maximum, whatever the scale.
      uint32_t pb[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float mx[2] = {fmaxf(s[t][0], s[t][2]), fmaxf(s[t][1], s[t][3])};
        if (__any_sync(0xffffffffu, (mx[0] - m[t][0]) * p.scale_log2 > 8.f || (mx[1] - m[t][1]) * p.scale_log2 > 8.f)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], w));
            const bool move = (mx[e] - m[t][e]) * p.scale_log2 > 8.f;
            const float alpha = move ? exp2f((m[t][e] - mx[e]) * p.scale_log2) : 1.f;
            if (move) m[t][e] = mx[e];
            l[t][e] *= alpha;
#pragma unroll
            for (int j = 0; j < VJ; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                o[t][j][i][e] *= alpha;
                o[t][j][i][e + 2] *= alpha;
              }
          }
        }
        const float r0 = m[t][0] == -CUDART_INF_F ? 0.f : m[t][0], r1 = m[t][1] == -CUDART_INF_F ? 0.f : m[t][1];
        float w[4] = {s[t][0] - r0, s[t][1] - r1, s[t][2] - r0, s[t][3] - r1};
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = exp2f(fmaf(w[e], p.scale_log2, T::WEIGHT_LOG2));
        if (key + 16 > key_end) {   // (-inf times a scale of 0 is no number)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key + r + (e >> 1) * 8 >= key_end) w[e] = 0.f;
        }
        l[t][0] += w[0] + w[2];
        l[t][1] += w[1] + w[3];
        // P in the cache's type, as the instruction wants it: half a step of relative error a weight, where fp16 has normal
        // numbers (from 2^-21 of the reference on; below, half a step of those, 2^-32 of the reference).  l sums the unrounded ones.
        pb[t][0] = transpose8x8(T::pack(w[0], w[1]));
        pb[t][1] = transpose8x8(T::pack(w[2], w[3]));
      }
#pragma unroll
      for (int j = 0; j < VJ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // rows 64 j + 8 r + 2 i and + 1 of V^T
          const uint32_t a0 = __byte_perm(vr[0][j][i], vr[1][j][i], 0x5410), a1 = __byte_perm(vr[0][j][i], vr[1][j][i], 0x7632);
          const uint32_t a2 = __byte_perm(vr[2][j][i], vr[3][j][i], 0x5410), a3 = __byte_perm(vr[2][j][i], vr[3][j][i], 0x7632);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma16816<T>(o[t][j][i], a0, a1, a2, a3, pb[t][0], pb[t][1]);
        }
      if (next < key_end) load_v(next, step);
    }

    done = true;
    done_b = b, done_hb = hb, done_t0 = t0, done_t1 = t1, done_units = n_units, done_end = key_end;
    u = next_u;
    if (u < u_end) {
      __syncwarp();
      const int4 run = *reinterpret_cast<const int4*>(next_run[warp]), more = *reinterpret_cast<const int4*>(next_run[warp] + 4);
      n_units = run.x, hb = run.y, t0 = run.z, t1 = run.w, key_from = more.x, key_end = more.y, b = more.z;
      pages = next_pages;
    }
  }
  if (threadIdx.x == 0 && p.open) p.open[blockIdx.x] = opened;
}

// Block (i, y): joins the parts of the pair that CTA i began, if it began one, for the query heads [y HB, (y + 1) HB).  A head
// at a time (HB = 1) where the pairs are few, so that many parts each are read side by side.
constexpr int JOIN_THREADS = 256;
template <typename T, int D, int NT, int HB>
__global__ void __launch_bounds__(JOIN_THREADS) decode_join_kernel(const DecParams p) {
  using Cfg = DecCfg<D, NT>;
  constexpr int LANES = D / 4, GROUPS = JOIN_THREADS / (LANES * HB), PART_LANES = JOIN_THREADS / HB;   // threads of a head
  constexpr int EARLY = 4;   // parts of O a thread asks for before it knows their weights
  __shared__ float4 acc_of[HB][GROUPS][LANES];
  __shared__ float red[HB][PART_LANES / 32], sum_of[HB][GROUPS];
  pdl_launch_dependents();
  pdl_wait();
  const int4 pair = p.open[blockIdx.x];
  if (pair.x < 0) return;
  const int mine = threadIdx.x / PART_LANES, tid = threadIdx.x % PART_LANES;
  const int h = blockIdx.y * HB + mine, h0 = pair.y % p.chunks * Cfg::HEADS, hk = pair.y / p.chunks;
  const int begin = blockIdx.x, parts = pair.z - begin + 1;
  auto slot = [&](int i) { return p.parts + (2ll * (begin + i) + (i == 0)) * Cfg::SLOT; };
  const int lane = tid % LANES, g = tid / LANES;
  struct Part {
    float4 o;
    float m, l;
  };
  auto fetch = [&](int i) -> Part {
    const float* at = slot(i);
    return {reinterpret_cast<const float4*>(at + h * D)[lane], at[Cfg::HEADS * D + h], at[Cfg::HEADS * (D + 1) + h]};
  };
  Part early[EARLY];
#pragma unroll
  for (int i = 0; i < EARLY; ++i)
    if (g + i * GROUPS < parts) early[i] = fetch(g + i * GROUPS);
  float top = -CUDART_INF_F;
  for (int i = tid; i < parts; i += PART_LANES) top = fmaxf(top, slot(i)[Cfg::HEADS * D + h]);
#pragma unroll
  for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
  if (PART_LANES > 32) {
    if ((tid & 31) == 0) red[mine][tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PART_LANES / 32; ++w) top = fmaxf(top, red[mine][w]);
  }
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  auto add = [&](const Part& a) {
    const float f = a.m == top ? 1.f : exp2f((a.m - top) * p.scale_log2);
    sum += f * a.l;
    acc = make_float4(acc.x + f * a.o.x, acc.y + f * a.o.y, acc.z + f * a.o.z, acc.w + f * a.o.w);
  };
#pragma unroll
  for (int i = 0; i < EARLY; ++i)
    if (g + i * GROUPS < parts) add(early[i]);
#pragma unroll 4
  for (int i = g + EARLY * GROUPS; i < parts; i += GROUPS) add(fetch(i));
  if (GROUPS > 1) {
    acc_of[mine][g][lane] = acc;
    if (lane == 0) sum_of[mine][g] = sum;
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int w = 1; w < GROUPS; ++w) {
      const float4 v = acc_of[mine][w][lane];
      acc = make_float4(acc.x + v.x, acc.y + v.y, acc.z + v.z, acc.w + v.w);
      sum += sum_of[mine][w];
    }
  }
  if (h >= p.group - h0) return;
  const float inv = 1.f / sum;
  *reinterpret_cast<uint2*>(p.out + ((long long)pair.x * p.c.Hq + hk * p.group + h0 + h) * D + lane * 4) =
      make_uint2(T::pack(acc.x * inv, acc.y * inv), T::pack(acc.z * inv, acc.w * inv));
}

// Loads in flight hold lines of the L1 cache, so the main kernel wants no more shared memory than its CTAs use, and the
// joining kernel has to ask for the same split: a kernel that starts while another one runs keeps the split that it finds.
// 256 sequences of up to 16384 tokens, 32 / 4 heads of 64: 339 us, 435 where the joining kernel took what it liked; with
// the most shared memory 128 sequences of up to 8192, 24 / 8 heads of 128, take 467 in place of 332 us.
template <typename Kern>
static bool shared_split(Kern kern, int bytes, PerDeviceFlags& flags) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const bool tracked = dev >= 0 && dev < kMaxDevicesPerProcess;
  if (tracked && __atomic_load_n(&flags.set[dev], __ATOMIC_ACQUIRE)) return true;
  const int percent = (bytes * 100 + 228 * 1024 - 1) / (228 * 1024);
  if (cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, percent) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  if (tracked) __atomic_store_n(&flags.set[dev], (unsigned char)1, __ATOMIC_RELEASE);
  return true;
}

struct DecPlan {
  int grid, chunks, unit;
  bool splits;   // whether a pair can cross CTAs
  long long bytes;
};

template <int D, int NT>
static DecPlan dec_plan(const incin_paged_desc* d) {
  using Cfg = DecCfg<D, NT>;
  DecPlan pl;
  pl.chunks = (d->Hq / d->Hkv + Cfg::HEADS - 1) / Cfg::HEADS;
  const long long seqs = d->seqs < DEC_SEQS ? d->seqs : DEC_SEQS;
  const long long steps = ((long long)d->table_width * d->page_size + DEC_STEP - 1) / DEC_STEP;
  const long long room = (long long)device_sm_count() * Cfg::CTAS_PER_SM, pairs = seqs * d->Hkv * pl.chunks;
  // Where the table holds up to four steps and every pair has a CTA, it stays with it and the joining kernel is not needed: one
  // sequence of 77 tokens, 12 heads of 64, 6.0 -> 4.5 us.  (With eight steps the join is worth it: 8 sequences of up to 500,
  // 32 / 4 heads of 64, 9.5 us a pair per CTA, 8.0 us split.  With several pairs a CTA it is, too: 256 sequences of up to 250,
  // 24 / 8 heads of 128, 42.7 us and 36.7.)
  const bool whole = steps <= 4 && pairs <= room;
  pl.unit = DEC_STEP * (whole ? (int)steps : 1);
  const long long per_pair = whole ? 1 : steps, most = pairs * per_pair;
  pl.grid = (int)(most < room ? most : room);
  pl.splits = per_pair > 1;
  pl.bytes = pl.splits ? (long long)pl.grid * (16 + 2 * Cfg::SLOT * 4) : 0;
  return pl;
}

template <typename T, int D, int NT>
static int launch_decode(const incin_paged_desc* d, cudaStream_t stream) {
  using Cfg = DecCfg<D, NT>;
  const DecPlan pl = dec_plan<D, NT>(d);
  if (pl.splits && !d->workspace) return INCIN_ERR_ARGUMENT;
  // units and the elements of 128 tokens are counted in 32 bits
  const long long per_seq = ((long long)d->table_width * d->page_size / pl.unit + 2) * d->Hkv * pl.chunks;
  if (per_seq >= (1ll << 30) || d->k_stride_token >= (1 << 23) || d->v_stride_token >= (1 << 23)) return INCIN_ERR_TOO_LARGE;
  const int slice = (int)(per_seq * DEC_SEQS < (1ll << 31) ? DEC_SEQS : ((1ll << 31) - 1) / per_seq);
  DecParams p = {paged_view(d), (const uint16_t*)d->x, d->x_stride_row, d->x_stride_head, (uint16_t*)d->out, d->scale * 1.4426950408889634f,
                 pl.unit, d->Hq / d->Hkv, pl.chunks, pl.splits ? (int4*)d->workspace : nullptr, (float*)((char*)d->workspace + 16ll * pl.grid)};
  p.c.offsets = nullptr;
  static PerDeviceFlags main_set, join_set, wide_join_set;
  if (!shared_split(decode_attention_kernel<T, D, NT>, Cfg::SHARED, main_set) || !shared_split(decode_join_kernel<T, D, NT, 1>, Cfg::SHARED, join_set) ||
      !shared_split(decode_join_kernel<T, D, NT, 8>, Cfg::SHARED, wide_join_set))
    return INCIN_ERR_LAUNCH;
  for (int s0 = 0; s0 < d->seqs; s0 += slice) {
    DecParams q = p;
    q.c.seqs = q.c.rows = d->seqs - s0 < slice ? d->seqs - s0 : slice;
    q.c.table += s0 * d->table_stride;
    q.c.lengths += s0;
    q.x += s0 * d->x_stride_row;
    q.out += (long long)s0 * d->Hq * D;
    // The main kernel is launched the ordinary way: 64 sequences of up to 4096, 32 / 4 heads of 64, 30.7 us, with programmatic
    // launches of both kernels 36.9.
    cudaError_t e = launch_pdl(decode_attention_kernel<T, D, NT>, dim3(pl.grid), dim3(DEC_WARPS * 32), 0, stream, q);
    if (e != cudaSuccess) return INCIN_ERR_LAUNCH;
    if (!pl.splits) continue;
    const bool few = (long long)q.c.seqs * d->Hkv * pl.chunks * 16 <= pl.grid;
    e = few ? launch_pdl<true>(decode_join_kernel<T, D, NT, 1>, dim3(pl.grid, Cfg::HEADS), dim3(JOIN_THREADS), 0, stream, q)
            : launch_pdl<true>(decode_join_kernel<T, D, NT, 8>, dim3(pl.grid, NT), dim3(JOIN_THREADS), 0, stream, q);
    if (e != cudaSuccess) return INCIN_ERR_LAUNCH;
  }
  return INCIN_OK;
}

}  // namespace incin

extern "C" long long incin_decode_attention_workspace(const incin_paged_desc* d) {
  using namespace incin;
  if (!d || d->Hkv <= 0 || d->Hq <= 0) return 0;
  const bool one = d->Hq / d->Hkv <= 8;
  if (d->D == 64) return one ? dec_plan<64, 1>(d).bytes : dec_plan<64, 2>(d).bytes;
  return one ? dec_plan<128, 1>(d).bytes : dec_plan<128, 2>(d).bytes;
}

extern "C" int incin_decode_attention(const incin_paged_desc* d, void* stream) {
  using namespace incin;
  const int rc = check_paged_attention(d);
  if (rc) return rc;
  if (d->rows != d->seqs) return INCIN_ERR_ARGUMENT;
  const cudaStream_t s = (cudaStream_t)stream;
  const bool one = d->Hq / d->Hkv <= 8;
  auto run = [&](auto t) {
    using T = decltype(t);
    if (d->D == 64) return one ? launch_decode<T, 64, 1>(d, s) : launch_decode<T, 64, 2>(d, s);
    return one ? launch_decode<T, 128, 1>(d, s) : launch_decode<T, 128, 2>(d, s);
  };
  return d->dtype == INCIN_GEMM_IN_FP16 ? run(Fp16()) : run(Bf16());
}
