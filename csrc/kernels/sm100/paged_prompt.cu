// Causal attention of packed runs of new tokens over a paged key-value cache.
//
// One persistent CTA per SM works on items: up to two 128-row query tiles of one sequence and key head, over a range of its
// keys.  The rows of a tile are (new token, query head of the key head), so that grouped heads share every key that is
// loaded and a run of a few tokens still fills a tile: with G query heads a key head a tile holds 128 / G tokens.  Where that is
// not a whole number two tiles share the heads of a token (256 tokens of 24 / 8 heads fill 6 tiles in place of 7: 126 -> 99 us
// behind 32768; 8191 alone 335 -> 325).  A box of the query map is {64 elements, G heads, the tokens that lie whole in a tile},
// one copy a half; the shared tokens' rows are fetched by the two warps that otherwise look over V tiles (by one-row copies they
// cost 2 us a tile at G = 12).  K and V tiles are 128 keys, fetched page
// by page (a box is one page of one head); the lanes of the producer warp hold the page numbers.
//
// The arithmetic and its schedule are those of the dense causal kernel (attention_fwd.cu): S_w = Q_w K^T into tensor memory, a
// softmax thread a row, P_w over S_w's columns, O_w += P_w V from tensor memory, the other tile's products meanwhile.  What
// is different here:
// - Items come from lengths that only the device knows.  The producer warp walks the sequences, 32 at a time by a scan
//   across its lanes, and hands items to the other warps through a ring.
// - Few rows over many keys: the keys of an item are split among `splits` CTAs, which leave fp32 parts (O, m, l) that a second
//   kernel joins in a fixed order.
// - The last page of a sequence has slots without tokens, and a tile's keys go past its first rows' own positions.  Scores
//   there are replaced by -inf, but P = 0 times a NaN or an infinity in V would still be NaN.  So two warps look over the V
//   tiles that hold such keys before the product reads them: rows behind the sequence become zeros, and non-finite
//   elements of keys that some row must not see become zeros and are added back, row by row, at the end (an item that had
//   any reads them from the cache again; a weight is positive, so the element itself is what the sum takes from it).
// - A CTA takes the next item when it has done its own (clusterlaunchcontrol: it takes over a CTA of the grid that has not
//   started).  Dealt out in advance, 16 runs of 8000 tokens in all took 119 us in place of 102, 32 / 4 heads of 64.
//
// Measured, and in operations a second: one run of 8191, 24 / 8 heads of 128, 327 to 335 us in short bursts, 1.23 to 1.26 PFLOP/s,
// 386 us, 1.07, call after call under the power cap (990 W; the dense kernel 317 and 368); 16 runs of 8000 in all, 32 / 4 heads of
// 64, 107 and 109 us, 0.49 (1965 MHz, 840 W); 256 tokens behind 32768, 24 / 8 heads of 128, 100 and 118 us, 1.03 and 0.87; 37
// tokens 7 us.
// What bounds it: a K / V tile takes a pair of query tiles 1.5 to 1.6 us at either head_dim, of which the tensor pipe, the
// special-function unit and tensor memory are each busy two thirds (ncu at head_dim 128: 62, 62 and 64 %); a warp's
// row takes 1420-1650 clocks for its exponentials (1024 at the unit's rate), 470-640 for its maximum, and waits 540-990 for its scores.
// Tried and slower, with that time in view: exponentials before the maximum is known (340 -> 355 us); the two warps of a
// scheduler taking turns with theirs (331 -> 393 us at head_dim 64); P in columns of its own at head_dim 64 and the next scores
// ahead of the product (331 -> 410); three regions for scores there, in turn, with the same aim (346 -> 361); masked tiles
// without the products and exponentials of keys that no row sees (102 -> 118); an eighth of the exponentials by a polynomial on the
// multiply-add units (326 -> 337, a quarter 342); the first scores of the next item between the last products of this one's tiles
// (104 -> 108); rows written as whole lines by four lanes each (nothing, without the cost of the exchange).
// 16 runs of 8000 in all: outside its tiles an item takes 4000 clocks, 16 % of the time (next item 800, first scores 1000, last product
// 350, epilogue 1700; head_dim 128: epilogue 3000, 6000 where it leaves fp32 parts).
// Without any maximum, as a limit, 1 % is gained.
#include "paged.cuh"

#include <math_constants.h>

namespace incin {

int make_operand_map(CUtensorMap* out, const void* ptr, long long inner, long long rows, long long ld, long long batch_lo,
                     long long stride_lo, long long batch_hi, long long stride_hi, int box_inner, int box_rows);
int make_operand_map_box(CUtensorMap* out, const void* ptr, long long inner, long long rows, long long ld, long long batch_lo,
                         long long stride_lo, long long batch_hi, long long stride_hi, int box_inner, int box_rows, int box_lo);

constexpr int PR_BM = 128;        // rows of a query tile, keys of a K / V tile
constexpr int PR_THREADS = 384;   // warp 0: items and TMA, 1: tcgen05 issue, 2-3: V tiles, 4-7 / 8-11: softmax of tile 0 / 1
// 384 threads are launched with 168 registers each: 128 x (104 + 200 + 200) = 64512.  (88 and 208: the producer's walk over the
// sequences spills, 8 runs of 8000 in all, 12 heads of 64, 57.5 us in place of 54.8; 120 and 192: 57.9.)
constexpr int PR_REGS_ISSUE = 104, PR_REGS_SOFTMAX = 200;
constexpr int PR_ITEMS = 3;       // slots of the item ring
constexpr float PR_FAR = 64.f;    // references past this, times scale log2(e), are taken off the scores in an instruction of their own

template <int D>
struct PrCfg {
  static constexpr int TILE_BYTES = PR_BM * D * 2;
  // Rings of K and of V tiles.  They are two because the warps that look over V tiles wait on each of a ring's barriers in
  // turn: a barrier tells its phases apart by parity alone, so who waits on it has to see every phase.
  static constexpr int K_STAGES = D == 128 ? 2 : 4, V_STAGES = D == 128 ? 3 : 4;
  static constexpr int OFF_K = 2 * TILE_BYTES, OFF_V = OFF_K + K_STAGES * TILE_BYTES;
  static constexpr int OFF_BAR = OFF_V + V_STAGES * TILE_BYTES;
  static constexpr int SMEM_BYTES = OFF_BAR + 1024 + 1024;
  // tensor memory: S_w (P_w in its first 64 columns) at [128 w, 128 w + 128), O_w at 256 + D w
  static constexpr int TMEM_COLS = 512, COL_O = 256;
  static constexpr int PART = 96;   // columns of P_w after which the first products of O_w += P_w V are let go
  static_assert(SMEM_BYTES <= 227 * 1024, "shared-memory plan");
};

struct PrItem {
  int seq, head;     // key head; -1 ends the list
  int row0, tokens;  // packed row of tile 0's first token, new tokens from there to the end of the sequence's run
  int head0;         // query head of the key head in tile 0's first row
  int pos0;          // position of that token (negative: more new tokens than the sequence has)
  int length;        // tokens of the sequence
  int lo, hi[2];     // K / V tiles [lo, hi[w]) for tile w
  int split;
  int direct;        // the keys are not split after all: the first split writes the result itself
  int odd;           // set when a non-finite element of a late key was taken out of a V tile
};

struct PrParams {
  PagedView c;
  const uint16_t* x;
  long long x_row, x_head;
  uint16_t* out;
  float scale_log2;
  int group;           // query heads of a key head
  uint32_t by_group;   // n / group = n by_group >> (31 + by_shift) for 0 <= n < 2^31: 2^by_shift is the next power of two from
  int by_shift;        // group on, by_group = 2^(31 + by_shift) / group, rounded up, so that the excess stays below 1 / group
  int tile_rows;       // rows of a tile that are used
  int box_tokens;      // tokens of tmQ's box
  int tiles;           // query tiles of an item: 2, or 1 where twice as many items are wanted
  int splits;
  float* part_o;       // [splits][rows][Hq][D]
  float2* part_ml;     // [splits][rows][Hq]: m (a score before its scale) and l; l = -1 for a row without a position, -2 in the first split of one that is done
};

template <typename T>
struct PrType;
template <>
struct PrType<Bf16> {
  static constexpr uint32_t FORMAT = 1, EXPONENT = 0x7f807f80u;
};
template <>
struct PrType<Fp16> {
  static constexpr uint32_t FORMAT = 0, EXPONENT = 0x7c007c00u;
};
// Whether either half of a word is an infinity or NaN: its exponent bits are all ones.
template <typename T>
__device__ __forceinline__ bool odd_word(uint32_t w) {
  return __vcmpeq2(w & PrType<T>::EXPONENT, PrType<T>::EXPONENT) != 0;
}

// Position in a ring of N stages.
template <int N>
struct PrRing {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == N) {
      stage = 0;
      phase ^= 1;
    }
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(PR_THREADS, 1)
prompt_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                        const PrParams p) {
  using Cfg = PrCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sK = smem + Cfg::OFF_K, *sV = smem + Cfg::OFF_V;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t *k_full = bars, *v_full = bars + 4;        // [STAGES <= 4] a K or V tile has landed
  uint64_t *k_empty = bars + 8, *v_empty = bars + 12;   // the products that read it have finished
  uint64_t* clean = bars + 16;        // [V_STAGES] a V tile has been looked over (two warps)
  uint64_t* q_full = bars + 24;       // [2] query tile w has landed
  uint64_t* q_empty = bars + 26;      // [2] the last score product of query tile w has finished
  uint64_t* s_full = bars + 28;       // [2] S_w is in tensor memory (and every earlier product has finished)
  uint64_t* p_full = bars + 30;       // [2] P_w is in tensor memory, O_w rescaled
  uint64_t* o_full = bars + 32;       // [2] O_w of this item is complete
  uint64_t* p_part = bars + 34;       // [2] the first PART columns of P_w are in tensor memory
  uint64_t* item_full = bars + 36;    // [PR_ITEMS]
  uint64_t* item_empty = bars + 40;   // [PR_ITEMS] one arrival a warp
  uint64_t* stolen = bars + 43;       // the answer about the next item has landed
  uint4* answer = reinterpret_cast<uint4*>(bars + 44);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 46);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  PrItem* items = reinterpret_cast<PrItem*>(bars + 48);   // [PR_ITEMS]

  const PagedView& c = p.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto by_group = [&](int n) { return (int)(__umulhi(2u * (uint32_t)n, p.by_group) >> p.by_shift); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < 4; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
      mbar_init(&clean[s], 2);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&q_full[w], 3);   // the box, single rows by two warps
      mbar_init(&q_empty[w], 1);
      mbar_init(&s_full[w], 1);
      mbar_init(&p_full[w], 4);
      mbar_init(&o_full[w], 1);
      mbar_init(&p_part[w], 4);
    }
    mbar_init(stolen, 1);
    for (int i = 0; i < PR_ITEMS; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 11);   // every warp but the producer
    }
    *abort_flag = 0;
    mbar_init_fence();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();   // tensor memory is held; a successor may be scheduled as CTAs retire
  pdl_wait();                // no global memory was touched above

  // The next item, for every warp but the producer: returned by value, `slot` kept until the warp lets go of it.
  auto take_item = [&](int i, PrItem& it) -> bool {
    const int slot = i % PR_ITEMS;
    if (!mbar_wait(&item_full[slot], (i / PR_ITEMS) & 1, abort_flag, c.status, kStatusTimeoutFull)) return false;
    it = items[slot];
    return it.head >= 0;
  };
  auto drop_item = [&](int i) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[i % PR_ITEMS]);
  };
  // Keys from this one on are not seen by every row of the item.
  auto late_from = [&](const PrItem& it) { return it.pos0 + 1; };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PR_REGS_ISSUE));
    if (warp == 0) {
      // ---------------------------------------------------------------- items and loads; warp-uniform, lanes issue copies
      const bool leader = elect_one() != 0;
      PrRing<Cfg::K_STAGES> k_at;
      PrRing<Cfg::V_STAGES> v_at;
      uint32_t q_phase[2] = {0, 0};
      bool ok = true;
      const int per_tile = PR_BM >> c.page_shift;   // pages of a K / V tile
      // sequences [chunk, chunk + 32): a lane's items and those in front of them
      int chunk = -32, before = 0, total = 0, my_items = 0, my_pairs = 0, my_upto = 0, my_row = 0, my_new = 0, my_len = 0;
      const int item_rows = p.tiles * p.tile_rows, group = p.group, per = c.Hkv * p.splits;
      // (offsets that overlap could name more items than fit; the grid has fewer indices)
      auto most_items = [](int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, 0x7fffffffu); };
      // An item per CTA of the grid; CTAs that run take over those that have not started.
      int idx = (int)blockIdx.x;
      const int begin = min(max(c.offsets[0], 0), c.rows), end = min(max(c.offsets[c.seqs], begin), c.rows);
      const long long row_vecs = (long long)c.Hq * (D / 8), outside = (long long)(begin + c.rows - end) * row_vecs;
      uint32_t steal_phase = 0;
      int published = 0;
      while (ok) {
        if (idx >= 0 && idx < before) chunk = -32, before = total = 0;   // (indices come in rising order)
        while (idx >= 0 && chunk < c.seqs && idx >= most_items(before, total)) {
          chunk += 32;
          before = most_items(before, total);
          const int s = chunk + lane;
          my_items = my_pairs = my_row = my_new = my_len = 0;
          if (s < c.seqs) {
            const int a = c.offsets[s], b = c.offsets[s + 1];
            my_row = min(max(a, 0), c.rows);
            my_new = min(max(b, my_row), c.rows) - my_row;
            my_len = paged_length(c, s);
            if (my_new > my_len || bad_offsets(c, a, b)) flag_bad_index(c.status);
            my_pairs = (my_new * group + item_rows - 1) / item_rows;
            my_items = my_pairs * per;
          }
          my_upto = my_items;
#pragma unroll
          for (int w = 1; w < 32; w <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, my_upto, w);
            if (lane >= w) my_upto = most_items(my_upto, other);
          }
          total = __shfl_sync(0xffffffffu, my_upto, 31);
        }
        PrItem it = {};
        it.head = -1;
        const bool there = idx >= 0 && chunk < c.seqs;   // the grid has an index for every item that there could be
        if (there) {
          const int at = idx - before;
          const int owner = __ffs(__ballot_sync(0xffffffffu, at < my_upto)) - 1;
          const int first = __shfl_sync(0xffffffffu, my_upto - my_items, owner), pairs = __shfl_sync(0xffffffffu, my_pairs, owner);
          const int row = __shfl_sync(0xffffffffu, my_row, owner), fresh = __shfl_sync(0xffffffffu, my_new, owner);
          it.length = __shfl_sync(0xffffffffu, my_len, owner);
          it.seq = chunk + owner;
          const int rest = at - first, behind = rest / per, k = rest - behind * per;
          const int pair = pairs - 1 - behind;   // the longest first
          it.head = p.splits == 1 ? k : k / p.splits;
          it.split = k - it.head * p.splits;
          const int t0 = by_group(pair * item_rows);
          it.head0 = pair * item_rows - t0 * group;
          it.row0 = row + t0;
          it.tokens = fresh - t0;
          it.pos0 = it.length - fresh + t0;
          int n[2];
#pragma unroll
          for (int w = 0; w < 2; ++w) {   // tiles up to the last row's own position
            const int at0 = it.head0 + w * p.tile_rows, last = it.pos0 + min(by_group(at0 + p.tile_rows - 1), it.tokens - 1);
            n[w] = w < p.tiles && by_group(at0) < it.tokens && last >= 0 ? last / PR_BM + 1 : 0;
          }
          // the host splits by what the table holds; at least three tiles a split are worth it
          const int most = max(n[0], n[1]), splits = min(p.splits, max(1, most / 3)), mine = min(it.split, splits);
          it.direct = splits == 1;
          it.lo = splits == 1 ? most * mine : (unsigned)(most * mine) / splits;
          const int hi = splits == 1 ? most : (unsigned)(most * min(mine + 1, splits)) / splits;   // (32 splits of 2^23 tiles at most)
          it.hi[0] = min(hi, n[0]);
          it.hi[1] = min(hi, n[1]);
        }
        if (there || idx < 0) {
          const int slot = published % PR_ITEMS;
          if (!mbar_wait(&item_empty[slot], ((published / PR_ITEMS) & 1) ^ 1, abort_flag, c.status, kStatusTimeoutEmpty)) break;
          if (lane == 0) {
            items[slot] = it;
            mbar_arrive(&item_full[slot]);
          }
          ++published;
          __syncwarp();
        }
        if (idx < 0) break;
        auto steal = [&]() {
          if (leader) {
            mbar_expect_tx(stolen, 16);
            steal_cta(answer, stolen);
          }
          __syncwarp();
        };
        const int hi = max(it.hi[0], it.hi[1]);
        const int entries = (it.length + (1 << c.page_shift) - 1) >> c.page_shift;   // pages with tokens
        auto load_q = [&](int w) -> bool {
          if (!mbar_wait(&q_empty[w], q_phase[w] ^ 1, abort_flag, c.status, kStatusTimeoutEmpty)) return false;
          q_phase[w] ^= 1;
          const int at0 = it.head0 + w * p.tile_rows, first_token = by_group(at0), first_head = at0 - first_token * group;
          const int front = first_head ? group - first_head : 0;
          if (leader) {
            mbar_expect_tx(&q_full[w], p.box_tokens * group * D * 2);
#pragma unroll
            for (int ch = 0; ch < D / 64; ++ch)
              tma_load_4d(smem + w * Cfg::TILE_BYTES + ch * (PR_BM * 128) + front * 128, &tmQ, &q_full[w], ch * 64, it.head * group,
                          it.row0 + first_token + (front > 0), 0);
          }
          __syncwarp();
          return true;
        };
        // a lane holds one of the next 32 page numbers; `pages` (out of range: zeros are filled in) where there is none
        int held_from = it.lo * per_tile, held;
        auto hold = [&](int from) {
          const int e = from + lane;
          const int page = e < entries ? paged_page(c, it.seq, e) : -1;
          return page < 0 ? c.pages : page;
        };
        held = hold(held_from);
        int ahead = hold(held_from + 32);
        auto load_kv = [&](const CUtensorMap* tm, uint8_t* ring, uint64_t* full, uint64_t* empty, auto& pos, int j) -> bool {
          if (!mbar_wait(&empty[pos.stage], pos.phase ^ 1, abort_flag, c.status, kStatusTimeoutEmpty)) return false;
          if (leader) mbar_expect_tx(&full[pos.stage], Cfg::TILE_BYTES);
          __syncwarp();
          const int box = lane % per_tile, ch = lane / per_tile;
          const int page = __shfl_sync(0xffffffffu, held, j * per_tile - held_from + box);
          if (ch < D / 64)
            tma_load_4d(ring + pos.stage * Cfg::TILE_BYTES + ch * (PR_BM * 128) + (box << c.page_shift) * 128, tm, &full[pos.stage], ch * 64, 0, it.head,
                        page);
          __syncwarp();
          pos.next();
          return true;
        };
        if (hi - it.lo <= 2) steal();
        if (hi > it.lo) {
          bool first_q = it.hi[0] > it.lo, second_q = it.hi[1] > it.lo;
          for (int j = it.lo; j < hi && ok; ++j) {
            if (j == hi - 2 && j > it.lo) steal();   // late, so that who is done first takes the next item
            if (j * per_tile >= held_from + 32) {
              held = ahead;
              held_from += 32;
              ahead = hold(held_from + 32);
            }
            if (first_q) ok = load_q(0);
            ok = ok && load_kv(&tmK, sK, k_full, k_empty, k_at, j);
            if (second_q) ok = ok && load_q(1);
            ok = ok && load_kv(&tmV, sV, v_full, v_empty, v_at, j);
            first_q = second_q = false;
          }
        }
        // rows outside every sequence give zeros: an equal share with every index of the grid, items or not
        for (long long z = (long long)idx * 32 + lane; z < outside; z += (long long)gridDim.x * 32) {
          const long long r = z / row_vecs, row = r < begin ? r : end + (r - begin);
          reinterpret_cast<uint4*>(p.out)[row * row_vecs + z % row_vecs] = make_uint4(0, 0, 0, 0);
        }
        ok = ok && mbar_wait(stolen, steal_phase, abort_flag, c.status, kStatusTimeoutFull);
        steal_phase ^= 1;
        if (ok) idx = stolen_cta(answer);
        fence_proxy_async_smem();   // the answer has been read before the next one is written
        __syncwarp();
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- products: one elected lane issues.  S_w(j+1) follows
      // O_w += P_w(j) V_j although it overwrites P_w: products of one issuing thread run in order (see attention_fwd.cu).
      const bool leader = elect_one() != 0;
      constexpr uint32_t idesc_s = idesc_with_format(make_idesc_bf16(PR_BM, PR_BM, false, false), PrType<T>::FORMAT);
      constexpr uint32_t idesc_o = idesc_with_format(make_idesc_bf16(PR_BM, D, false, true), PrType<T>::FORMAT);
      constexpr uint32_t kDescHi = ((1024u >> 4) & 0x3FFF) | (1u << 14) | (2u << 29);   // SBO 1024, version, SWIZZLE_128B
      constexpr uint32_t kLoK = (16u >> 4) << 16;                                       // K-major: LBO 16
      constexpr uint32_t kLoMN = ((uint32_t)(PR_BM * 128) >> 4) << 16;                  // MN-major V: 64-column chunks 16 KB apart
      auto desc = [&](uint32_t lo) -> uint64_t { return (static_cast<uint64_t>(kDescHi) << 32) | lo; };
      const uint32_t q16 = (smem_u32(smem) & 0x3FFFF) >> 4, k16 = (smem_u32(sK) & 0x3FFFF) >> 4, v16 = (smem_u32(sV) & 0x3FFFF) >> 4;
      uint32_t q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
      PrRing<Cfg::K_STAGES> k_at;
      PrRing<Cfg::V_STAGES> v_at;
      bool ok = true;
      auto scores = [&](int w, int k_stage) {   // S_w = Q_w K^T
        const uint32_t a = q16 + w * (Cfg::TILE_BYTES >> 4), bk = k16 + k_stage * (Cfg::TILE_BYTES >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * (PR_BM * 128 >> 4) + (kk & 3) * 2;
          if (leader) umma_f16_ss(tmem_base + w * PR_BM, desc(a + off + kLoK), desc(bk + off + kLoK), idesc_s, kk > 0 ? 1u : 0u);
        }
        if (leader) umma_commit(&s_full[w]);
        __syncwarp();
      };
      auto take = [&](uint64_t* full, auto& pos, int& my_stage) -> bool {   // next tile of a ring
        if (!mbar_wait(&full[pos.stage], pos.phase, abort_flag, c.status, kStatusTimeoutFull)) return false;
        my_stage = pos.stage;
        pos.next();
        return true;
      };
      auto take_v = [&](int& my_stage) -> bool {   // landed and looked over
        return mbar_wait(&clean[v_at.stage], v_at.phase, abort_flag, c.status, kStatusTimeoutFull) && take(v_full, v_at, my_stage);
      };
      PrItem it;
      for (int i = 0; ok && take_item(i, it); ++i) {
        const int lo = it.lo, hi = max(it.hi[0], it.hi[1]);
        if (hi > lo) {
          int k_stage = 0, v_stage = 0;
          ok = take(k_full, k_at, k_stage);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            if (!ok || it.hi[w] <= lo) continue;
            ok = mbar_wait(&q_full[w], q_phase[w], abort_flag, c.status, kStatusTimeoutFull);
            if (!ok) continue;
            q_phase[w] ^= 1;
            tc_fence_after();
            scores(w, k_stage);
            if (leader && it.hi[w] == lo + 1) umma_commit(&q_empty[w]);
          }
          if (ok && leader) umma_commit(&k_empty[k_stage]);
          for (int j = lo; j < hi && ok; ++j) {
            ok = take_v(v_stage);
            if (ok && j + 1 < hi) ok = take(k_full, k_at, k_stage);
            if (!ok) break;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              if (!ok || j >= it.hi[w]) continue;
              const uint32_t bv = v16 + v_stage * (Cfg::TILE_BYTES >> 4);
              // O_w += P_w V: 16 keys per product, P_w from tensor memory, the first products before all of P_w is there
              ok = mbar_wait(&p_part[w], p_phase[w], abort_flag, c.status, kStatusTimeoutTmemFull);
              if (!ok) continue;
              tc_fence_after();
#pragma unroll
              for (int kk = 0; kk < PR_BM / 16; ++kk) {
                if (kk == Cfg::PART / 16) {
                  ok = mbar_wait(&p_full[w], p_phase[w], abort_flag, c.status, kStatusTimeoutTmemFull);
                  if (!ok) break;
                  tc_fence_after();
                }
                if (leader) umma_f16_ts(tmem_base + Cfg::COL_O + w * D, tmem_base + w * PR_BM + kk * 8, desc(bv + kk * 128 + kLoMN), idesc_o,
                                        (j > lo || kk > 0) ? 1u : 0u);
              }
              if (!ok) continue;
              p_phase[w] ^= 1;
              if (j + 1 < it.hi[w]) {
                scores(w, k_stage);
                if (leader && j + 2 == it.hi[w]) umma_commit(&q_empty[w]);
              } else if (leader) {
                umma_commit(&o_full[w]);
              }
              __syncwarp();
            }
            if (ok && leader) {
              umma_commit(&v_empty[v_stage]);
              if (j + 1 < hi) umma_commit(&k_empty[k_stage]);
            }
            __syncwarp();
          }
        }
        drop_item(i);
      }
    } else {
      // ---------------------------------------------------------------- V tiles with late keys, and single query rows: 64 threads
      const int tid = (warp - 2) * 32 + lane;
      uint32_t q_phase = 0;   // a bit a tile
      PrRing<Cfg::V_STAGES> v_at;
      bool ok = true;
      PrItem it;
      for (int i = 0; ok && take_item(i, it); ++i) {
        // query rows in front of the box and behind it: heads of tokens that two tiles share
#pragma unroll 1
        for (int w = 0; w < 2 && ok; ++w) {
          if ((w ? it.hi[1] : it.hi[0]) <= it.lo) continue;
          ok = mbar_wait(&q_empty[w], (q_phase >> w & 1) ^ 1, abort_flag, c.status, kStatusTimeoutEmpty);
          if (!ok) break;
          q_phase ^= 1 << w;
          const int at0 = it.head0 + w * p.tile_rows, first_head = at0 - by_group(at0) * p.group;
          const int front = first_head ? p.group - first_head : 0, boxed = p.box_tokens * p.group;
          const int rows = front + min(max(it.tokens * p.group - at0 - front - boxed, 0), p.tile_rows - front - boxed);
#pragma unroll 4
          for (int i = tid; i < rows * (D / 8); i += 64) {
            const int u = i % (D / 8), r = i / (D / 8) < front ? i / (D / 8) : i / (D / 8) + boxed, token = by_group(at0 + r);
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(p.x + (it.row0 + token) * p.x_row +
                                                                 (it.head * p.group + at0 + r - token * p.group) * p.x_head + u * 8));
            *reinterpret_cast<uint4*>(smem + w * Cfg::TILE_BYTES + (u >> 3) * (PR_BM * 128) + r * 128 + (((u & 7) ^ (r & 7)) << 4)) = x;
          }
          if (rows) fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[w]);
        }
        const int hi = max(it.hi[0], it.hi[1]), late = late_from(it);
        for (int j = it.lo; j < hi && ok; ++j) {
          const int v_stage = v_at.stage;
          ok = mbar_wait(&v_full[v_stage], v_at.phase, abort_flag, c.status, kStatusTimeoutFull);
          if (!ok) break;
          v_at.next();
          if ((j + 1) * PR_BM <= late) {
            if (lane == 0) mbar_arrive(&clean[v_stage]);
            continue;
          }
          uint8_t* tile = sV + v_stage * Cfg::TILE_BYTES;
#pragma unroll 1
          for (int row = tid; row < PR_BM; row += 64) {
            const int key = j * PR_BM + row;
            if (key < late) continue;
            auto vec = [&](int ch, int u) { return reinterpret_cast<uint4*>(tile + ch * (PR_BM * 128) + row * 128 + ((u ^ (row & 7)) << 4)); };
            if (key >= it.length) {
#pragma unroll
              for (int u = 0; u < D / 8; ++u) *vec(u >> 3, u & 7) = make_uint4(0, 0, 0, 0);
              continue;
            }
            bool odd = false;
#pragma unroll
            for (int u = 0; u < D / 8; ++u) {
              const uint4 x = *vec(u >> 3, u & 7);
              odd |= odd_word<T>(x.x) || odd_word<T>(x.y) || odd_word<T>(x.z) || odd_word<T>(x.w);
            }
            if (odd) {
              items[i % PR_ITEMS].odd = 1;
              for (int u = 0; u < D / 8; ++u) {
                uint4 x = *vec(u >> 3, u & 7);
                uint32_t* xs = &x.x;
                for (int e = 0; e < 4; ++e) xs[e] &= ~__vcmpeq2(xs[e] & PrType<T>::EXPONENT, PrType<T>::EXPONENT);
                *vec(u >> 3, u & 7) = x;
              }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&clean[v_stage]);
        }
        drop_item(i);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PR_REGS_SOFTMAX));
    // ------------------------------------------------------------------ softmax / rescale / epilogue of query tile w
    const int w = (warp >> 2) - 1;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;  // row inside the tile == TMEM lane
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tmem_S = tmem_base + w * PR_BM + lane_addr, tmem_O = tmem_base + Cfg::COL_O + w * D + lane_addr;
    uint32_t s_phase = 0, o_phase = 0;
    bool ok = true;
    PrItem it;
    for (int i = 0; ok && take_item(i, it); ++i) {
      const int lo = it.lo, hi = it.hi[w];
      const int at0 = it.head0 + w * p.tile_rows, first_token = by_group(at0);
      const int mine = by_group(at0 + row), g = at0 + row - mine * p.group;   // token of the item and its query head
      const bool live_row = w < p.tiles && row < p.tile_rows && mine < it.tokens;
      const int limit = it.pos0 + (live_row ? mine : min(first_token, it.tokens - 1));   // the last key that the row sees
      const int all_see = it.pos0 + first_token;                 // ... and the last one that every row of the tile sees
      float m_ref = -CUDART_INF_F;   // a score before its scale
      float bias = T::WEIGHT_LOG2;   // less scale m_ref, where that is not taken off the scores themselves
      bool far = false;              // ... which the whole warp does when the reference of one of its rows is far from 0
      float2 l2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      for (int j = lo; j < hi; ++j) {
        if (!mbar_wait(&s_full[w], s_phase, abort_flag, c.status, kStatusTimeoutTmemFull)) { ok = false; break; }
        s_phase ^= 1;
        tc_fence_after();
        // whole S row into registers with back-to-back TMEM loads and a single wait
        uint32_t s[PR_BM];
#pragma unroll
        for (int ch = 0; ch < PR_BM / 32; ++ch) tmem_ld_32x32(tmem_S + ch * 32, reinterpret_cast<uint32_t(&)[32]>(s[ch * 32]));
        tmem_ld_wait();
        if (j * PR_BM + PR_BM - 1 > all_see) {   // masked scores become -inf
          const int last = limit - j * PR_BM;
#pragma unroll
          for (int e = 0; e < PR_BM; ++e)
            if (e > last) s[e] = __float_as_uint(-CUDART_INF_F);
        }
        float mx4[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};   // four chains, three-input maxima
#pragma unroll
        for (int e = 0; e < PR_BM; e += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k) mx4[k] = fmaxf(fmaxf(mx4[k], __uint_as_float(s[e + k * 2])), __uint_as_float(s[e + k * 2 + 1]));
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        // lazy rescale: only move the reference when the maximum grew by more than 2^8.  P = exp2(scale (s - m_ref)) as one
        // instruction, scale s - scale m_ref, is off by half a step of the rounded product, 2^-18 at most below PR_FAR;
        // past it, where it could be any power of 2, the difference comes first.  (16 runs of 8000 in all, 32 / 4
        // heads of 64: 104.6 us without it, 107.0 as it is; 113 with far references in a branch of their own in front of the
        // exponentials, 111 with scale times difference everywhere, 107.5 with the differences taken in tensor memory.)
        const bool need = (mx - m_ref) * p.scale_log2 > 8.0f, moves = __any_sync(0xffffffffu, need);
        if (moves || far) {
          const float alpha = need ? exp2f((m_ref - mx) * p.scale_log2) : 1.0f;   // 0 the first time
          if (need) m_ref = mx;
          const float ref = m_ref == -CUDART_INF_F ? 0.f : m_ref;   // a row that has only seen scores of -inf weighs them 0
          // (rows that hold no query have no say: what is in them changes from call to call)
          far = __any_sync(0xffffffffu, live_row && !(fabsf(ref * p.scale_log2) <= PR_FAR));
          bias = far ? T::WEIGHT_LOG2 : T::WEIGHT_LOG2 - ref * p.scale_log2;
          if (far) {
#pragma unroll
            for (int e = 0; e < PR_BM; ++e) s[e] = __float_as_uint(__uint_as_float(s[e]) - ref);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            l2[e].x *= alpha;
            l2[e].y *= alpha;
          }
          if (j > lo && moves) {   // s_full covers O_w += P_w(j-1) V_{j-1}: O_w is at rest
#pragma unroll 1
            for (int ch = 0; ch < D / 32; ++ch) {
              uint32_t o[32];
              tmem_ld_32x32(tmem_O + ch * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st_32x32(tmem_O + ch * 32, o);
            }
          }
        }
        // P in the cache's type over the first half of S_w's columns (half a step of relative error a weight; fp16 below 2^-21 of
        // the reference half a step of that, 2^-32), sums of the unrounded weights in fp32
        const float2 sc2 = make_float2(p.scale_log2, p.scale_log2), nm2 = make_float2(bias, bias);
#pragma unroll
        for (int ch = 0; ch < PR_BM / 32; ++ch) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 x = fma2(make_float2(__uint_as_float(s[ch * 32 + e]), __uint_as_float(s[ch * 32 + e + 1])), sc2, nm2);
            const float2 y = make_float2(exp2f(x.x), exp2f(x.y));
            l2[(e >> 1) & 1] = add2(l2[(e >> 1) & 1], y);
            pk[e >> 1] = T::pack(y.x, y.y);
          }
          tmem_st_32x16(tmem_S + ch * 16, pk);
          if ((ch + 1) * 32 == Cfg::PART) {
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_part[w]);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();                        // every lane's stores and fences precede the single arrival of its warp
        if (lane == 0) mbar_arrive(&p_full[w]);
      }
      const bool ran = hi > lo;
      if (ran) {
        if (!ok || !mbar_wait(&o_full[w], o_phase, abort_flag, c.status, kStatusTimeoutTmemFull)) { ok = false; break; }
        o_phase ^= 1;
        tc_fence_after();
      }
      const float l_sum = (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
      const long long out_row = (long long)(it.row0 + mine) * c.Hq + it.head * p.group + g;
      const bool odd = ran && *reinterpret_cast<volatile int*>(&items[i % PR_ITEMS].odd);
      const bool parts = p.splits > 1 && !(it.direct && it.split == 0), empty_part = it.direct && it.split > 0;
      const float inv = limit < 0 ? 0.f : parts ? 1.f : 1.0f / l_sum;
#pragma unroll 1
      for (int ch = 0; ch < (empty_part ? 0 : D / 32); ++ch) {
        uint32_t o[32];
        if (ran) {
          tmem_ld_32x32(tmem_O + ch * 32, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * inv);
        if (odd && live_row) {   // non-finite elements of late keys, left out of the products
          for (int key = max(late_from(it), lo * PR_BM); key <= min(limit, hi * PR_BM - 1); ++key) {
            const int page = paged_page(c, it.seq, key >> c.page_shift);
            if (page < 0) continue;
            const uint16_t* v = c.v + page * c.v_page + it.head * c.v_head + (key & ((1 << c.page_shift) - 1)) * c.v_token + ch * 32;
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const uint32_t x = *reinterpret_cast<const uint32_t*>(v + e);
              const uint32_t bad = __vcmpeq2(x & PrType<T>::EXPONENT, PrType<T>::EXPONENT);
              const float2 y = T::unpack(x);
              if (bad & 0xffffu) o[e] = __float_as_uint(__uint_as_float(o[e]) + y.x);
              if (bad >> 16) o[e + 1] = __float_as_uint(__uint_as_float(o[e + 1]) + y.y);
            }
          }
        }
        if (live_row && parts) {
          float* dst = p.part_o + ((long long)it.split * c.rows * c.Hq + out_row) * D + ch * 32;   // whole sectors, as below
#pragma unroll
          for (int u = 0; u < 4; ++u) st_global_b256(dst + u * 8, reinterpret_cast<uint32_t(&)[8]>(o[u * 8]));
        } else if (live_row) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) pk[e] = T::pack(__uint_as_float(o[e * 2]), __uint_as_float(o[e * 2 + 1]));
          uint16_t* dst = p.out + out_row * D + ch * 32;
          if (aligned32(dst)) {   // 32 bytes per store: whole sectors of the row
            st_global_b256(dst, reinterpret_cast<uint32_t(&)[8]>(pk[0]));
            st_global_b256(dst + 16, reinterpret_cast<uint32_t(&)[8]>(pk[8]));
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              *reinterpret_cast<uint4*>(dst + u * 8) = make_uint4(pk[u * 4], pk[u * 4 + 1], pk[u * 4 + 2], pk[u * 4 + 3]);
          }
        }
        __syncwarp();
      }
      if (live_row && p.splits > 1)
        p.part_ml[(long long)it.split * c.rows * c.Hq + out_row] = parts ? make_float2(m_ref, limit < 0 ? -1.f : l_sum) : make_float2(-CUDART_INF_F, -2.f);
      tc_fence_before();   // O_w has been read before the next item's first product, which follows this warp's p_part
      drop_item(i);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

// Joins the parts of a row and query head: a warp each.
template <typename T, int D>
__global__ void __launch_bounds__(256) prompt_join_kernel(const PrParams p) {
  constexpr int PER = D / 32;
  pdl_launch_dependents();
  pdl_wait();
  const PagedView& c = p.c;
  const long long n = (long long)c.rows * c.Hq, at = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int begin = min(max(c.offsets[0], 0), c.rows), end = min(max(c.offsets[c.seqs], begin), c.rows);
  if (at >= n || at / c.Hq < begin || at / c.Hq >= end) return;
  const float2 ml = lane < p.splits ? p.part_ml[lane * n + at] : make_float2(-CUDART_INF_F, 0.f);
  float top = ml.x;
#pragma unroll
  for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
  const float weight = ml.x == -CUDART_INF_F ? 0.f : ml.x == top ? 1.f : exp2f((ml.x - top) * p.scale_log2);
  if (__any_sync(0xffffffffu, ml.y == -2.f)) return;
  const bool nowhere = __any_sync(0xffffffffu, ml.y < 0.f);
  float sum = weight * ml.y, acc[PER] = {};
#pragma unroll
  for (int w = 16; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
  for (int i0 = 0; i0 < p.splits; i0 += 8) {   // eight parts on their way at a time
    float part[8][PER];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u < p.splits) {
#pragma unroll
        for (int e = 0; e < PER; e += 2) *reinterpret_cast<float2*>(&part[u][e]) = *reinterpret_cast<const float2*>(p.part_o + ((i0 + u) * n + at) * D + lane * PER + e);
      }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float f = __shfl_sync(0xffffffffu, weight, (i0 + u) & 31);
      if (i0 + u < p.splits) {   // one without weight, too: 0 times a value that is not finite is not 0
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] += f * part[u][e];
      }
    }
  }
  const float inv = nowhere ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < PER; e += 2) reinterpret_cast<uint32_t*>(p.out + at * D + lane * PER)[e / 2] = T::pack(acc[e] * inv, acc[e + 1] * inv);
}

struct PrPlan {
  int tile_rows, box_tokens, tiles, splits;
  long long items, bytes;
};

// Query tiles of an item and CTAs that share its keys, by the time that the longest items take in all, in ns.  Measured at
// head_dim 128 (24 / 8 heads) and 64 (32 / 4): a K / V tile takes a pair of query tiles 1580 and a single one 1460, an item's
// beginning and end 1500, the joining kernel 3500 and its parts' bytes.  256 tokens behind 32768: single tiles and two splits
// 217 us, pairs and four 129, six (the rule's) 100, nine 128; 500 tokens alone: single tiles 13.9 us, pairs 15.0, two splits 19.5.
static PrPlan pr_plan(const incin_paged_desc* d) {
  PrPlan pl = {};
  const int sms = device_sm_count();
  const int group = d->Hq / d->Hkv;
  // Groups that do not divide 128 fill all rows of a tile, too, up to 2 group - 2 of them one by one.  Large groups keep to whole
  // tokens.  Whole and shared, one run of 6000, two key heads of 128: 3 heads each 86.3 and 85.8 us, 12: 194 and 184, 24: 380 and
  // 363, 40: 640 and 608; one of 1000: 18.8 and 18.2, 22.7 and 22.6, 25.3 and 25.5, 39.7 and 44.8.
  const bool dense = PR_BM % group != 0 && group <= 24;
  pl.box_tokens = dense ? (PR_BM - group + 1) / group : PR_BM / group;
  pl.tile_rows = dense ? PR_BM : pl.box_tokens * group;
  const long long rows = (long long)d->rows * group;
  const long long keys = ((long long)d->table_width * d->page_size + PR_BM - 1) / PR_BM;   // K / V tiles of a sequence at most
  double best = 0;
  for (int tiles = 1; tiles <= 2; ++tiles)
    for (int splits = 1; splits <= 32 && (splits == 1 || splits * 2 <= keys); ++splits) {
      const long long n = ((rows + tiles * pl.tile_rows - 1) / (tiles * pl.tile_rows) + (d->seqs - 1) / 2) * d->Hkv * splits;
      if (splits > 1 && n > 2 * sms) break;
      const double rounds = n <= 3 * sms ? (double)((n + sms - 1) / sms) : (double)n / sms + 0.5;
      double time = rounds * ((double)((keys + splits - 1) / splits) * (tiles == 2 ? 1580 : 1460) + 1500);
      if (splits > 1) time += 3500 + (double)splits * d->rows * d->Hq * d->D * 8 / 2500;
      if (pl.tiles == 0 || time < best) best = time, pl.tiles = tiles, pl.splits = splits;
    }
  pl.items = (rows / (pl.tiles * pl.tile_rows) + d->seqs) * d->Hkv * pl.splits;   // at most
  pl.bytes = pl.splits > 1 ? (long long)pl.splits * d->rows * d->Hq * (d->D * 4 + 8) : 0;
  return pl;
}

template <typename T, int D>
static int launch_prompt(const incin_paged_desc* d, cudaStream_t stream) {
  using Cfg = PrCfg<D>;
  const PrPlan pl = pr_plan(d);
  if (pl.items > (1ll << 30) || (long long)d->rows * (d->Hq / d->Hkv) > 0x7fffff00) return INCIN_ERR_TOO_LARGE;   // counted in 32 bits
  if (pl.bytes && !d->workspace) return INCIN_ERR_ARGUMENT;
  const int group = d->Hq / d->Hkv;
  CUtensorMap tq, tk, tv;
  int rc = make_operand_map_box(&tq, d->x, D, d->Hq, d->Hq > 1 ? d->x_stride_head : D, d->rows, d->x_stride_row, 1, 0, 64, group, pl.box_tokens);
  if (rc) return rc;
  rc = make_operand_map(&tk, d->k_pages, D, d->page_size, d->k_stride_token, d->Hkv, d->k_stride_head, d->pages, d->k_stride_page, 64, d->page_size);
  if (rc) return rc;
  rc = make_operand_map(&tv, d->v_pages, D, d->page_size, d->v_stride_token, d->Hkv, d->v_stride_head, d->pages, d->v_stride_page, 64, d->page_size);
  if (rc) return rc;
  auto kern = prompt_attention_kernel<T, D>;
  static PerDeviceFlags attr;
  if (!ensure_dynamic_smem(kern, Cfg::SMEM_BYTES, attr)) return INCIN_ERR_LAUNCH;
  const long long n = (long long)d->rows * d->Hq;
  // A masked score of -inf times 0 would be NaN.  Scores below 2^100 times the least normal number change no weight.
  const float scale_log2 = fmaxf(d->scale * 1.4426950408889634f, 0x1p-126f);
  int by_shift = 0;
  while (1 << by_shift < group) ++by_shift;
  const PrParams p = {paged_view(d), (const uint16_t*)d->x, d->x_stride_row, d->x_stride_head, (uint16_t*)d->out, scale_log2,
                      group, (uint32_t)(((1ull << (31 + by_shift)) + group - 1) / group), by_shift, pl.tile_rows, pl.box_tokens, pl.tiles, pl.splits,
                      (float*)d->workspace, (float2*)((float*)d->workspace + pl.splits * n * D)};
  if (launch_pdl<true>(kern, dim3((unsigned)pl.items), dim3(PR_THREADS), Cfg::SMEM_BYTES, stream, tq, tk, tv, p) != cudaSuccess)
    return INCIN_ERR_LAUNCH;
  if (pl.splits > 1 &&
      launch_pdl<true>(prompt_join_kernel<T, D>, dim3((unsigned)((n + 7) / 8)), dim3(256), 0, stream, p) != cudaSuccess)
    return INCIN_ERR_LAUNCH;
  return INCIN_OK;
}

}  // namespace incin

extern "C" long long incin_prompt_attention_workspace(const incin_paged_desc* d) {
  if (!d || d->Hkv <= 0 || d->Hq < d->Hkv || d->Hq / d->Hkv > 128) return 0;
  return incin::pr_plan(d).bytes;
}

extern "C" int incin_prompt_attention(const incin_paged_desc* d, void* stream) {
  using namespace incin;
  const int rc = check_paged_attention(d);
  if (rc) return rc;
  if (!d->offsets) return INCIN_ERR_ARGUMENT;
  const cudaStream_t s = (cudaStream_t)stream;
  if (d->dtype == INCIN_GEMM_IN_FP16) return d->D == 64 ? launch_prompt<Fp16, 64>(d, s) : launch_prompt<Fp16, 128>(d, s);
  return d->D == 64 ? launch_prompt<Bf16, 64>(d, s) : launch_prompt<Bf16, 128>(d, s);
}
