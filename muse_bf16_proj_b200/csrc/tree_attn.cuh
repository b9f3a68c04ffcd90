// Attention of drafted tokens over a paged cache. Row (token t of request b, query head h) sees the request's
// cached tokens l < context[b], and drafted token j of its request (cached at context[b] + j) where bit j of
// its mask row is set (without a mask: j up to itself). With s_l = scale * q . K_l over what it sees,
//   out = sum_l exp(s_l) V_l / sum_l exp(s_l)   (0 where it sees nothing), times sigmoid(gate) if given.
//
// Bound: the cache is read once (4 * dim bytes a token and kv head), so up to a few dozen rows a kv head the kernel
// is a stream of K and V tiles from HBM; the matrix products only have to keep up.
//
// Shape. The rows of a request that share a kv head (tokens x heads / kv_heads) are one operand, cut into row tiles of
// kRows (16, 32, 64 or 128). Tokens are the tensor cores' M: a tile of 128 cached tokens gives
//   S^T [128 tokens x kRows] = K [128 x dim] . Q^T        (UMMA M = 128, N = kRows; K as stored, K-major)
//   O^T [dim x kRows]       += V^T [dim x 128] . P^T      (UMMA M = 128, N = kRows; V as stored, M-major)
// so both operands from the cache enter as the TMA wrote them, few rows cost few columns (N = 16) instead of
// idle lanes of a 128-row tile, and every softmax thread owns one token and all rows: with 8 rows a thread
// takes 8 exponentials a tile where a row-per-thread layout takes 128 on 8 lanes. dim = 64 runs the second
// product with M = 128 on 64 dims twice over (the copy's half is not read back).
//
// Softmax. P is taken against a reference maximum per row that only has to be within 2^8 of the true running
// maximum (P then stays below 256, exact enough in both 16-bit types and far from overflow in FP32 sums). A
// tile first checks whether any score passes its reference by more than that, one barrier reduction; only then are
// the row maxima reduced across the 128 tokens, the references moved and O^T and the sums rescaled. That happens on a
// run's first tile and rarely after. Sums of P are kept a thread (token) in FP32 and joined at the end of a run;
// they add the rounded 16-bit values that the second product uses, so that the rounding of P cancels in the
// quotient of rows that one token dominates.
//
// Split. One CTA an SM; all (request, row tile, kv head, token tile) units in that order are cut into equal
// contiguous runs, one a CTA, from lengths read on the device (no host synchronisation, graph-safe). A row tile
// that lies inside one CTA's run is finished there. One that crosses runs leaves (max, sum, O^T) FP32 partials in
// scratch, at most two a CTA, which tree_attn_join_kernel adds in run order: deterministic, no atomics.
//
// Warps: 0 producer (a lane a TMA box: boxes of min(page, 128) tokens x 64 dims, so any page size of 8 or more
// and any page order), 1 UMMA issue, then 4 (8 at kRows = 128) softmax warps of 32 TMEM lanes each.
//
// Entries that no row may see: tokens past the request's end are not loaded (or are whatever the page holds)
// and their V rows are zeroed in shared memory, because 0 x NaN is NaN; drafted tokens, which some rows see and
// others not, have non-finite V entries replaced by zero and added back at the end to the rows that do see them.
#pragma once

#include "ptx.cuh"
#include "rope_append.cuh"

namespace muse {

constexpr unsigned int kErrAttnDraft = 0xB01, kErrAttnTable = 0xB02, kErrAttnPage = 0xB03;
constexpr unsigned int kErrAttnProducer = 0xB11, kErrAttnMma = 0xB12, kErrAttnSoftmax = 0xB13, kErrAttnDrain = 0xB14;

constexpr int kAttnTok = 128;       // cached tokens a tile
constexpr float kAttnSlack = 8.f;   // log2 of how far a score may pass its row's reference maximum
constexpr float kAttnUnseen = -1e30f;  // reference of a row that has seen nothing: below every score, and finite

struct AttnArgs {
  const uint16_t *q, *gate, *k_pages, *v_pages;
  uint16_t* out;
  const int32_t *table, *context, *starts;
  const uint32_t* mask;
  long long q_token, q_head, gate_token, gate_head, out_token, out_head;
  long long k_page, k_head, k_slot, v_page, v_head, v_slot;
  long long table_row, mask_row;
  long long pages;
  int requests, tokens, max_draft, table_cols, heads, kv_heads, page, mask_words;
  float scale_log2;  // scale * log2(e)
  long long* prefix;  // scratch: [requests + 1] tiles before each request
  float2* part_ml;    // scratch: [ctas][2][kRows] (reference maximum, sum)
  float* part_o;      // scratch: [ctas][2][kRows][dim]
};

// Shared memory of a variant: K and V rings, Q, P, then the small arrays.
template <int kDim, int kRows>
struct AttnShape {
  static constexpr int kHalves = kDim / 64;
  static constexpr int kStage = kAttnTok * kDim * 2;           // one K or V tile
  static constexpr int kQ = kRows * kDim * 2;
  static constexpr int kP = kAttnTok * kRows * 2;
  static constexpr int kNP = kRows == 128 && kDim == 128 ? 1 : 2;  // P buffers
  static constexpr int kNK = kDim == 64 ? (kRows <= 32 ? 6 : (kRows == 64 ? 5 : 4)) : (kRows <= 64 ? 3 : 2);
  static constexpr int kNV = kDim == 64 ? kNK : (kRows <= 32 ? 3 : 2);
  static constexpr int kGroups = kRows == 128 ? 2 : 1;         // softmax warpgroups, each its own columns
  static constexpr int kCols = kRows / kGroups;                // columns (rows of Q) a group
  static constexpr int kThreads = 64 + 128 * kGroups;
  static constexpr int kTmem = kRows == 16 ? 64 : (kRows == 32 ? 128 : (kRows == 64 ? 256 : 512));
  static constexpr int kOffV = kNK * kStage, kOffQ = kOffV + kNV * kStage, kOffP = kOffQ + kQ, kOffSmall = kOffP + kNP * kP;
  // ref, rescale, 1 / sum and row ids [kRows]; red [4][kRows]; mask words [kRows][8]; barriers.
  static constexpr int kSmall = kRows * 4 * 4 + 4 * kRows * 4 + kRows * 32 + (2 * kNK + 2 * kNV + 9) * 8 + 64;
  static constexpr int kSmem = 1024 + kOffSmall + kSmall;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

struct AttnReq {
  int first, drafted, ctx, kv, tiles, rows;  // first token, drafted tokens, context, entries, token tiles, rows a kv head
  long long units;                           // kv heads x row tiles
};

// A request's sizes, clamped to what may be touched whatever the device arrays hold.
template <int kRows>
__device__ __forceinline__ AttnReq attn_request(const AttnArgs& a, int b, bool report) {
  AttnReq r;
  const int lo = a.starts[b], hi = a.starts[b + 1], ctx = a.context[b];
  r.first = min(max(lo, 0), a.tokens);
  int t = min(max(hi, r.first), a.tokens) - r.first;
  if (report && (r.first != lo || t != hi - lo || t > a.max_draft || ctx < 0)) report_error(kErrAttnDraft);
  t = min(t, a.max_draft);
  r.drafted = t;
  r.ctx = max(ctx, 0);
  const long long have = static_cast<long long>(a.table_cols) * a.page, want = static_cast<long long>(r.ctx) + t;
  if (report && t > 0 && want > have) report_error(kErrAttnTable);
  r.kv = static_cast<int>(min(want, have));
  r.tiles = t > 0 ? (r.kv + kAttnTok - 1) / kAttnTok : 0;
  r.rows = t * (a.heads / a.kv_heads);
  r.units = static_cast<long long>(a.kv_heads) * ((r.rows + kRows - 1) / kRows);
  return r;
}

// `total` tiles over at most `ctas` runs of at least one tile: how many runs, where run c starts, and
// which run holds tile w (the largest c that starts at or before it).
__device__ __forceinline__ int attn_runs(long long total, int ctas) { return static_cast<int>(min(total, static_cast<long long>(ctas))); }
__device__ __forceinline__ long long attn_run_start(long long total, int c, int runs) { return total * c / runs; }
__device__ __forceinline__ int attn_run_of(long long total, long long w, int runs) {
  return static_cast<int>(((w + 1) * runs - 1) / total);
}

// Walks a CTA's run segment by segment (a segment: consecutive token tiles of one row tile and kv head).
struct AttnSeg {
  int b, head, row0, i0, i1;  // request, kv head, first row, token tiles [i0, i1)
  long long unit0;            // tiles before this unit, over all requests
  AttnReq r;
};
template <int kRows>
struct AttnWalk {
  long long left, base;  // tiles left in the run; tiles before request b
  long long unit;
  int b, i;
  AttnReq r;
  __device__ __forceinline__ AttnWalk(const AttnArgs& a, int b0, long long base0, long long w0, long long w1)
      : left(w1 - w0), base(base0), unit(0), b(b0), i(0) {
    if (left > 0) {
      r = attn_request<kRows>(a, b, false);
      const long long off = w0 - base;
      unit = off / r.tiles;
      i = static_cast<int>(off - unit * r.tiles);
    }
  }
  __device__ __forceinline__ bool next(const AttnArgs& a, AttnSeg& s) {
    if (left <= 0) return false;
    while (unit >= r.units || r.tiles == 0) {
      base += r.units * r.tiles;
      if (++b >= a.requests) return false;
      r = attn_request<kRows>(a, b, false);
      unit = 0;
      i = 0;
    }
    s.b = b;
    s.r = r;
    // Row tiles of one kv head follow one another, so that CTAs that share cached tokens run side by side.
    const int row_tiles = (r.rows + kRows - 1) / kRows;
    s.head = static_cast<int>(unit / row_tiles);
    s.row0 = static_cast<int>(unit % row_tiles) * kRows;
    s.unit0 = base + unit * r.tiles;
    s.i0 = i;
    s.i1 = static_cast<int>(min(static_cast<long long>(r.tiles), i + left));
    left -= s.i1 - s.i0;
    ++unit;
    i = 0;
    return true;
  }
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3,
                                            uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "l"(policy)
      : "memory");
}

// 16 columns of this warp's 32 TMEM lanes, not waited for; attn_ld_wait ties the registers to the wait.
__device__ __forceinline__ void attn_ld16(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr));
}
__device__ __forceinline__ void attn_ld_wait(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                 "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])::"memory");
}
__device__ __forceinline__ void attn_st16(uint32_t taddr, const float* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
      "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
      : "memory");
}
__device__ __forceinline__ void attn_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void bar_named(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
// Barrier that also tells every thread whether any had `p`.
__device__ __forceinline__ bool bar_any(int id, int threads, bool p) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbarrier.cta.red.or.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"(static_cast<uint32_t>(p))
      : "memory");
  return r != 0u;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// lo += p.lo, hi += p.hi for a packed pair of 16-bit values.
template <bool kHalf>
__device__ __forceinline__ void add16x2(uint32_t p, float& lo, float& hi) {
  if constexpr (kHalf) {
    asm("{\n\t.reg .b16 a, b, o;\n\tmov.b32 {a, b}, %2;\n\tmov.b16 o, 0x3C00;\n\t"
        "fma.rn.f32.f16 %0, a, o, %0;\n\tfma.rn.f32.f16 %1, b, o, %1;\n\t}"
        : "+f"(lo), "+f"(hi)
        : "r"(p));
  } else {
    fma_bf16x2(p, 0x3F803F80u, lo, hi);
  }
}

// kN (32 or 16) values a lane reduced over the warp's lanes by halving: afterwards lane l holds column l
// (32) or l / 2 (16) in v[0].
template <int kN, bool kMax>
__device__ __forceinline__ void warp_fold(float* v, int lane) {
  int n = kN;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool up = (lane & o) != 0;
#pragma unroll
      for (int j = 0; j < kN / 2; ++j) {
        if (j < n) {
          const float give = up ? v[j] : v[j + n], keep = up ? v[j + n] : v[j];
          const float got = __shfl_xor_sync(0xffffffffu, give, o);
          v[j] = kMax ? fmaxf(keep, got) : keep + got;
        }
      }
    } else {
      const float got = __shfl_xor_sync(0xffffffffu, v[0], o);
      v[0] = kMax ? fmaxf(v[0], got) : v[0] + got;
    }
  }
}

// UMMA descriptor of an M- or N-major 16-bit operand: `row` bytes of M/N entries a k row (swizzled at that width),
// groups of 8 k rows 8 * row apart, `chunk` bytes between runs of 64 M/N entries.
__host__ __device__ constexpr uint64_t attn_mn_desc_bits(int row, int chunk) {
  return (static_cast<uint64_t>(chunk >> 4) << 16) | (static_cast<uint64_t>((8 * row) >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
         (static_cast<uint64_t>(row == 128 ? 2 : (row == 64 ? 4 : 6)) << 61);
}

template <bool kHalf, int kDim, int kRows>
__global__ void __launch_bounds__(AttnShape<kDim, kRows>::kThreads, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const AttnArgs a) {
  using Sh = AttnShape<kDim, kRows>;
  constexpr int kHalves = Sh::kHalves, kNK = Sh::kNK, kNV = Sh::kNV, kNP = Sh::kNP, kCols = Sh::kCols;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_align<1024>(smem_raw);
  uint8_t* ring_k = smem;
  uint8_t* ring_v = smem + Sh::kOffV;
  uint8_t* q_s = smem + Sh::kOffQ;
  uint8_t* p_s = smem + Sh::kOffP;
  float* ref = reinterpret_cast<float*>(smem + Sh::kOffSmall);  // reference maximum (scaled, log2)
  float* rescale = ref + kRows;
  float* inv = rescale + kRows;
  int* row_id = reinterpret_cast<int*>(inv + kRows);             // token of the request << 16 | query head
  float* red = reinterpret_cast<float*>(row_id + kRows);         // [4][kRows]
  uint32_t* words = reinterpret_cast<uint32_t*>(red + 4 * kRows);  // [kRows][8]: drafted tokens a row sees
  uint64_t* k_full = reinterpret_cast<uint64_t*>(words + kRows * 8);
  uint64_t* k_empty = k_full + kNK;
  uint64_t* v_full = k_empty + kNK;
  uint64_t* v_empty = v_full + kNV;
  uint64_t* s_full = v_empty + kNV;  // [2]
  uint64_t* p_full = s_full + 2;     // [2]
  // [2], by tile parity: a softmax thread may look at a phase up to two tiles late, and one barrier's parity
  // would by then name the next phase.
  uint64_t* pv_done = p_full + 2;
  uint64_t* q_full = pv_done + 2;
  uint64_t* fin = q_full + 1;
  long long* start_s = reinterpret_cast<long long*>(fin + 1);  // first request's tiles before it
  int* start_b = reinterpret_cast<int*>(start_s + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(start_b + 1);
  int* odd_v = reinterpret_cast<int*>(tmem_slot + 1);  // a drafted token of this segment has a non-finite V entry

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&tmk);
    prefetch_tensormap(&tmv);
    for (int i = 0; i < kNK; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < kNV; ++i) mbar_init(&v_full[i], 1), mbar_init(&v_empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 128 * Sh::kGroups), mbar_init(&pv_done[i], 1);
    mbar_init(q_full, 128 * Sh::kGroups);
    mbar_init(fin, 1);
    fence_mbar_init();
    *start_b = a.requests;
    *odd_v = 0;
  }
  if (warp == 1) tmem_alloc(tmem_slot, Sh::kTmem);
  pdl_launch_dependents();
  pdl_wait();

  // Tiles before each request: a scan over the requests by the whole CTA, a run of requests a thread.
  long long total = 0, before = 0;
  const int each = (a.requests + Sh::kThreads - 1) / Sh::kThreads;
  const int b_lo = min(static_cast<int>(threadIdx.x) * each, a.requests), b_hi = min(b_lo + each, a.requests);
  {
    long long* sums = reinterpret_cast<long long*>(red);
    long long mine = 0;
    for (int b = b_lo; b < b_hi; ++b) {
      const AttnReq r = attn_request<kRows>(a, b, blockIdx.x == 0);
      mine += r.units * r.tiles;
    }
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    for (int w = 0; w < Sh::kThreads / 32; ++w) {
      if (w < warp) before += sums[w];
      total += sums[w];
    }
    before += upto - mine;
    __syncthreads();
  }
  const int runs = attn_runs(total, gridDim.x);
  long long w0 = 0, w1 = 0;
  if (static_cast<int>(blockIdx.x) < runs) w0 = attn_run_start(total, blockIdx.x, runs), w1 = attn_run_start(total, blockIdx.x + 1, runs);
  {
    long long at = before;
    for (int b = b_lo; b < b_hi; ++b) {
      const AttnReq r = attn_request<kRows>(a, b, false);
      if (blockIdx.x == 0) a.prefix[b] = at;
      const long long end = at + r.units * r.tiles;
      if (at <= w0 && w0 < end) *start_s = at, *start_b = b;
      at = end;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.prefix[a.requests] = total;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int b0 = *start_b;
  const bool work = w0 < w1 && b0 < a.requests;
  const uint32_t tmem_o = tmem + 2 * kRows;

  if (warp == 0) {
    // ---- producer: lane = one box ------------------------------------------------------------------
    if (work) {
      int issued_k = 0, issued_v = 0;
      AttnWalk<kRows> walk(a, b0, *start_s, w0, w1);
      AttnSeg s;
      const int box = min(a.page, kAttnTok), boxes = kAttnTok / box;
      const int mine = lane % boxes, half = lane / boxes;  // this lane's box of the tile and 64-dim half
      // Tokens that several row tiles read stay in L2; a request's only reader streams them.
      const uint64_t stream = policy_evict_first(), keep = policy_evict_normal();
      Ring rk, rv;
      bool ok = true;
      while (ok && walk.next(a, s)) {
        const uint64_t policy = s.r.rows > kRows ? keep : stream;
        const int32_t* row = a.table + s.b * a.table_row;
        int page = 0;
        bool have = false;
        auto lookup = [&](int i) {
          const int pos = i * kAttnTok + mine * box;
          have = half < kHalves && pos < s.r.kv;
          page = have ? row[pos / a.page] : 0;
        };
        lookup(s.i0);
        for (int i = s.i0; i < s.i1; ++i) {
          const int now = page, in = (i * kAttnTok + mine * box) % a.page;
          const bool go = have;
          if (go && (now < 0 || now >= a.pages)) report_error(kErrAttnPage);  // reads as zeros: outside the map
          if (i + 1 < s.i1) lookup(i + 1);
          const uint32_t bytes = static_cast<uint32_t>(__popc(__ballot_sync(0xffffffffu, go)) * box * 128);
          const uint32_t off = static_cast<uint32_t>(half * (kAttnTok * 128) + mine * box * 128);
          ok = mbar_wait(&k_empty[rk.slot], rk.phase ^ 1u, kErrAttnProducer);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          if (lane == 0) mbar_expect_tx(&k_full[rk.slot], bytes);
          __syncwarp();
          if (go) tma_load_4d(ring_k + rk.slot * Sh::kStage + off, &tmk, &k_full[rk.slot], half * 64, in, s.head, now, policy);
          rk.next(kNK);
          ++issued_k;
          ok = mbar_wait(&v_empty[rv.slot], rv.phase ^ 1u, kErrAttnProducer);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          if (lane == 0) mbar_expect_tx(&v_full[rv.slot], bytes);
          __syncwarp();
          if (go) tma_load_4d(ring_v + rv.slot * Sh::kStage + off, &tmv, &v_full[rv.slot], half * 64, in, s.head, now, policy);
          rv.next(kNV);
          ++issued_v;
        }
      }
      // No copy may be in flight when the CTA ends, whichever way it does.
      for (int n = max(issued_k - kNK, 0); n < issued_k; ++n)
        mbar_wait(&k_full[n % kNK], static_cast<uint32_t>((n / kNK) & 1), kErrAttnDrain, kWaitLimitNs / 100);
      for (int n = max(issued_v - kNV, 0); n < issued_v; ++n)
        mbar_wait(&v_full[n % kNV], static_cast<uint32_t>((n / kNV) & 1), kErrAttnDrain, kWaitLimitNs / 100);
    }
  } else if (warp == 1) {
    // ---- UMMA issue --------------------------------------------------------------------------------
    if (work && lane == 0) {
      AttnWalk<kRows> walk(a, b0, *start_s, w0, w1);
      AttnSeg s;
      constexpr uint32_t kType = kHalf ? 0u : ((1u << 7) | (1u << 10));
      constexpr uint32_t kShape = (1u << 4) | (static_cast<uint32_t>(kRows >> 3) << 17) | (8u << 24);
      constexpr uint32_t idesc_s = kShape | kType, idesc_o = kShape | kType | (1u << 15) | (1u << 16);
      constexpr int kPRow = kRows >= 64 ? 128 : kRows * 2;  // bytes of a token's row of P
      constexpr uint64_t v_bits = attn_mn_desc_bits(128, kDim == 128 ? kAttnTok * 128 : 0);
      constexpr uint64_t p_bits = attn_mn_desc_bits(kPRow, kRows == 128 ? kAttnTok * 128 : 0);
      Ring rk, rv;
      uint32_t seg_phase = 0, n = 0;
      bool ok = true;
      auto issue_s = [&](uint32_t m) {
        if (!mbar_wait(&k_full[rk.slot], rk.phase, kErrAttnMma)) return false;
        tc_fence_after();
        const uint64_t dk = umma_desc_sw128(smem_u32(ring_k + rk.slot * Sh::kStage)), dq = umma_desc_sw128(smem_u32(q_s));
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_bf16(tmem + (m & 1u) * kRows, dk + ((h * kAttnTok * 128) >> 4) + 2 * k, dq + ((h * kRows * 128) >> 4) + 2 * k, idesc_s,
                      (h | k) != 0);
        umma_commit(&k_empty[rk.slot]);
        umma_commit(&s_full[m & 1u]);
        rk.next(kNK);
        return true;
      };
      while (ok && walk.next(a, s)) {
        ok = mbar_wait(q_full, seg_phase, kErrAttnMma);
        seg_phase ^= 1u;
        if (!ok) break;
        tc_fence_after();
        ok = issue_s(n);
        for (int i = s.i0; ok && i < s.i1; ++i, ++n) {
          // The next tile's scores are under way while the softmax of this one runs.
          if (i + 1 < s.i1 && !(ok = issue_s(n + 1))) break;
          ok = mbar_wait(&p_full[n & 1u], (n >> 1) & 1u, kErrAttnMma) && mbar_wait(&v_full[rv.slot], rv.phase, kErrAttnMma);
          if (!ok) break;
          tc_fence_after();
          const uint64_t dv = v_bits | ((smem_u32(ring_v + rv.slot * Sh::kStage) & 0x3FFFFu) >> 4);
          const uint64_t dp = p_bits | ((smem_u32(p_s + (n % kNP) * Sh::kP) & 0x3FFFFu) >> 4);
#pragma unroll
          for (int k = 0; k < kAttnTok / 16; ++k)
            umma_bf16(tmem_o, dv + ((k * 16 * 128) >> 4), dp + ((k * 16 * kPRow) >> 4), idesc_o, (i > s.i0 || k > 0) ? 1u : 0u);
          umma_commit(&v_empty[rv.slot]);
          umma_commit(&pv_done[n & 1u]);
          rv.next(kNV);
        }
      }
      umma_commit(fin);
      mbar_wait(fin, 0u, kErrAttnDrain, kWaitLimitNs / 10);  // nothing of the tensor cores is under way past here
    }
    __syncwarp();
  } else if (work) {
    // ---- softmax: thread = one token of the tile (TMEM lane), all columns of its group --------------
    const int tid = static_cast<int>(threadIdx.x) - 64, group = tid >> 7;
    const int quarter = warp & 3, token = quarter * 32 + lane, gtid = tid & 127;
    const int c0 = group * kCols;
    const int bar = 1 + group;
    constexpr int kAll = 128 * Sh::kGroups;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const int g = a.heads / a.kv_heads;
    const float kNegInf = __int_as_float(0xff800000);
    const float c = a.scale_log2;
    AttnWalk<kRows> walk(a, b0, *start_s, w0, w1);
    AttnSeg s;
    uint32_t n = 0;  // tiles done in this run
    uint32_t v_slot = 0, v_phase = 0;
    bool ok = true;
    float l[kCols];
    while (ok && walk.next(a, s)) {
      // ---- the segment's rows: Q, mask words, references -------------------------------------------
      const int rows = min(kRows, s.r.rows - s.row0);
      const int full = min(kRows, (rows + 15) & ~15);  // columns that are computed
      const int live = min(max(full - c0, 0), kCols);  // of this group
      bar_named(3, kAll);                              // every thread is done with the last segment's arrays
      for (int i = tid; i < full * (kDim / 8); i += kAll) {
        const int r = i / (kDim / 8), ch = i % (kDim / 8);
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows) {
          const int row = s.row0 + r, t = row / g;
          v = ldg_cg_v4(a.q + (s.r.first + t) * a.q_token + (s.head * g + row - t * g) * a.q_head + ch * 8);
        }
        const uint32_t at = smem_u32(q_s) + (ch >> 3) * (kRows * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
        st_shared_v4u(at, v.x, v.y, v.z, v.w);
      }
      const int nw = (s.r.drafted + 31) >> 5;
      for (int i = tid; i < full * nw; i += kAll) {
        const int r = i / nw, w = i - r * nw;
        uint32_t v = 0u;
        if (r < rows) {
          const int t = (s.row0 + r) / g;
          // Bits up to the token itself without a mask; nothing past the request's tokens.
          const int last = a.mask ? s.r.drafted : t + 1;
          v = a.mask ? a.mask[(s.r.first + t) * a.mask_row + w] : 0xffffffffu;
          const int nb = min(last, s.r.drafted) - w * 32;
          v &= nb >= 32 ? 0xffffffffu : (nb <= 0 ? 0u : (1u << nb) - 1u);
        }
        words[r * 8 + w] = v;
      }
      if (tid < kRows) {
        const int row = min(s.row0 + tid, s.r.rows - 1), t = row / g;
        ref[tid] = kAttnUnseen;
        row_id[tid] = (t << 16) | (s.head * g + row - t * g);
      }
      if (tid == 0) *odd_v = 0;
      fence_proxy_async_shared();
      mbar_arrive(q_full);
      bar_named(3, kAll);
#pragma unroll
      for (int j = 0; j < kCols; ++j) l[j] = 0.f;

      // ---- tiles -----------------------------------------------------------------------------------
      for (int i = s.i0; ok && i < s.i1; ++i, ++n) {
        ok = mbar_wait(&s_full[n & 1u], (n >> 1) & 1u, kErrAttnSoftmax);
        // P's buffer is free, and with two of them PV of two tiles ago is done, once this has passed.
        if (n >= static_cast<uint32_t>(kNP)) ok = mbar_wait(&pv_done[(n - kNP) & 1u], ((n - kNP) >> 1) & 1u, kErrAttnSoftmax) && ok;
        tc_fence_after();
        float x[kCols];
        const uint32_t ts = tmem + (n & 1u) * kRows + c0 + lanes;
#pragma unroll
        for (int cc = 0; cc < kCols; cc += 16)
          if (cc < live) attn_ld16(ts + cc, x + cc);
#pragma unroll
        for (int cc = 0; cc < kCols; cc += 16)
          if (cc < live) attn_ld_wait(x + cc);
        const int pos = i * kAttnTok + token;
        const bool edge = (i + 1) * kAttnTok > s.r.ctx;  // the tile reaches past the context
        const float cm = edge ? 1.f : c;                 // scores of an edge tile are scaled here, with their mask
        if (edge) {
          const int j = pos - s.r.ctx;
#pragma unroll
          for (int k = 0; k < kCols; ++k) {
            if (k < live) {
              const bool seen = j < 0 || (pos < s.r.kv && ((words[(c0 + k) * 8 + (j >> 5)] >> (j & 31)) & 1u));
              x[k] = seen ? x[k] * c : kNegInf;
            }
          }
        }
        bool past = false;
#pragma unroll
        for (int cc = 0; cc < kCols; cc += 4) {
          if (cc < live) {
            const float4 m = *reinterpret_cast<const float4*>(ref + c0 + cc);
            past |= fmaf(x[cc], cm, -m.x) > kAttnSlack;
            past |= fmaf(x[cc + 1], cm, -m.y) > kAttnSlack;
            past |= fmaf(x[cc + 2], cm, -m.z) > kAttnSlack;
            past |= fmaf(x[cc + 3], cm, -m.w) > kAttnSlack;
          }
        }
        if (bar_any(bar, 128, past || !ok)) {
          if (bar_any(bar, 128, !ok)) {
            ok = false;
            break;
          }
          // Move the references to the true maxima and rescale what was summed against the old ones.
          constexpr int kFold = kCols < 32 ? kCols : 32;
#pragma unroll
          for (int cc = 0; cc < kCols; cc += kFold) {
            float top[kFold];
#pragma unroll
            for (int j = 0; j < kFold; ++j) top[j] = cc + j < live ? x[cc + j] * cm : kNegInf;
            warp_fold<kFold, true>(top, lane);
            if (kFold == 32 || !(lane & 1)) red[quarter * kRows + c0 + cc + (kFold == 32 ? lane : lane >> 1)] = top[0];
          }
          bar_named(bar, 128);
          if (gtid < kCols) {
            const int col = c0 + gtid;
            const float old = ref[col];
            const float now = fmaxf(fmaxf(fmaxf(red[col], red[kRows + col]), fmaxf(red[2 * kRows + col], red[3 * kRows + col])), old);
            ref[col] = now;
            rescale[col] = ex2(old - now);
          }
          bar_named(bar, 128);
#pragma unroll
          for (int j = 0; j < kCols; ++j)
            if (j < live) l[j] *= rescale[c0 + j];
          if (i > s.i0) {
            ok = mbar_wait(&pv_done[(n - 1) & 1u], ((n - 1) >> 1) & 1u, kErrAttnSoftmax);
            tc_fence_after();
#pragma unroll
            for (int cc = 0; cc < kCols; cc += 16) {
              if (cc < live) {
                float o[16];
                attn_ld16(tmem_o + c0 + cc + lanes, o);
                attn_ld_wait(o);
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] *= rescale[c0 + cc + k];
                attn_st16(tmem_o + c0 + cc + lanes, o);
              }
            }
            attn_st_wait();
          }
        }
        // P, rounded, as the second product reads it (a score that is not seen is -inf, its P zero).
        const uint32_t pt = smem_u32(p_s + (n % kNP) * Sh::kP);
#pragma unroll
        for (int cc = 0; cc < kCols; cc += 8) {
          if (cc < live) {
            const float4 m0 = *reinterpret_cast<const float4*>(ref + c0 + cc), m1 = *reinterpret_cast<const float4*>(ref + c0 + cc + 4);
            const float m[8] = {m0.x, m0.y, m0.z, m0.w, m1.x, m1.y, m1.z, m1.w};
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              w[k] = pack16x2<kHalf>(ex2(fmaf(x[cc + 2 * k], cm, -m[2 * k])), ex2(fmaf(x[cc + 2 * k + 1], cm, -m[2 * k + 1])));
              add16x2<kHalf>(w[k], l[cc + 2 * k], l[cc + 2 * k + 1]);
            }
            const int ch = (c0 + cc) >> 3;
            uint32_t at;
            if constexpr (kRows == 16) at = token * 32 + ((ch ^ ((token >> 2) & 1)) << 4);
            else if constexpr (kRows == 32) at = token * 64 + ((ch ^ ((token >> 1) & 3)) << 4);
            else at = (ch >> 3) * (kAttnTok * 128) + token * 128 + (((ch & 7) ^ (token & 7)) << 4);
            st_shared_v4u(pt + at, w[0], w[1], w[2], w[3]);
          }
        }
        if (group == 0) {
          // V rows that not every row sees (see above). They are in the last tile or two of a request.
          const bool ragged = (i + 1) * kAttnTok > s.r.kv, drafted = edge && s.r.drafted > 1;
          if (ragged || drafted) {
            ok = mbar_wait(&v_full[v_slot], v_phase, kErrAttnSoftmax);
            const uint32_t vt = smem_u32(ring_v + v_slot * Sh::kStage) + token * 128;
            if (pos >= s.r.kv) {
#pragma unroll
              for (int ch = 0; ch < kDim / 8; ++ch) st_shared_v4u(vt + (ch >> 3) * (kAttnTok * 128) + (ch & 7) * 16, 0u, 0u, 0u, 0u);
            } else if (drafted && pos >= s.r.ctx) {
              constexpr uint32_t kExp = kHalf ? 0x7C00u : 0x7F80u;
#pragma unroll
              for (int ch = 0; ch < kDim / 8; ++ch) {
                const uint32_t at = vt + (ch >> 3) * (kAttnTok * 128) + (ch & 7) * 16;
                const uint4 v = ld_shared_v4u(at);
                uint32_t e[4] = {v.x, v.y, v.z, v.w};
                bool odd = false;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  if ((e[k] & kExp) == kExp) e[k] &= 0xFFFF0000u, odd = true;
                  if ((e[k] & (kExp << 16)) == (kExp << 16)) e[k] &= 0x0000FFFFu, odd = true;
                }
                if (odd) {
                  st_shared_v4u(at, e[0], e[1], e[2], e[3]);
                  *odd_v = 1;
                }
              }
            }
          }
        }
        if (++v_slot == kNV) v_slot = 0, v_phase ^= 1u;
        fence_proxy_async_shared();
        tc_fence_before();
        mbar_arrive(&p_full[n & 1u]);
      }
      ok = !bar_any(3, kAll, !ok);
      if (!ok) break;

      // ---- end of the segment: finish the row tile, or leave a partial -----------------------------
      constexpr int kFold = kCols < 32 ? kCols : 32;
#pragma unroll
      for (int cc = 0; cc < kCols; cc += kFold) {
        warp_fold<kFold, false>(l + cc, lane);
        if (kFold == 32 || !(lane & 1)) red[quarter * kRows + c0 + cc + (kFold == 32 ? lane : lane >> 1)] = l[cc];
      }
      bar_named(bar, 128);
      const bool whole = s.i0 == 0 && s.i1 == s.r.tiles;
      // The run that starts inside a row tile keeps its partial first, the one that ends inside it second.
      const long long slot = (static_cast<long long>(blockIdx.x) * 2 + (s.i0 > 0 ? 0 : 1)) * kRows;
      if (gtid < kCols) {
        const int col = c0 + gtid;
        const float sum = (red[col] + red[kRows + col]) + (red[2 * kRows + col] + red[3 * kRows + col]);
        inv[col] = sum == 0.f ? 0.f : 1.f / sum;
        if (!whole && col < rows) a.part_ml[slot + col] = make_float2(ref[col], sum);
      }
      ok = mbar_wait(&pv_done[(n - 1) & 1u], ((n - 1) >> 1) & 1u, kErrAttnSoftmax);
      ok = !bar_any(3, kAll, !ok);
      if (!ok) break;
      tc_fence_after();
      const int odd = *odd_v;
#pragma unroll
      for (int cc = 0; cc < kCols; cc += 16) {
        if (cc < live) {
          float o[16];
          attn_ld16(tmem_o + c0 + cc + lanes, o);
          attn_ld_wait(o);
          if (token < kDim) {
            if (odd) {
              // Put the non-finite entries back for the rows that see them.
              const int j0 = max(s.i0 * kAttnTok - s.r.ctx, 0), j1 = min(min(s.i1 * kAttnTok, s.r.kv) - s.r.ctx, s.r.drafted);
              for (int j = j0; j < j1; ++j) {
                const int p = s.r.ctx + j;
                const long long page = a.table[s.b * a.table_row + p / a.page];
                if (page < 0 || page >= a.pages) continue;
                const float v = lo16<kHalf>(a.v_pages[page * a.v_page + s.head * a.v_head + (p % a.page) * a.v_slot + token]);
                if (!(fabsf(v) < __int_as_float(0x7f800000)))
#pragma unroll
                  for (int k = 0; k < 16; ++k)
                    if ((words[(c0 + cc + k) * 8 + (j >> 5)] >> (j & 31)) & 1u) o[k] += v;
              }
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const int col = c0 + cc + k;
              if (col < rows) {
                if (whole) {
                  const int id = row_id[col], t = id >> 16, h = id & 0xFFFF;
                  float v = o[k] * inv[col];
                  if (a.gate) v /= 1.f + __expf(-lo16<kHalf>(a.gate[(s.r.first + t) * a.gate_token + h * a.gate_head + token]));
                  a.out[(s.r.first + t) * a.out_token + h * a.out_head + token] =
                      static_cast<uint16_t>(pack16x2<kHalf>(v, v) & 0xFFFFu);
                } else {
                  a.part_o[(slot + col) * kDim + token] = o[k];
                }
              }
            }
          }
        }
      }
      tc_fence_before();
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Sh::kTmem);
  }
}

// Joins the partials of the row tiles that cross runs: one warp an output row. Weighs each partial by
// 2^(its reference - the largest), in run order.
template <bool kHalf, int kDim, int kRows>
__global__ void __launch_bounds__(128) tree_attn_join_kernel(const AttnArgs a, int ctas) {
  constexpr int kN = kDim / 32;
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long at = static_cast<long long>(blockIdx.x) * 4 + warp;
  if (at >= static_cast<long long>(a.tokens) * a.heads) return;
  const int t = static_cast<int>(at / a.heads), h = static_cast<int>(at % a.heads);
  // The request with starts[b] <= t < starts[b + 1], 32 candidates a step.
  int lo = 0, hi = a.requests;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int cand = lo + lane * step;
    const unsigned int below = __ballot_sync(0xffffffffu, cand < hi && a.starts[cand] <= t);
    const int k = 31 - __clz(static_cast<int>(below | 1u));
    lo += k * step;
    hi = min(hi, lo + step);
  }
  const long long total = a.prefix[a.requests];
  const AttnReq r = attn_request<kRows>(a, lo, false);
  const int inner = t - r.first;
  if (inner < 0 || inner >= r.drafted) return;
  const int g = a.heads / a.kv_heads, head = h / g, row = inner * g + h - head * g;
  const int row_tiles = (r.rows + kRows - 1) / kRows;
  const long long w0 = a.prefix[lo] + (static_cast<long long>(head) * row_tiles + row / kRows) * r.tiles, w1 = w0 + r.tiles;
  const int runs = attn_runs(total, ctas);
  const int c0 = attn_run_of(total, w0, runs), c1 = attn_run_of(total, w1 - 1, runs);
  if (c0 == c1) return;  // finished by its CTA
  const int col = row % kRows;
  auto slot = [&](int c) { return (static_cast<long long>(c) * 2 + (attn_run_start(total, c, runs) > w0 ? 0 : 1)) * kRows + col; };
  float top = kAttnUnseen;
  for (int c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, a.part_ml[slot(c)].x);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float acc[kN], sum = 0.f;
#pragma unroll
  for (int i = 0; i < kN; ++i) acc[i] = 0.f;
  for (int c = c0; c <= c1; c += 32) {
    float w = 0.f, part = 0.f;
    long long mine = 0;
    if (c + lane <= c1) {
      mine = slot(c + lane);
      const float2 ml = a.part_ml[mine];
      w = ex2(ml.x - top);  // 0 for a partial that saw nothing beside one that saw something
      part = ml.y * w;
    }
    const int n = min(32, c1 - c + 1);
#pragma unroll 8
    for (int k = 0; k < n; ++k) {
      const float wk = __shfl_sync(0xffffffffu, w, k);
      sum += __shfl_sync(0xffffffffu, part, k);
      const float* src = a.part_o + __shfl_sync(0xffffffffu, mine, k) * kDim + lane * kN;
      if constexpr (kN == 4) {
        const float4 v = *reinterpret_cast<const float4*>(src);
        acc[0] += wk * v.x, acc[1] += wk * v.y, acc[2] += wk * v.z, acc[3] += wk * v.w;
      } else {
        const float2 v = *reinterpret_cast<const float2*>(src);
        acc[0] += wk * v.x, acc[1] += wk * v.y;
      }
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint32_t packed[kN / 2];
#pragma unroll
  for (int i = 0; i < kN; i += 2) {
    float v[2] = {acc[i] * inv, acc[i + 1] * inv};
    if (a.gate) {
      const uint32_t gw = *reinterpret_cast<const uint32_t*>(a.gate + t * a.gate_token + h * a.gate_head + lane * kN + i);
      v[0] /= 1.f + __expf(-lo16<kHalf>(gw));
      v[1] /= 1.f + __expf(-hi16<kHalf>(gw));
    }
    packed[i / 2] = pack16x2<kHalf>(v[0], v[1]);
  }
  uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + t * a.out_token + h * a.out_head + lane * kN);
  if constexpr (kN == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(packed[0], packed[1]);
  else dst[0] = packed[0];
}

}  // namespace muse
