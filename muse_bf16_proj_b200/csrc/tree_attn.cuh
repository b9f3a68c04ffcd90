// Attention of drafted tokens over a paged cache. Row (token t of request b, query head h) sees the request's
// cached tokens l < context[b], and drafted token j of its request (cached at context[b] + j) where bit j of
// its mask row is set (without a mask: j up to itself). With s_l = scale * q . K_l over what it sees,
//   out = sum_l exp(s_l) V_l / sum_l exp(s_l)   (0 where it sees nothing), times sigmoid(gate) if given.
//
// Bound: the cache is read once (4 * dim bytes a token and kv head), so up to a few dozen rows a kv head the kernel
// is a stream of K and V tiles from HBM; the matrix products only have to keep up. Measured with the join, 8 kv heads of
// 128, bf16, device time of a call: 537 MB of cache (one token of 64 heads over 131072 entries) in 83.6 us = 6.42 TB/s, 0.98
// of a plain copy's rate; 336 MB (32 requests of 1024 to 4096 entries, pages of 16) in 58.1 us = 5.78 TB/s, 0.88: about 3 us
// pass before the first tile and 3 us in the join. Short calls are latency: 700 entries of 2 heads of 64 take 9.1 us, of
// which the cut of the runs is 1 us, the first Q and K 2 us and the join 2.4 us.
//
// Shape. The rows of a request that share a kv head (tokens x heads / kv_heads) are one operand, cut into row tiles of
// kRows (16 or 32; more rows take the rows-as-M kernel of tree_attn_wide.cuh). Tokens are the tensor cores'
// M: a tile of 128 cached tokens (256 at dim 64) gives
//   S^T [128 tokens x kRows] = K [128 x dim] . Q^T        (UMMA M = 128, N = kRows; K as stored, K-major)
//   O^T [dim x kRows]       += V^T [dim x 128] . P^T      (UMMA M = 128, N = kRows; V as stored, M-major)
// so both operands from the cache enter as the TMA wrote them, few rows cost few columns (N = 16) instead of
// idle lanes of a 128-row tile, and every softmax thread owns one token and all rows: with 8 rows a thread
// takes 8 exponentials a tile where a row-per-thread layout takes 128 on 8 lanes. dim = 64 runs the second
// product with M = 128 on 64 dims twice over (the copy's half is not read back).
//
// Softmax. P is taken against a reference per row that only has to be within 2^8 of the true running maximum (P then
// stays below 256 and its sums far from overflow in FP32). FP16 holds little below 1 (halving steps end at 2^-24, and the
// many small weights of a long context may add up to a share of the result), so its reference is set 2^7 below the
// maximum: P stays within 2^15, weights down to 2^-31 of the largest keep a bit, and the factor cancels in the quotient. A
// tile first checks whether any score passes its reference by more than allowed, one barrier reduction; only then are
// the row maxima reduced across the 128 tokens, the references moved and O^T and the sums rescaled. That happens on a
// run's first tile and rarely after. P is rounded to the cache's type because the second product's operands have one
// type, which is V's; its weights are then off by up to 2^-9 (BF16) or 2^-12 (FP16) each, and results are 1.1 to 1.4 times
// as far from the exact ones as with P in FP32 (one token over 131072 entries 2.3e-3 against 1.7e-3, of which the output's
// own rounding is 1.7e-3). Sums of P are kept a thread (token) in FP32 and joined at the end of a run; they add the rounded
// values that the second product uses, so that the rounding of P cancels in the quotient of rows that one token dominates.
// ex2.approx (about 2^-22) and, in the gate, __expf and __fdividef (under 2^-18 up to |gate| = 20) are far below either.
//
// Split. One CTA an SM; all (request, row tile, kv head, token tile) units in that order are cut into equal
// contiguous runs, one a CTA, from lengths read on the device (no host synchronisation, graph-safe). A row tile
// that lies inside one CTA's run is finished there. One that crosses runs leaves (max, sum, O^T) FP32 partials in
// scratch, at most two a CTA, which tree_attn_join_kernel adds in run order: deterministic, no atomics.
//
// Warps: 0 brings K and V (a lane a TMA box of min(page, tile) tokens: any page size of 8 or more and any page order),
// 1 issues the UMMAs, then 4 or 8 softmax warps of 32 TMEM lanes each, then the row loader. All but the producer wait
// asleep (mbar_wait_idle): polling warps take issue slots from those at work (11 x 13: 29.4 us polling, 28.6 asleep).
//
// Entries that no row may see: tokens past the request's end are not loaded (or are whatever the page holds)
// and their V rows are zeroed in shared memory, because 0 x NaN is NaN; drafted tokens, which some rows see and
// others not (a mask may hide a request's only one from all of them), have non-finite V entries replaced by zero and
// added back at the end to the rows that do see them.
#pragma once

#include "ptx.cuh"
#include "rope_append.cuh"

namespace muse {

constexpr unsigned int kErrAttnDraft = 0xB01, kErrAttnTable = 0xB02, kErrAttnPage = 0xB03;
constexpr unsigned int kErrAttnProducer = 0xB11, kErrAttnMma = 0xB12, kErrAttnSoftmax = 0xB13, kErrAttnDrain = 0xB14,
                       kErrAttnLoader = 0xB15;

// log2 of how far below a row's maximum its reference is set, and of how far above the reference a score may be.
template <bool kHalf>
constexpr float kAttnBelow = kHalf ? 7.f : 0.f;
template <bool kHalf>
constexpr float kAttnSlack = 8.f + kAttnBelow<kHalf>;
constexpr int kAttnEnds = 2;        // what a row tile's beginning and end cost, in token tiles, when runs are cut
constexpr float kAttnUnseen = -1e30f;  // reference of a row that has seen nothing: below every score, and finite

struct AttnArgs {
  const uint16_t *q, *gate, *v_pages;  // K is reached through its tensor map alone
  uint16_t* out;
  const int32_t *table, *context, *starts;
  const uint32_t* mask;
  long long q_token, q_head, gate_token, gate_head, out_token, out_head;
  long long v_page, v_head, v_slot;
  long long table_row, mask_row;
  long long pages;
  int requests, tokens, max_draft, table_cols, heads, kv_heads, page;
  int k_combo, v_combo;      // page stride / head stride: a (page, head) pair is one coordinate of the maps
  unsigned int group_magic;  // row / (heads / kv_heads) = umulhi(row, magic); 0: the group is one head
  float scale_log2;          // |scale| * log2(e)
  uint32_t q_flip;           // 0x80008000 where scale is negative: q is taken with the other sign
  struct AttnCross* cross;   // scratch: [ctas]
  float2* part_ml;           // scratch: [ctas][2][kRows] (reference, sum)
  float* part_o;             // scratch: [ctas][2][kRows][dim]
};

// The row tile that starts in a CTA's run and goes on in the next ones: its rows, and the last run of it.
struct AttnCross {
  int first, row0, rows, head;  // request's first token, first row, rows (0: no such tile), kv head
  int last, pad0, pad1, pad2;
};
static_assert(sizeof(AttnCross) == 32, "AttnCross layout");

// (token of the request, head of the group) of a row.
__device__ __forceinline__ int attn_token(const AttnArgs& a, int row) {
  return a.group_magic ? static_cast<int>(__umulhi(static_cast<unsigned int>(row), a.group_magic)) : row;
}

// One variant: threads, rings, Q, P, then the small arrays in shared memory.
template <int kDim, int kRows>
struct AttnShape {
  static constexpr int kHalves = kDim / 64;
  static_assert(kRows == 16 || kRows == 32, "rows");
  static constexpr int kTG = kDim == 64 ? 2 : 1;                  // 128-token groups a tile
  static constexpr int kTok = 128 * kTG;                          // cached tokens a tile
  static constexpr int kSoft = 128 * kTG;                         // softmax threads
  static constexpr int kThreads = 64 + kSoft + 32;                // producer, UMMA, softmax, row loader
  static constexpr int kStage = kTok * kDim * 2;                  // one K or V tile
  static constexpr int kQ = kRows * kDim * 2;
  static constexpr int kP = kTok * kRows * 2;
  static constexpr int kNP = 2;                                   // P buffers
  static constexpr int kNK = 3;
  static constexpr int kNV = kDim == 64 && kRows == 32 ? 2 : 3;
  static constexpr int kTmemO = 2 * kTG * kRows;                  // after two buffers of S^T
  static constexpr int kTmem = kTmemO + kRows <= 64 ? 64 : (kTmemO + kRows <= 128 ? 128 : 256);
  static constexpr int kOffV = kNK * kStage, kOffQ = kOffV + kNV * kStage, kOffP = kOffQ + kQ, kOffSmall = kOffP + kNP * kP;
  // ref, rescale, 1 / sum [kRows]; row ids [2][kRows]; red [4 kTG][kRows]; mask words [2][kRows][9]; segments; barriers.
  static constexpr int kSmall = kRows * 4 * 5 + 4 * kTG * kRows * 4 + kRows * 72 + 128 + (2 * kNK + 2 * kNV + 13) * 8 + 64;
  static constexpr int kSmem = 1024 + kOffSmall + kSmall;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

struct AttnReq {
  int first, drafted, ctx, kv, tiles, rows;  // first token, drafted tokens, context, entries, token tiles, rows a kv head
  int units;                                 // kv heads x row tiles
  int cost;                                  // of a unit, in token tiles (0: nothing to do)
};

// A request's sizes, clamped to what may be touched whatever the device arrays hold.
template <int kTok, int kRows>
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
  r.tiles = t > 0 ? (r.kv + kTok - 1) / kTok : 0;
  r.cost = r.tiles > 0 ? r.tiles + kAttnEnds : 0;
  r.rows = t * (a.heads / a.kv_heads);
  r.units = a.kv_heads * ((r.rows + kRows - 1) / kRows);
  return r;
}

// `total` of cost over at most `ctas` runs, the first `more` one longer.
struct AttnRuns {
  int runs, per, more;
  __device__ __forceinline__ AttnRuns(int total, int ctas) : runs(min(total, ctas)), per(0), more(0) {
    if (runs > 0) per = total / runs, more = total - per * runs;
  }
  __device__ __forceinline__ int start(int c) const { return c * per + min(c, more); }
  // The run that holds position w.
  __device__ __forceinline__ int of(int w) const {
    const int longer = more * (per + 1);
    return w < longer ? w / (per + 1) : more + (w - longer) / per;
  }
};

// Walks a CTA's run segment by segment (a segment: consecutive token tiles of one row tile and kv head). A unit's
// positions are kAttnEnds of its ends, then its tiles.
struct AttnSeg {
  int b, head, row0, i0, i1;  // request, kv head, first row, token tiles [i0, i1)
  int unit0;                  // position of the unit's first tile
  AttnReq r;
};
template <int kTok, int kRows>
struct AttnWalk {
  int left, base;  // of the run; positions before request b
  int unit, b, at;  // unit of the request, position in it
  AttnReq r;
  __device__ __forceinline__ AttnWalk(const AttnArgs& a, int b0, int base0, int w0, int w1)
      : left(w1 - w0), base(base0), unit(0), b(b0), at(0) {
    r = attn_request<kTok, kRows>(a, b, false);
    const int off = w0 - base;
    unit = off / r.cost;
    at = off - unit * r.cost;
  }
  __device__ __forceinline__ bool next(const AttnArgs& a, AttnSeg& s) {
    while (left > 0) {
      while (unit >= r.units || r.cost == 0) {
        base += r.units * r.cost;
        if (++b >= a.requests) return false;
        r = attn_request<kTok, kRows>(a, b, false);
        unit = 0;
        at = 0;
      }
      const int take = min(left, r.cost - at);
      s.i0 = max(at - kAttnEnds, 0);
      s.i1 = max(at + take - kAttnEnds, 0);
      s.b = b;
      s.r = r;
      // Row tiles of one kv head follow one another, so that CTAs that share cached tokens run side by side.
      const int row_tiles = (r.rows + kRows - 1) / kRows;
      s.head = row_tiles == 1 ? unit : unit / row_tiles;
      s.row0 = (unit - s.head * row_tiles) * kRows;
      s.unit0 = base + unit * r.cost + kAttnEnds;
      left -= take;
      ++unit;
      at = 0;
      if (s.i1 > s.i0) return true;
    }
    return false;
  }
};

__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, uint64_t* bar, int c3, int c4, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %3, %3, %4, %5}], [%2], %6;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(c3), "r"(c4), "l"(policy)
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

// One lane of a converged warp. The UMMA warp runs its loop with all lanes, on values made uniform with a
// shuffle, and elects a lane around the tcgen05 instructions alone: descriptors then live in uniform registers. With
// the whole loop under `lane == 0` each UMMA took about 105 cycles to issue, more than the 64 an N = 128 one runs for.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0u;
}
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

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

// 16 values a lane reduced over the warp's lanes by halving (16 shuffles in all): afterwards lane l holds
// column l / 2 in v[0].
template <bool kMax>
__device__ __forceinline__ void warp_fold16(float* v, int lane) {
#pragma unroll
  for (int n = 8, o = 16; n; n >>= 1, o >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j < n) {
        const float give = up ? v[j] : v[j + n], keep = up ? v[j + n] : v[j];
        const float got = __shfl_xor_sync(0xffffffffu, give, o);
        v[j] = kMax ? fmaxf(keep, got) : keep + got;
      }
    }
  }
  const float got = __shfl_xor_sync(0xffffffffu, v[0], 1);
  v[0] = kMax ? fmaxf(v[0], got) : v[0] + got;
}

// UMMA descriptor but for its address: `row` bytes of a swizzled row, `group` bytes between groups of 8 rows,
// `chunk` bytes between runs of 64 M/N entries (M- or N-major operands; 0: one run, or the same one again).
__host__ __device__ constexpr uint64_t attn_desc_bits(int row, int group, int chunk) {
  return (static_cast<uint64_t>(chunk >> 4) << 16) | (static_cast<uint64_t>(group >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
         (static_cast<uint64_t>(row == 128 ? 2 : (row == 64 ? 4 : 6)) << 61);
}

// The cached tokens of a tile in shared memory: groups of 8 tokens, each kHalves blocks (64 dims) of 8 rows of 128
// bytes, swizzled within a block: what one TMA box {64 dims, 8 tokens, halves, groups} writes. A page's (or a
// tile's) share is one box, its 2 * dim bytes a token contiguous in the cache as a rule.
__device__ __forceinline__ uint32_t attn_row(int token, int halves) { return static_cast<uint32_t>((token >> 3) * 1024 * halves + (token & 7) * 128); }

// Where a CTA's run starts: every CTA scans the requests (a run of requests a thread), none waits for another.
struct AttnPlan {
  AttnRuns runs;
  int w0, w1, b0, s0;  // the run [w0, w1); its first request and the positions before that
  bool work;
};
template <int kThreads, int kTok, int kRows>
__device__ __forceinline__ AttnPlan attn_plan(const AttnArgs& a, int* sums, int* start) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int total = 0, before = 0, mine = 0;
  const int each = (a.requests + kThreads - 1) / kThreads;
  const int b_lo = min(static_cast<int>(threadIdx.x) * each, a.requests), b_hi = min(b_lo + each, a.requests);
  for (int b = b_lo; b < b_hi; ++b) {
    const AttnReq r = attn_request<kTok, kRows>(a, b, blockIdx.x == 0);
    mine += r.units * r.cost;
  }
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  before += upto - mine;
  AttnPlan p = {AttnRuns(total, gridDim.x), 0, 0, 0, 0, false};
  p.work = static_cast<int>(blockIdx.x) < p.runs.runs;
  if (p.work) p.w0 = p.runs.start(blockIdx.x), p.w1 = p.runs.start(blockIdx.x + 1);
  if (p.work && before <= p.w0 && p.w0 < before + mine) {
    int at = before, b = b_lo;
    if (each > 1) {
      for (;; ++b) {
        const AttnReq r = attn_request<kTok, kRows>(a, b, false);
        if (p.w0 < at + r.units * r.cost) break;
        at += r.units * r.cost;
      }
    }
    start[0] = b, start[1] = at;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  p.b0 = start[0], p.s0 = start[1];
  return p;
}

// The producer warp: K and V tiles of the run into their rings, a lane a box. Ends with no copy in flight.
template <int kTok, int kRows, int kDim, int kNK, int kNV>
__device__ __forceinline__ void attn_produce(const AttnArgs& a, const AttnPlan& plan, const CUtensorMap* tmk, const CUtensorMap* tmv,
                                             uint8_t* ring_k, uint8_t* ring_v, uint64_t* k_full, uint64_t* k_empty, uint64_t* v_full,
                                             uint64_t* v_empty) {
  static_assert(kTok / 8 <= 32, "a lane a box");
  constexpr int kStage = kTok * kDim * 2;
  const int lane = threadIdx.x & 31;
  int issued_k = 0, issued_v = 0;
  AttnWalk<kTok, kRows> walk(a, plan.b0, plan.s0, plan.w0, plan.w1);
  AttnSeg s;
  const int box = min(a.page, kTok), boxes = kTok / box;
  const uint32_t off = static_cast<uint32_t>(lane * box * kDim * 2), box_bytes = static_cast<uint32_t>(box * kDim * 2);
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
      const int pos = i * kTok + lane * box;
      have = lane < boxes && pos < s.r.kv;
      page = have ? row[static_cast<unsigned int>(pos) / static_cast<unsigned int>(a.page)] : 0;
    };
    lookup(s.i0);
    for (int i = s.i0; i < s.i1; ++i) {
      int now = page;
      const int in = ((i * kTok + lane * box) & (a.page - 1)) >> 3;
      const bool go = have;
      if (go && (now < 0 || now >= a.pages)) report_error(kErrAttnPage), now = 0;
      if (i + 1 < s.i1) lookup(i + 1);
      const uint32_t bytes = static_cast<uint32_t>(__popc(__ballot_sync(0xffffffffu, go))) * box_bytes;
      ok = mbar_wait(&k_empty[rk.slot], rk.phase ^ 1u, kErrAttnProducer);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      if (lane == 0) mbar_expect_tx(&k_full[rk.slot], bytes);
      __syncwarp();
      if (go) tma_load_5d(ring_k + rk.slot * kStage + off, tmk, &k_full[rk.slot], in, now * a.k_combo + s.head, policy);
      rk.next(kNK);
      ++issued_k;
      ok = mbar_wait(&v_empty[rv.slot], rv.phase ^ 1u, kErrAttnProducer);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      if (lane == 0) mbar_expect_tx(&v_full[rv.slot], bytes);
      __syncwarp();
      if (go) tma_load_5d(ring_v + rv.slot * kStage + off, tmv, &v_full[rv.slot], in, now * a.v_combo + s.head, policy);
      rv.next(kNV);
      ++issued_v;
    }
  }
  for (int n = max(issued_k - kNK, 0); n < issued_k; ++n)
    mbar_wait(&k_full[n % kNK], static_cast<uint32_t>((n / kNK) & 1), kErrAttnDrain, kWaitLimitNs / 100);
  for (int n = max(issued_v - kNV, 0); n < issued_v; ++n)
    mbar_wait(&v_full[n % kNV], static_cast<uint32_t>((n / kNV) & 1), kErrAttnDrain, kWaitLimitNs / 100);
}

// V rows that not every row of Q may see, before the second product reads them (0 x NaN is NaN): this thread's
// token is zeroed past the request's end; a drafted one has non-finite entries zeroed and *odd set.
__device__ __forceinline__ uint4* attn_shared16(uint32_t addr) { return reinterpret_cast<uint4*>(__cvta_shared_to_generic(addr)); }

template <bool kHalf, int kDim>
__device__ __forceinline__ void attn_clean_v(uint32_t tile, int token, bool beyond, bool drafted, int* odd_v) {
  constexpr int kHalves = kDim / 64;
  const uint32_t row = tile + attn_row(token, kHalves);
  if (beyond) {
#pragma unroll
    for (int ch = 0; ch < kDim / 8; ++ch) st_shared_v4u(row + (ch >> 3) * 1024 + (ch & 7) * 16, 0u, 0u, 0u, 0u);
  } else if (drafted) {
    constexpr uint32_t kExp = kHalf ? 0x7C00u : 0x7F80u;
    constexpr uint32_t kBit = kHalf ? 0x04000400u : 0x00800080u;  // an exponent of all ones carries into the sign's place
#pragma unroll 1
    for (int c0 = 0; c0 < kDim / 8; c0 += 4) {
      uint4 v[4];
      uint32_t any = 0u;
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = *attn_shared16(row + ((c0 + u) >> 3) * 1024 + ((c0 + u) & 7) * 16);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t e[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) any |= (e[k] & (kExp * 0x10001u)) + kBit;
      }
      if (!(any & 0x80008000u)) continue;
      *odd_v = 1;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        uint32_t e[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if ((e[k] & kExp) == kExp) e[k] &= 0xFFFF0000u;
          if ((e[k] & (kExp << 16)) == (kExp << 16)) e[k] &= 0x0000FFFFu;
        }
        *attn_shared16(row + ((c0 + u) >> 3) * 1024 + ((c0 + u) & 7) * 16) = make_uint4(e[0], e[1], e[2], e[3]);
      }
    }
  }
}

// Word w of the drafted tokens that row `t` of request r sees: its mask's bits (or itself and every earlier token),
// nothing past the request's tokens.
__device__ __forceinline__ uint32_t attn_seen_word(const AttnArgs& a, const AttnReq& r, int t, int w) {
  const uint32_t v = a.mask ? a.mask[(r.first + t) * a.mask_row + w] : 0xffffffffu;
  const int n = (a.mask ? r.drafted : min(t + 1, r.drafted)) - w * 32;
  return v & (n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u));
}

// 16 bytes from global to shared memory without a register; zeros where `live` is false.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// The row loader (kLanes threads of their own): for each segment of the run its description, mask words and row ids
// (two places in turn) and Q, as soon as the last product that reads the segment before's Q is done: while that segment's
// softmax, second products and end still run (a segment's first scores wait for it no longer than that). q_full and
// seg_done are two barriers each, by segment parity: their waiters may come a whole segment late, and one barrier's parity
// would then name the next phase. q_full tells the others (kLanes arrivals); a segment without tiles ends
// the run. Q is [row tiles of kTile rows][halves][kTile][64 dims] swizzled; every row that is computed with is written, a
// multiple of kFill, zeros past the rows (what stood there would have a say in when the references move).
template <int kTok, int kRows, int kTile, int kFill, int kDim, int kLanes>
__device__ __forceinline__ void attn_load_rows(const AttnArgs& a, const AttnPlan& plan, int me, uint8_t* q_s, AttnSeg* segs, uint32_t* words,
                                               int* row_id, uint64_t* q_full, uint64_t* q_empty, uint64_t* seg_done) {
  constexpr int kChunks = kDim / 8;
  const int g = a.heads / a.kv_heads;
  AttnWalk<kTok, kRows> walk(a, plan.b0, plan.s0, plan.w0, plan.w1);
  AttnSeg s;
  for (int k = 0;; ++k) {
    const bool more = walk.next(a, s);
    if (!more) s.i0 = s.i1 = 0;
    // This place's last user, two segments ago, is done with it.
    if (k > 1 && !mbar_wait_idle(&seg_done[k & 1], ((k >> 1) - 1) & 1, kErrAttnLoader)) break;
    if (more) {
      const int rows = min(kRows, s.r.rows - s.row0), fill = min(kRows, (rows + kFill - 1) / kFill * kFill);
      if (k > 0 && !mbar_wait_idle(q_empty, (k - 1) & 1, kErrAttnLoader)) break;
      auto at = [&](int r, int ch) {
        return smem_u32(q_s) + (r / kTile) * (kTile * kDim * 2) + (ch >> 3) * (kTile * 128) + (r & (kTile - 1)) * 128 +
               (((ch & 7) ^ (r & 7)) << 4);
      };
#pragma unroll 4
      for (int i = me; i < fill * kChunks; i += kLanes) {
        const int r = i / kChunks, ch = i % kChunks, row = s.row0 + min(r, rows - 1), t = attn_token(a, row);
        cp_async16(at(r, ch), a.q + (s.r.first + t) * a.q_token + (s.head * g + row - t * g) * a.q_head + ch * 8, r < rows);
      }
      uint32_t* w = words + (k & 1) * kRows * 9;
      int* id = row_id + (k & 1) * kRows;
      const int nw = (s.r.drafted + 31) >> 5;
      for (int r = me; r < fill; r += kLanes) {
        const int row = s.row0 + min(r, rows - 1), t = attn_token(a, row);
        id[r] = (t << 16) | (s.head * g + row - t * g);
        for (int j = 0; j < nw; ++j) w[r * 9 + j] = r < rows ? attn_seen_word(a, s.r, t, j) : 0u;
        for (int j = nw; j < 9; ++j) w[r * 9 + j] = 0u;
      }
      cp_async_wait();
      if (a.q_flip) {  // a negative scale: this thread's own chunks with the other sign
        for (int i = me; i < fill * kChunks; i += kLanes) {
          const uint32_t to = at(i / kChunks, i % kChunks);
          const uint4 v = ld_shared_v4u(to);
          st_shared_v4u(to, v.x ^ a.q_flip, v.y ^ a.q_flip, v.z ^ a.q_flip, v.w ^ a.q_flip);
        }
      }
      fence_proxy_async_shared();
    }
    if (me == 0) segs[k & 1] = s;
    mbar_arrive(&q_full[k & 1]);
    if (!more) break;
  }
}

template <bool kHalf, int kDim, int kRows>
__global__ void __launch_bounds__(AttnShape<kDim, kRows>::kThreads, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const AttnArgs a) {
  using Sh = AttnShape<kDim, kRows>;
  constexpr int kHalves = Sh::kHalves, kNK = Sh::kNK, kNV = Sh::kNV, kNP = Sh::kNP, kTok = Sh::kTok;
  constexpr int kTG = Sh::kTG, kSoft = Sh::kSoft;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_align<1024>(smem_raw);
  uint8_t* ring_k = smem;
  uint8_t* ring_v = smem + Sh::kOffV;
  uint8_t* q_s = smem + Sh::kOffQ;
  uint8_t* p_s = smem + Sh::kOffP;
  float* ref = reinterpret_cast<float*>(smem + Sh::kOffSmall);  // reference (scaled, log2)
  float* rescale = ref + kRows;
  float* inv = rescale + kRows;
  int* row_ids = reinterpret_cast<int*>(inv + kRows);            // [2][kRows]: token of the request << 16 | query head
  float* red = reinterpret_cast<float*>(row_ids + 2 * kRows);    // [4 kTG][kRows]
  uint32_t* all_words = reinterpret_cast<uint32_t*>(red + 4 * kTG * kRows);  // [2][kRows][9]: drafted tokens a row sees
  AttnSeg* segs = reinterpret_cast<AttnSeg*>(all_words + 2 * kRows * 9);     // [2]
  uint64_t* k_full = reinterpret_cast<uint64_t*>(segs) + 16;
  uint64_t* k_empty = k_full + kNK;
  uint64_t* v_full = k_empty + kNK;
  uint64_t* v_empty = v_full + kNV;
  uint64_t* s_full = v_empty + kNV;  // [2]
  uint64_t* p_full = s_full + 2;     // [2]
  // [2], by tile parity: a softmax thread may look at a phase up to two tiles late, and one barrier's parity
  // would by then name the next phase.
  uint64_t* pv_done = p_full + 2;
  uint64_t* q_full = pv_done + 2;
  uint64_t* q_empty = q_full + 2;    // q_full [2], seg_done [2]: by segment parity
  uint64_t* seg_done = q_empty + 1;
  uint64_t* fin = seg_done + 2;
  int* start_b = reinterpret_cast<int*>(fin + 1);  // [2]: the run's first request, and the tiles before it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(start_b + 2);
  int* odd_vs = reinterpret_cast<int*>(tmem_slot + 1);  // [2], by segment: a drafted token has a non-finite V entry

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&tmk);
    prefetch_tensormap(&tmv);
    for (int i = 0; i < kNK; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < kNV; ++i) mbar_init(&v_full[i], 1), mbar_init(&v_empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], kSoft), mbar_init(&pv_done[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&q_full[i], 32), mbar_init(&seg_done[i], kSoft);
    mbar_init(q_empty, 1);
    odd_vs[0] = odd_vs[1] = 0;
    mbar_init(fin, 1);
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, Sh::kTmem);
  pdl_launch_dependents();
  pdl_wait();

  const AttnPlan plan = attn_plan<Sh::kThreads, kTok, kRows>(a, reinterpret_cast<int*>(red), start_b);
  const uint32_t tmem = static_cast<uint32_t>(uniform(static_cast<int>(*tmem_slot)));
  const uint32_t tmem_o = tmem + Sh::kTmemO;

  if (warp == 0) {
    if (plan.work)
      attn_produce<kTok, kRows, kDim, kNK, kNV>(a, plan, &tmk, &tmv, ring_k, ring_v, k_full, k_empty, v_full, v_empty);
  } else if (warp == 1) {
    // ---- UMMA issue --------------------------------------------------------------------------------
    if (uniform(plan.work)) {
      constexpr uint32_t kType = kHalf ? 0u : ((1u << 7) | (1u << 10));
      constexpr uint32_t kShape = (1u << 4) | (static_cast<uint32_t>(kRows >> 3) << 17) | (8u << 24);
      constexpr uint32_t idesc_s = kShape | kType, idesc_o = kShape | kType | (1u << 15) | (1u << 16);
      constexpr int kPRow = kRows * 2;  // bytes of a token's row of P
      constexpr uint64_t k_bits = attn_desc_bits(128, 1024 * kHalves, 16);
      constexpr uint64_t v_bits = attn_desc_bits(128, 1024 * kHalves, kHalves > 1 ? 1024 : 0);
      constexpr uint64_t p_bits = attn_desc_bits(kPRow, 8 * kPRow, 0);
      Ring rk, rv;
      uint32_t n = 0;
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_idle(bar, parity, kErrAttnMma)) != 0; };
      auto issue_s = [&](uint32_t m, bool last) {
        if (!wait(&k_full[rk.slot], rk.phase)) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t dk = k_bits | ((smem_u32(ring_k + rk.slot * Sh::kStage) & 0x3FFFFu) >> 4), dq = umma_desc_sw128(smem_u32(q_s));
#pragma unroll
          for (int t = 0; t < kTG; ++t)
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_bf16(tmem + ((m & 1u) * kTG + t) * kRows, dk + ((h * 1024 + t * 128 * kDim * 2) >> 4) + 2 * k,
                          dq + ((h * kRows * 128) >> 4) + 2 * k, idesc_s, (h | k) != 0);
          umma_commit(&k_empty[rk.slot]);
          umma_commit(&s_full[m & 1u]);
          if (last) umma_commit(q_empty);
        }
        __syncwarp();
        rk.next(kNK);
        return true;
      };
      for (int k = 0;; ++k) {
        if (!(ok = wait(&q_full[k & 1], (k >> 1) & 1))) break;
        const int tiles = uniform(segs[k & 1].i1 - segs[k & 1].i0);
        if (tiles == 0) break;
        tc_fence_after();
        ok = issue_s(n, tiles == 1);
        for (int i = 0; ok && i < tiles; ++i, ++n) {
          // The next tile's scores are under way while the softmax of this one runs.
          if (i + 1 < tiles && !(ok = issue_s(n + 1, i + 2 == tiles))) break;
          ok = wait(&p_full[n & 1u], (n >> 1) & 1u) && wait(&v_full[rv.slot], rv.phase);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t dv = v_bits | ((smem_u32(ring_v + rv.slot * Sh::kStage) & 0x3FFFFu) >> 4);
            const uint64_t dp = p_bits | ((smem_u32(p_s + (n % kNP) * Sh::kP) & 0x3FFFFu) >> 4);
#pragma unroll
            for (int k = 0; k < kTok / 16; ++k)
              umma_bf16(tmem_o, dv + ((k * 16 * kDim * 2) >> 4), dp + ((k * 16 * kPRow) >> 4), idesc_o, (i > 0 || k > 0) ? 1u : 0u);
            umma_commit(&v_empty[rv.slot]);
            umma_commit(&pv_done[n & 1u]);
          }
          __syncwarp();
          rv.next(kNV);
        }
        if (!ok) break;
      }
      if (elect_one()) umma_commit(fin);
      __syncwarp();
      mbar_wait(fin, 0u, kErrAttnDrain, kWaitLimitNs / 10);  // nothing of the tensor cores is under way past here
    }
    __syncwarp();
  } else if (warp == Sh::kThreads / 32 - 1) {
    if (plan.work)
      attn_load_rows<kTok, kRows, kRows, 16, kDim, 32>(a, plan, lane, q_s, segs, all_words, row_ids, q_full, q_empty, seg_done);
  } else {
    // ---- softmax: thread = one token of the tile (a TMEM lane of its token group), all rows ----
    const int tid = static_cast<int>(threadIdx.x) - 64;
    const int tg = tid >> 7;
    const int quarter = warp & 3, tl = quarter * 32 + lane, token = tg * 128 + tl;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const float kNegInf = __int_as_float(0xff800000);
    const float c = a.scale_log2;
    AttnCross cross = {};
    if (plan.work) {
      uint32_t n = 0;  // tiles done in this run
      uint32_t v_slot = 0, v_phase = 0;
      bool ok = true;
      float l[kRows];
      for (int k = 0;; ++k) {
        // ---- the segment's rows --------------------------------------------------------------------
        ok = mbar_wait_idle(&q_full[k & 1], (k >> 1) & 1, kErrAttnSoftmax);
        if (bar_any(8, kSoft, !ok)) break;  // every thread is done with the last segment's arrays, too
        const AttnSeg s = segs[k & 1];
        if (s.i1 <= s.i0) break;
        const int rows = min(kRows, s.r.rows - s.row0);
        const int live = min(kRows, (rows + 15) & ~15);  // columns that are computed
        const uint32_t* words = all_words + (k & 1) * kRows * 9;
        const int* row_id = row_ids + (k & 1) * kRows;
        int* odd_v = odd_vs + (k & 1);
        if (tid < kRows) ref[tid] = kAttnUnseen;
        if (tid == 0) odd_vs[(k + 1) & 1] = 0;
        bar_named(8, kSoft);
#pragma unroll
        for (int j = 0; j < kRows; ++j) l[j] = 0.f;
        const bool lone = s.r.drafted == 1 && !a.mask;  // one token, which sees itself

        // ---- tiles ---------------------------------------------------------------------------------
        // A wait that gave up is carried to the next barrier reduction: the loop's end has to be the same for all.
        for (int i = s.i0; i < s.i1; ++i, ++n) {
          ok = mbar_wait_idle(&s_full[n & 1u], (n >> 1) & 1u, kErrAttnSoftmax) && ok;
          // P's buffer is free, and with two of them PV of two tiles ago is done, once this has passed.
          if (n >= static_cast<uint32_t>(kNP)) ok = mbar_wait_idle(&pv_done[(n - kNP) & 1u], ((n - kNP) >> 1) & 1u, kErrAttnSoftmax) && ok;
          tc_fence_after();
          float x[kRows];
          const uint32_t ts = tmem + ((n & 1u) * kTG + tg) * kRows + lanes;
#pragma unroll
          for (int cc = 0; cc < kRows; cc += 16)
            if (cc < live) attn_ld16(ts + cc, x + cc);
#pragma unroll
          for (int cc = 0; cc < kRows; cc += 16)
            if (cc < live) attn_ld_wait(x + cc);
          const int pos = i * kTok + token;
          const bool edge = (i + 1) * kTok > s.r.ctx;  // the tile reaches past the context
          const float cm = edge ? 1.f : c;             // scores of an edge tile are scaled here, with their mask
          if (edge) {
            // Bit k: this token is seen by column k.
            uint32_t seen = pos < s.r.kv ? 0xffffffffu : 0u;
            const int j = pos - s.r.ctx;
            if (!lone && seen && j >= 0) {
              seen = 0u;
#pragma unroll
              for (int k = 0; k < kRows; ++k)
                if (k < live) seen |= ((words[k * 9 + (j >> 5)] >> (j & 31)) & 1u) << k;
            }
#pragma unroll
            for (int k = 0; k < kRows; ++k) x[k] = (seen >> k) & 1u ? x[k] * c : kNegInf;
          }
          float over[4] = {kNegInf, kNegInf, kNegInf, kNegInf};  // how far a score passes its reference
#pragma unroll
          for (int cc = 0; cc < kRows; cc += 4) {
            if (cc < live) {
              const float4 m = *reinterpret_cast<const float4*>(ref + cc);
              over[0] = fmaxf(over[0], fmaf(x[cc], cm, -m.x));
              over[1] = fmaxf(over[1], fmaf(x[cc + 1], cm, -m.y));
              over[2] = fmaxf(over[2], fmaf(x[cc + 2], cm, -m.z));
              over[3] = fmaxf(over[3], fmaf(x[cc + 3], cm, -m.w));
            }
          }
          const bool past = fmaxf(fmaxf(over[0], over[1]), fmaxf(over[2], over[3])) > kAttnSlack<kHalf>;
          if (bar_any(8, kSoft, past || !ok)) {
            if (bar_any(8, kSoft, !ok)) {
              ok = false;
              break;
            }
            // Move the references after the true maxima and rescale what was summed against the old ones.
#pragma unroll
            for (int cc = 0; cc < kRows; cc += 16) {
              float top[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) top[j] = cc < live ? x[cc + j] * cm : kNegInf;
              warp_fold16<true>(top, lane);
              if (!(lane & 1)) red[(tg * 4 + quarter) * kRows + cc + (lane >> 1)] = top[0];
            }
            bar_named(8, kSoft);
            if (tid < kRows) {
              const int col = tid;
              const float old = ref[col];
              float now = old;
#pragma unroll
              for (int w = 0; w < 4 * kTG; ++w) now = fmaxf(now, red[w * kRows + col] - kAttnBelow<kHalf>);
              ref[col] = now;
              rescale[col] = ex2(old - now);
            }
            bar_named(8, kSoft);
            if (i > s.i0) {
#pragma unroll
              for (int j = 0; j < kRows; ++j)
                if (j < live) l[j] *= rescale[j];
              ok = mbar_wait_idle(&pv_done[(n - 1) & 1u], ((n - 1) >> 1) & 1u, kErrAttnSoftmax) && ok;
              tc_fence_after();
#pragma unroll
              for (int cc = 0; cc < kRows; cc += 16) {
                if (cc < live && ((cc >> 4) & (kTG - 1)) == tg) {
                  float o[16];
                  attn_ld16(tmem_o + cc + lanes, o);
                  attn_ld_wait(o);
#pragma unroll
                  for (int k = 0; k < 16; ++k) o[k] *= rescale[cc + k];
                  attn_st16(tmem_o + cc + lanes, o);
                }
              }
              attn_st_wait();
            }
          }
          // P, rounded, as the second product reads it (a score that is not seen is -inf, its P zero).
          const uint32_t pt = smem_u32(p_s + (n % kNP) * Sh::kP);
#pragma unroll
          for (int cc = 0; cc < kRows; cc += 8) {
            if (cc < live) {
              const float4 m0 = *reinterpret_cast<const float4*>(ref + cc), m1 = *reinterpret_cast<const float4*>(ref + cc + 4);
              const float m[8] = {m0.x, m0.y, m0.z, m0.w, m1.x, m1.y, m1.z, m1.w};
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                w[k] = pack16x2<kHalf>(ex2(fmaf(x[cc + 2 * k], cm, -m[2 * k])), ex2(fmaf(x[cc + 2 * k + 1], cm, -m[2 * k + 1])));
                add16x2<kHalf>(w[k], l[cc + 2 * k], l[cc + 2 * k + 1]);
              }
              const int ch = cc >> 3;
              uint32_t at;
              if constexpr (kRows == 16) at = token * 32 + ((ch ^ ((token >> 2) & 1)) << 4);
              else at = token * 64 + ((ch ^ ((token >> 1) & 3)) << 4);
              st_shared_v4u(pt + at, w[0], w[1], w[2], w[3]);
            }
          }
          // In the last tile or two of a request. A lone token sees itself: only then is no drafted entry hidden from a row.
          const bool ragged = (i + 1) * kTok > s.r.kv, drafted = edge && !lone;
          if (ragged || drafted) {
            ok = mbar_wait_idle(&v_full[v_slot], v_phase, kErrAttnSoftmax) && ok;
            attn_clean_v<kHalf, kDim>(smem_u32(ring_v + v_slot * Sh::kStage), token, pos >= s.r.kv, drafted && pos >= s.r.ctx, odd_v);
          }
          if (++v_slot == kNV) v_slot = 0, v_phase ^= 1u;
          fence_proxy_async_shared();
          tc_fence_before();
          mbar_arrive(&p_full[n & 1u]);
        }

        // ---- end of the segment: finish the row tile, or leave a partial ---------------------------
        const bool whole = s.i0 == 0 && s.i1 == s.r.tiles;
#pragma unroll
        for (int cc = 0; cc < kRows; cc += 16) {
          warp_fold16<false>(l + cc, lane);
          if (!(lane & 1)) red[(tg * 4 + quarter) * kRows + cc + (lane >> 1)] = l[cc];
        }
        if (ok) ok = mbar_wait_idle(&pv_done[(n - 1) & 1u], ((n - 1) >> 1) & 1u, kErrAttnSoftmax);
        ok = !bar_any(8, kSoft, !ok);
        if (!ok) break;
        tc_fence_after();
        // The run that starts inside a row tile keeps its partial first, the one that ends inside it second.
        const int slot = (blockIdx.x * 2 + (s.i0 > 0 ? 0 : 1)) * kRows;
        if (tid < kRows) {
          const int col = tid;
          float sum = 0.f;
#pragma unroll
          for (int w = 0; w < 4 * kTG; ++w) sum += red[w * kRows + col];
          inv[col] = sum == 0.f ? 0.f : 1.f / sum;
          if (!whole && col < rows) a.part_ml[slot + col] = make_float2(ref[col], sum);
        }
        if (!whole && s.i0 == 0) {
          cross.first = s.r.first, cross.row0 = s.row0, cross.rows = rows, cross.head = s.head;
          cross.last = plan.runs.of(s.unit0 + s.r.tiles - 1);
        }
        bar_named(8, kSoft);
        const int odd = *odd_v;
#pragma unroll
        for (int cc = 0; cc < kRows; cc += 16) {
          if (cc < live && ((cc >> 4) & (kTG - 1)) == tg) {
            float o[16];
            attn_ld16(tmem_o + cc + lanes, o);
            uint16_t gv[16];
            const bool mine_o = tl < kDim;
            if (whole && a.gate && mine_o) {
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                const int id = row_id[cc + k];
                gv[k] = __ldg(a.gate + (s.r.first + (id >> 16)) * a.gate_token + (id & 0xFFFF) * a.gate_head + tl);
              }
            }
            attn_ld_wait(o);
            if (mine_o) {
              if (odd) {
                // Put the non-finite entries back for the rows that see them.
                const int j0 = max(s.i0 * kTok - s.r.ctx, 0), j1 = min(min(s.i1 * kTok, s.r.kv) - s.r.ctx, s.r.drafted);
                for (int j = j0; j < j1; ++j) {
                  const int p = s.r.ctx + j;
                  const long long page = a.table[s.b * a.table_row + p / a.page];
                  if (page < 0 || page >= a.pages) continue;
                  const float v = lo16<kHalf>(a.v_pages[page * a.v_page + s.head * a.v_head + (p % a.page) * a.v_slot + tl]);
                  if (!(fabsf(v) < __int_as_float(0x7f800000)))
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                      if ((words[(cc + k) * 9 + (j >> 5)] >> (j & 31)) & 1u) o[k] += v;
                }
              }
              if (whole) {
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                  const int col = cc + k, id = row_id[col];
                  float v = o[k] * inv[col];
                  if (a.gate) v = __fdividef(v, 1.f + __expf(-lo16<kHalf>(gv[k])));
                  if (col < rows)
                    a.out[(s.r.first + (id >> 16)) * a.out_token + (id & 0xFFFF) * a.out_head + tl] =
                        static_cast<uint16_t>(pack16x2<kHalf>(v, v) & 0xFFFFu);
                }
              } else {
#pragma unroll
                for (int k = 0; k < 16; ++k)
                  if (cc + k < rows) a.part_o[static_cast<long long>(slot + cc + k) * kDim + tl] = o[k];
              }
            }
          }
        }
        tc_fence_before();
        mbar_arrive(&seg_done[k & 1]);
      }
    }
    if (tid == 0) a.cross[blockIdx.x] = cross;
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Sh::kTmem);
  }
}

// Rows that belong to no request, before the first one's and past the last one's (what a fixed-size step carries without a
// token), become 0: by the join, each of whose CTAs takes a share. Two loads a CTA beside its own first one where there are
// none; where there are, the least and the largest of all starts bound them, so that in a batch whose starts are out of
// order (0xB01) no row that some request has is touched.
template <int kDim>
__device__ __forceinline__ void attn_clear_outside(const AttnArgs& a, int first, int last) {
  if (first <= 0 && last >= a.tokens) return;  // the same for the whole grid
  __shared__ int bounds[16];
  int lo = a.tokens, hi = 0;
  for (int b = threadIdx.x; b <= a.requests; b += 256) {
    const int at = min(max(a.starts[b], 0), a.tokens);
    lo = min(lo, at), hi = max(hi, at);
  }
  lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi);
  if ((threadIdx.x & 31) == 0) bounds[threadIdx.x >> 5] = lo, bounds[8 + (threadIdx.x >> 5)] = hi;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) lo = min(lo, bounds[w]), hi = max(hi, bounds[8 + w]);
  const long long pieces = static_cast<long long>(a.heads) * (kDim / 8), all = (static_cast<long long>(lo) + a.tokens - hi) * pieces;
  const long long step = static_cast<long long>(gridDim.x) * gridDim.y * 256;
  for (long long i = (static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x) * 256 + threadIdx.x; i < all; i += step) {
    const long long at = i / pieces, rest = i - at * pieces, token = at < lo ? at : at - lo + hi, head = rest / (kDim / 8);
    *reinterpret_cast<uint4*>(a.out + token * a.out_token + head * a.out_head + (rest - head * (kDim / 8)) * 8) = make_uint4(0u, 0u, 0u, 0u);
  }
}

__host__ __device__ constexpr int attn_join_rows(int rows) { return rows >= 128 ? 8 : rows / 16; }  // rows a CTA

// Joins the partials of the row tiles that cross runs: grid (runs, parts of the rows), 8 warps, of which each
// row has 8 (16 rows) to 1 (128 and more) that take the runs in turn, four partials on their way at once. A
// partial weighs 2^(its reference - the largest); the order of the sums is fixed. Latency is its cost: one load of
// what crosses here, then everything else together (2.4 us after one token over 700 entries, 4 us with 52 rows; 14 us
// for the 38 MB of partials of 256-row tiles). A CTA takes few rows: with four rows a warp 8 requests x 16 tokens took
// 21 us in all, 17 so.
template <bool kHalf, int kDim, int kRows>
__global__ void __launch_bounds__(256) tree_attn_join_kernel(const AttnArgs a) {
  constexpr int kN = kDim / 32, kBlock = attn_join_rows(kRows), kPerRow = 8 / kBlock;
  __shared__ float sums[8][kDim + 2];
  pdl_launch_dependents();
  pdl_wait();
  const AttnCross x = a.cross[blockIdx.x];
  attn_clear_outside<kDim>(a, a.starts[0], a.starts[a.requests]);
  const int r0 = blockIdx.y * kBlock;
  if (r0 >= x.rows) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % kPerRow, col = r0 + warp / kPerRow;
  const int c0 = blockIdx.x, n = x.last - c0 + 1;
  const bool live = col < x.rows;
  const int row = x.row0 + col, t = attn_token(a, row), g = a.heads / a.kv_heads;
  const long long token = x.first + t, h = x.head * g + row - t * g;
  uint32_t gw[kN / 2] = {};
  if (a.gate && live) {
#pragma unroll
    for (int i = 0; i < kN / 2; ++i)
      gw[i] = __ldg(reinterpret_cast<const uint32_t*>(a.gate + token * a.gate_token + h * a.gate_head + lane * kN) + i);
  }
  float acc[kN], sum = 0.f, top = kAttnUnseen;
#pragma unroll
  for (int i = 0; i < kN; ++i) acc[i] = 0.f;
  if (live) {
    for (int k0 = part; k0 < n; k0 += 4 * kPerRow) {
      float2 ml[4];
      float o[4][kN];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int k = k0 + u * kPerRow;
        ml[u] = make_float2(kAttnUnseen, 0.f);
#pragma unroll
        for (int i = 0; i < kN; ++i) o[u][i] = 0.f;
        if (k < n) {
          // Run c0 holds the tile's beginning in its second partial, the others their share in their first.
          const long long slot = static_cast<long long>((c0 + k) * 2 + (k == 0 ? 1 : 0)) * kRows + col;
          ml[u] = a.part_ml[slot];
          const float* src = a.part_o + slot * kDim + lane * kN;
          if constexpr (kN == 4) {
            const float4 v = *reinterpret_cast<const float4*>(src);
            o[u][0] = v.x, o[u][1] = v.y, o[u][2] = v.z, o[u][3] = v.w;
          } else {
            const float2 v = *reinterpret_cast<const float2*>(src);
            o[u][0] = v.x, o[u][1] = v.y;
          }
        }
      }
      const float now = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), top), f = ex2(top - now);
      top = now;
      sum *= f;
#pragma unroll
      for (int i = 0; i < kN; ++i) acc[i] *= f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float w = ex2(ml[u].x - now);
        sum += ml[u].y * w;
#pragma unroll
        for (int i = 0; i < kN; ++i) acc[i] += w * o[u][i];
      }
    }
  }
  if constexpr (kPerRow > 1) {
#pragma unroll
    for (int i = 0; i < kN; ++i) sums[warp][lane * kN + i] = acc[i];
    if (lane == 0) sums[warp][kDim] = sum, sums[warp][kDim + 1] = top;
    __syncthreads();
    if (part != 0) return;
    float now = top;
#pragma unroll
    for (int w = 1; w < kPerRow; ++w) now = fmaxf(now, sums[warp + w][kDim + 1]);
    const float f = ex2(top - now);
    sum *= f;
#pragma unroll
    for (int i = 0; i < kN; ++i) acc[i] *= f;
#pragma unroll
    for (int w = 1; w < kPerRow; ++w) {
      const float fw = ex2(sums[warp + w][kDim + 1] - now);
#pragma unroll
      for (int i = 0; i < kN; ++i) acc[i] += fw * sums[warp + w][lane * kN + i];
      sum += fw * sums[warp + w][kDim];
    }
  }
  if (!live) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint32_t packed[kN / 2];
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) {
    float v[2] = {acc[2 * i] * inv, acc[2 * i + 1] * inv};
    if (a.gate) {
      v[0] = __fdividef(v[0], 1.f + __expf(-lo16<kHalf>(gw[i])));
      v[1] = __fdividef(v[1], 1.f + __expf(-hi16<kHalf>(gw[i])));
    }
    packed[i] = pack16x2<kHalf>(v[0], v[1]);
  }
  uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + token * a.out_token + h * a.out_head + lane * kN);
  if constexpr (kN == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(packed[0], packed[1]);
  else dst[0] = packed[0];
}

}  // namespace muse
