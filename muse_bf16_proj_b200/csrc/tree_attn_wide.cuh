// tree_attention with many rows a kv head (more than 32): rows as the tensor cores' M.
//
// A unit is up to 256 rows (tokens x heads of a group) of one request and kv head: one or two row tiles of 128, which
// share every K and V tile that is brought in. For a row tile and 128 cached tokens
//   S [128 rows x 128 tokens] = Q . K^T            (both K-major from shared memory)
//   O [128 rows x dim]       += P . V              (P from tensor memory over S's columns, V as stored, N-major)
// A row is a TMEM lane and one softmax thread's, so its maximum, its references and its sums need no other thread,
// and P never passes through shared memory. Bound: at 2 x 128 rows the two products of both take 2048 tensor cycles a tile at
// dim 128 and the 32768 exponentials as many cycles of the exponential unit, so the two bind alike; K and V come in once for
// both row tiles. Measured: 16 requests of 64 tokens, 64 heads over 8 of 128, up to 8192 entries (174 GFLOP) in 205 us with
// the join in short runs = 850 TFLOP/s, 0.51 of a dense product's rate; in calls one after another 244 to 255 us = 710 to
// 680 TFLOP/s, where the power limit holds the SM clock near 1630 of 1965 MHz (241 us a call from a graph at that clock). The
// tensor cores are busy 44 % of the cycles: one S at a time passes from the products to a softmax and back, and each of those
// hand-offs is on the chain (TMEM has no room for a second S at dim 128). A softmax thread of the 256-row variants holds 128
// scores under the 168 registers that 384 threads leave it and spills 132 or 136 bytes (the 128-row ones none). 33 to 128 rows over 822 MB of cache take 132 to 141 us = 6.2 to 5.8 TB/s; 52 rows over 84 MB
// (11 requests of up to 13 tokens) take 25 us against 12.7 of bytes: the start, the row tiles' ends and the join.
//
// Two row tiles alternate ("pair"): while one's softmax runs, the tensor cores do the other's products. Each has its
// own warpgroup and O. One row tile ("lone"): each warpgroup takes 64 of a tile's 128 tokens of every row; the two
// threads of a row share its reference (moved together, through shared memory) and O, and add their sums at the end.
// Either way there is one S, which is free again as soon as its scores are in registers, and two places for P (product
// v of the sequence uses place v % 2): S of v + 1 is issued once S of v has been read, before PV of v - 1, so the next
// scores are under way through the whole of a softmax. (With P over S in two buffers, S of v + 2 had to wait for PV of
// v: 1.1 us of each 2.5 us were spent waiting for it.)
//
// References, partials, runs and entries that must not be seen are as in tree_attn.cuh.
#pragma once

#include <type_traits>

#include "tree_attn.cuh"

namespace muse {

// kRows: 256, or 128 where no request has more (one row tile: Q's second place goes to the ring).
template <int kDim, int kRows_>
struct WideShape {
  static constexpr int kRows = kRows_, kTok = 128;
  static constexpr int kHalves = kDim / 64;
  static constexpr int kThreads = 64 + 256 + 64;  // producer, UMMA, softmax, row loaders
  static constexpr int kStage = kTok * kDim * 2;
  static constexpr int kQ = 128 * kDim * 2;  // one row tile
  static constexpr int kNK = kDim == 64 ? 5 : (kRows == 128 ? 3 : 2), kNV = kDim == 64 ? 5 : (kRows == 128 ? 2 : 2);
  static constexpr int kTmem = 512;          // S [128], P [2][64], O [2][kDim]
  static constexpr int kOffV = kNK * kStage, kOffQ = kOffV + kNV * kStage, kOffSmall = kOffQ + kRows / 128 * kQ;
  // mask words [2][kRows][9] (the ninth zero), row ids [2][kRows], exchange [2][128], scan sums, segments, barriers
  static constexpr int kSmall = 2 * kRows * 9 * 4 + 2 * kRows * 4 + 2 * 128 * 4 + 64 + 128 + (2 * kNK + 2 * kNV + 15) * 8 + 64;
  static constexpr int kSmem = 1024 + kOffSmall + kSmall;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

// One tensor's tiles of a run into its ring of kN, a lane a box.
template <int kTok, int kRows, int kDim, int kN>
struct WideFeed {
  static constexpr int kStage = kTok * kDim * 2;
  const CUtensorMap* map;
  uint8_t* ring;
  uint64_t *full, *empty;
  int combo, box, lane;
  AttnWalk<kTok, kRows> walk;
  AttnSeg s;
  Ring at;
  int i, issued, page;
  bool have, more;
  __device__ __forceinline__ WideFeed(const AttnArgs& a, const AttnPlan& p, const CUtensorMap* map, int combo, uint8_t* ring, uint64_t* full,
                                      uint64_t* empty)
      : map(map), ring(ring), full(full), empty(empty), combo(combo), box(min(a.page, kTok)), lane(threadIdx.x & 31),
        walk(a, p.b0, p.s0, p.w0, p.w1), i(0), issued(0), page(0), have(false) {
    segment(a);
  }
  __device__ __forceinline__ void lookup(const AttnArgs& a) {
    const int pos = i * kTok + lane * box;
    have = lane < kTok / box && pos < s.r.kv;
    page = have ? a.table[s.b * a.table_row + static_cast<unsigned int>(pos) / static_cast<unsigned int>(a.page)] : 0;
  }
  __device__ __forceinline__ void segment(const AttnArgs& a) {
    more = walk.next(a, s);
    i = s.i0;
    if (more) lookup(a);
  }
  __device__ __forceinline__ bool ready() const { return __all_sync(0xffffffffu, mbar_test(smem_u32(&empty[at.slot]), at.phase ^ 1u)); }
  // Issues the current tile and moves on (the next tile's page is on its way while its place is waited for).
  __device__ __forceinline__ void issue(const AttnArgs& a, uint64_t stream, uint64_t keep) {
    const int now = page, in = ((i * kTok + lane * box) & (a.page - 1)) >> 3;
    const bool wrong = have && (now < 0 || now >= a.pages);
    if (wrong) report_error(kErrAttnPage);
    const uint32_t bytes = static_cast<uint32_t>(__popc(__ballot_sync(0xffffffffu, have))) * static_cast<uint32_t>(box * kDim * 2);
    if (lane == 0) mbar_expect_tx(&full[at.slot], bytes);
    __syncwarp();
    // Tokens that several row tiles read stay in L2; a request's only reader streams them.
    if (have)
      tma_load_5d(ring + at.slot * kStage + lane * box * kDim * 2, map, &full[at.slot], in, (wrong ? 0 : now) * combo + s.head,
                  s.r.rows > kRows ? keep : stream);
    at.next(kN);
    ++issued;
    if (++i < s.i1) lookup(a);
    else segment(a);
  }
  // The copies still under way land before the CTA may end.
  __device__ __forceinline__ void drain() {
    for (int n = max(issued - kN, 0); n < issued; ++n)
      mbar_wait(&full[n % kN], static_cast<uint32_t>((n / kN) & 1), kErrAttnDrain, kWaitLimitNs / 100);
  }
};

// The producer warp: K and V tiles in the order K, V, K, V while both have places free, else whichever has. A K tile is
// needed a whole softmax before its V tile, and with two V places the one-after-the-other order of attn_produce held back
// the scores that would free them: 242 us at 128 rows, dim 128 and 822 MB, 141 so. (The tokens-as-M kernel, with three
// places and every tile waiting on HBM, is faster with that order: 59 us at 32 x 4096, 64 so.)
template <int kTok, int kRows, int kDim, int kNK, int kNV>
__device__ __forceinline__ void wide_produce(const AttnArgs& a, const AttnPlan& plan, const CUtensorMap* tmk, const CUtensorMap* tmv,
                                             uint8_t* ring_k, uint8_t* ring_v, uint64_t* k_full, uint64_t* k_empty, uint64_t* v_full,
                                             uint64_t* v_empty) {
  static_assert(kTok / 8 <= 32, "a lane a box");
  WideFeed<kTok, kRows, kDim, kNK> k(a, plan, tmk, a.k_combo, ring_k, k_full, k_empty);
  WideFeed<kTok, kRows, kDim, kNV> v(a, plan, tmv, a.v_combo, ring_v, v_full, v_empty);
  const uint64_t stream = policy_evict_first(), keep = policy_evict_normal();
  unsigned long long since = 0;  // of a wait under way
  while (v.more) {
    bool idle = true;
    if (k.more && k.ready()) k.issue(a, stream, keep), idle = false;
    if (v.issued < k.issued && v.ready()) v.issue(a, stream, keep), idle = false;
    if (!idle) {
      since = 0;
      continue;
    }
    __nanosleep(40);
    const unsigned long long now = globaltimer();
    if (since == 0) since = now;
    if (now - since > kErrPollNs) {
      const bool late = now - since > kWaitLimitNs;
      if (late) report_error(kErrAttnProducer);
      if (__any_sync(0xffffffffu, late || error_raised())) break;
    }
  }
  k.drain();
  v.drain();
}

// kN columns of this warp's lanes.
template <int kN>
__device__ __forceinline__ void wide_ld(uint32_t taddr, float (&v)[kN]) {
#pragma unroll
  for (int i = 0; i < kN; i += 16) attn_ld16(taddr + i, v + i);
#pragma unroll
  for (int i = 0; i < kN; i += 16) attn_ld_wait(v + i);
}

// Two FP32 fused multiply-adds (or sums) an instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// 32 bytes, 32-byte aligned.
__device__ __forceinline__ void st_global_v8(float* p, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
               "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// D (+)= A . B with A [128 x 16] in tensor memory (16-bit pairs), B from shared memory.
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, uint32_t n) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(n) : "memory");
}

// Bits k = 0 .. 31: whether tokens pos0 + k (pos0 = first of a 32-token part) are seen, from the row's words.
__device__ __forceinline__ uint32_t wide_seen(const uint32_t* row_words, int j0) {
  if (j0 <= -32) return 0xffffffffu;
  if (j0 < 0) return (row_words[0] << -j0) | ((1u << -j0) - 1u);
  if (j0 >= 256) return 0u;
  return __funnelshift_r(row_words[j0 >> 5], row_words[(j0 >> 5) + 1], j0 & 31);
}

template <bool kHalf, int kDim, int kRows>
__global__ void __launch_bounds__(WideShape<kDim, kRows>::kThreads, 1)
    tree_attn_wide_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const AttnArgs a) {
  using Sh = WideShape<kDim, kRows>;
  constexpr int kHalves = Sh::kHalves, kNK = Sh::kNK, kNV = Sh::kNV, kTok = Sh::kTok;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_align<1024>(smem_raw);
  uint8_t* ring_k = smem;
  uint8_t* ring_v = smem + Sh::kOffV;
  uint8_t* q_s = smem + Sh::kOffQ;
  uint32_t* all_words = reinterpret_cast<uint32_t*>(smem + Sh::kOffSmall);  // [2][kRows][9]
  int* row_ids = reinterpret_cast<int*>(all_words + 2 * kRows * 9);         // [2][kRows]
  float* swap = reinterpret_cast<float*>(row_ids + 2 * kRows);              // [2][128]
  int* sums = reinterpret_cast<int*>(swap + 256);
  AttnSeg* segs = reinterpret_cast<AttnSeg*>(sums + 16);                    // [2]
  uint64_t* k_full = reinterpret_cast<uint64_t*>(segs) + 16;
  uint64_t* k_empty = k_full + kNK;
  uint64_t* v_full = k_empty + kNK;
  uint64_t* v_empty = v_full + kNV;
  uint64_t* s_full = v_empty + kNV;  // [2]
  uint64_t* p_full = s_full + 2;     // [2], 256 arrivals: one a thread (lone) or two (pair)
  uint64_t* pv_done = p_full + 2;    // [2]
  uint64_t* s_read = pv_done + 2;    // 256 arrivals as p_full's
  uint64_t* q_full = s_read + 1;
  uint64_t* q_empty = q_full + 2;    // q_full [2], seg_done [2]: by segment parity
  uint64_t* seg_done = q_empty + 1;
  uint64_t* fin = seg_done + 2;
  int* start = reinterpret_cast<int*>(fin + 1);  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(start + 2);
  int* odd_vs = reinterpret_cast<int*>(tmem_slot + 1);  // [2]

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&tmk);
    prefetch_tensormap(&tmv);
    for (int i = 0; i < kNK; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < kNV; ++i) mbar_init(&v_full[i], 1), mbar_init(&v_empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 256), mbar_init(&pv_done[i], 1);
    mbar_init(s_read, 256);
    for (int i = 0; i < 2; ++i) mbar_init(&q_full[i], 64), mbar_init(&seg_done[i], 256);
    mbar_init(q_empty, 1);
    odd_vs[0] = odd_vs[1] = 0;
    mbar_init(fin, 1);
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, Sh::kTmem);
  pdl_launch_dependents();
  pdl_wait();
  const AttnPlan plan = attn_plan<Sh::kThreads, kTok, kRows>(a, sums, start);
  const uint32_t tmem = static_cast<uint32_t>(uniform(static_cast<int>(*tmem_slot)));
  const uint32_t tmem_p = tmem + 128, tmem_o = tmem + 256;

  if (warp == 0) {
    if (plan.work)
      wide_produce<kTok, kRows, kDim, kNK, kNV>(a, plan, &tmk, &tmv, ring_k, ring_v, k_full, k_empty, v_full, v_empty);
  } else if (warp == 1) {
    // ---- UMMA issue --------------------------------------------------------------------------------
    if (uniform(plan.work)) {
      constexpr uint32_t kType = (1u << 4) | (8u << 24) | (kHalf ? 0u : ((1u << 7) | (1u << 10)));
      constexpr uint32_t idesc_s = kType | (static_cast<uint32_t>(kTok >> 3) << 17);
      constexpr uint32_t idesc_o = kType | (static_cast<uint32_t>(kDim >> 3) << 17) | (1u << 16);
      constexpr uint64_t k_bits = attn_desc_bits(128, 1024 * kHalves, 16);
      constexpr uint64_t v_bits = attn_desc_bits(128, 1024 * kHalves, kHalves > 1 ? 1024 : 0);
      Ring rk, rv;
      uint32_t v0 = 0;  // products before this segment
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_idle(bar, parity, kErrAttnMma)) != 0; };
      for (int k = 0;; ++k) {
        if (!(ok = wait(&q_full[k & 1], (k >> 1) & 1))) break;
        const AttnSeg& s = segs[k & 1];
        const int pair = kRows > 128 ? uniform(s.r.rows - s.row0 > 128 ? 1 : 0) : 0;
        const int products = uniform((s.i1 - s.i0) << pair);
        if (products == 0) break;
        tc_fence_after();
        // The first (or only) row tile's product waits for a K tile, the last releases it; V alike.
        auto issue_s = [&](int v) {
          const int tile = pair & v;
          if (tile == 0 && !wait(&k_full[rk.slot], rk.phase)) return false;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t dk = k_bits | ((smem_u32(ring_k + rk.slot * Sh::kStage) & 0x3FFFFu) >> 4);
            const uint64_t dq = umma_desc_sw128(smem_u32(q_s + tile * Sh::kQ));
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_bf16(tmem, dq + ((h * 128 * 128) >> 4) + 2 * k, dk + ((h * 1024) >> 4) + 2 * k, idesc_s, (h | k) != 0);
            if (tile == pair) umma_commit(&k_empty[rk.slot]);
            umma_commit(&s_full[(v0 + v) & 1u]);
            if (v + 1 == products) umma_commit(q_empty);
          }
          __syncwarp();
          if (tile == pair) rk.next(kNK);
          return true;
        };
        // S holds the last scores of the segment before until they have been read.
        ok = (k == 0 || wait(s_read, (v0 - 1) & 1u)) && issue_s(0);
        for (int u = 0; ok && u <= products; ++u) {
          if (u + 1 < products) {
            ok = wait(s_read, (v0 + u) & 1u) && issue_s(u + 1);
            if (!ok) break;
          }
          if (u == 0) continue;
          const int v = u - 1, tile = pair & v;
          const uint32_t n = v0 + v, buffer = n & 1u;
          ok = wait(&p_full[buffer], (n >> 1) & 1u) && (tile != 0 || wait(&v_full[rv.slot], rv.phase));
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t dv = v_bits | ((smem_u32(ring_v + rv.slot * Sh::kStage) & 0x3FFFFu) >> 4);
#pragma unroll
            for (int k = 0; k < kTok / 16; ++k)
              umma_ts(tmem_o + tile * kDim, tmem_p + buffer * 64 + k * 8, dv + ((k * 16 * kDim * 2) >> 4), idesc_o,
                      (v > pair || k > 0) ? 1u : 0u);
            if (tile == pair) umma_commit(&v_empty[rv.slot]);
            umma_commit(&pv_done[buffer]);
          }
          __syncwarp();
          if (tile == pair) rv.next(kNV);
        }
        v0 += products;
        if (!ok) break;
      }
      if (elect_one()) umma_commit(fin);
      __syncwarp();
      mbar_wait(fin, 0u, kErrAttnDrain, kWaitLimitNs / 10);  // nothing of the tensor cores is under way past here
    }
    __syncwarp();
  } else if (warp >= 10) {
    if (plan.work)
      attn_load_rows<kTok, kRows, 128, 128, kDim, 64>(a, plan, static_cast<int>(threadIdx.x) - 320, q_s, segs, all_words, row_ids, q_full,
                                                     q_empty, seg_done);
  } else {
    // ---- softmax: thread = one row -----------------------------------------------------------------
    const int tid = static_cast<int>(threadIdx.x) - 64, wg = tid >> 7;
    const int quarter = warp & 3, tl = quarter * 32 + lane;  // TMEM lane = row of the row tile
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const float kNegInf = __int_as_float(0xff800000);
    const float c = a.scale_log2;
    AttnCross cross = {};
    if (plan.work) {
      uint32_t v0 = 0, v_slot = 0, v_phase = 0;
      bool ok = true;
      for (int k = 0;; ++k) {
        ok = mbar_wait_idle(&q_full[k & 1], (k >> 1) & 1, kErrAttnSoftmax);
        if (bar_any(8, 256, !ok)) break;  // every thread is done with the last segment's arrays, too
        const AttnSeg s = segs[k & 1];
        if (s.i1 <= s.i0) break;
        const int rows = min(kRows, s.r.rows - s.row0);
        const bool pair = kRows > 128 && rows > 128;
        const int row = pair ? wg * 128 + tl : tl;  // this thread's row of the unit
        const bool mine = row < rows;
        const uint32_t* words = all_words + (k & 1) * kRows * 9;
        int* odd_v = odd_vs + (k & 1);
        if (tid == 0) odd_vs[(k + 1) & 1] = 0;

        // The products of this thread's row tile in the sequence, and its row's running values.
        const int step = pair ? 2 : 1, products = (s.i1 - s.i0) << (pair ? 1 : 0);
        const uint32_t o_base = tmem_o + (pair ? wg * kDim : 0) + lanes;
        float ref = kAttnUnseen, l = 0.f;
        // One product's softmax over this thread's kN columns (128: pair, 64: lone). False: a wait gave up, for all
        // threads that share a vote (a warp, or both warpgroups).
        auto product = [&](auto columns, int v) {
          constexpr int kN = decltype(columns)::value;
          constexpr bool kPair = kN == 128;
          const uint32_t n = v0 + v, buffer = n & 1u;
          const int i = s.i0 + (kPair ? v >> 1 : v), col0 = kPair ? 0 : wg * 64;
          const bool edge = (i + 1) * kTok > s.r.ctx;  // the tile reaches past the context
          if (wg == 0 && edge) {
            // One token without a mask sees itself: only then is no drafted entry hidden from a row.
            const bool ragged = (i + 1) * kTok > s.r.kv, drafted = s.r.drafted > 1 || a.mask;
            if (ragged || drafted) {
              // The place's fill before is complete once PV of two products ago is: only then does the parity name this fill.
              if (v >= 2) ok = mbar_wait_idle(&pv_done[buffer], ((n - 2) >> 1) & 1u, kErrAttnSoftmax) && ok;
              ok = mbar_wait_idle(&v_full[v_slot], v_phase, kErrAttnSoftmax) && ok;
              const int pos = i * kTok + tl;
              attn_clean_v<kHalf, kDim>(smem_u32(ring_v + v_slot * Sh::kStage), tl, pos >= s.r.kv, drafted && pos >= s.r.ctx, odd_v);
              fence_proxy_async_shared();
            }
          }
          ok = mbar_wait_idle(&s_full[buffer], (n >> 1) & 1u, kErrAttnSoftmax) && ok;
          tc_fence_after();
          float x[kN];
          wide_ld<kN>(tmem + col0 + lanes, x);
          tc_fence_before();
          if (kPair) mbar_arrive_n(s_read, 2);
          else mbar_arrive(s_read);
          if (edge) {
#pragma unroll
            for (int cc = 0; cc < kN; cc += 32) {
              const uint32_t seen = wide_seen(words + row * 9, i * kTok + col0 + cc - s.r.ctx);
#pragma unroll
              for (int k = 0; k < 32; ++k) x[cc + k] = (seen >> k) & 1u ? x[cc + k] : kNegInf;
            }
          }
          float m[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
          for (int k = 4; k < kN; ++k) m[k & 3] = fmaxf(m[k & 3], x[k]);
          float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * c;
          // Whether this warp (pair) or any softmax thread (lone) has a reference to move.
          const bool past = top - ref > kAttnSlack<kHalf> || !ok;
          if (kPair ? __any_sync(0xffffffffu, past) : bar_any(8, 256, past)) {
            if (kPair ? __any_sync(0xffffffffu, !ok) : bar_any(8, 256, !ok)) return false;
            if (!kPair) {
              swap[wg * 128 + tl] = top;
              bar_named(8, 256);
              top = fmaxf(top, swap[(wg ^ 1) * 128 + tl]);
              bar_named(8, 256);
            }
            const float now = fmaxf(ref, top - kAttnBelow<kHalf>), f = ex2(ref - now);
            ref = now;
            l *= f;
            if (v >= step) {
              // O has to be whole up to this row tile's product before.
              ok = mbar_wait_idle(&pv_done[(n - step) & 1u], ((n - step) >> 1) & 1u, kErrAttnSoftmax) && ok;
              tc_fence_after();
              const int d0 = kPair ? 0 : wg * (kDim / 2), d1 = kPair ? kDim : d0 + kDim / 2;
#pragma unroll 1
              for (int d = d0; d < d1; d += 16) {
                float o[16];
                wide_ld<16>(o_base + d, o);
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] *= f;
                attn_st16(o_base + d, o);
              }
              attn_st_wait();
            }
          }
          // P, rounded, once its place is free: 32 scores become 16 words.
          if (v >= 2) ok = mbar_wait_idle(&pv_done[buffer], ((n - 2) >> 1) & 1u, kErrAttnSoftmax) && ok;
          tc_fence_after();
          float2 sum = {0.f, 0.f};
          const float2 cc2 = {c, c}, mm2 = {-ref, -ref};
#pragma unroll
          for (int cc = 0; cc < kN; cc += 32) {
            float p[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float2 e = fma2({x[cc + 2 * k], x[cc + 2 * k + 1]}, cc2, mm2);
              const uint32_t w = pack16x2<kHalf>(ex2(e.x), ex2(e.y));
              add16x2<kHalf>(w, sum.x, sum.y);
              p[k] = __uint_as_float(w);
            }
            attn_st16(tmem_p + buffer * 64 + ((col0 + cc) >> 1) + lanes, p);
          }
          l += sum.x + sum.y;
          attn_st_wait();
          if (++v_slot == kNV) v_slot = 0, v_phase ^= 1u;
          tc_fence_before();
          if (kPair) mbar_arrive_n(&p_full[buffer], 2);
          else mbar_arrive(&p_full[buffer]);
          return true;
        };
        // A wait that gave up is carried to the next vote: the loop's end has to be the same for all that vote.
        if (pair) {
          for (int v = wg; v < products; v += 2)
            if (!product(std::integral_constant<int, 128>{}, v)) break;
        } else {
          for (int v = 0; v < products; ++v)
            if (!product(std::integral_constant<int, 64>{}, v)) break;
        }

        // ---- end of the segment: finish the rows, or leave a partial ---------------------------------
        if (ok) {
          const uint32_t n = v0 + products - (pair ? 2 - wg : 1);
          ok = mbar_wait_idle(&pv_done[n & 1u], (n >> 1) & 1u, kErrAttnSoftmax);
        }
        swap[wg * 128 + tl] = l;
        ok = !bar_any(8, 256, !ok);
        if (!ok) break;
        tc_fence_after();
        v0 += products;
        if (!pair) l += swap[(wg ^ 1) * 128 + tl];
        const bool whole = s.i0 == 0 && s.i1 == s.r.tiles;
        const long long slot = (static_cast<long long>(blockIdx.x) * 2 + (s.i0 > 0 ? 0 : 1)) * kRows + row;
        if (!whole && mine && (pair || wg == 0)) a.part_ml[slot] = make_float2(ref, l);
        if (!whole && s.i0 == 0) {
          cross.first = s.r.first, cross.row0 = s.row0, cross.rows = rows, cross.head = s.head;
          cross.last = plan.runs.of(s.unit0 + s.r.tiles - 1);
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int odd = *odd_v;
        // A thread writes its own row.
        const int id = row_ids[(k & 1) * kRows + row], t = id >> 16, h = id & 0xFFFF;
        const int d0 = pair ? 0 : wg * (kDim / 2), d1 = pair ? kDim : d0 + kDim / 2;
        uint16_t* out = a.out + (s.r.first + t) * a.out_token + h * a.out_head;
        const uint16_t* gate = a.gate ? a.gate + (s.r.first + t) * a.gate_token + h * a.gate_head : nullptr;
        float* part = a.part_o + slot * kDim;
#pragma unroll 1
        for (int d = d0; d < d1; d += 16) {
          uint4 g0 = make_uint4(0u, 0u, 0u, 0u), g1 = g0;
          if (whole && gate && mine) g0 = __ldg(reinterpret_cast<const uint4*>(gate + d)), g1 = __ldg(reinterpret_cast<const uint4*>(gate + d) + 1);
          float o[16];
          wide_ld<16>(o_base + d, o);
          if (!mine) continue;
          if (odd) {
            // Put the non-finite entries back for the rows that see them.
            const int j0 = max(s.i0 * kTok - s.r.ctx, 0), j1 = min(min(s.i1 * kTok, s.r.kv) - s.r.ctx, s.r.drafted);
            for (int j = j0; j < j1; ++j) {
              if (!((words[row * 9 + (j >> 5)] >> (j & 31)) & 1u)) continue;
              const int p = s.r.ctx + j;
              const long long page = a.table[s.b * a.table_row + p / a.page];
              if (page < 0 || page >= a.pages) continue;
              const uint16_t* src = a.v_pages + page * a.v_page + s.head * a.v_head + (p % a.page) * a.v_slot + d;
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                const float x = lo16<kHalf>(src[k]);
                if (!(fabsf(x) < __int_as_float(0x7f800000))) o[k] += x;
              }
            }
          }
          if (whole) {
            const uint32_t gw[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
            uint32_t w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              float e0 = o[2 * k] * inv, e1 = o[2 * k + 1] * inv;
              if (gate) {
                e0 = __fdividef(e0, 1.f + __expf(-lo16<kHalf>(gw[k])));
                e1 = __fdividef(e1, 1.f + __expf(-hi16<kHalf>(gw[k])));
              }
              w[k] = pack16x2<kHalf>(e0, e1);
            }
            // out is 16-byte aligned, not 32: two stores.
            reinterpret_cast<uint4*>(out + d)[0] = make_uint4(w[0], w[1], w[2], w[3]);
            reinterpret_cast<uint4*>(out + d)[1] = make_uint4(w[4], w[5], w[6], w[7]);
          } else {
            st_global_v8(part + d, o);
            st_global_v8(part + d + 8, o + 8);
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

}  // namespace muse
