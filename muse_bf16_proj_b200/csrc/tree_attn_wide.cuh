// tree_attention with many rows a kv head (more than 64): rows as the tensor cores' M.
//
// A unit is up to 256 rows (tokens x heads of a group) of one request and kv head: one or two row tiles of 128, which
// share every K and V tile that is brought in. For a row tile and 128 cached tokens
//   S [128 rows x 128 tokens] = Q . K^T            (both K-major from shared memory)
//   O [128 rows x dim]       += P . V              (P from tensor memory over S's columns, V as stored, N-major)
// A row is a TMEM lane and one softmax thread's, so its maximum, its references and its sums need no other thread,
// and P never passes through shared memory. Bound: at 2 x 128 rows the two products take 1024 tensor cycles a tile at
// dim 128 and its 16384 exponentials as many cycles of the exponential unit; K and V come in once for both.
//
// Two row tiles alternate ("pair"): while one's softmax runs, the tensor cores do the other's products. Each has its
// own warpgroup, S buffer and O. One row tile ("lone"): the S buffers take turns over the token tiles and each
// warpgroup takes 64 of a tile's 128 tokens of every row; the two threads of a row share its reference (moved
// together, through shared memory) and O, and add their sums at the end. Either way product v of the sequence uses S
// buffer v % 2, and S of v + 2 is issued right after PV of v, whose P stands in that buffer.
//
// References, partials, runs and entries that must not be seen are as in tree_attn.cuh.
#pragma once

#include "tree_attn.cuh"

namespace muse {

template <int kDim>
struct WideShape {
  static constexpr int kRows = 256, kTok = 128;
  static constexpr int kHalves = kDim / 64;
  static constexpr int kThreads = 64 + 256;
  static constexpr int kStage = kTok * kDim * 2;
  static constexpr int kQ = 128 * kDim * 2;  // one row tile
  static constexpr int kNK = kDim == 64 ? 4 : 2, kNV = kNK;
  static constexpr int kTmem = 512;          // S [2][128], O [2][kDim]
  static constexpr int kOffV = kNK * kStage, kOffQ = kOffV + kNV * kStage, kOffSmall = kOffQ + 2 * kQ;
  // mask words [256][9] (the ninth zero), exchange [2][128], scan sums, barriers
  static constexpr int kSmall = 256 * 9 * 4 + 2 * 128 * 4 + 64 + (2 * kNK + 2 * kNV + 10) * 8 + 64;
  static constexpr int kSmem = 1024 + kOffSmall + kSmall;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

// 32 columns of this warp's lanes, not waited for, and the wait that the registers depend on.
__device__ __forceinline__ void attn_ld32(uint32_t taddr, float (&v)[32]) {
  attn_ld16(taddr, v);
  attn_ld16(taddr + 16, v + 16);
}
__device__ __forceinline__ void attn_ld32_wait(float (&v)[32]) {
  attn_ld_wait(v);
  attn_ld_wait(v + 16);
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

template <bool kHalf, int kDim>
__global__ void __launch_bounds__(WideShape<kDim>::kThreads, 1)
    tree_attn_wide_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const AttnArgs a) {
  using Sh = WideShape<kDim>;
  using Walk = AttnWalk<Sh::kTok, Sh::kRows>;
  constexpr int kHalves = Sh::kHalves, kNK = Sh::kNK, kNV = Sh::kNV, kTok = Sh::kTok;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_align<1024>(smem_raw);
  uint8_t* ring_k = smem;
  uint8_t* ring_v = smem + Sh::kOffV;
  uint8_t* q_s = smem + Sh::kOffQ;
  uint32_t* words = reinterpret_cast<uint32_t*>(smem + Sh::kOffSmall);  // [256][9]
  float* swap = reinterpret_cast<float*>(words + 256 * 9);              // [2][128]
  int* sums = reinterpret_cast<int*>(swap + 256);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(sums + 16);
  uint64_t* k_empty = k_full + kNK;
  uint64_t* v_full = k_empty + kNK;
  uint64_t* v_empty = v_full + kNV;
  uint64_t* s_full = v_empty + kNV;  // [2]
  uint64_t* p_full = s_full + 2;     // [2], 256 arrivals: one a thread (lone) or two (pair)
  uint64_t* pv_done = p_full + 2;    // [2]
  uint64_t* q_full = pv_done + 2;
  uint64_t* fin = q_full + 1;
  int* start = reinterpret_cast<int*>(fin + 1);  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(start + 2);
  int* odd_v = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&tmk);
    prefetch_tensormap(&tmv);
    for (int i = 0; i < kNK; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < kNV; ++i) mbar_init(&v_full[i], 1), mbar_init(&v_empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 256), mbar_init(&pv_done[i], 1);
    mbar_init(q_full, 256);
    mbar_init(fin, 1);
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, Sh::kTmem);
  pdl_launch_dependents();
  pdl_wait();
  const AttnPlan plan = attn_plan<Sh::kThreads, kTok, Sh::kRows>(a, sums, start);
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_o = tmem + 256;

  if (warp == 0) {
    if (plan.work)
      attn_produce<kTok, Sh::kRows, kDim, kNK, kNV>(a, plan, &tmk, &tmv, ring_k, ring_v, k_full, k_empty, v_full, v_empty);
  } else if (warp == 1) {
    // ---- UMMA issue --------------------------------------------------------------------------------
    if (plan.work && lane == 0) {
      Walk walk(a, plan.b0, plan.s0, plan.w0, plan.w1);
      AttnSeg s;
      constexpr uint32_t kType = (1u << 4) | (8u << 24) | (kHalf ? 0u : ((1u << 7) | (1u << 10)));
      constexpr uint32_t idesc_s = kType | (static_cast<uint32_t>(kTok >> 3) << 17);
      constexpr uint32_t idesc_o = kType | (static_cast<uint32_t>(kDim >> 3) << 17) | (1u << 16);
      constexpr uint64_t k_bits = attn_desc_bits(128, 1024 * kHalves, 16);
      constexpr uint64_t v_bits = attn_desc_bits(128, 1024 * kHalves, kHalves > 1 ? 1024 : 0);
      Ring rk, rv;
      uint32_t seg_phase = 0, v0 = 0;  // products before this segment
      bool ok = true;
      while (ok && walk.next(a, s)) {
        ok = mbar_wait(q_full, seg_phase, kErrAttnMma);
        seg_phase ^= 1u;
        if (!ok) break;
        tc_fence_after();
        const int pair = s.r.rows - s.row0 > 128 ? 1 : 0;
        const int products = (s.i1 - s.i0) << pair;
        // The first (or only) row tile's product waits for a K tile, the last releases it; V alike.
        auto issue_s = [&](int v) {
          const int tile = pair & v;
          if (tile == 0 && !mbar_wait(&k_full[rk.slot], rk.phase, kErrAttnMma)) return false;
          tc_fence_after();
          const uint64_t dk = k_bits | ((smem_u32(ring_k + rk.slot * Sh::kStage) & 0x3FFFFu) >> 4);
          const uint64_t dq = umma_desc_sw128(smem_u32(q_s + tile * Sh::kQ));
          const uint32_t buffer = (v0 + v) & 1u;
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_bf16(tmem + buffer * 128, dq + ((h * 128 * 128) >> 4) + 2 * k, dk + ((h * 1024) >> 4) + 2 * k, idesc_s, (h | k) != 0);
          if (tile == pair) {
            umma_commit(&k_empty[rk.slot]);
            rk.next(kNK);
          }
          umma_commit(&s_full[buffer]);
          return true;
        };
        ok = issue_s(0) && (products < 2 || issue_s(1));
        for (int v = 0; ok && v < products; ++v) {
          const int tile = pair & v;
          const uint32_t n = v0 + v, buffer = n & 1u;
          ok = mbar_wait(&p_full[buffer], (n >> 1) & 1u, kErrAttnMma) && (tile != 0 || mbar_wait(&v_full[rv.slot], rv.phase, kErrAttnMma));
          if (!ok) break;
          tc_fence_after();
          const uint64_t dv = v_bits | ((smem_u32(ring_v + rv.slot * Sh::kStage) & 0x3FFFFu) >> 4);
#pragma unroll
          for (int k = 0; k < kTok / 16; ++k)
            umma_ts(tmem_o + tile * kDim, tmem + buffer * 128 + k * 8, dv + ((k * 16 * kDim * 2) >> 4), idesc_o,
                    (v > pair || k > 0) ? 1u : 0u);
          if (tile == pair) {
            umma_commit(&v_empty[rv.slot]);
            rv.next(kNV);
          }
          umma_commit(&pv_done[buffer]);
          if (v + 2 < products) ok = issue_s(v + 2);
        }
        v0 += products;
      }
      umma_commit(fin);
      mbar_wait(fin, 0u, kErrAttnDrain, kWaitLimitNs / 10);  // nothing of the tensor cores is under way past here
    }
    __syncwarp();
  } else {
    // ---- softmax: thread = one row -----------------------------------------------------------------
    const int tid = static_cast<int>(threadIdx.x) - 64, wg = tid >> 7;
    const int quarter = warp & 3, tl = quarter * 32 + lane;  // TMEM lane = row of the row tile
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const int g = a.heads / a.kv_heads;
    const float kNegInf = __int_as_float(0xff800000);
    const float c = a.scale_log2;
    AttnCross cross = {};
    if (plan.work) {
      Walk walk(a, plan.b0, plan.s0, plan.w0, plan.w1);
      AttnSeg s;
      uint32_t v0 = 0, v_slot = 0, v_phase = 0;
      bool ok = true;
      while (ok && walk.next(a, s)) {
        const int rows = min(Sh::kRows, s.r.rows - s.row0);
        const bool pair = rows > 128;
        const int row = pair ? wg * 128 + tl : tl;                   // this thread's row of the unit
        const bool mine = row < rows;
        const int t = mine ? attn_token(a, s.row0 + row) : 0, h = s.head * g + s.row0 + row - t * g;
        bar_named(8, 256);  // every thread is done with the last segment's arrays
        // Q: each warp brings whole rows, 16 (8) lanes a row, eight loads in flight.
        const int q_rows = pair ? 256 : 128;
        constexpr int kChunks = kDim / 8, kBatch = 8;
        for (int base = 0; base < q_rows * kChunks; base += 256 * kBatch) {
          uint4 qv[kBatch];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            const int i = base + tid + u * 256, r = i / kChunks, ch = i % kChunks;
            qv[u] = make_uint4(0u, 0u, 0u, 0u);
            if (r < rows) {
              const int tr = attn_token(a, s.row0 + r);
              qv[u] = __ldg(reinterpret_cast<const uint4*>(a.q + (s.r.first + tr) * a.q_token +
                                                           (s.head * g + s.row0 + r - tr * g) * a.q_head + ch * 8));
            }
          }
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            const int i = base + tid + u * 256, r = i / kChunks, ch = i % kChunks;
            if (r < q_rows)
              st_shared_v4u(smem_u32(q_s) + (r >> 7) * Sh::kQ + (ch >> 3) * (128 * 128) + (r & 127) * 128 + (((ch & 7) ^ (r & 7)) << 4),
                            qv[u].x ^ a.q_flip, qv[u].y ^ a.q_flip, qv[u].z ^ a.q_flip, qv[u].w ^ a.q_flip);
          }
        }
        if (wg == 0 || pair) {
          const int nw = (s.r.drafted + 31) >> 5;
          for (int w = 0; w < nw; ++w) words[row * 9 + w] = mine ? attn_seen_word(a, s.r, t, w) : 0u;
          for (int w = nw; w < 9; ++w) words[row * 9 + w] = 0u;
        }
        if (tid == 0) *odd_v = 0;
        fence_proxy_async_shared();
        mbar_arrive(q_full);
        bar_named(8, 256);

        // A thread's columns of a product, its products in the sequence, and its row's running values.
        const int col0 = pair ? 0 : wg * 64, col1 = pair ? 128 : col0 + 64;
        const int step = pair ? 2 : 1, products = (s.i1 - s.i0) << (pair ? 1 : 0);
        const uint32_t o_base = tmem_o + (pair ? wg * kDim : 0) + lanes;
        float ref = kAttnUnseen, l = 0.f;
        // A wait that gave up is carried to the next vote: the loop's end has to be the same for a warp (pair) or all (lone).
        for (int v = pair ? wg : 0; v < products; v += step) {
          const uint32_t n = v0 + v, buffer = n & 1u;
          const int i = s.i0 + (pair ? v >> 1 : v);
          ok = mbar_wait(&s_full[buffer], (n >> 1) & 1u, kErrAttnSoftmax) && ok;
          tc_fence_after();
          const uint32_t ts = tmem + buffer * 128 + lanes;
          const bool edge = (i + 1) * kTok > s.r.ctx;  // the tile reaches past the context
          // Largest score of the row (of this thread's columns).
          float top = kNegInf;
          for (int cc = col0; cc < col1; cc += 32) {
            float x[32];
            attn_ld32(ts + cc, x);
            attn_ld32_wait(x);
            if (edge) {
              const uint32_t seen = wide_seen(words + row * 9, i * kTok + cc - s.r.ctx);
#pragma unroll
              for (int k = 0; k < 32; ++k) x[k] = (seen >> k) & 1u ? x[k] : kNegInf;
            }
            float m[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
            for (int k = 4; k < 32; ++k) m[k & 3] = fmaxf(m[k & 3], x[k]);
            top = fmaxf(top, fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
          }
          top *= c;
          const bool past = top - ref > kAttnSlack;
          // Whether this warp (pair) or the CTA's softmax threads (lone) have a reference to move.
          const bool move = pair ? __any_sync(0xffffffffu, past || !ok) : bar_any(8, 256, past || !ok);
          if (move) {
            if (pair ? __any_sync(0xffffffffu, !ok) : bar_any(8, 256, !ok)) {
              ok = false;
              break;
            }
            if (!pair) {
              swap[wg * 128 + tl] = top;
              bar_named(8, 256);
              top = fmaxf(top, swap[(wg ^ 1) * 128 + tl]);
              bar_named(8, 256);
            }
            const float now = fmaxf(ref, top), f = ex2(ref - now);
            ref = now;
            l *= f;
            if (v >= step) {
              // O is whole up to the product before: the pair's last of this row tile came before S, the lone one's not.
              if (!pair) {
                ok = mbar_wait(&pv_done[(n - 1) & 1u], ((n - 1) >> 1) & 1u, kErrAttnSoftmax) && ok;
                tc_fence_after();
              }
              const int d0 = pair ? 0 : wg * (kDim / 2), d1 = pair ? kDim : d0 + kDim / 2;
              for (int d = d0; d < d1; d += 32) {
                float o[32];
                attn_ld32(o_base + d, o);
                attn_ld32_wait(o);
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] *= f;
                attn_st16(o_base + d, o);
                attn_st16(o_base + d + 16, o + 16);
              }
              attn_st_wait();
            }
          }
          // P over S's columns, rounded; 32 scores become 16 words, behind what is still to be read. (Lone: the
          // second warpgroup writes over columns the first may still have to read, so it waits for it below.)
          uint32_t w[2][16];
          for (int cc = col0; cc < col1; cc += 32) {
            float x[32];
            attn_ld32(ts + cc, x);
            attn_ld32_wait(x);
            if (edge) {
              const uint32_t seen = wide_seen(words + row * 9, i * kTok + cc - s.r.ctx);
#pragma unroll
              for (int k = 0; k < 32; ++k) x[k] = (seen >> k) & 1u ? x[k] : kNegInf;
            }
            float l0 = 0.f, l1 = 0.f;
            uint32_t p[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              p[k] = pack16x2<kHalf>(ex2(fmaf(x[2 * k], c, -ref)), ex2(fmaf(x[2 * k + 1], c, -ref)));
              add16x2<kHalf>(p[k], l0, l1);
            }
            l += l0 + l1;
            if (pair) {
              attn_st16(ts + (cc >> 1), reinterpret_cast<const float*>(p));
            } else {
#pragma unroll
              for (int k = 0; k < 16; ++k) w[0][k] = cc == col0 ? p[k] : w[0][k], w[1][k] = p[k];
            }
          }
          if (!pair) {
            bar_named(8, 256);  // both warpgroups have read all of S
            attn_st16(ts + (col0 >> 1), reinterpret_cast<const float*>(w[0]));
            attn_st16(ts + (col0 >> 1) + 16, reinterpret_cast<const float*>(w[1]));
          }
          attn_st_wait();
          if (wg == 0) {
            const bool ragged = (i + 1) * kTok > s.r.kv, drafted = edge && s.r.drafted > 1;
            if (ragged || drafted) {
              ok = mbar_wait(&v_full[v_slot], v_phase, kErrAttnSoftmax) && ok;
              const int pos = i * kTok + tl;
              attn_clean_v<kHalf, kDim>(smem_u32(ring_v + v_slot * Sh::kStage), tl, pos >= s.r.kv, drafted && pos >= s.r.ctx, odd_v);
              fence_proxy_async_shared();
            }
          }
          if (++v_slot == kNV) v_slot = 0, v_phase ^= 1u;
          tc_fence_before();
          if (pair) mbar_arrive_n(&p_full[buffer], 2);
          else mbar_arrive(&p_full[buffer]);
        }

        // ---- end of the segment: finish the rows, or leave a partial ---------------------------------
        if (ok) {
          const uint32_t n = v0 + products - (pair ? 2 - wg : 1);
          ok = mbar_wait(&pv_done[n & 1u], (n >> 1) & 1u, kErrAttnSoftmax);
        }
        swap[wg * 128 + tl] = l;
        ok = !bar_any(8, 256, !ok);
        if (!ok) break;
        tc_fence_after();
        v0 += products;
        if (!pair) l += swap[(wg ^ 1) * 128 + tl];
        const bool whole = s.i0 == 0 && s.i1 == s.r.tiles;
        const long long slot = (static_cast<long long>(blockIdx.x) * 2 + (s.i0 > 0 ? 0 : 1)) * Sh::kRows + row;
        if (!whole && mine && (pair || wg == 0)) a.part_ml[slot] = make_float2(ref, l);
        if (!whole && s.i0 == 0) {
          cross.first = s.r.first, cross.row0 = s.row0, cross.rows = rows, cross.head = s.head;
          cross.last = plan.runs.of(s.unit0 + s.r.tiles - 1);
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int odd = *odd_v;
        const int d0 = pair ? 0 : wg * (kDim / 2), d1 = pair ? kDim : d0 + kDim / 2;
        for (int d = d0; d < d1; d += 32) {
          float o[32];
          attn_ld32(o_base + d, o);
          uint4 gv[4];
          if (whole && a.gate && mine) {
            const uint4* src = reinterpret_cast<const uint4*>(a.gate + (s.r.first + t) * a.gate_token + h * a.gate_head + d);
#pragma unroll
            for (int k = 0; k < 4; ++k) gv[k] = __ldg(src + k);
          }
          attn_ld32_wait(o);
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
              for (int k = 0; k < 32; ++k) {
                const float e = lo16<kHalf>(src[k]);
                if (!(fabsf(e) < __int_as_float(0x7f800000))) o[k] += e;
              }
            }
          }
          if (whole) {
            uint32_t p[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float e0 = o[2 * k] * inv, e1 = o[2 * k + 1] * inv;
              if (a.gate) {
                const uint4 q4 = gv[k >> 2];
                const uint32_t gw = (k & 3) == 0 ? q4.x : ((k & 3) == 1 ? q4.y : ((k & 3) == 2 ? q4.z : q4.w));
                e0 = __fdividef(e0, 1.f + __expf(-lo16<kHalf>(gw)));
                e1 = __fdividef(e1, 1.f + __expf(-hi16<kHalf>(gw)));
              }
              p[k] = pack16x2<kHalf>(e0, e1);
            }
            uint4* dst = reinterpret_cast<uint4*>(a.out + (s.r.first + t) * a.out_token + h * a.out_head + d);
#pragma unroll
            for (int k = 0; k < 4; ++k) dst[k] = make_uint4(p[4 * k], p[4 * k + 1], p[4 * k + 2], p[4 * k + 3]);
          } else {
            float4* dst = reinterpret_cast<float4*>(a.part_o + slot * kDim + d);
#pragma unroll
            for (int k = 0; k < 8; ++k) dst[k] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          }
        }
        tc_fence_before();
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
