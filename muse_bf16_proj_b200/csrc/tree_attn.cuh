// Attention of drafted tokens over a paged cache. Row (token t of request b, query head h) sees the request's
// cached tokens l < context[b], and drafted token j of its request (cached at context[b] + j) where bit j of
// its mask row is set (without a mask: j up to itself). With s_l = scale * q . K_l over what it sees,
//   out = sum_l exp(s_l) V_l / sum_l exp(s_l)   (0 where it sees nothing), times sigmoid(gate) if given.
// The softmax statistics and sums are FP32.
#pragma once

#include "ptx.cuh"
#include "rope_append.cuh"

namespace muse {

constexpr unsigned int kErrAttnDraft = 0xB01, kErrAttnTable = 0xB02, kErrAttnPage = 0xB03;

struct AttnArgs {
  const uint16_t *q, *gate, *k_pages, *v_pages;
  uint16_t* out;
  const int32_t *table, *context, *starts;
  const uint32_t* mask;
  long long q_token, q_head, gate_token, gate_head, out_token, out_head;
  long long k_page, k_head, k_slot, v_page, v_head, v_slot;
  long long table_row, mask_row;
  long long pages;
  int requests, tokens, max_draft, table_cols, heads, kv_heads, page;
  float scale_log2;  // scale * log2(e)
};

// Simple form: one warp a row, a lane owning dim / 32 entries.
template <bool kHalf, int kDim>
__global__ void __launch_bounds__(128) tree_attn_simple_kernel(const AttnArgs a) {
  constexpr int kN = kDim / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * 4 + warp;
  if (row >= static_cast<long long>(a.tokens) * a.heads) return;
  const int t = static_cast<int>(row / a.heads), h = static_cast<int>(row % a.heads);
  int lo = 0, hi = a.requests;  // the request with starts[lo] <= t < starts[lo + 1]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.starts[mid] <= t) lo = mid; else hi = mid;
  }
  while (lo + 1 < a.requests && a.starts[lo + 1] <= t) ++lo;
  const int inner = t - a.starts[lo], drafted = a.starts[lo + 1] - a.starts[lo];
  if (inner < 0 || inner >= a.max_draft || drafted > a.max_draft) {
    if (lane == 0) report_error(kErrAttnDraft);
    return;
  }
  const int ctx = max(a.context[lo], 0);
  const int g = h / (a.heads / a.kv_heads);
  float q[kN], acc[kN], m = __int_as_float(0xff800000), l = 0.f;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    q[i] = lo16<kHalf>(a.q[t * a.q_token + h * a.q_head + lane * kN + i]) * a.scale_log2;
    acc[i] = 0.f;
  }
  for (int pos = 0; pos < ctx + drafted; ++pos) {
    if (pos >= ctx) {
      const int j = pos - ctx;
      const bool seen = a.mask ? (a.mask[t * a.mask_row + (j >> 5)] >> (j & 31)) & 1u : j <= inner;
      if (!seen) continue;
    }
    const int col = pos / a.page;
    if (col >= a.table_cols) {
      if (lane == 0) report_error(kErrAttnTable);
      break;
    }
    const long long page = a.table[lo * a.table_row + col];
    if (page < 0 || page >= a.pages) {
      if (lane == 0) report_error(kErrAttnPage);
      continue;
    }
    const uint16_t* k = a.k_pages + page * a.k_page + g * a.k_head + (pos % a.page) * a.k_slot + lane * kN;
    const uint16_t* v = a.v_pages + page * a.v_page + g * a.v_head + (pos % a.page) * a.v_slot + lane * kN;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kN; ++i) s += q[i] * lo16<kHalf>(k[i]);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float top = fmaxf(m, s);
    const float keep = m == top ? 1.f : exp2f(m - top), p = exp2f(s - top);
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < kN; ++i) acc[i] = acc[i] * keep + p * lo16<kHalf>(v[i]);
    m = top;
  }
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    float o = l == 0.f ? 0.f : acc[i] / l;
    if (a.gate) o /= 1.f + expf(-lo16<kHalf>(a.gate[t * a.gate_token + h * a.gate_head + lane * kN + i]));
    a.out[t * a.out_token + h * a.out_head + lane * kN + i] = static_cast<uint16_t>(pack16x2<kHalf>(o, o) & 0xFFFFu);
  }
}

}  // namespace muse
