// Experts of each token from the router's logits: scores (softmax over the experts, or sigmoid), the choice
// (logits when there is no bias, whose order is the scores' order; score + bias otherwise, the bias entering
// the choice only), group-limited selection (a group is worth its best choice, or with a bias the sum of its
// best two; the best `top_groups` groups stay), top-k by choice, ties to the lowest index, and the chosen
// scores as weights, renormalised to sum to one and scaled.
//
// One warp a token, everything in registers: lane l holds experts 128 j + 4 l + i, so a token's logits are
// one coalesced 16-byte (8-byte) load a lane for each 128 experts. A choice becomes an unsigned key in its
// order, and a lane keeps its best two with their places; each of the k rounds is one warp-wide maximum of the
// lanes' best keys and one warp-wide minimum of the index among its holders, after which the holder's second moves
// up (17.0 us for 8192 tokens of 256 experts where the holder searched its eight again, 14 so). Lane r then
// computes the r-th expert's weight from its logit, so the k weights cost one pass. Bound: latency of that chain
// (5 us for one token at k = 8, 3 us of them the launch) until enough tokens are there to fill the SMs' warps, then
// the issue of its instructions (66 % of all slots at 8192 tokens); the bytes (4 a logit, 8.9 MB and 1.4 us there)
// are far below it.
//
// Scores are computed with expf and IEEE division, each operation rounded once, so that a sigmoid's score + bias has
// the bits of the same elementary operations anywhere else, and near ties fall the same way; with softmax the sum over the
// experts is added in the warp's own order, and near ties under a bias may fall otherwise. NaN logits
// count as -inf; an expert of -inf is chosen after every other, lowest index first, and weighs 0. A token
// whose chosen scores sum to 0 has weights 0.
#pragma once

#include "ptx.cuh"
#include "rope_append.cuh"

namespace muse {

constexpr int kRouteWarps = 4;
constexpr int kRouteMaxExperts = 1024, kRouteMaxTopK = 32, kRouteMaxGroups = 32;
enum RouteType { kRouteF32 = 0, kRouteBf16 = 1, kRouteF16 = 2 };

struct RouteArgs {
  const void* logits;
  const float* bias;  // null: none
  float* weights;     // [tokens, top_k]
  int32_t* experts;   // [tokens, top_k]
  long long row;      // logits row stride in elements
  int tokens, count, top_k, groups, top_groups, group_size;
  int group_lanes;           // lanes of a group where it is a power of two of lanes, else 0: one group, or scanned in shared memory
  unsigned int group_magic;  // e / group_size = (e * group_magic) >> 20 for e < 1024
  int sigmoid, renormalize, vector, bias_vector;
  float scale;
};

template <int kType>
__device__ __forceinline__ float route_logit(const void* p, long long i) {
  if constexpr (kType == kRouteF32) return static_cast<const float*>(p)[i];
  const uint32_t w = static_cast<const uint16_t*>(p)[i];
  return lo16<kType == kRouteF16>(w);
}

__device__ __forceinline__ float clean_logit(float x) { return x != x ? __int_as_float(0xff800000) : x; }

// Order-preserving unsigned key of a float without NaN; -0 and +0 alike. Every key is above 0, which
// marks a taken or excluded expert.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A group's worth by its best two choices. An infinite best one is the worth itself: with a bias of +inf and the rest of the
// group masked the sum would be NaN, which no rank counts, and a group more than top_groups would stay.
__device__ __forceinline__ float group_worth(float best, float second) {
  return fabsf(best) == __int_as_float(0x7f800000) ? best : best + second;
}

// kJ: 128-expert blocks (count <= 128 * kJ).
template <int kType, int kJ>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const RouteArgs a) {
  constexpr int kN = kJ * 4;
  __shared__ float choices[kRouteWarps][kJ * 128];  // group scan only
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float kNegInf = __int_as_float(0xff800000);
  pdl_wait();
  pdl_launch_dependents();
  const int token = blockIdx.x * kRouteWarps + warp;
  if (token >= a.tokens) return;
  const long long base = token * a.row;
  float bias[kN];
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
    const int e = j * 128 + lane * 4;
    if (a.bias_vector) {
      const float4 b = e < a.count ? __ldg(reinterpret_cast<const float4*>(a.bias + e)) : make_float4(0.f, 0.f, 0.f, 0.f);
      bias[j * 4] = b.x, bias[j * 4 + 1] = b.y, bias[j * 4 + 2] = b.z, bias[j * 4 + 3] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) bias[j * 4 + i] = a.bias && e + i < a.count ? __ldg(a.bias + e + i) : 0.f;
    }
  }

  float x[kN];
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
    const int e = j * 128 + lane * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[j * 4 + i] = kNegInf;
    if (a.vector) {
      if (e < a.count) {
        if constexpr (kType == kRouteF32) {
          const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(a.logits) + base + e);
          x[j * 4] = v.x, x[j * 4 + 1] = v.y, x[j * 4 + 2] = v.z, x[j * 4 + 3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.logits) + base + e);
          constexpr bool h = kType == kRouteF16;
          x[j * 4] = lo16<h>(v.x), x[j * 4 + 1] = hi16<h>(v.x), x[j * 4 + 2] = lo16<h>(v.y), x[j * 4 + 3] = hi16<h>(v.y);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (e + i < a.count) x[j * 4 + i] = route_logit<kType>(a.logits, base + e + i);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[j * 4 + i] = clean_logit(x[j * 4 + i]);
  }

  // Softmax statistics where a probability itself is needed (the choice with a bias, or weights that are
  // not renormalised); otherwise only the maximum of the chosen matters and it is the row's.
  float top = kNegInf, total = 1.f;
  if (!a.sigmoid) {
#pragma unroll
    for (int i = 0; i < kN; ++i) top = fmaxf(top, x[i]);
    top = warp_max(top);
    if (top == kNegInf) top = 0.f;  // nothing but -inf: every score is 0
    if (a.bias || !a.renormalize) {
      total = 0.f;
#pragma unroll
      for (int i = 0; i < kN; ++i) total += expf(x[i] - top);
      total = warp_sum(total);
      if (total == 0.f) total = 1.f;
    }
  }

  uint32_t key[kN];
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = j * 128 + lane * 4 + i, n = j * 4 + i;
      float choice = x[n];
      if (a.bias) {
        const float score = a.sigmoid ? 1.0f / (1.0f + expf(-x[n])) : expf(x[n] - top) / total;
        // An expert of -inf stays behind every other whatever its bias.
        choice = x[n] == kNegInf ? kNegInf : clean_logit(score + bias[n]);
      }
      key[n] = e < a.count ? order_key(choice) : 0u;
    }
  }

  if (a.group_lanes > 0) {
    // A group is 4 x 2^i experts of one 128-block: the lanes that hold it fold their two best by shuffles.
    float worth[kJ];
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      uint32_t b1 = max(key[j * 4], key[j * 4 + 1]), b2 = min(key[j * 4], key[j * 4 + 1]);
      const uint32_t c1 = max(key[j * 4 + 2], key[j * 4 + 3]), c2 = min(key[j * 4 + 2], key[j * 4 + 3]);
      b2 = max(max(b2, c2), min(b1, c1));
      b1 = max(b1, c1);
      for (int o = a.group_lanes >> 1; o; o >>= 1) {
        const uint32_t d1 = __shfl_xor_sync(0xffffffffu, b1, o), d2 = __shfl_xor_sync(0xffffffffu, b2, o);
        b2 = max(max(b2, d2), min(b1, d1));
        b1 = max(b1, d1);
      }
      worth[j] = a.bias ? group_worth(key_value(b1), key_value(b2)) : key_value(b1);
    }
    // Rank of each held group: groups of a block follow one another over its lanes.
    const int in_block = 32 / a.group_lanes, mine = lane / a.group_lanes;
    int rank[kJ] = {};
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      for (int o = 0; o < in_block; ++o) {
        if (j * in_block + o >= a.groups) break;
        const float w = __shfl_sync(0xffffffffu, worth[j], o * a.group_lanes);
#pragma unroll
        for (int k = 0; k < kJ; ++k) rank[k] += (w > worth[k]) || (w == worth[k] && (j < k || (j == k && o < mine)));
      }
    }
#pragma unroll
    for (int n = 0; n < kN; ++n)
      if (rank[n >> 2] >= a.top_groups) key[n] = 0u;
  } else if (a.groups > 1) {
    // Each group's worth: `per` lanes (a power of two) scan one group from shared memory.
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = j * 128 + lane * 4 + i;
        if (e < a.count) choices[warp][e] = key_value(key[j * 4 + i]);
      }
    }
    __syncwarp();
    int per = 1;
    while (per * 2 * a.groups <= 32) per *= 2;
    const int g = lane / per, sub = lane - g * per;
    float b1 = kNegInf, b2 = kNegInf;
    if (g < a.groups) {
      // Lanes start at different members so that their banks differ; the two largest do not depend on order.
      int m = sub + per * (g % ((a.group_size + per - 1) / per));
      if (m >= a.group_size) m = sub;
      for (int n = sub; n < a.group_size; n += per) {
        const float v = choices[warp][g * a.group_size + m];
        b2 = fmaxf(b2, fminf(b1, v));
        b1 = fmaxf(b1, v);
        m += per;
        if (m >= a.group_size) m = sub;
      }
    }
    for (int o = per >> 1; o; o >>= 1) {
      const float c1 = __shfl_xor_sync(0xffffffffu, b1, o), c2 = __shfl_xor_sync(0xffffffffu, b2, o);
      b2 = fmaxf(fmaxf(b2, c2), fminf(b1, c1));
      b1 = fmaxf(b1, c1);
    }
    const float worth = a.bias && a.group_size > 1 ? group_worth(b1, b2) : b1;
    int rank = 0;
    for (int o = 0; o < a.groups; ++o) {
      const float w = __shfl_sync(0xffffffffu, worth, o * per);
      rank += (w > worth) || (w == worth && o < g);
    }
    const uint32_t mine = __ballot_sync(0xffffffffu, g < a.groups && sub == 0 && rank < a.top_groups);
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned int e = j * 128 + lane * 4 + i;
        const int of = static_cast<int>((e * a.group_magic) >> 20);
        if (!((mine >> ((of * per) & 31)) & 1u)) key[j * 4 + i] = 0u;
      }
    }
  }

  // Top-k: this lane's best two keys and their places; on a win the second moves up, and a lane that wins again
  // (under one a token at k = 8) looks through what it has left.
  uint32_t best, next, gone = 0u;
  int at, after;
  auto look = [&]() {
    best = next = 0u;
    at = after = 0;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const uint32_t k = (gone >> n) & 1u ? 0u : key[n];
      const bool first = k > best, second = k > next;
      next = first ? best : (second ? k : next);
      after = first ? at : (second ? n : after);
      best = first ? k : best;
      at = first ? n : at;
    }
  };
  look();
  bool spare = true;  // `next` is this lane's second best
  int chosen = 0;
  for (int r = 0; r < a.top_k; ++r) {
    const uint32_t m = __reduce_max_sync(0xffffffffu, best);
    const int mine = (at >> 2) * 128 + lane * 4 + (at & 3);
    const int e = __reduce_min_sync(0xffffffffu, best == m ? mine : 0x7FFFFFFF);
    if (lane == r) chosen = e;
    if (best == m && mine == e) {
      gone |= 1u << at;
      if (spare) {
        best = next, at = after, spare = false;
      } else {
        look();
        spare = true;
      }
    }
  }

  float w = 0.f;
  if (lane < a.top_k) {
    const float v = clean_logit(route_logit<kType>(a.logits, base + chosen));
    w = a.sigmoid ? 1.0f / (1.0f + expf(-v)) : expf(v - top) / total;
  }
  if (a.renormalize) {
    const float sum = warp_sum(w);
    w = sum > 0.f ? w / sum : (sum != sum ? sum : 0.f);
  }
  if (lane < a.top_k) {
    a.weights[static_cast<long long>(token) * a.top_k + lane] = w * a.scale;
    a.experts[static_cast<long long>(token) * a.top_k + lane] = chosen;
  }
}

}  // namespace muse
