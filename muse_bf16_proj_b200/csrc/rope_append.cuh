// Rotary positions on q and k, and k and v appended to a paged cache, in one pass over the projection's
// rows: for token t with table row (c, s) of its position and each rotated pair (a, b) of a q or k head
//   (a, b) -> (a c - b s, b c + a s)
// in FP32, rounded once to the 16-bit type (v and the entries past `rotary` are copied). A pair is
// (2i, 2i + 1) (interleaved) or (i, i + rotary / 2). The table is FP32 and built in 64 bits by the
// caller: an FP32 position * frequency is off by 0.008 rad at position 131072.
//
// Bound: bytes (q, k, v in; q and the cache rows out), 16-byte accesses throughout. A thread owns one
// 16-element piece of a head (eight pairs) and walks heads with it, so its table entries are loaded
// once a token and stay in registers; a CTA covers 8 (dim 128) or 16 (dim 64) heads at a time.
// Rotary sizes that are no multiple of 16, strides or pointers that rule out 16-byte accesses take the scalar kernel
// for the whole row, one pair a thread. Measured, device time: 4096 tokens of 64 + 2 x 8 heads of 128 (170 MB) in 29.0 us =
// 5.85 TB/s, 0.89 of a plain copy's rate, at rotary 128 and 64 and for both kinds of pairs; in 111 us by the scalar kernel
// (rotary 36 and 20); 201 tokens in 3.0 us and one in 2.3 us, which is the launch.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace muse {

constexpr unsigned int kErrRopePosition = 0xA01, kErrRopeSlot = 0xA02;
constexpr int kRopeThreads = 64;  // 4096 tokens x 80 heads of 128: 29.4 us, 31.2 with 128 threads, 36.0 with 256

struct RopeArgs {
  const uint16_t *q, *k, *v;
  uint16_t *q_out, *k_pages, *v_pages;
  const float* rope;         // [positions, rotary]: rotary / 2 cosines, then as many sines
  const int32_t* position;   // [tokens]
  const int64_t* slot;       // [tokens]: page * page size + entry; negative: not appended
  long long q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head;
  long long kp_page, kp_head, kp_slot, vp_page, vp_head, vp_slot;
  long long positions, slots;  // bounds
  int tokens, heads, kv_heads, dim, rotary, page, interleaved;
};

template <bool kHalf>
__device__ __forceinline__ float lo16(uint32_t w) {
  if constexpr (kHalf) return __half2float(__ushort_as_half(static_cast<unsigned short>(w & 0xFFFFu)));
  return bf16lo(w);
}
template <bool kHalf>
__device__ __forceinline__ float hi16(uint32_t w) {
  if constexpr (kHalf) return __half2float(__ushort_as_half(static_cast<unsigned short>(w >> 16)));
  return bf16hi(w);
}
// Two FP32 values to two 16-bit ones (lo in the low half), round to nearest even.
template <bool kHalf>
__device__ __forceinline__ uint32_t pack16x2(float lo, float hi) {
  if constexpr (kHalf) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  return pack_bf16x2(lo, hi);
}

// Where a token's row of one head goes and comes from: heads [0, heads) are q, then k, then v.
struct RopeRow {
  const uint16_t* src;
  uint16_t* dst;  // null: nothing is stored (k or v of a row without a slot)
  bool turn;
};

__device__ __forceinline__ RopeRow rope_row(const RopeArgs& a, int token, int h, long long page, long long entry) {
  RopeRow r;
  if (h < a.heads) {
    r.src = a.q + token * a.q_token + h * a.q_head;
    r.dst = a.q_out + token * a.out_token + h * a.out_head;
    r.turn = true;
  } else if (h < a.heads + a.kv_heads) {
    const int i = h - a.heads;
    r.src = a.k + token * a.k_token + i * a.k_head;
    r.dst = page < 0 ? nullptr : a.k_pages + page * a.kp_page + i * a.kp_head + entry * a.kp_slot;
    r.turn = true;
  } else {
    const int i = h - a.heads - a.kv_heads;
    r.src = a.v + token * a.v_token + i * a.v_head;
    r.dst = page < 0 ? nullptr : a.v_pages + page * a.vp_page + i * a.vp_head + entry * a.vp_slot;
    r.turn = false;
  }
  return r;
}

// The token's slot as (page, entry); page -1 where nothing is appended. A position or slot outside its
// range is recorded in the device error word (by one thread a token), its token is not appended, and a
// bad position turns by nothing (false).
__device__ __forceinline__ bool rope_token(const RopeArgs& a, int token, bool report, long long& pos, long long& page,
                                           long long& entry) {
  pos = a.position[token];
  const long long slot = a.slot[token];
  page = -1;
  entry = 0;
  bool ok = true;
  if (pos < 0 || pos >= a.positions) {
    if (report) report_error(kErrRopePosition);
    ok = false;
  }
  if (slot >= a.slots) {
    if (report) report_error(kErrRopeSlot);
  } else if (slot >= 0 && ok) {
    page = slot / a.page;
    entry = slot - page * a.page;
  }
  return ok;
}

template <bool kHalf>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const RopeArgs a) {
  pdl_wait();  // q, k and v are usually the previous grid's output
  pdl_launch_dependents();
  const int token = blockIdx.x;
  const int pieces = a.dim / 16, per = kRopeThreads / pieces;  // heads a pass of the CTA
  const int piece = threadIdx.x % pieces;
  long long pos, page, entry;
  const bool ok = rope_token(a, token, threadIdx.x == 0 && blockIdx.y == 0, pos, page, entry);
  const int half = a.rotary / 2;
  // This piece's two 16-byte parts, and whether it is turned: eight pairs of the rotary part, else a copy.
  const bool turned = ok && piece * 16 < a.rotary;
  const bool split = !a.interleaved && piece * 16 < a.rotary;
  const int o0 = split ? piece * 8 : piece * 16;
  const int o1 = split ? half + piece * 8 : o0 + 8;
  float c[8], s[8];
  if (turned) {
    const float* row = a.rope + pos * a.rotary + piece * 8;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(row + i);
      const float4 y = *reinterpret_cast<const float4*>(row + half + i);
      c[i] = x.x, c[i + 1] = x.y, c[i + 2] = x.z, c[i + 3] = x.w;
      s[i] = y.x, s[i + 1] = y.y, s[i + 2] = y.z, s[i + 3] = y.w;
    }
  }
  const int all = a.heads + 2 * a.kv_heads;
  for (int h0 = blockIdx.y * per + threadIdx.x / pieces; h0 < all; h0 += per * gridDim.y * 2) {
    // Two heads' loads in flight together.
    RopeRow r[2];
    uint4 x[2], y[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int h = h0 + u * per * gridDim.y;
      r[u].dst = nullptr;
      if (h < all) {
        r[u] = rope_row(a, token, h, page, entry);
        if (r[u].dst) {
          x[u] = *reinterpret_cast<const uint4*>(r[u].src + o0);
          y[u] = *reinterpret_cast<const uint4*>(r[u].src + o1);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (!r[u].dst) continue;
      if (r[u].turn && turned) {
        uint32_t xs[4] = {x[u].x, x[u].y, x[u].z, x[u].w}, ys[4] = {y[u].x, y[u].y, y[u].z, y[u].w};
        if (a.interleaved) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = lo16<kHalf>(xs[i]), q = hi16<kHalf>(xs[i]);
            xs[i] = pack16x2<kHalf>(p * c[i] - q * s[i], q * c[i] + p * s[i]);
            const float v = lo16<kHalf>(ys[i]), w = hi16<kHalf>(ys[i]);
            ys[i] = pack16x2<kHalf>(v * c[4 + i] - w * s[4 + i], w * c[4 + i] + v * s[4 + i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = lo16<kHalf>(xs[i]), q = hi16<kHalf>(xs[i]);
            const float v = lo16<kHalf>(ys[i]), w = hi16<kHalf>(ys[i]);
            xs[i] = pack16x2<kHalf>(p * c[2 * i] - v * s[2 * i], q * c[2 * i + 1] - w * s[2 * i + 1]);
            ys[i] = pack16x2<kHalf>(v * c[2 * i] + p * s[2 * i], w * c[2 * i + 1] + q * s[2 * i + 1]);
          }
        }
        x[u] = make_uint4(xs[0], xs[1], xs[2], xs[3]);
        y[u] = make_uint4(ys[0], ys[1], ys[2], ys[3]);
      }
      *reinterpret_cast<uint4*>(r[u].dst + o0) = x[u];
      *reinterpret_cast<uint4*>(r[u].dst + o1) = y[u];
    }
  }
}

// Any rotary size, stride and alignment: one pair (or two copied entries) a thread.
template <bool kHalf>
__global__ void __launch_bounds__(kRopeThreads) rope_append_any_kernel(const RopeArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int token = blockIdx.x;
  long long pos, page, entry;
  const bool ok = rope_token(a, token, threadIdx.x == 0 && blockIdx.y == 0, pos, page, entry);
  const int half = a.rotary / 2, pairs = a.dim / 2, all = (a.heads + 2 * a.kv_heads) * pairs;
  for (int i = blockIdx.y * kRopeThreads + threadIdx.x; i < all; i += kRopeThreads * gridDim.y) {
    const int h = i / pairs, p = i - h * pairs;
    const RopeRow r = rope_row(a, token, h, page, entry);
    if (!r.dst) continue;
    const bool rotary = p < half;
    const int o0 = rotary && !a.interleaved ? p : 2 * p;
    const int o1 = rotary && !a.interleaved ? half + p : 2 * p + 1;
    uint16_t x = r.src[o0], y = r.src[o1];
    if (r.turn && rotary && ok) {
      const float c = a.rope[pos * a.rotary + p], s = a.rope[pos * a.rotary + half + p];
      const float v = lo16<kHalf>(x), w = lo16<kHalf>(y);
      const uint32_t both = pack16x2<kHalf>(v * c - w * s, w * c + v * s);
      x = static_cast<uint16_t>(both & 0xFFFFu);
      y = static_cast<uint16_t>(both >> 16);
    }
    r.dst[o0] = x;
    r.dst[o1] = y;
  }
}

}  // namespace muse
