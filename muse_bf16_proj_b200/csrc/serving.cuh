// Host side of the operators between the projections: argument checks and launches (included by capi.cu).
#pragma once

namespace {

// A kernel launch with programmatic dependent launch.
template <typename K, typename... A>
int launch_pdl(const char* what, K kern, dim3 grid, int threads, int smem, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) return fail(MUSE_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return MUSE_OK;
}

bool aligned_to(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool all_multiples(std::initializer_list<int64_t> v, int64_t n) {
  for (int64_t x : v)
    if (x % n) return false;
  return true;
}

// Checks shared by the two cache operators: heads, dim, type and the cache's geometry.
int check_heads(const char* op, int32_t heads, int32_t kv_heads, int32_t dim, int32_t type) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads || heads > 4096)
    return fail(MUSE_ERR_SHAPE, "%s: heads must be 1..4096 and a multiple of kv_heads (got %d and %d)", op, heads, kv_heads);
  if (dim != 64 && dim != 128) return fail(MUSE_ERR_SHAPE, "%s: dim must be 64 or 128 (got %d)", op, dim);
  if (type != MUSE_BF16 && type != MUSE_F16) return fail(MUSE_ERR_INVALID, "%s: type must be MUSE_BF16 or MUSE_F16 (got %d)", op, type);
  return MUSE_OK;
}

}  // namespace

extern "C" int muse_rope_append(const MuseRopeAppend* p, void* stream) {
  muse::clear_error();
  if (!p) return fail(MUSE_ERR_INVALID, "rope_append: null arguments");
  if (p->tokens < 0) return fail(MUSE_ERR_INVALID, "rope_append: negative tokens");
  if (int rc = check_heads("rope_append", p->heads, p->kv_heads, p->dim, p->type)) return rc;
  if (p->rotary < 2 || p->rotary > p->dim || p->rotary % 2)
    return fail(MUSE_ERR_SHAPE, "rope_append: rotary must be even, 2..dim (got %d)", p->rotary);
  if (p->page_size < 1 || p->pages < 1 || p->positions < 1)
    return fail(MUSE_ERR_INVALID, "rope_append: page_size, pages and positions must be positive");
  if (p->tokens == 0) return MUSE_OK;
  if (!p->q || !p->k || !p->v || !p->q_out || !p->k_pages || !p->v_pages || !p->rope || !p->position || !p->slot)
    return fail(MUSE_ERR_INVALID, "rope_append: null pointer");
  if (!aligned_to(p->q, 2) || !aligned_to(p->k, 2) || !aligned_to(p->v, 2) || !aligned_to(p->q_out, 2) ||
      !aligned_to(p->k_pages, 2) || !aligned_to(p->v_pages, 2) || !aligned_to(p->rope, 4) || !aligned_to(p->position, 4) ||
      !aligned_to(p->slot, 8))
    return fail(MUSE_ERR_ALIGN, "rope_append: pointers must be aligned to their elements");
  DeviceInfo* d;
  if (int rc = device_info(&d)) return rc;
  muse::RopeArgs a;
  a.q = static_cast<const uint16_t*>(p->q);
  a.k = static_cast<const uint16_t*>(p->k);
  a.v = static_cast<const uint16_t*>(p->v);
  a.q_out = static_cast<uint16_t*>(p->q_out);
  a.k_pages = static_cast<uint16_t*>(p->k_pages);
  a.v_pages = static_cast<uint16_t*>(p->v_pages);
  a.rope = p->rope;
  a.position = p->position;
  a.slot = p->slot;
  a.q_token = p->q_token, a.q_head = p->q_head, a.k_token = p->k_token, a.k_head = p->k_head;
  a.v_token = p->v_token, a.v_head = p->v_head, a.out_token = p->out_token, a.out_head = p->out_head;
  a.kp_page = p->k_page, a.kp_head = p->k_page_head, a.kp_slot = p->k_entry;
  a.vp_page = p->v_page, a.vp_head = p->v_page_head, a.vp_slot = p->v_entry;
  a.positions = p->positions;
  a.slots = p->pages * p->page_size;
  a.tokens = p->tokens, a.heads = p->heads, a.kv_heads = p->kv_heads, a.dim = p->dim, a.rotary = p->rotary;
  a.page = p->page_size, a.interleaved = p->interleaved ? 1 : 0;
  const bool wide = p->rotary % 16 == 0 && aligned16(p->q) && aligned16(p->k) && aligned16(p->v) && aligned16(p->q_out) &&
                    aligned16(p->k_pages) && aligned16(p->v_pages) && aligned16(p->rope) &&
                    all_multiples({a.q_token, a.q_head, a.k_token, a.k_head, a.v_token, a.v_head, a.out_token, a.out_head,
                                   a.kp_page, a.kp_head, a.kp_slot, a.vp_page, a.vp_head, a.vp_slot}, 8);
  // Few tokens: more CTAs a token, down to one pass of its threads over the heads; many: one CTA a token.
  const int64_t items = static_cast<int64_t>(a.heads + 2 * a.kv_heads) * (wide ? a.dim / 16 : a.dim / 2);
  const int64_t passes = (items + muse::kRopeThreads - 1) / muse::kRopeThreads;
  const int64_t split = std::min<int64_t>(passes, std::max<int64_t>(1, (8 * d->sms + a.tokens - 1) / a.tokens));
  const dim3 grid(static_cast<unsigned>(a.tokens), static_cast<unsigned>(split), 1);
  const bool half = p->type == MUSE_F16;
  auto kern = wide ? (half ? muse::rope_append_kernel<true> : muse::rope_append_kernel<false>)
                   : (half ? muse::rope_append_any_kernel<true> : muse::rope_append_any_kernel<false>);
  return launch_pdl("rope_append", kern, grid, muse::kRopeThreads, 0, static_cast<cudaStream_t>(stream), a);
}

namespace {

int check_attention(const MuseTreeAttention* p) {
  if (!p) return fail(MUSE_ERR_INVALID, "tree_attention: null arguments");
  if (int rc = check_heads("tree_attention", p->heads, p->kv_heads, p->dim, p->type)) return rc;
  if (p->tokens < 0 || p->requests < 0) return fail(MUSE_ERR_INVALID, "tree_attention: negative tokens or requests");
  if (!std::isfinite(p->scale) || p->scale == 0.f) return fail(MUSE_ERR_INVALID, "tree_attention: scale must be finite and not 0");
  if (p->max_draft < 1 || p->max_draft > 256)
    return fail(MUSE_ERR_SHAPE, "tree_attention: max_draft must be 1..256 (got %d)", p->max_draft);
  return MUSE_OK;
}

// Rows of a unit: those that share a kv head, rounded up to a variant. Tokens-as-M up to 32 rows, rows-as-M past that.
// Measured, tokens-as-M and rows-as-M, at 1 x 700, 1 x 20000, 8 x 3000 and 16 x 20000 (requests x entries), 8 kv heads of
// 128: 20 rows 12.1 and 12.6, 22.1 and 25.2, 20.8 and 21.0, 132 and 132 us; 64 rows (a softmax thread a token and 32
// columns; that variant is gone) 14.9 and 13.4, 27.5 and 26.4, 26.9 and 24.4, 142 and 133 us. 2 kv heads of 64, these four
// and 32 x 4096 and 64 x 1000: 20 rows 10.9 and 9.5, 14.1 and 20.0, 13.1 and 13.0, 27.6 and 37.1, 20.0 and 22.0, 19.2 and
// 18.6 us; 32 rows 11.7 and 9.7, 14.7 and 20.2, 13.9 and 13.3, 28.5 and 37.3, 20.8 and 22.0, 20.0 and 18.7 us. There neither
// side wins throughout: tokens-as-M gives up 2 us at most and gains up to 9, and the lengths that decide are the device's.
int attention_rows(const MuseTreeAttention* p) {
  const int64_t rows = static_cast<int64_t>(p->max_draft) * (p->heads / p->kv_heads);
  return rows <= 16 ? 16 : (rows <= 32 ? 32 : (rows <= 128 ? 128 : 256));
}

int attention_tokens(int dim, int rows) {  // cached tokens a tile (AttnShape::kTok, WideShape::kTok)
  return dim == 64 && rows <= 32 ? 256 : 128;
}

struct AttentionScratch {
  int64_t ml, o, bytes;  // offsets of the partials' statistics and sums, and the whole
};
AttentionScratch attention_scratch(int rows, int dim, int ctas) {
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  AttentionScratch s;
  s.ml = up(static_cast<int64_t>(ctas) * sizeof(muse::AttnCross));
  s.o = s.ml + up(static_cast<int64_t>(ctas) * 2 * rows * 8);
  s.bytes = s.o + static_cast<int64_t>(ctas) * 2 * rows * dim * 4;
  return s;
}

// 5-D map of one cache tensor: 64 dims, 8 entries, the halves of dim, groups of 8 entries in a page, and (page, kv head)
// pairs as one coordinate, the head stride apart. A box is `entries` entries of one page and head, all of dim.
int make_cache_map(CUtensorMap* map, const void* base, const MuseTreeAttention* p, int64_t head, int64_t entry, int64_t combo, int entries) {
  auto fn = encode_fn();
  if (!fn) return fail(MUSE_ERR_CUDA, "cuTensorMapEncodeTiled entry point not found");
  const cuuint64_t pairs = static_cast<cuuint64_t>((p->pages - 1) * combo + p->kv_heads);
  cuuint64_t dims[5] = {64, 8, static_cast<cuuint64_t>(p->dim / 64), static_cast<cuuint64_t>(p->page_size / 8), pairs};
  cuuint64_t strides[4] = {static_cast<cuuint64_t>(entry * 2), 128, static_cast<cuuint64_t>(entry * 16), static_cast<cuuint64_t>(head * 2)};
  cuuint32_t boxes[5] = {64u, 8u, static_cast<cuuint32_t>(p->dim / 64), static_cast<cuuint32_t>(entries / 8), 1u};
  cuuint32_t estr[5] = {1u, 1u, 1u, 1u, 1u};
  const CUresult r = fn(map, p->type == MUSE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
                        const_cast<void*>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MUSE_ERR_CUDA, "cuTensorMapEncodeTiled of the cache failed (%d)", static_cast<int>(r));
  return MUSE_OK;
}

template <bool kHalf, int kDim, int kRows, typename Kern>
int launch_attention_t(Kern kern, int threads, int smem, const CUtensorMap& tmk, const CUtensorMap& tmv, const muse::AttnArgs& a, int ctas,
                       cudaStream_t st) {
  const int group = a.heads / a.kv_heads, rows = std::min(kRows, a.max_draft > kRows / group ? kRows : a.max_draft * group);
  static bool configured[kMaxDevices] = {};
  int dev;
  if (int rc = current_device(&dev)) return rc;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return fail(MUSE_ERR_CUDA, "cudaFuncSetAttribute(tree_attention): %s", cudaGetErrorString(e));
    configured[dev] = true;
  }
  if (int rc = launch_pdl("tree_attention", kern, dim3(static_cast<unsigned>(ctas)), threads, smem, st, tmk, tmv, a)) return rc;
  return launch_pdl("tree_attention join", muse::tree_attn_join_kernel<kHalf, kDim, kRows>,
                    dim3(static_cast<unsigned>(ctas), static_cast<unsigned>((rows - 1) / muse::attn_join_rows(kRows) + 1)), 256, 0, st, a);
}

template <bool kHalf, int kDim, int kRows>
int launch_attention(const CUtensorMap& tmk, const CUtensorMap& tmv, const muse::AttnArgs& a, int ctas, cudaStream_t st) {
  using Sh = muse::AttnShape<kDim, kRows>;
  return launch_attention_t<kHalf, kDim, kRows>(muse::tree_attn_kernel<kHalf, kDim, kRows>, Sh::kThreads, Sh::kSmem, tmk, tmv, a, ctas, st);
}

template <bool kHalf, int kDim, int kRows>
int launch_attention_wide(const CUtensorMap& tmk, const CUtensorMap& tmv, const muse::AttnArgs& a, int ctas, cudaStream_t st) {
  using Sh = muse::WideShape<kDim, kRows>;
  return launch_attention_t<kHalf, kDim, kRows>(muse::tree_attn_wide_kernel<kHalf, kDim, kRows>, Sh::kThreads, Sh::kSmem, tmk, tmv, a, ctas, st);
}

template <bool kHalf, int kDim>
int launch_attention_rows(int rows, const CUtensorMap& tmk, const CUtensorMap& tmv, const muse::AttnArgs& a, int ctas, cudaStream_t st) {
  if (rows == 16) return launch_attention<kHalf, kDim, 16>(tmk, tmv, a, ctas, st);
  if (rows == 32) return launch_attention<kHalf, kDim, 32>(tmk, tmv, a, ctas, st);
  if (rows == 128) return launch_attention_wide<kHalf, kDim, 128>(tmk, tmv, a, ctas, st);
  return launch_attention_wide<kHalf, kDim, 256>(tmk, tmv, a, ctas, st);
}

}  // namespace

extern "C" int muse_tree_attention_scratch_bytes(const MuseTreeAttention* p, int64_t* bytes) {
  muse::clear_error();
  if (!bytes) return fail(MUSE_ERR_INVALID, "tree_attention_scratch_bytes: null output");
  if (int rc = check_attention(p)) return rc;
  DeviceInfo* d;
  if (int rc = device_info(&d)) return rc;
  *bytes = attention_scratch(attention_rows(p), p->dim, d->sms).bytes;
  return MUSE_OK;
}

extern "C" int muse_tree_attention(const MuseTreeAttention* p, void* stream) {
  muse::clear_error();
  if (int rc = check_attention(p)) return rc;
  if (p->page_size < 8 || p->page_size > 1024 || (p->page_size & (p->page_size - 1)))
    return fail(MUSE_ERR_SHAPE, "tree_attention: page_size must be a power of two, 8..1024 (got %d)", p->page_size);
  if (p->mask && static_cast<int64_t>(p->mask_words) * 32 < p->max_draft)
    return fail(MUSE_ERR_SHAPE, "tree_attention: %d mask words do not cover max_draft %d", p->mask_words, p->max_draft);
  if (p->pages < 1 || p->table_cols < 1) return fail(MUSE_ERR_INVALID, "tree_attention: pages and table_cols must be positive");
  if (static_cast<int64_t>(p->table_cols) * p->page_size > (int64_t(1) << 30) || p->pages > (int64_t(1) << 31) - 1)
    return fail(MUSE_ERR_SHAPE, "tree_attention: a request's pages must hold at most 2^30 entries, the cache fewer than 2^31 pages");
  const int64_t tiles = static_cast<int64_t>(p->table_cols) * p->page_size / 128 + 1 + muse::kAttnEnds;
  const int64_t units = static_cast<int64_t>(p->kv_heads) * (static_cast<int64_t>(p->max_draft) * (p->heads / p->kv_heads) / 128 + 1);
  if (p->requests > 0 && tiles * units > ((int64_t(1) << 31) - 1) / p->requests)
    return fail(MUSE_ERR_SHAPE, "tree_attention: requests x page table x kv_heads x max_draft is too large (more than 2^31 tiles)");
  if (p->tokens == 0 || p->requests == 0) return MUSE_OK;
  if (!p->q || !p->out || !p->k_pages || !p->v_pages || !p->table || !p->context || !p->starts || !p->scratch)
    return fail(MUSE_ERR_INVALID, "tree_attention: null pointer");
  if (!aligned16(p->q) || !aligned16(p->out) || !aligned16(p->k_pages) || !aligned16(p->v_pages) || !aligned16(p->gate) ||
      !all_multiples({p->q_token, p->q_head, p->out_token, p->out_head, p->k_page, p->k_page_head, p->k_entry, p->v_page,
                      p->v_page_head, p->v_entry}, 8) ||
      (p->gate && !all_multiples({p->gate_token, p->gate_head}, 8)))
    return fail(MUSE_ERR_ALIGN, "tree_attention: q, gate, out and the cache must be 16-byte aligned, rows included");
  if (!aligned_to(p->table, 4) || !aligned_to(p->context, 4) || !aligned_to(p->starts, 4) || !aligned_to(p->mask, 4))
    return fail(MUSE_ERR_ALIGN, "tree_attention: table, context, starts and mask must be 4-byte aligned");
  for (int64_t x : {p->k_page, p->k_page_head, p->k_entry, p->v_page, p->v_page_head, p->v_entry})
    if (x < 1 || x >= (int64_t(1) << 35)) return fail(MUSE_ERR_SHAPE, "tree_attention: cache strides must be 1..2^35 (got %lld)", (long long)x);
  // One kv head: the head stride is free, a page's takes its place.
  const int64_t k_head = p->kv_heads == 1 ? p->k_page : p->k_page_head, v_head = p->kv_heads == 1 ? p->v_page : p->v_page_head;
  const int64_t k_combo = p->pages == 1 ? p->kv_heads : p->k_page / k_head, v_combo = p->pages == 1 ? p->kv_heads : p->v_page / v_head;
  if (p->pages > 1 && (p->k_page % k_head || p->v_page % v_head || k_combo < 1 || v_combo < 1))
    return fail(MUSE_ERR_SHAPE, "tree_attention: the cache's page stride must be a multiple of its head stride");
  if (p->pages > ((int64_t(1) << 31) - 1) / std::max(k_combo, v_combo) - 1)
    return fail(MUSE_ERR_SHAPE, "tree_attention: the cache has too many pages (2^31 head strides)");
  DeviceInfo* d;
  if (int rc = device_info(&d)) return rc;
  const int tile = attention_rows(p);
  const AttentionScratch sc = attention_scratch(tile, p->dim, d->sms);
  if (p->scratch_bytes < sc.bytes)
    return fail(MUSE_ERR_CAPACITY, "tree_attention: needs %lld bytes of scratch (got %lld)", (long long)sc.bytes, (long long)p->scratch_bytes);
  if (!aligned_to(p->scratch, 256)) return fail(MUSE_ERR_ALIGN, "tree_attention: scratch must be 256-byte aligned");
  const int box = std::min(p->page_size, attention_tokens(p->dim, tile));
  CUtensorMap tmk, tmv;
  if (int rc = make_cache_map(&tmk, p->k_pages, p, k_head, p->k_entry, k_combo, box)) return rc;
  if (int rc = make_cache_map(&tmv, p->v_pages, p, v_head, p->v_entry, v_combo, box)) return rc;
  muse::AttnArgs a;
  a.q = static_cast<const uint16_t*>(p->q);
  a.gate = static_cast<const uint16_t*>(p->gate);
  a.v_pages = static_cast<const uint16_t*>(p->v_pages);
  a.out = static_cast<uint16_t*>(p->out);
  a.table = p->table, a.context = p->context, a.starts = p->starts, a.mask = p->mask;
  a.q_token = p->q_token, a.q_head = p->q_head, a.gate_token = p->gate_token, a.gate_head = p->gate_head;
  a.out_token = p->out_token, a.out_head = p->out_head;
  a.v_page = p->v_page, a.v_head = p->v_page_head, a.v_slot = p->v_entry;
  a.table_row = p->table_row, a.mask_row = p->mask_row, a.pages = p->pages;
  a.requests = p->requests, a.tokens = p->tokens, a.max_draft = p->max_draft, a.table_cols = p->table_cols;
  a.heads = p->heads, a.kv_heads = p->kv_heads, a.page = p->page_size;
  a.scale_log2 = std::fabs(p->scale) * 1.4426950408889634f;
  a.q_flip = p->scale < 0.f ? 0x80008000u : 0u;
  a.k_combo = static_cast<int>(k_combo), a.v_combo = static_cast<int>(v_combo);
  const unsigned int group = static_cast<unsigned int>(p->heads / p->kv_heads);
  a.group_magic = group == 1 ? 0u : static_cast<unsigned int>(((uint64_t(1) << 32) + group - 1) / group);
  uint8_t* base = static_cast<uint8_t*>(p->scratch);
  a.cross = reinterpret_cast<muse::AttnCross*>(base);
  a.part_ml = reinterpret_cast<float2*>(base + sc.ml);
  a.part_o = reinterpret_cast<float*>(base + sc.o);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->type == MUSE_F16)
    return p->dim == 64 ? launch_attention_rows<true, 64>(tile, tmk, tmv, a, d->sms, st)
                        : launch_attention_rows<true, 128>(tile, tmk, tmv, a, d->sms, st);
  return p->dim == 64 ? launch_attention_rows<false, 64>(tile, tmk, tmv, a, d->sms, st)
                      : launch_attention_rows<false, 128>(tile, tmk, tmv, a, d->sms, st);
}

namespace {

template <int kType>
int launch_route(const muse::RouteArgs& a, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>((a.tokens + muse::kRouteWarps - 1) / muse::kRouteWarps));
  const int threads = muse::kRouteWarps * 32;
  if (a.count <= 128) return launch_pdl("route", muse::route_kernel<kType, 1>, grid, threads, 0, st, a);
  if (a.count <= 256) return launch_pdl("route", muse::route_kernel<kType, 2>, grid, threads, 0, st, a);
  if (a.count <= 512) return launch_pdl("route", muse::route_kernel<kType, 4>, grid, threads, 0, st, a);
  return launch_pdl("route", muse::route_kernel<kType, 8>, grid, threads, 0, st, a);
}

}  // namespace

extern "C" int muse_route(const MuseRoute* p, void* stream) {
  muse::clear_error();
  if (!p) return fail(MUSE_ERR_INVALID, "route: null arguments");
  if (p->tokens < 0) return fail(MUSE_ERR_INVALID, "route: negative tokens");
  if (p->experts < 1 || p->experts > muse::kRouteMaxExperts)
    return fail(MUSE_ERR_SHAPE, "route: experts must be 1..%d (got %d)", muse::kRouteMaxExperts, p->experts);
  if (p->groups < 1 || p->groups > muse::kRouteMaxGroups || p->experts % p->groups || p->top_groups < 1 || p->top_groups > p->groups)
    return fail(MUSE_ERR_SHAPE, "route: groups must divide experts, 1..%d, and 1 <= top_groups <= groups (got %d, %d)",
                muse::kRouteMaxGroups, p->groups, p->top_groups);
  if (p->top_k < 1 || p->top_k > muse::kRouteMaxTopK || p->top_k > p->experts / p->groups * p->top_groups)
    return fail(MUSE_ERR_SHAPE, "route: top_k must be 1..%d and at most the %d experts of top_groups groups (got %d)",
                muse::kRouteMaxTopK, p->experts / p->groups * p->top_groups, p->top_k);
  if (p->type != MUSE_BF16 && p->type != MUSE_F16 && p->type != MUSE_F32)
    return fail(MUSE_ERR_INVALID, "route: type must be MUSE_BF16, MUSE_F16 or MUSE_F32 (got %d)", p->type);
  if (p->tokens == 0) return MUSE_OK;
  if (!p->logits || !p->weights || !p->expert_ids) return fail(MUSE_ERR_INVALID, "route: null pointer");
  const int size = p->type == MUSE_F32 ? 4 : 2;
  if (!aligned_to(p->logits, size) || !aligned_to(p->bias, 4) || !aligned_to(p->weights, 4) || !aligned_to(p->expert_ids, 4))
    return fail(MUSE_ERR_ALIGN, "route: pointers must be aligned to their elements");
  DeviceInfo* d;
  if (int rc = device_info(&d)) return rc;
  muse::RouteArgs a;
  a.logits = p->logits;
  a.bias = p->bias;
  a.weights = p->weights;
  a.experts = p->expert_ids;
  a.row = p->row;
  a.tokens = p->tokens, a.count = p->experts, a.top_k = p->top_k, a.groups = p->groups, a.top_groups = p->top_groups;
  a.group_size = p->experts / p->groups;
  a.group_magic = (1u << 20) / static_cast<unsigned>(a.group_size) + 1u;
  const int lanes = a.group_size / 4;
  a.group_lanes = p->groups > 1 && a.group_size % 4 == 0 && lanes <= 32 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
  a.sigmoid = p->sigmoid ? 1 : 0, a.renormalize = p->renormalize ? 1 : 0;
  // Four logits a load where every lane's four are in one row and aligned together.
  a.vector = p->experts % 4 == 0 && p->row % 4 == 0 && aligned_to(p->logits, static_cast<unsigned>(4 * size));
  a.bias_vector = p->bias && p->experts % 4 == 0 && aligned16(p->bias);
  a.scale = p->scale;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->type == MUSE_F32) return launch_route<muse::kRouteF32>(a, st);
  if (p->type == MUSE_BF16) return launch_route<muse::kRouteBf16>(a, st);
  return launch_route<muse::kRouteF16>(a, st);
}
