// C ABI of the cache of pages and of packed attention (declared in include/cats_gemv.h): argument checks, launch shapes and dispatch on dtype.
// No allocation, no synchronisation, everything on the caller's stream.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "cats_gemv.h"
#include "cats_launch_paged.h"

namespace cats {

template <> hipError_t launch_paged_append<F16>(int, bool, const PagedAppendArgs&, hipStream_t);
template <> hipError_t launch_paged_append<BF16>(int, bool, const PagedAppendArgs&, hipStream_t);
template <> hipError_t launch_packed_attn<F16>(int, const PackedPlan*, PackedAttnArgs, hipStream_t);
template <> hipError_t launch_packed_attn<BF16>(int, const PackedPlan*, PackedAttnArgs, hipStream_t);

namespace {

bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

constexpr int kMaxHeads = 65535, kMaxSequences = 1 << 20;

int check_packed(int N, int B, int heads, int kv_heads, int D, int dtype) {
  if (dtype != CATS_F16 && dtype != CATS_BF16) return CATS_ERR_DTYPE;
  if (B < 1 || B > kMaxSequences) return CATS_ERR_BATCH;
  if (N < 1 || N > CATS_PAGED_MAX_TOKENS || kv_heads < 1 || kv_heads > kMaxHeads || heads < 0 || heads > kMaxHeads) return CATS_ERR_SHAPE;
  if (D != 32 && D != 64 && D != 128 && D != 256) return CATS_ERR_SHAPE;
  return (long long)N * heads <= 1 << 30 && (long long)N * kv_heads <= 1 << 30 ? CATS_OK : CATS_ERR_SHAPE;
}

int check_pool(int page, int pages, int width, int kv_heads) {
  if (page < 16 || page > 1024 || (page & (page - 1)) != 0 || pages < 1 || width < 1) return CATS_ERR_SHAPE;
  return (long long)width * page <= 1 << 30 && (long long)pages * kv_heads <= INT_MAX ? CATS_OK : CATS_ERR_SHAPE;
}

// Vectors of 16 bytes are read wherever a token's head starts; a tile of tokens spans less than 2^31 bytes.
int check_strides(const void* p, const int64_t* strides) {
  if (!p || !strides) return CATS_ERR_NULL;
  if (!aligned(p, 16)) return CATS_ERR_ALIGN;
  for (int i = 0; i < 2; i++)
    if (strides[i] < 0 || strides[i] % 8 != 0) return CATS_ERR_ALIGN;
  return strides[0] <= 1 << 23 ? CATS_OK : CATS_ERR_SHAPE;
}

int check_words(const int64_t* w) { return !w ? CATS_ERR_NULL : aligned(w, 8) ? CATS_OK : CATS_ERR_ALIGN; }

int fill_pool(Pool& pool, const void* k_pages, const void* v_pages, const int32_t* table, int64_t table_stride, int kv_heads, int page, int pages, int width) {
  if (!k_pages || !v_pages || !table) return CATS_ERR_NULL;
  if (!aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(table, 4)) return CATS_ERR_ALIGN;
  if (table_stride < 0) return CATS_ERR_SHAPE;
  pool = {(uint16_t*)k_pages, (uint16_t*)v_pages, table, table_stride, kv_heads, __builtin_ctz((unsigned)page), pages, width};
  return CATS_OK;
}

// A window that no sequence exceeds is none.
int window_of(int window) { return window >= 1 << 30 ? 0 : window; }

// Workgroups of a launch, whose threads have to be fewer than 2^32.  Those of a join are four rows each, and where there are many rows there is one only for groups.
bool grid_ok(int N, int B, int heads, int kv_heads, int members = 1) {
  return (long long)N * heads / 16 + (B + 2ll) * kv_heads < 1 << (members > 1 ? 21 : 24);
}

// The rule goes by what the host knows: how many tokens there are, and how long a sequence can be at most.
//   tiles   More than one workgroup's 16 rows a sequence (8 x 5 tokens x 4 heads behind 4000: 39 us with the kernel of few tokens, 34 with that of many; 8 x 8 tokens
//           39 and 34), or a group (8 groups of 8 sequences behind 2048: 34 us and 30).
//   splits  As many as bring workgroups to two a CU, whose loads cover for each other (1 row behind 131072 with two 87 us, 6.2 TB/s), and to one where
//           the matrix cores bound (piece of 512 behind 7680 with two 131 us, with one 117), or where keys are shared: a sequence's own ones are few then (4 x 8 beams
//           on 2000 with two 39 us, with one 37; 4 rows behind 8192 21 and 16).  Sequences of 17 to 64 rows, which memory bounds, go by the same rule and have not
//           been measured with two.  No part is of fewer than 128 or 256 keys, and 1024 are not split: the join, and the
//           writing and reading of parts, would cost what they give (1 row behind 1000 takes 9 us whole).
PackedPlan paged_plan(int N, int B, int heads, int kv_heads, int page, int width, int window, int members) {
  const int cus = current_device_cus(), group = heads / kv_heads;
  const long long room = (long long)width * page, keys = window ? std::min(room, window + 64ll) : room;
  const long long rows = ((long long)N * group + B - 1) / B;  // of a sequence, on average
  auto splits = [&](bool tiles, long long sets, long long set_rows) {
    const int most = tiles ? kTileRows : kStepRows;
    const long long groups = kv_heads * sets * ((set_rows + most - 1) / most), want = ((tiles || members > 1 ? 1ll : 2ll) * cus + groups - 1) / groups;
    return keys <= 1024 ? 1 : (int)std::min(want, keys / (tiles ? kSplitTiles * kTileKeys : 128));
  };
  PackedPlan plan = {};
  plan.tiles = rows > kStepRows;
  plan.splits = splits(plan.tiles, B, rows);
  if (members > 1 && !plan.tiles) {
    plan.group_tiles = rows * members > kStepRows;
    plan.group_splits = splits(plan.group_tiles, B / members, rows * members);
  }
  return plan;
}
// What the splits leave, for the join.
size_t paged_bytes(const PackedPlan& plan, int N, int heads, int D) {
  const int n = plan.splits + plan.group_splits;
  return n == 1 ? 0 : (size_t)N * heads * n * (D + 2) * sizeof(float);
}

bool scale_ok(float scale) { return scale >= 0x1p-64f && scale <= 0x1p64f; }

}  // namespace
}  // namespace cats

using namespace cats;

extern "C" {

int cats_paged_append(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                      const int64_t* offsets, const int64_t* start, const void* cos_table, const void* sin_table, int rot, int positions,
                      int table_dtype, void* q_out, void* k_pages, void* v_pages, const int32_t* table, int64_t table_stride, int N, int B, int heads,
                      int kv_heads, int D, int page, int pages, int width, int dtype, void* stream) {
  if (int st = check_packed(N, B, heads, kv_heads, D, dtype)) return st;
  if (int st = check_pool(page, pages, width, kv_heads)) return st;
  if (rot < 0 || rot > D || rot % 16 != 0 || (rot && positions < 1)) return CATS_ERR_SHAPE;
  if (rot && table_dtype != CATS_F32 && table_dtype != dtype) return CATS_ERR_DTYPE;
  if (!q != !q_out || !q != (heads == 0)) return CATS_ERR_NULL;
  PagedAppendArgs a = {};
  if (q) {
    if (int st = check_strides(q, q_strides)) return st;
    if (!aligned(q_out, 16)) return CATS_ERR_ALIGN;
    a.q_tok = q_strides[0], a.q_head = q_strides[1];
  }
  if (int st = check_strides(k, k_strides)) return st;
  if (int st = check_strides(v, v_strides)) return st;
  if (int st = check_words(offsets)) return st;
  if (int st = check_words(start)) return st;
  if (rot && (!cos_table || !sin_table)) return CATS_ERR_NULL;
  if (rot && (!aligned(cos_table, 16) || !aligned(sin_table, 16))) return CATS_ERR_ALIGN;
  if (int st = fill_pool(a.pool, k_pages, v_pages, table, table_stride, kv_heads, page, pages, width)) return st;
  a.q = (const uint16_t*)q;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.k_tok = k_strides[0], a.k_head = k_strides[1];
  a.v_tok = v_strides[0], a.v_head = v_strides[1];
  a.q_out = (uint16_t*)q_out;
  a.seq = {offsets, B, N};
  a.start = start;
  a.cos = cos_table;
  a.sin = sin_table;
  a.rot = rot;
  a.positions = positions;
  a.heads = heads;
  a.per = N < 16 * current_device_cus() ? 1 : kAppendTokens;
  const bool wide = table_dtype == CATS_F32;
  const hipError_t e = dtype == CATS_F16 ? launch_paged_append<F16>(D, wide, a, (hipStream_t)stream) : launch_paged_append<BF16>(D, wide, a, (hipStream_t)stream);
  return e == hipSuccess ? CATS_OK : CATS_ERR_LAUNCH;
}

size_t cats_paged_attention_scratch_bytes(int N, int B, int heads, int kv_heads, int D, int page, int width, int window, int group) {
  if (check_packed(N, B, heads, kv_heads, D, CATS_F16) || check_pool(page, 1, width, kv_heads) || heads < kv_heads || heads % kv_heads != 0 || window < 0 || group < 1 ||
      B % group != 0)
    return 0;
  return paged_bytes(paged_plan(N, B, heads, kv_heads, page, width, window_of(window), group), N, heads, D);
}

int cats_paged_attention(const void* q, const int64_t* q_strides, const int64_t* offsets, const int64_t* start, const void* k_pages, const void* v_pages,
                         const int32_t* table, int64_t table_stride, float scale, int window, int group, const int64_t* shared, int shared_step,
                         void* out, int N, int B, int heads, int kv_heads, int D, int page, int pages, int width, int dtype, void* scratch,
                         size_t scratch_bytes, void* stream) {
  if (int st = check_packed(N, B, heads, kv_heads, D, dtype)) return st;
  if (int st = check_pool(page, pages, width, kv_heads)) return st;
  if (heads < kv_heads || heads % kv_heads != 0 || window < 0 || !scale_ok(scale) || !grid_ok(N, B, heads, kv_heads, group)) return CATS_ERR_SHAPE;
  if (group < 1 || B % group != 0 || (shared_step != 0 && shared_step != 1)) return CATS_ERR_SHAPE;
  if (int st = check_strides(q, q_strides)) return st;
  if (int st = check_words(offsets)) return st;
  if (int st = check_words(start)) return st;
  if (group > 1)
    if (int st = check_words(shared)) return st;
  if (!out) return CATS_ERR_NULL;
  if (!aligned(out, 16)) return CATS_ERR_ALIGN;
  PackedAttnArgs a = {};
  if (int st = fill_pool(a.pool, k_pages, v_pages, table, table_stride, kv_heads, page, pages, width)) return st;
  a.q = (const uint16_t*)q;
  a.q_tok = q_strides[0], a.q_head = q_strides[1];
  a.out = (uint16_t*)out;
  a.seq = {offsets, B, N};
  a.start = start;
  a.shared = group > 1 ? shared : nullptr;
  a.shared_step = shared_step;
  a.members = group;
  a.scale = 1.44269504088896341f * scale;
  a.kv_heads = kv_heads;
  a.group = heads / kv_heads;
  a.window = window_of(window);
  const PackedPlan plan = paged_plan(N, B, heads, kv_heads, page, width, a.window, group);
  const size_t bytes = paged_bytes(plan, N, heads, D);
  if (bytes && (!scratch || !aligned(scratch, 16) || scratch_bytes < bytes)) return CATS_ERR_WORKSPACE;
  a.part = (float*)scratch;
  const hipError_t e = dtype == CATS_F16 ? launch_packed_attn<F16>(D, &plan, a, (hipStream_t)stream) : launch_packed_attn<BF16>(D, &plan, a, (hipStream_t)stream);
  return e == hipSuccess ? CATS_OK : CATS_ERR_LAUNCH;
}

int cats_prompt_attention(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                          const int64_t* offsets, const int64_t* k_offsets, float scale, int window, void* out, int N, int M, int B, int heads,
                          int kv_heads, int D, int dtype, void* stream) {
  if (int st = check_packed(N, B, heads, kv_heads, D, dtype)) return st;
  if (M < 1 || M > CATS_PAGED_MAX_TOKENS || (!k_offsets && M != N)) return CATS_ERR_SHAPE;
  if (heads < kv_heads || heads % kv_heads != 0 || window < 0 || !scale_ok(scale) || !grid_ok(N, B, heads, kv_heads)) return CATS_ERR_SHAPE;
  if (int st = check_strides(q, q_strides)) return st;
  if (int st = check_strides(k, k_strides)) return st;
  if (int st = check_strides(v, v_strides)) return st;
  if (int st = check_words(offsets)) return st;
  if (!aligned(k_offsets, 8) || !aligned(out, 16)) return CATS_ERR_ALIGN;
  if (!out) return CATS_ERR_NULL;
  PackedAttnArgs a = {};
  a.q = (const uint16_t*)q;
  a.q_tok = q_strides[0], a.q_head = q_strides[1];
  a.out = (uint16_t*)out;
  a.seq = {offsets, B, N};
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.k_tok = k_strides[0], a.k_head = k_strides[1];
  a.v_tok = v_strides[0], a.v_head = v_strides[1];
  a.keys = {k_offsets ? k_offsets : offsets, B, M};
  a.scale = 1.44269504088896341f * scale;
  a.kv_heads = kv_heads;
  a.group = heads / kv_heads;
  a.window = window_of(window);
  const hipError_t e = dtype == CATS_F16 ? launch_packed_attn<F16>(D, nullptr, a, (hipStream_t)stream) : launch_packed_attn<BF16>(D, nullptr, a, (hipStream_t)stream);
  return e == hipSuccess ? CATS_OK : CATS_ERR_LAUNCH;
}

}  // extern "C"
