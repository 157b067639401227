// C ABI of the cache in 8 bits and of beam search (declared in include/cats_gemv.h): argument checks, launch shapes and dispatch on dtype.
// No allocation, no synchronisation, everything on the caller's stream.
#include <hip/hip_runtime.h>
#include <math.h>
#include <string.h>

#include "cats_gemv.h"
#include "cats_launch_cache.h"

namespace cats {

template <> hipError_t launch_kv8_append<F16>(int, const KvAppendArgs&, int, hipStream_t);
template <> hipError_t launch_kv8_append<BF16>(int, const KvAppendArgs&, int, hipStream_t);
template <> hipError_t launch_kv8_attn<F16>(int, const KvAttnPlan&, KvAttnArgs, hipStream_t);
template <> hipError_t launch_kv8_attn<BF16>(int, const KvAttnPlan&, KvAttnArgs, hipStream_t);
template <> hipError_t launch_beam_rows<F16>(int, const BeamArgs&, int, hipStream_t);
template <> hipError_t launch_beam_rows<BF16>(int, const BeamArgs&, int, hipStream_t);
template <> hipError_t launch_beam_rows<F32>(int, const BeamArgs&, int, hipStream_t);

namespace {

bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// One workgroup's share of the grid's y and z
constexpr int kMaxGrid = 65535;

int check_cache(int B, int T, int kv_heads, int D, int blocks, int dtype) {
  if (dtype != CATS_F16 && dtype != CATS_BF16) return CATS_ERR_DTYPE;
  if (B < 1 || B > kMaxGrid) return CATS_ERR_BATCH;
  if (T < 1 || kv_heads < 1 || kv_heads > kMaxGrid || blocks < 1 || blocks > CATS_KV8_MAX_BLOCKS) return CATS_ERR_SHAPE;
  if (D != 32 && D != 64 && D != 128 && D != 256) return CATS_ERR_SHAPE;
  if ((long long)T > (long long)blocks * kKvBlock || (long long)B * kv_heads > (1 << 24)) return CATS_ERR_SHAPE;
  return CATS_OK;
}

int fill_cache(KvCache& c, void* k8, void* v8, float* ks, float* vs, void* kt, void* vt, int heads, int blocks) {
  if (!k8 || !v8 || !ks || !vs || !kt || !vt) return CATS_ERR_NULL;
  for (const void* p : {k8, v8, kt, vt})
    if (!aligned(p, 16)) return CATS_ERR_ALIGN;
  if (!aligned(ks, 4) || !aligned(vs, 4)) return CATS_ERR_ALIGN;
  c = {(uint8_t*)k8, (uint8_t*)v8, ks, vs, (uint16_t*)kt, (uint16_t*)vt, heads, blocks};
  return CATS_OK;
}

// Vectors of 16 bytes are read wherever a token's head starts.
int check_strides(const void* p, const int64_t* strides) {
  if (!p || !strides) return CATS_ERR_NULL;
  if (!aligned(p, 16)) return CATS_ERR_ALIGN;
  for (int i = 0; i < 3; i++)
    if (strides[i] < 0 || strides[i] % 8 != 0) return CATS_ERR_ALIGN;
  return CATS_OK;
}

int check_span(const int64_t* start, int start_step, const int64_t* count, int count_step) {
  if (!start) return CATS_ERR_NULL;
  if (!aligned(start, 8) || !aligned(count, 8)) return CATS_ERR_ALIGN;
  return (start_step == 0 || start_step == 1) && (count_step == 0 || count_step == 1) ? CATS_OK : CATS_ERR_SHAPE;
}

// Which kernel, and how many splits of a row's cache.  Up to 16 rows of queries a cached head are one operand of the step's kernel; more of them are
// several of its workgroups, each of which reads the cache, or the prompt's kernel.  That one pays for LDS and for few splits of short caches, so
// the line is drawn by the work, (row, cached head) pairs x 16 rows x tiles of the cache.  Step / prompt in us, heads of 128, bf16:
//   8 pairs, 256 rows, 20 tiles (2560) 15.5 / 17.8     8, 128, 59 (3776) 18.2 / 20.2     8, 192, 59 (5664) 21.4 / 20.8     8, 256, 59 (7552) 20.2 / 21.0
//   128, 32, 10 (2560) 10.4 / 13.6     8, 1024, 5 (2560) 9.4 / 11.4     8, 2048, 10 (10240) 16.2 / 14.1     64, 24, 79 (10112) 27.7 / 22.3
// A second launch costs more than it gives for short caches, up to 16 tiles for the step's kernel (one row, 32 heads, 8 cached, 300 tokens 9.5 with,
// 6.7 without; 16 rows of 32 at 600 tokens 23.2 and 18.8; one row at 600 tokens 9.5 and 9.0), up to 32 for the prompt's (512 tokens of 32 heads
// over 8, 10 tiles, 17.6 with two splits, 14.0 with one; 256 behind 768, 20 tiles, 21.3 and 18.3; 256 behind 1144, 28 tiles, 24.1 and 21.3).  Beyond that
// the step's is to have two workgroups a CU (with four: 64 rows of 8 heads at 1000 tokens 26.3 against 23.1, 16 rows of 32 at 2000 49.2 against
// 45.7, one row of 8 at 3000 tokens the same), the prompt's one, and 16 tiles a split (two a CU and 8 tiles: 512 behind 3584 54.0, 48.1; 128
// behind 3172 32.4, 24.9; 100 behind 7900 39.8, 37.0).
constexpr int kStepRows = 16, kStepWork = 5000, kStepAlone = 16, kPromptAlone = 32;

}  // namespace

KvAttnPlan kv8_attn_plan(int B, int T, int heads, int kv_heads, int blocks, int window) {
  const int cus = current_device_cus(), rows = T * (heads / kv_heads);
  // tiles that a workgroup's queries see at most
  const int tiles = window ? (int)min((long long)blocks, ((long long)window + kKvPromptRows + 2 * kKvBlock) / kKvBlock) : blocks;
  const long long pairs = (long long)B * kv_heads, step_groups = pairs * ((rows + 15) / 16);
  KvAttnPlan plan = {rows > kStepRows && step_groups * tiles > kStepWork, 1, false};
  const int unit = plan.prompt ? kKvPromptUnit : kKvStepWaves;
  const long long groups = plan.prompt ? pairs * ((rows + kKvPromptRows - 1) / kKvPromptRows) : step_groups;
  const long long want = ((plan.prompt ? 1ll : 2ll) * cus + groups - 1) / groups;
  if (tiles > (plan.prompt ? kPromptAlone : kStepAlone)) plan.splits = (int)max(1ll, min(want, (long long)(tiles + unit - 1) / unit));
  return plan;
}

namespace {

// A window that no cache of so many blocks exceeds is none.
int window_of(int window, int blocks) { return window >= (long long)blocks * kKvBlock ? 0 : window; }

bool attn_shape_ok(int T, int heads, int kv_heads) {
  return heads >= kv_heads && heads % kv_heads == 0 && (long long)T * (heads / kv_heads) <= 16ll * kMaxGrid;
}

size_t attn_bytes(const KvAttnPlan& plan, int B, int T, int heads, int kv_heads, int D) {
  return plan.splits == 1 ? 0 : (size_t)B * T * heads * plan.splits * (D + 2) * sizeof(float);
}

}  // namespace
}  // namespace cats

using namespace cats;

extern "C" {

int cats_kv8_append(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, const int64_t* start, int start_step,
                    const int64_t* count, int count_step, void* k8, void* v8, float* k_scale, float* v_scale, void* k_tail, void* v_tail, int B,
                    int T, int kv_heads, int D, int blocks, int dtype, void* stream) {
  if (int st = check_cache(B, T, kv_heads, D, blocks, dtype)) return st;
  if (int st = check_strides(k, k_strides)) return st;
  if (int st = check_strides(v, v_strides)) return st;
  if (int st = check_span(start, start_step, count, count_step)) return st;
  KvAppendArgs a;
  if (int st = fill_cache(a.c, k8, v8, k_scale, v_scale, k_tail, v_tail, kv_heads, blocks)) return st;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.k_row = k_strides[0], a.k_tok = k_strides[1], a.k_head = k_strides[2];
  a.v_row = v_strides[0], a.v_tok = v_strides[1], a.v_head = v_strides[2];
  a.span = {start, count, start_step, count_step, blocks * kKvBlock};
  a.T = T;
  const hipError_t e = dtype == CATS_F16 ? launch_kv8_append<F16>(D, a, B, (hipStream_t)stream) : launch_kv8_append<BF16>(D, a, B, (hipStream_t)stream);
  return e == hipSuccess ? CATS_OK : CATS_ERR_LAUNCH;
}

size_t cats_kv8_attention_scratch_bytes(int B, int T, int heads, int kv_heads, int D, int blocks, int window) {
  if (check_cache(B, T, kv_heads, D, blocks, CATS_F16) || !attn_shape_ok(T, heads, kv_heads) || window < 0) return 0;
  return attn_bytes(kv8_attn_plan(B, T, heads, kv_heads, blocks, window_of(window, blocks)), B, T, heads, kv_heads, D);
}

int cats_kv8_attention_plan(int B, int T, int heads, int kv_heads, int D, int blocks, int window, int* out) {
  if (int st = check_cache(B, T, kv_heads, D, blocks, CATS_F16)) return st;
  if (!attn_shape_ok(T, heads, kv_heads) || window < 0) return CATS_ERR_SHAPE;
  if (!out) return CATS_ERR_NULL;
  const KvAttnPlan plan = kv8_attn_plan(B, T, heads, kv_heads, blocks, window_of(window, blocks));
  out[0] = plan.prompt;
  out[1] = plan.splits;
  return CATS_OK;
}

int cats_kv8_attention(const void* q, const int64_t* q_strides, const int64_t* start, int start_step, const int64_t* count, int count_step,
                       const void* k8, const void* v8, const float* k_scale, const float* v_scale, const void* k_tail, const void* v_tail,
                       float scale, int window, void* out, int B, int T, int heads, int kv_heads, int D, int blocks, int dtype, void* scratch,
                       size_t scratch_bytes, void* stream) {
  if (int st = check_cache(B, T, kv_heads, D, blocks, dtype)) return st;
  if (!attn_shape_ok(T, heads, kv_heads) || window < 0 || !(scale >= 0x1p-64f && scale <= 0x1p64f)) return CATS_ERR_SHAPE;
  if (int st = check_strides(q, q_strides)) return st;
  if (int st = check_span(start, start_step, count, count_step)) return st;
  if (!out) return CATS_ERR_NULL;
  if (!aligned(out, 16)) return CATS_ERR_ALIGN;
  window = window_of(window, blocks);
  KvAttnArgs a;
  if (int st = fill_cache(a.c, (void*)k8, (void*)v8, (float*)k_scale, (float*)v_scale, (void*)k_tail, (void*)v_tail, kv_heads, blocks)) return st;
  const KvAttnPlan plan = kv8_attn_plan(B, T, heads, kv_heads, blocks, window);
  const size_t bytes = attn_bytes(plan, B, T, heads, kv_heads, D);
  if (bytes && (!scratch || !aligned(scratch, 16) || scratch_bytes < bytes)) return CATS_ERR_WORKSPACE;
  a.q = (const uint16_t*)q;
  a.q_row = q_strides[0], a.q_tok = q_strides[1], a.q_head = q_strides[2];
  a.out = (uint16_t*)out;
  a.span = {start, count, start_step, count_step, blocks * kKvBlock};
  a.part = (float*)scratch;
  a.scale = 1.44269504088896341f * scale;
  a.T = T;
  a.group = heads / kv_heads;
  a.window = window;
  a.pairs = B * kv_heads;
  const hipError_t e = dtype == CATS_F16 ? launch_kv8_attn<F16>(D, plan, a, (hipStream_t)stream) : launch_kv8_attn<BF16>(D, plan, a, (hipStream_t)stream);
  return e == hipSuccess ? CATS_OK : CATS_ERR_LAUNCH;
}

}  // extern "C"

namespace cats {
namespace {

// Elements a lane of beam_rows_kernel holds, and the pieces of 4 waves that a row makes.
struct BeamPlan {
  int per_lane, pieces;
};
// Eight elements a lane where that is up to four workgroups a CU and leaves the second launch 256 candidates a row at most, else 32.  Both launches, 8 / 32,
// in us, logits of 16 bits, keep = beams:
//   4 beams, 32000 words 9.2 / 10.2     8 x 4, 32000 9.8 / 10.6     4 x 8, 50257 11.9 / 12.3     8, 64000 10.5 / 11.6
//   8 x 4, 64000 11.0 / 10.8            4 x 16, 32000 17.2 / 15.9   16 x 8, 32000 14.6 / 13.8    8 x 8, 128000 (fp32) 18.7 / 16.2
//   8, 128000 (504 candidates) 11.3 / 11.9     16, 50257 (400) 17.9 / 15.9     16, 128000 (1008) 30.6 / 17.3
BeamPlan beam_plan(int groups, int beams, int V, int keep) {
  BeamPlan p;
  const long long small = ((long long)V + 4 * kWave * 8 - 1) / (4 * kWave * 8);
  p.per_lane = small * groups * beams <= 4ll * current_device_cus() && small * keep <= 256 ? 8 : 32;
  const int per = 4 * kWave * p.per_lane;
  p.pieces = (V - 1) / per + 1;
  return p;
}
bool beam_ok(int groups, int beams, int V, int keep) {
  return groups >= 1 && beams >= 1 && beams <= CATS_MAX_BEAMS && V >= 1 && V <= (1 << 30) && keep >= 1 && keep <= CATS_MAX_BEAMS &&
         (long long)groups * beams <= kMaxGrid && keep <= (long long)beams * V;
}
size_t beam_bytes(const BeamPlan& p, int groups, int beams, int keep) {
  return (size_t)groups * beams * p.pieces * (2 + 2 * (size_t)keep) * 4;
}

}  // namespace
}  // namespace cats

extern "C" {

size_t cats_beam_scratch_bytes(int groups, int beams, int V, int keep) {
  return beam_ok(groups, beams, V, keep) ? beam_bytes(beam_plan(groups, beams, V, keep), groups, beams, keep) : 0;
}

int cats_beam_select(const void* logits, int64_t row_stride, const float* scores, const uint8_t* finished, int64_t eos, float* scores_out,
                     int64_t* parents_out, int64_t* tokens_out, uint8_t* finished_out, int groups, int beams, int V, int keep, int dtype,
                     void* scratch, size_t scratch_bytes, void* stream) {
  if (dtype != CATS_F16 && dtype != CATS_BF16 && dtype != CATS_F32) return CATS_ERR_DTYPE;
  if (!beam_ok(groups, beams, V, keep) || row_stride < 0 || eos >= V || (finished && eos < 0)) return CATS_ERR_SHAPE;
  if (!logits || !scores || !scores_out || !parents_out || !tokens_out || !finished_out) return CATS_ERR_NULL;
  const size_t esz = dtype == CATS_F32 ? 4 : 2;
  if (!aligned(logits, esz) || !aligned(scores, 4) || !aligned(scores_out, 4) || !aligned(parents_out, 8) || !aligned(tokens_out, 8)) return CATS_ERR_ALIGN;
  const BeamPlan plan = beam_plan(groups, beams, V, keep);
  const size_t n = (size_t)groups * beams * plan.pieces;
  if (!scratch || !aligned(scratch, 16) || scratch_bytes < beam_bytes(plan, groups, beams, keep)) return CATS_ERR_WORKSPACE;
  BeamArgs a;
  a.logits = logits;
  a.row_stride = row_stride;
  a.scores = scores;
  a.finished = finished;
  a.eos = eos < 0 ? -1 : eos;
  a.scores_out = scores_out;
  a.parents_out = parents_out;
  a.tokens_out = tokens_out;
  a.finished_out = finished_out;
  a.ml = (float*)scratch;
  a.vals = a.ml + 2 * n;
  a.ids = (int*)(a.vals + n * keep);
  a.beams = beams;
  a.V = V;
  a.keep = keep;
  a.pieces = plan.pieces;
  const int rows = groups * beams;
  hipStream_t s = (hipStream_t)stream;
  hipError_t e = dtype == CATS_F16    ? launch_beam_rows<F16>(plan.per_lane, a, rows, s)
                 : dtype == CATS_BF16 ? launch_beam_rows<BF16>(plan.per_lane, a, rows, s)
                                      : launch_beam_rows<F32>(plan.per_lane, a, rows, s);
  if (e == hipSuccess) e = launch_kernel(beam_join_kernel<kBeamMax>, dim3(groups), dim3(1024), 0, s, a);
  return e == hipSuccess ? CATS_OK : CATS_ERR_LAUNCH;
}

int cats_cache_reorder(const cats_cache_t* caches, int n, const int64_t* parents, const int64_t* lengths, int lengths_step, int groups,
                       int beams, void* stream) {
  if (n < 1 || groups < 1 || groups > kMaxGrid || beams < 1 || beams > CATS_MAX_BEAMS || (lengths_step != 0 && lengths_step != 1)) return CATS_ERR_SHAPE;
  if (!caches || !parents) return CATS_ERR_NULL;
  if (!aligned(parents, 8) || !aligned(lengths, 8)) return CATS_ERR_ALIGN;
  for (int i = 0; i < n; i++) {
    const cats_cache_t& c = caches[i];
    if (c.heads < 1 || c.entries < 1 || c.slots < 0 || c.entry_bytes < 1 || c.entry_bytes > (1ll << 40) / c.entries / c.heads) return CATS_ERR_SHAPE;
    if (!c.data || (c.slots && !lengths)) return CATS_ERR_NULL;
    if (!aligned(c.data, 4) || c.entry_bytes % 4 != 0) return CATS_ERR_ALIGN;
  }
  if (beams == 1) return CATS_OK;  // nothing to move
  ReorderArgs a;
  memset(&a, 0, sizeof(a));
  a.parents = parents;
  a.lengths = lengths;
  a.lengths_step = lengths_step;
  a.beams = beams;
  for (int at = 0; at < n; at += kReorderCaches) {
    const int m = n - at < kReorderCaches ? n - at : kReorderCaches;
    long long steps = 1;  // of 256 units that the largest cache has room for
    for (int i = 0; i < m; i++) {
      const cats_cache_t& c = caches[at + i];
      const int unit = aligned(c.data, 16) && c.entry_bytes % 16 == 0 ? 16 : 4;
      a.c[i] = {(char*)c.data, c.entry_bytes, c.heads, c.entries, c.slots, unit};
      const long long per = (c.entries * c.entry_bytes / unit + 255) / 256 * c.heads;
      steps = steps > per ? steps : per;
    }
    // Workgroups in all: 64 a CU.  More of them, each with less to do one after the other, move faster, and those without a live step cost little (8 searches
    // of 4 beams, caches in 8 bits of 4000 tokens, 406 MB: 8 a CU 110.8 us, 16 90.2, 32 87.6, 64 82.9, 128 80.6; 4 beams of 300 tokens in room for
    // 384, 79 MB: 14.2, 14.6, 15.9, 15.9, 15.9).
    const long long share = (64ll * current_device_cus() + (long long)m * groups - 1) / ((long long)m * groups);
    const dim3 grid((unsigned)(steps < share ? steps : share), m, groups);
    auto kern = beams <= 4 ? cache_reorder_kernel<4> : beams <= 8 ? cache_reorder_kernel<8> : cache_reorder_kernel<16>;
    if (launch_kernel(kern, grid, dim3(256), 0, (hipStream_t)stream, a) != hipSuccess) return CATS_ERR_LAUNCH;
  }
  return CATS_OK;
}

}  // extern "C"
