// A cache of keys and values in 8 bits, and attention over it (16-bit models).
//
// Format.  A row (sequence) of the cache has `blocks` blocks of 64 tokens.  A block that is complete is held as e4m3 numbers with one
// power of two as scale for a head's keys and one for its values: the smallest that brings the block's largest finite magnitude within 448.
// e4m3 is a floating format, so a power of two costs no precision against a free scale, and scaling is exact: a value is rounded once
// (by at most 2^-4 of itself) and what the products use is what is stored.  Values that are not finite are stored as NaN.
//   k8 (B, kv_heads, blocks, 64, D)   v8 (B, kv_heads, blocks, D, 64)   scales (B, kv_heads, blocks) float
// The block that holds a row's last token, complete or not, is always read as it was given, from
//   k_tail (B, kv_heads, 64, D)       v_tail (B, kv_heads, D, 64)        slot = position % 64
// so every token is rounded once, from what was given, whatever pieces the tokens come in.
// Values lie with the tokens of one element side by side: that is the order in which the matrix cores want them, both as operand of
// v_mfma_f32_16x16x32 and of 32x32x16, where 64 tokens of one element are 16 bytes of each of four lanes.
#pragma once
#include <float.h>
#include <limits.h>

#include <type_traits>

#include "cats_down_mma.h"
#include "cats_rows_mma.h"

namespace cats {

constexpr int kKvBlock = 64;

struct KvCache {
  uint8_t* k8;
  uint8_t* v8;
  float* ks;
  float* vs;
  uint16_t* kt;
  uint16_t* vt;
  int heads;   // of the cache
  int blocks;  // of a row; at most 2^24, so that positions are ints
};

// Where a row's new tokens lie: positions start .. start + n - 1, as many of the call's T tokens as its count says.
struct KvSpan {
  const int64_t* start;
  const int64_t* count;  // nullptr: all T
  int start_step;        // 0: one start for all rows
  int count_step;
  int limit;             // positions lie below it
};
__device__ __forceinline__ bool kv_span(const KvSpan& s, int b, int T, int& start, int& n) {
  const long long a = s.start[(size_t)b * s.start_step], c = s.count ? s.count[(size_t)b * s.count_step] : T;
  n = (int)(c < 0 ? 0 : c > T ? T : c);
  const bool ok = a >= 0 && a <= (long long)s.limit - n;
  start = ok ? (int)a : 0;
  return ok;
}

// What differs between the two types.  HEAD: attention's weights are held as 2^HEAD times themselves: in fp16 the normal numbers reach down to 2^-29
// of the largest weight (2^-21 with SLACK), in bf16 2^32 values of the largest size add up within 32 bits.  SLACK: by how many powers of two weights may pass
// 2^HEAD's part before kv8_attn_prompt_kernel scales its sums again; they start that much lower (8 against 0: a prompt of 2048 tokens 58.8 / 61.3 us, heads of
// 256 behind 3300 tokens 70.9 / 73.7).
// VMAX: e4m3 values become operands as what they stand for, so sums have one unit, blocks and the tail alike, and weights are those of the softmax.  The
// conversion multiplies by a power of two.  In fp16 that is exact: values are multiples of 2^-24, so are those that e4m3 keeps four bits of, and the
// scale is 2^-32 or more; only 256 times a scale of 2^8 is too large.  In bf16 it is exact up to 2^73.  What a scale has beyond VMAX goes into the weights of its block (kv_over).
template <class DT> struct Kv;
template <> struct Kv<F16> {
  static constexpr uint32_t kExp = 0x7c00u, kOne = 0x3c00u;
  static constexpr float HEAD = 15.f, SLACK = 8.f, VMAX = 0x1p7f;
  template <bool HI>
  static __device__ __forceinline__ uint32_t cvt(uint32_t w, float scale) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI)); }
};
template <> struct Kv<BF16> {
  static constexpr uint32_t kExp = 0x7f80u, kOne = 0x3f80u;
  static constexpr float HEAD = -32.f, SLACK = 8.f, VMAX = 0x1p64f;
  template <bool HI>
  static __device__ __forceinline__ uint32_t cvt(uint32_t w, float scale) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI)); }
};
// Eight e4m3 numbers times a power of two as an operand of sixteen bits, exactly.
template <class DT>
__device__ __forceinline__ u32x4 kv_wide(uint32_t a, uint32_t b, float scale = 1.f) {
  typedef Kv<DT> F;
  return u32x4{F::template cvt<false>(a, scale), F::template cvt<true>(a, scale), F::template cvt<false>(b, scale), F::template cvt<true>(b, scale)};
}
template <class DT>
__device__ __forceinline__ float kv_over(float vs) { return fmaxf(vs * (1.f / Kv<DT>::VMAX), 1.f); }

// Places of numbers that are not finite.
template <class DT>
__device__ __forceinline__ uint32_t kv_nan16(uint32_t w) {  // bit 0 of each half: an exponent of ones carries into the sign's place
  constexpr uint32_t E = Kv<DT>::kExp * 0x10001u, L = (Kv<DT>::kExp & -Kv<DT>::kExp) * 0x10001u;
  return ((w & E) + L) >> 15 & 0x10001u;
}

// ---- storing ----------------------------------------------------------------------------------------------------------------------

// The smallest power of two with amax <= 448 * scale, between 2^-60 and 2^120 (values below 2^-70 become 0); 1 for a block of zeros.
__device__ __forceinline__ float kv_scale_of(float amax) {
  if (!(amax > 0.f)) return 1.f;
  const uint32_t bits = __float_as_uint(amax);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);  // 448 = 1.75 * 2^8
  e = e < -60 ? -60 : e;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// A block on its way into e4m3: 256 threads.  Of the keys thread 4 t + i holds elements i D / 4 .. of token t.  Of the values a thread holds four
// tokens of eight elements, which become one dword for each element; LDS turns them round.
template <int D>
struct KvBlockRegs {
  static constexpr int NK = D / 32, NV = D > 128 ? D / 128 : 1;
  u32x4 k[NK];
  u32x4 v[NV][4];
  static __device__ __forceinline__ int k_token() { return threadIdx.x / 4; }
  static __device__ __forceinline__ int k_first() { return threadIdx.x % 4 * (D / 4); }
  // item i of the thread: tokens 4 v_four .. + 3 of elements v_first .. + 7
  static __device__ __forceinline__ bool v_on(int i) { return (int)threadIdx.x + 256 * i < 2 * D; }
  static __device__ __forceinline__ int v_four(int i) { return (threadIdx.x + 256 * i) / (D / 8); }
  static __device__ __forceinline__ int v_first(int i) { return (threadIdx.x + 256 * i) % (D / 8) * 8; }
};
template <int D>
struct KvStage {
  uint32_t most[2][4];
  uint32_t v[D][kKvBlock / 4 + 1];
};
// What the tails hold.
template <int D>
__device__ __forceinline__ void kv_from_tails(KvBlockRegs<D>& r, const uint16_t* kt, const uint16_t* vt) {
#pragma unroll
  for (int i = 0; i < r.NK; i++) r.k[i] = ((const u32x4*)(kt + r.k_token() * D + r.k_first()))[i];
#pragma unroll
  for (int i = 0; i < r.NV; i++)
    if (r.v_on(i)) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const u32x2 lo = *(const u32x2*)(vt + (r.v_first(i) + e) * kKvBlock + 4 * r.v_four(i));
        const u32x2 hi = *(const u32x2*)(vt + (r.v_first(i) + e + 1) * kKvBlock + 4 * r.v_four(i));
#pragma unroll
        for (int j = 0; j < 4; j++) r.v[i][j][e / 2] = (lo[j / 2] >> (16 * (j & 1)) & 0xffffu) | (hi[j / 2] >> (16 * (j & 1)) << 16);
      }
    }
}
// Quantises block `blk` of a (row, cached head) pair.
template <class DT, int D>
__device__ __forceinline__ void kv_quantise(const KvCache& c, size_t pair, int blk, KvBlockRegs<D>& r, KvStage<D>& stage) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  const int tid = threadIdx.x;
  // magnitudes of 16-bit floats are ordered as integers
  auto larger = [](uint32_t m, uint32_t w) { return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, w & 0x7fff7fffu))); };
  auto finite = [](uint32_t w) { return w & ~(kv_nan16<DT>(w) * 0xffffu); };
  auto most = [&](bool all) {  // of keys in the first, of values in the second; all: also of what is not finite
    uint32_t m[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < r.NK; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) m[0] = larger(m[0], all ? r.k[i][e] : finite(r.k[i][e]));
#pragma unroll
    for (int i = 0; i < r.NV; i++)
      if (r.v_on(i)) {
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) m[1] = larger(m[1], all ? r.v[i][j][e] : finite(r.v[i][j][e]));
      }
#pragma unroll
    for (int a = 0; a < 2; a++) {
      m[a] = max(m[a] & 0xffffu, m[a] >> 16);
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) m[a] = max(m[a], (uint32_t)__shfl_xor((int)m[a], o, kWave));
      if (tid % kWave == 0) stage.most[a][tid / kWave] = m[a];
    }
    __syncthreads();
  };
  auto of_all = [&](int a) { return max(max(stage.most[a][0], stage.most[a][1]), max(stage.most[a][2], stage.most[a][3])); };
  most(true);
  const bool odd = max(of_all(0), of_all(1)) >= Kv<DT>::kExp;  // numbers that are not finite: rare
  if (odd) {
    __syncthreads();
    most(false);
  }
  const float ks = kv_scale_of(DT::tof((uint16_t)of_all(0))), vs = kv_scale_of(DT::tof((uint16_t)of_all(1)));
  const size_t block = pair * c.blocks + blk;
  if (tid == 0) {
    c.ks[block] = ks;
    c.vs[block] = vs;
  }
  const float ki = 1.f / ks, vi = 1.f / vs;  // powers of two
  auto four = [&](float a, float b, float x, float y) {  // in e4m3; NaN where a number is not finite
    if (odd) a = fmaf(a, 0.f, a), b = fmaf(b, 0.f, b), x = fmaf(x, 0.f, x), y = fmaf(y, 0.f, y);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, y, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
  };
  auto lo = [](uint32_t w) { return DT::tof((uint16_t)w); };
  auto hi = [](uint32_t w) { return DT::tof((uint16_t)(w >> 16)); };
  u32x2* k8 = (u32x2*)(c.k8 + block * kKvBlock * D + r.k_token() * D + r.k_first());
#pragma unroll
  for (int i = 0; i < r.NK; i++) {
    const u32x4 x = r.k[i];
    k8[i] = u32x2{four(lo(x[0]) * ki, hi(x[0]) * ki, lo(x[1]) * ki, hi(x[1]) * ki), four(lo(x[2]) * ki, hi(x[2]) * ki, lo(x[3]) * ki, hi(x[3]) * ki)};
  }
#pragma unroll
  for (int i = 0; i < r.NV; i++)
    if (r.v_on(i)) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const uint32_t w0 = r.v[i][0][e], w1 = r.v[i][1][e], w2 = r.v[i][2][e], w3 = r.v[i][3][e];
        stage.v[r.v_first(i) + 2 * e][r.v_four(i)] = four(lo(w0) * vi, lo(w1) * vi, lo(w2) * vi, lo(w3) * vi);
        stage.v[r.v_first(i) + 2 * e + 1][r.v_four(i)] = four(hi(w0) * vi, hi(w1) * vi, hi(w2) * vi, hi(w3) * vi);
      }
    }
  __syncthreads();
  u32x4* v8 = (u32x4*)(c.v8 + block * kKvBlock * D);
  for (int i = tid; i < D * 4; i += 256) {
    const uint32_t* s = &stage.v[i / 4][i % 4 * 4];
    v8[i] = u32x4{s[0], s[1], s[2], s[3]};
  }
}

struct KvAppendArgs {
  const uint16_t* k;  // (B, T, heads, D) in elements: strides of a row, a token and a head
  const uint16_t* v;
  long long k_row, k_tok, k_head, v_row, v_tok, v_head;
  KvSpan span;
  KvCache c;
  int T;
};

// Workgroup (i, head, row) quantises block start / 64 + i if these tokens complete it; the first one also stores the tail.  It is the only one that
// reads the tail (the tokens of the first block that were there before) and the only one that writes it, behind a barrier.
// Bound by memory, 2 bytes of a value read and one written: 8 prompts of 2048 tokens, 32 heads of 128, 93 us, 4.3 TB/s where a copy reaches 4.9 (with
// the values turned round a byte at a time in LDS 107).  A token each for 64 rows of 8 heads is the launch, 6.6 us.
template <class DT, int D>
__global__ __launch_bounds__(256) void kv8_append_kernel(KvAppendArgs p) {
  const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
  int start, n;
  if (!kv_span(p.span, b, p.T, start, n) || n == 0) return;
  const int end = start + n, last = (end - 1) / kKvBlock, blk = start / kKvBlock + blockIdx.x;
  if (blk > last) return;
  const size_t pair = (size_t)b * p.c.heads + h;
  uint16_t* kt = p.c.kt + pair * kKvBlock * D;
  uint16_t* vt = p.c.vt + pair * kKvBlock * D;
  const uint16_t* k = p.k + b * p.k_row + h * p.k_head;
  const uint16_t* v = p.v + b * p.v_row + h * p.v_head;

  __shared__ KvStage<D> stage;
  if ((blk + 1) * kKvBlock <= end) {
    KvBlockRegs<D> r;
    const int first = blk * kKvBlock - start;  // the new token that is the block's token 0
    if (first < 0) kv_from_tails<D>(r, kt, vt);
    if (first + r.k_token() >= 0) {
#pragma unroll
      for (int i = 0; i < r.NK; i++) r.k[i] = load_stream((const u32x4*)(k + (first + r.k_token()) * p.k_tok + r.k_first()) + i);
    }
#pragma unroll
    for (int i = 0; i < r.NV; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int t = first + 4 * r.v_four(i) + j;
        if (r.v_on(i) && t >= 0) r.v[i][j] = load_stream((const u32x4*)(v + t * p.v_tok + r.v_first(i)));
      }
    kv_quantise<DT, D>(p.c, pair, blk, r, stage);
  }
  if (blockIdx.x != 0) return;
  __syncthreads();  // what the tail held has been read
  const int from = max(start, last * kKvBlock), live = end - from;  // new tokens of the last block
  for (int i = tid; i < live * (D / 8); i += 256) {
    const int t = i / (D / 8), d = i % (D / 8) * 8;
    *(u32x4*)(kt + (from + t) % kKvBlock * D + d) = *(const u32x4*)(k + (from + t - start) * p.k_tok + d);
  }
  const int t = tid % kWave;
  if (t < live)
    for (int d = tid / kWave * 8; d < D; d += 32) {
      const u32x4 x = *(const u32x4*)(v + (from + t - start) * p.v_tok + d);
#pragma unroll
      for (int e = 0; e < 8; e++) vt[(d + e) * kKvBlock + (from + t) % kKvBlock] = (uint16_t)(x[e / 2] >> (16 * (e & 1)));
    }
}

// ---- attention ---------------------------------------------------------------------------------------------------------------------

struct KvAttnArgs {
  const uint16_t* q;  // (B, T, heads, D) in elements: strides of a row, a token and a head
  long long q_row, q_tok, q_head;
  uint16_t* out;      // (B, T, heads, D)
  KvSpan span;
  KvCache c;
  float* part;        // [pair][split][row][D] sums and, behind them, [pair][split][row][2] largest exponent and sum of weights
  float scale;        // log2(e) * the softmax's scale
  int T, group;       // group: query heads of a cached head
  int window;         // keys that a query sees, at most; 0: all
  int pairs, splits;  // pairs: rows x cached heads
};

// Row r of a (row, cached head) pair is head r % group of token r / group: the queries of a step that share a cached head are one
// operand of the matrix cores.  ROWS of them are a workgroup's; UNIT tiles of 64 tokens at a time are shared out over the splits.
struct KvTiles {
  int pos_lo, pos_hi;    // positions of the first and the last query
  int tile_lo, tile_hi;  // first and last tile of 64 keys
  int last;              // tile that is read from the tail
  int active;            // splits that have tiles
};
template <int ROWS, int UNIT>
__device__ __forceinline__ bool kv_tiles(const KvAttnArgs& p, int r0, int start, int n, KvTiles& t) {
  const int lo = r0 / p.group, hi = min((r0 + ROWS - 1) / p.group, n - 1);
  if (lo >= n) return false;
  t.pos_lo = start + lo;
  t.pos_hi = start + hi;
  t.tile_lo = p.window ? max(0, t.pos_lo - p.window + 1) / kKvBlock : 0;
  t.tile_hi = t.pos_hi / kKvBlock;
  t.last = (start + n - 1) / kKvBlock;
  t.active = min(p.splits, (t.tile_hi - t.tile_lo + UNIT) / UNIT);
  return true;
}

__device__ __forceinline__ uint16_t* kv_out_row(const KvAttnArgs& p, int pair, int r, int D) {
  const int b = pair / p.c.heads, h = pair - b * p.c.heads, t = r / p.group, g = r - t * p.group;
  return p.out + (((size_t)b * p.T + t) * p.c.heads * p.group + h * p.group + g) * D;
}

// Rows behind the last query are zeros, and all rows NaN where the row's tokens do not lie in the cache.
template <class DT>
__device__ __forceinline__ void kv_fill_rows(const KvAttnArgs& p, int pair, int r0, int rows, int n, bool ok, int D, int tid, int threads) {
  for (int i = tid; i < rows * (D / 8); i += threads) {
    const int r = r0 + i / (D / 8);
    if (r >= p.T * p.group) return;
    const uint32_t w = ok || r / p.group >= n ? 0u : DT::fromf(NAN) * 0x10001u;
    ((u32x4*)kv_out_row(p, pair, r, D))[i % (D / 8)] = u32x4{w, w, w, w};
  }
}

// A masked weight is 0, but 0 times a NaN is not.  So where keys are masked, numbers of V that are not finite are set to 0, and at the end, if there
// were any, the queries that see one are set to NaN: products of those places (1, and 0 elsewhere) and of what a query sees count them.
__device__ __forceinline__ uint32_t kv_nan8(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7; }  // bit 0 of each byte
// Sets them to 0; not 0 if there were any.
__device__ __forceinline__ uint32_t kv_fix8(u32x4& x) {
  uint32_t any = 0;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const uint32_t w = x[e], n = kv_nan8(w);
    x[e] = w & ~(n * 0xffu);
    any |= n;
  }
  return any;
}
template <class DT, class V>
__device__ __forceinline__ uint32_t kv_fix16(V& x) {
  uint32_t any = 0;
#pragma unroll
  for (int e = 0; e < (int)(sizeof(V) / 4); e++) {
    const uint32_t w = x[e], n = kv_nan16<DT>(w);
    x[e] = w & ~(n * 0xffffu);
    any |= n;
  }
  return any;
}
// Eight numbers' places as an operand.
template <class DT>
__device__ __forceinline__ u32x4 kv_bad8(const uint8_t* at) {
  const u32x2 w = *(const u32x2*)at;
  return kv_wide<DT>(kv_nan8(w[0]) * 0x38u, kv_nan8(w[1]) * 0x38u);  // 1 in e4m3
}
template <class DT>
__device__ __forceinline__ u32x4 kv_bad16(const uint16_t* at) {
  u32x4 w = *(const u32x4*)at;
#pragma unroll
  for (int e = 0; e < 4; e++) w[e] = kv_nan16<DT>(w[e]) * Kv<DT>::kOne;
  return w;
}

// Largest over the lanes that agree modulo 32, and modulo 16, in all of them: the halves of a wave, and its rows, change places.
__device__ __forceinline__ float max_mod32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_mod16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_mod32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

// A weight's exponent is s * sc - top.  Scores of 2^24 and more lie further apart than 1 in 32 bits, and then the product, rounded in `top` and not in
// the fma, may exceed it by any power of two: the largest weight would overflow.  So where a query's largest score is far from 0, scores are
// taken relative to the tile's largest, and that one's distance from the top, a difference of rounded products and not above 0 (or SLACK), is added.  Below
// this bound the rest is at most 2^-7 of an exponent, what 32 bits hold of such a score.
__device__ __forceinline__ bool kv_far(float top) { return fabsf(top) > 0x1p16f && top > -FLT_MAX; }
__device__ __forceinline__ float kv_scaled(float s, float sc) {  // rounded, whatever it is added to
#pragma clang fp contract(off)
  return s * sc;
}

// One new token, or a few: 16 rows of queries, the cache split over workgroups and over the four waves of each, the waves' results joined in LDS
// and the workgroups' by kv8_join_kernel.  Each wave takes 64 tokens at a time:
//   S^T = K . Q^T   tile i, row 4 g + e of the 16x16 result: token 16 g + 4 i + e, in lanes of group g = lane / 16; columns are queries
//   O^T += V^T . P  the weights of lane group g are those of tokens 16 g .. + 15 in order: what the lane has to supply as operand
// so weights go from one product into the other without leaving their lane, and every load of the cache is 16 bytes a lane of 1 KiB in a
// row (V) or of whole lines (K).  The next tile's keys are asked for when this one's have been used, and so are its values.  The numbers become
// 16-bit operands (two an instruction), the keys' scale goes into the exponent, the values' into the conversion: with w = s * ks * scale, weights are
// 2^(HEAD + w - max w), O sums them times the values, and both are divided at the end.
// The tail is four times sixteen tokens, for a wave each: tile `wave` of the four, and one product over sixteen tokens.
// Bound by the cache's bytes where it is long: one row of 131072 tokens, 8 heads of 128 for 32, 43 us, 6.2 TB/s where a read stream reaches 7.1, and 4.6
// for the join.  16 rows of 2048 to 4096 tokens take 23.0 us where the bytes take 14.5: four tiles a wave do not hide the way of the first and what
// the end costs.  100 tokens are the launch and three trips to memory one behind the other (positions, keys and values, the output), 6 us.
// MASK: queries that see different keys, or a window.  One token without a window sees all of every tile but the tail.
// SEAL: the tokens are in the tails and nowhere else yet.  One workgroup a pair more quantises the block that they complete; nobody reads that block
// in this launch.
constexpr int kKvStepWaves = 4;
// Waves a SIMD, as far as registers allow.
constexpr int kv_step_waves(int D) { return D == 256 ? 1 : D == 128 ? 3 : 4; }
template <class DT, int D, bool MASK, bool SEAL>
__global__ __launch_bounds__(256, kv_step_waves(D)) void kv8_attn_step_kernel(KvAttnArgs p) {
  constexpr bool AHEAD = D < 256 || !MASK;  // the next tile's keys over this one's values: registers
  constexpr int W = kKvStepWaves, ROWS = 16, NU = D / 16, NK = D >= 64 ? D / 64 : 1, NV = D >= 64 ? 2 : 1;
  typedef Kv<DT> F;
  const int lane = threadIdx.x & (kWave - 1), m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pair = blockIdx.x, split = blockIdx.y, r0 = blockIdx.z * ROWS, rows = p.T * p.group;
  const int b = pair / p.c.heads;
  int start, n;
  KvTiles t;
  const bool ok = kv_span(p.span, b, p.T, start, n);
  if constexpr (SEAL) {
    if (split == p.splits) {
      __shared__ KvStage<D> stage;
      if (!ok || (start + n) % kKvBlock != 0 || n == 0 || blockIdx.z != 0) return;
      KvBlockRegs<D> r;
      kv_from_tails<D>(r, p.c.kt + (size_t)pair * kKvBlock * D, p.c.vt + (size_t)pair * kKvBlock * D);
      kv_quantise<DT, D>(p.c, pair, (start + n) / kKvBlock - 1, r, stage);
      return;
    }
  }
  if (!kv_tiles<ROWS, W>(p, r0, start, n, t) || !ok) {
    if (split == 0) kv_fill_rows<DT>(p, pair, r0, ROWS, n, ok, D, threadIdx.x, 256);
    return;
  }
  if (split >= t.active) return;

  // queries: operand of step (c, v) is elements 64 c + 16 g + 8 v .. + 7 (of 32 elements: 8 g .. + 7)
  const int row = min(r0 + m, rows - 1), tok = min(row / p.group, n - 1), pos = start + tok;
  const int first = MASK && p.window ? pos - p.window : -1;  // the query sees first + 1 .. pos
  const int d0 = D >= 64 ? 16 * g : 8 * g;
  u32x4 qf[NK][NV];
  {
    const uint16_t* q = p.q + b * p.q_row + (row / p.group) * p.q_tok + ((pair - b * p.c.heads) * p.group + row % p.group) * p.q_head;
#pragma unroll
    for (int c = 0; c < NK; c++)
#pragma unroll
      for (int v = 0; v < NV; v++) qf[c][v] = *(const u32x4*)(q + 64 * c + d0 + 8 * v);
  }
  const int ktok = 16 * (m >> 2) + (m & 3);  // token of this lane's row of K in tile 0; 4 more in each of the next
  const uint8_t* k8 = p.c.k8 + (size_t)pair * p.c.blocks * kKvBlock * D + ktok * D + d0;
  const uint8_t* v8 = p.c.v8 + (size_t)pair * p.c.blocks * kKvBlock * D + m * kKvBlock + 16 * g;
  const float* kscale = p.c.ks + (size_t)pair * p.c.blocks;
  const float* vscale = p.c.vs + (size_t)pair * p.c.blocks;

  u32x4 kk[4][NK], vv[NU];
  auto fetch_k = [&](int tile) {
    const uint8_t* k = k8 + (size_t)tile * kKvBlock * D;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int c = 0; c < NK; c++) {
        if constexpr (D >= 64) {
          kk[i][c] = load_stream((const u32x4*)(k + 4 * i * D + 64 * c));
        } else {
          const u32x2 w = *(const u32x2*)(k + 4 * i * D);
          kk[i][c] = u32x4{w[0], w[1], 0u, 0u};
        }
      }
  };
  auto fetch_v = [&](int tile) {
    const uint8_t* v = v8 + (size_t)tile * kKvBlock * D;
#pragma unroll
    for (int u = 0; u < NU; u++) vv[u] = load_stream((const u32x4*)(v + 16 * u * kKvBlock));
  };
  const int step = t.active * W, end8 = min(t.tile_hi, t.last - 1);  // last tile in 8 bits
  int tile = t.tile_lo + split * W + wave;

  float top = -FLT_MAX, sum = 0.f;
  bool far = false;   // whether some query's scores are
  uint32_t some = 0;  // whether a tile that is seen in part had numbers of V that are not finite
  f32x4 o[NU];
#pragma unroll
  for (int u = 0; u < NU; u++) o[u] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto seen = [&](int key) { return key <= pos && (!MASK || key > first); };
  // weights of this lane's N x 4 scores, in place; the lanes of a query agree on their largest
  auto weigh = [&](f32x4* s, int N, float ks, float over) {
    const float sc = p.scale * ks, lv = __builtin_amdgcn_logf(over);
    float mx = s[0][0];
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) mx = fmaxf(mx, s[i][e]);
    mx = max_mod16(mx);
    const float at = kv_scaled(mx, sc), now = fmaxf(top, at + lv);
    float off = lv + F::HEAD - now;
    if (__any(now > top)) {
      const float keep = __builtin_amdgcn_exp2f(top - now);
      sum *= keep;
#pragma unroll
      for (int u = 0; u < NU; u++) o[u] *= keep;
      top = now;
      far = __any(kv_far(top));
    }
    if (far) {
      const float ref = fmaxf(mx, -FLT_MAX);
      off = fminf(at - now + lv, 0.f) + F::HEAD;
#pragma unroll
      for (int i = 0; i < N; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[i][e] -= ref;
    }
    float add = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        s[i][e] = __builtin_amdgcn_exp2f(fmaf(s[i][e], sc, off));
        add += s[i][e];
      }
    sum = fmaf(add, __builtin_amdgcn_rcpf(over), sum);
    asm volatile("" : "+v"(sum));  // here: the weights' registers are wanted
  };

  auto part_tile = [&](int at) {  // whether some query does not see all of it
    return at * kKvBlock + kKvBlock - 1 > t.pos_lo || (p.window && at * kKvBlock <= t.pos_hi - p.window);
  };
  // the tail, by the split whose turn it would be: its loads go ahead of the first tile's, whose way from memory hides what the tail takes
  const bool tail = t.tile_hi == t.last && (t.last - t.tile_lo) / W % t.active == split;
  u32x4 kq[NK][NV];
  u32x2 vq[NU];
  if (tail) {
    const uint16_t* kt = p.c.kt + (size_t)pair * kKvBlock * D + (ktok + 4 * wave) * D + d0;
    const uint16_t* vt = p.c.vt + (size_t)pair * kKvBlock * D + m * kKvBlock + 16 * g + 4 * wave;
#pragma unroll
    for (int c = 0; c < NK; c++)
#pragma unroll
      for (int v = 0; v < NV; v++) kq[c][v] = *(const u32x4*)(kt + 64 * c + 8 * v);
#pragma unroll
    for (int u = 0; u < NU; u++) vq[u] = *(const u32x2*)(vt + 16 * u * kKvBlock);
  }
  __builtin_amdgcn_sched_barrier(0);
  if (tile <= end8) {
    fetch_k(tile);
    fetch_v(tile);
  }
  __builtin_amdgcn_sched_barrier(0);
  if (tail) {
    f32x4 s[1] = {f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int c = 0; c < NK; c++)
#pragma unroll
      for (int v = 0; v < NV; v++) s[0] = Mma<DT>::run(kq[c][v], qf[c][v], s[0]);
    const int key = t.last * kKvBlock + 16 * g + 4 * wave;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float x = fmaf(s[0][e], 0.f, s[0][e]);  // a key that is not finite makes the score NaN, as in e4m3
      s[0][e] = seen(key + e) ? x : -INFINITY;
    }
    weigh(s, 1, 1.f, 1.f);
    const u32x2 pf = u32x2{DT::pack(s[0][0], s[0][1]), DT::pack(s[0][2], s[0][3])};
#pragma unroll
    for (int u = 0; u < NU; u++) {
      some |= kv_fix16<DT>(vq[u]);
      o[u] = DownMma<DT>::run(vq[u], pf, o[u]);
    }
  }
  // What the next tile would need is asked for under a condition and not behind a way out of the loop: with that (and heads of 32, MASK) this compiler took
  // parts of vv for undefined and gave their registers to others.
  while (tile <= end8) {
    const float ks = kscale[tile], vs = vscale[tile], vm = fminf(vs, F::VMAX);
    f32x4 s[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      __builtin_amdgcn_sched_barrier(0);
      s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NK; c++)
#pragma unroll
        for (int v = 0; v < NV; v++) s[i] = Mma<DT>::run(kv_wide<DT>(kk[i][c][2 * v], kk[i][c][2 * v + 1]), qf[c][v], s[i]);
    }
    const bool more = tile + step <= end8;
    __builtin_amdgcn_sched_barrier(0);
    if (AHEAD && more) fetch_k(tile + step);
    __builtin_amdgcn_sched_barrier(0);
    const int key0 = tile * kKvBlock + 16 * g;  // of this lane's weights
    const bool part = MASK && part_tile(tile);
    if (part) {
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[i][e] = seen(key0 + 4 * i + e) ? s[i][e] : -INFINITY;
    }
    weigh(s, 4, ks, kv_over<DT>(vs));
    u32x4 pf[2];  // the weights, rounded to the type the products take: half a step each, independent of one another
#pragma unroll
    for (int v = 0; v < 2; v++)
      pf[v] = u32x4{DT::pack(s[2 * v][0], s[2 * v][1]), DT::pack(s[2 * v][2], s[2 * v][3]), DT::pack(s[2 * v + 1][0], s[2 * v + 1][1]),
                    DT::pack(s[2 * v + 1][2], s[2 * v + 1][3])};
    if (part) {
#pragma unroll
      for (int u = 0; u < NU; u++) some |= kv_fix8(vv[u]);
    }
#pragma unroll
    for (int u = 0; u < NU; u++) {
      if (u % 4 == 0) __builtin_amdgcn_sched_barrier(0);  // operands of four products at a time
      o[u] = Mma<DT>::run(kv_wide<DT>(vv[u][0], vv[u][1], vm), pf[0], o[u]);
      o[u] = Mma<DT>::run(kv_wide<DT>(vv[u][2], vv[u][3], vm), pf[1], o[u]);
    }
    __builtin_amdgcn_sched_barrier(0);
    tile += step;
    if (more) {
      if (!AHEAD) fetch_k(tile);
      fetch_v(tile);
    }
  }

  if (__any(some != 0)) {  // the queries that see a number that is not finite
    auto spoil = [&](int tile, auto load) {
#pragma unroll
      for (int u = 0; u < NU; u++) {
        f32x4 z = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < 2; v++) {
          const int key = tile * kKvBlock + 16 * g + 8 * v;
          u32x4 one;
#pragma unroll
          for (int e = 0; e < 4; e++) one[e] = (seen(key + 2 * e) ? F::kOne : 0u) | (seen(key + 2 * e + 1) ? F::kOne << 16 : 0u);
          z = Mma<DT>::run(load(16 * u + m, 16 * g + 8 * v), one, z);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) o[u][e] = z[e] > 0.f ? NAN : o[u][e];
      }
    };
    if constexpr (MASK)
      for (tile = t.tile_lo + split * W + wave; tile <= end8; tile += step)
        if (part_tile(tile)) spoil(tile, [&](int d, int key) { return kv_bad8<DT>(p.c.v8 + ((size_t)pair * p.c.blocks + tile) * kKvBlock * D + d * kKvBlock + key); });
    if (tail) spoil(t.last, [&](int d, int key) { return kv_bad16<DT>(p.c.vt + ((size_t)pair * D + d) * kKvBlock + key); });
  }
  sum += __shfl_xor(sum, 16, kWave);
  sum += __shfl_xor(sum, 32, kWave);

  // the four waves' results
  __shared__ __align__(16) float s_o[W][ROWS][D + 4];
  __shared__ float s_top[W][ROWS], s_sum[W][ROWS];
#pragma unroll
  for (int u = 0; u < NU; u++) *(f32x4*)&s_o[wave][m][16 * u + 4 * g] = o[u];
  if (g == 0) {
    s_top[wave][m] = top;
    s_sum[wave][m] = sum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < ROWS * (D / 4); i += 256) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    if (r0 + r >= rows) break;
    float most = s_top[0][r];
#pragma unroll
    for (int w = 1; w < W; w++) most = fmaxf(most, s_top[w][r]);
    f32x4 num = f32x4{0.f, 0.f, 0.f, 0.f};
    float den = 0.f;
#pragma unroll
    for (int w = 0; w < W; w++) {
      const float f = __builtin_amdgcn_exp2f(s_top[w][r] - most);
      const f32x4 x = *(const f32x4*)&s_o[w][r][d];
#pragma unroll
      for (int e = 0; e < 4; e++) num[e] = fmaf(f, x[e], num[e]);
      den = fmaf(f, s_sum[w][r], den);
    }
    if (t.active == 1) {
      const bool dead = (r0 + r) / p.group >= n;
#pragma unroll
      for (int e = 0; e < 4; e++) num[e] = dead ? 0.f : num[e] / den;
      *(u32x2*)(kv_out_row(p, pair, r0 + r, D) + d) = u32x2{DT::pack(num[0], num[1]), DT::pack(num[2], num[3])};
    } else {
      const size_t at = ((size_t)pair * p.splits + split) * rows + r0 + r;
      *(f32x4*)(p.part + at * D + d) = num;
      if (d == 0) {
        float* ml = p.part + (size_t)p.pairs * p.splits * rows * D + 2 * at;
        ml[0] = most;
        ml[1] = den;
      }
    }
  }
}

// Many new tokens: 64 rows of queries a workgroup and two tiles of 64 keys at a time, a wave for each 32 rows and tile; what the two halves of the keys
// give is joined in LDS at the end.  The tiles come into LDS in 8 bits, straight from memory, the next two while the weights of these are computed.
// The same steps as above with v_mfma_f32_32x32x16:
//   S^T   tile u, row 8 a + 4 h + i of the result: token 32 u + 16 h + 4 a + i, in lanes of half h = lane / 32; columns are queries
//   O^T   operand of step (u, v): tokens 32 u + 16 h + 8 v .. + 7, again those whose weights the lane has
// Rows of LDS are 16-byte pieces, exchanged within a row so that any 16 lanes in order find the 64 banks once each.
// Workgroups with the most keys start first.
// Bound by what a SIMD issues: a tile is 32 products a wave (1024 cycles of the matrix cores with heads of 128) and some 310 other instructions, of which 128
// turn e4m3 into operands and 32 are exponentials, and the two overlap only in part (a loop of each, alone 1189 and 1169 cycles, on one SIMD 1570); a third
// wave a SIMD, which heads of 64 have room for, is worth 2 to 6 %.  A prompt of 2048 tokens, 32 heads of 128, takes 50 us, 690 TFLOP/s of what is
// seen; two pieces of 512 behind 7680 tokens 118 us, 880 (a large product 1125 to 1180); other cards 51 and 123.
// 128 rows a workgroup need the registers of one wave a SIMD and were slower.
typedef float f32x16 __attribute__((ext_vector_type(16)));
template <class DT> struct Mma32;
template <> struct Mma32<F16> {
  static __device__ __forceinline__ f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <> struct Mma32<BF16> {
  static __device__ __forceinline__ f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
// Which piece of token t's row of K is exchanged with piece 0: of the lanes that read together, tokens differ in bits 0, 1, 4 and 2.
template <int D>
__device__ __forceinline__ int kv_swap_k(int t) {
  if (D == 256) return (t & 3) | (t >> 4 & 1) << 2 | (t >> 2 & 1) << 3;
  if (D == 128) return (t >> 1 & 1) | (t >> 4 & 1) << 1 | (t >> 2 & 1) << 2;
  if (D == 64) return (t >> 4 & 1) | (t >> 2 & 1) << 1;
  return t >> 4 & 1;
}
__device__ __forceinline__ int kv_swap_v(int d) { return d >> 2 & 3; }

constexpr int kKvPromptRows = 64, kKvPromptUnit = 16;  // rows of a workgroup; tiles that make a split worth while
template <class DT, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void kv8_attn_prompt_kernel(KvAttnArgs p) {
  constexpr int ROWS = kKvPromptRows, C = D / 32, NW = D / 32, PK = D / 16;
  constexpr int kVecs = D * kKvBlock / 16;  // of a tile's keys, and of its values
  typedef Kv<DT> F;
  __shared__ u32x4 s_kv[2][2][2][kVecs];  // [buffer][tile][keys, values]
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 31, h = lane >> 5;
  const int rw = wave & 1, kh = wave >> 1;  // the wave's rows and its tile of two
  const int pair = blockIdx.x, r0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * ROWS, split = blockIdx.z, rows = p.T * p.group;
  const int b = pair / p.c.heads;
  int start, n;
  KvTiles t;
  const bool ok = kv_span(p.span, b, p.T, start, n);
  if (!kv_tiles<ROWS, kKvPromptUnit>(p, r0, start, n, t) || !ok) {
    if (split == 0) kv_fill_rows<DT>(p, pair, r0, ROWS, n, ok, D, tid, 256);
    return;
  }
  if (split >= t.active) return;

  const int mine = r0 + 32 * rw + m, row = min(mine, rows - 1), pos = start + min(row / p.group, n - 1);
  const int first = p.window ? pos - p.window : -1;  // the query sees first + 1 .. pos
  // the wave's own keys
  const int lo_pos = start + min((r0 + 32 * rw) / p.group, n - 1), hi_pos = start + min((r0 + 32 * rw + 31) / p.group, n - 1);
  u32x4 qf[C][2];
  {
    const uint16_t* q = p.q + b * p.q_row + (row / p.group) * p.q_tok + ((pair - b * p.c.heads) * p.group + row % p.group) * p.q_head;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int v = 0; v < 2; v++) qf[c][v] = *(const u32x4*)(q + 32 * c + 16 * h + 8 * v);
  }
  const u32x4* k8 = (const u32x4*)p.c.k8 + (size_t)pair * p.c.blocks * kVecs;
  const u32x4* v8 = (const u32x4*)p.c.v8 + (size_t)pair * p.c.blocks * kVecs;
  const float* kscale = p.c.ks + (size_t)pair * p.c.blocks;
  const float* vscale = p.c.vs + (size_t)pair * p.c.blocks;

  // A wave brings half of the rows of keys and of values of its tile, 1 KiB at a time: lane l of load j writes piece 64 j + l and reads what belongs
  // there.  What is exchanged goes by bits of the row, so load j differs from load 0 by constants, and reads of LDS differ by constants too: four
  // offsets in bytes are kept over the loop, hidden from the compiler, which would keep every address that follows from them.
  unsigned k_from = (lane / PK * PK + ((lane % PK) ^ kv_swap_k<D>(lane / PK))) * 16, v_from = (lane / 4 * 4 + ((lane % 4) ^ kv_swap_v(lane / 4))) * 16;
  const int ktok = 16 * (m >> 2 & 1) + 4 * (m >> 3) + (m & 3);  // token of this lane's row of K in tile 0; 32 more in tile 1
  unsigned k_at = (ktok * PK + (h ^ kv_swap_k<D>(ktok))) * 16, v_at = (m * 4 + (h ^ kv_swap_v(m))) * 16;
  asm volatile("" : "+v"(k_from), "+v"(v_from), "+v"(k_at), "+v"(v_at));
  const int end8 = min(t.tile_hi, t.last - 1);  // last tile in 8 bits; behind it the last one comes again
  float ks = 1.f, vs = 1.f, ks1 = 1.f, vs1 = 1.f;  // scales of the wave's tile and of the next one
  auto bring = [&](int tile, int buf) {
    const int at = min(tile + kh, end8);
    ks1 = kscale[at];
    vs1 = vscale[at];
    const u32x4* kf = k8 + (size_t)at * kVecs + rw * (kVecs / 2);
    const u32x4* vf = v8 + (size_t)at * kVecs + rw * (kVecs / 2);
    u32x4* to = s_kv[buf][kh][0] + rw * (kVecs / 2);
#pragma unroll
    for (int j = 0; j < kVecs / 2 / kWave; j++) {
      const char *kj = (const char*)(kf + j * kWave), *vj = (const char*)(vf + j * kWave);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(kj + (size_t)(k_from ^ (16u * kv_swap_k<D>(j * kWave / PK)))),
                                       (__attribute__((address_space(3))) void*)(to + j * kWave), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(vj + (size_t)v_from),
                                       (__attribute__((address_space(3))) void*)(to + kVecs + j * kWave), 16, 0, 0);
    }
  };

  float top = -FLT_MAX, sum = 0.f;
  bool far = false;   // whether some query's scores are
  uint32_t some = 0;  // whether a tile that is seen in part had numbers of V that are not finite
  f32x16 o[NW];
  auto zeros = [] {
    f32x16 z;
#pragma unroll
    for (int e = 0; e < 16; e++) z[e] = 0.f;
    return z;
  };
#pragma unroll
  for (int w = 0; w < NW; w++) o[w] = zeros();

  // weights of a tile from its scores; returns them as operands
  auto weigh = [&](f32x16 (&s)[2], float ks, float over, u32x4 (&pf)[2][2]) {
    const float sc = p.scale * ks, lv = __builtin_amdgcn_logf(over);
    float mx = s[0][0];
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int e = 0; e < 16; e++) mx = fmaxf(mx, s[u][e]);
    mx = max_mod32(mx);
    const float at = kv_scaled(mx, sc), now = fmaxf(top, at + lv);
    if (__any(now > top + F::SLACK)) {
      const float keep = __builtin_amdgcn_exp2f(top - now);
      sum *= keep;
#pragma unroll
      for (int w = 0; w < NW; w++) o[w] *= keep;
      top = now;
      far = __any(kv_far(top));
    }
    float off = lv + F::HEAD - F::SLACK - top;
    if (far) {
      const float ref = fmaxf(mx, -FLT_MAX);
      off = fminf(at - top + lv, F::SLACK) + F::HEAD - F::SLACK;
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int e = 0; e < 16; e++) s[u][e] -= ref;
    }
    float add = 0.f;
#pragma unroll
    for (int u = 0; u < 2; u++) {
#pragma unroll
      for (int e = 0; e < 16; e++) {
        s[u][e] = __builtin_amdgcn_exp2f(fmaf(s[u][e], sc, off));
        add += s[u][e];
      }
#pragma unroll
      for (int v = 0; v < 2; v++)
#pragma unroll
        for (int e = 0; e < 4; e++) pf[u][v][e] = DT::pack(s[u][8 * v + 2 * e], s[u][8 * v + 2 * e + 1]);
    }
    sum = fmaf(add, __builtin_amdgcn_rcpf(over), sum);
    asm volatile("" : "+v"(sum));  // here: the weights' registers are wanted
  };
  auto seen = [&](int key) { return key <= pos && key > first; };
  auto mask = [&](f32x16 (&s)[2], int tile) {
    const int most = pos - tile * kKvBlock - 16 * h;  // of 32 u + e
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int e = 0; e < 16; e++) s[u][e] = 32 * u + e <= most ? s[u][e] : -INFINITY;
    if (p.window) {
      const int least = max(most, -kKvBlock) - p.window;  // a tile that is none has most near INT_MIN
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int e = 0; e < 16; e++) s[u][e] = 32 * u + e > least ? s[u][e] : -INFINITY;
    }
  };
  // one tile of 64 keys from LDS; PART: some query of the wave does not see all of them
  auto take = [&](auto PART, int tile, int buf, auto behind) {
    // All of a tile's keys are asked for at once, and its values before the weights are computed: what LDS takes to answer is as long as eight
    // products each time.  (Heads of 256 elements do not have the registers.)
    constexpr bool ASK = D <= 128;
    f32x16 s[2] = {zeros(), zeros()};
    const char* tile_kv = (const char*)s_kv[buf][kh][0];
    auto keys = [&](int c, int u) { return *(const u32x4*)(tile_kv + (k_at ^ 32u * c) + 32 * u * PK * 16); };
    auto values = [&](int w, int u) { return *(const u32x4*)(tile_kv + (v_at ^ 32u * u) + (kVecs + 32 * w * 4) * 16); };
    u32x4 x[ASK ? 2 * NW : 1];  // C is NW
    if constexpr (ASK) {
#pragma unroll
      for (int c = 0; c < C; c++)
#pragma unroll
        for (int u = 0; u < 2; u++) x[2 * c + u] = keys(c, u);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const u32x4 kk = ASK ? x[ASK ? 2 * c + u : 0] : keys(c, u);
        s[u] = Mma32<DT>::run(kv_wide<DT>(kk[0], kk[1]), qf[c][0], s[u]);
        s[u] = Mma32<DT>::run(kv_wide<DT>(kk[2], kk[3]), qf[c][1], s[u]);
      }
    if constexpr (ASK) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int w = 0; w < NW; w++)
#pragma unroll
        for (int u = 0; u < 2; u++) x[2 * w + u] = values(w, u);
      __builtin_amdgcn_sched_barrier(0);
      behind();
    }
    // The other wave's products before this one's weights: two pieces of 512 behind 7680 tokens 146 us, without 151; a prompt of 2048 58.8 and 57.3.
    __builtin_amdgcn_s_setprio(0);
    if constexpr (PART) {
      mask(s, tile);
      if constexpr (ASK) {
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < 2 * NW; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) bad |= (x[i][e] & 0x7f7f7f7fu) + 0x01010101u;
        if (__any((bad & 0x80808080u) != 0)) {
          some = 1;
#pragma unroll
          for (int i = 0; i < 2 * NW; i++) kv_fix8(x[i]);
        }
      }
    }
    u32x4 pf[2][2];
    const float vm = fminf(vs, F::VMAX);
    weigh(s, ks, kv_over<DT>(vs), pf);
    __builtin_amdgcn_s_setprio(1);
    if constexpr (ASK) {
      // Sums of different w in turn, and each operand made while the product before it runs: otherwise the products wait for theirs (a prompt of 2048
      // tokens 50.6, 49.6 us; two pieces of 512 behind 7680 119.7, 118.0; the same for the scores gains nothing).
      auto wide = [&](int i) {
        const u32x4 vv = x[2 * (i % NW) + i / (2 * NW)];
        return i / NW & 1 ? kv_wide<DT>(vv[2], vv[3], vm) : kv_wide<DT>(vv[0], vv[1], vm);
      };
      __builtin_amdgcn_sched_barrier(0);
      u32x4 operand = wide(0);
#pragma unroll
      for (int i = 0; i < 4 * NW; i++) {
        const u32x4 now = operand;
        if (i + 1 < 4 * NW) operand = wide(i + 1);
        o[i % NW] = Mma32<DT>::run(now, pf[i / (2 * NW)][i / NW & 1], o[i % NW]);
      }
      __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);  // four conversions are an operand
#pragma unroll
      for (int i = 0; i < 4 * NW; i++) {
        __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    } else {
#pragma unroll
      for (int w = 0; w < NW; w++)
#pragma unroll
        for (int u = 0; u < 2; u++) {
          u32x4 vv = values(w, u);
          if constexpr (PART) some |= kv_fix8(vv);
          o[w] = Mma32<DT>::run(kv_wide<DT>(vv[0], vv[1], vm), pf[u][0], o[w]);
          o[w] = Mma32<DT>::run(kv_wide<DT>(vv[2], vv[3], vm), pf[u][1], o[w]);
        }
      behind();
    }
  };

  auto seen_tile = [&](int tile) {  // whether some query of the wave sees some of it
    return tile * kKvBlock <= hi_pos && !(p.window && tile * kKvBlock + kKvBlock - 1 <= lo_pos - p.window);
  };
  const int step = 2 * t.active;
  int tile = t.tile_lo + 2 * split, buf = 0;  // the first of the two
  if (t.tile_lo <= end8) bring(tile, 0);
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): in LDS
  ks = ks1, vs = vs1;
  lds_barrier();
  auto run = [&](auto PART, int to) {
    for (; tile <= to; tile += step, buf ^= 1) {
      // Behind the last read of this buffer: a read of LDS behind these loads would wait for them.  A second tile behind the last one has no key
      // that is seen: it is the last one again.
      take(PART, tile + kh <= end8 ? tile + kh : INT_MAX / kKvBlock, buf, [&] { bring(tile + step, buf ^ 1); });
      __builtin_amdgcn_s_waitcnt(0x0f70);
      ks = ks1, vs = vs1;
      lds_barrier();
    }
  };
  // tiles that a window cuts, tiles that all of the workgroup's queries see, tiles that hold some of their own keys
  const int cut = p.window && t.pos_hi >= p.window ? (t.pos_hi - p.window) / kKvBlock : -1, own = (t.pos_lo + 1) / kKvBlock;  // last and first of them
  run(std::true_type(), min(cut, end8));
  run(std::false_type(), min(own - 2, end8 - 1));
  run(std::true_type(), end8);
  // the tail, by the split whose turn it would be, from memory: one tile of the last rows only
  const bool tail = t.tile_hi == t.last && (t.last - t.tile_lo) / 2 % t.active == split && (t.last - t.tile_lo) % 2 == kh && t.last * kKvBlock <= hi_pos;
  if (tail) {
    const uint16_t* kt = p.c.kt + (size_t)pair * kKvBlock * D;
    const uint16_t* vt = p.c.vt + (size_t)pair * kKvBlock * D;
    f32x16 s[2] = {zeros(), zeros()};
#pragma unroll
    for (int u = 0; u < 2; u++) {
#pragma unroll
      for (int c = 0; c < C; c++)
#pragma unroll
        for (int v = 0; v < 2; v++) s[u] = Mma32<DT>::run(*(const u32x4*)(kt + (ktok + 32 * u) * D + 32 * c + 16 * h + 8 * v), qf[c][v], s[u]);
#pragma unroll
      for (int e = 0; e < 16; e++) s[u][e] = fmaf(s[u][e], 0.f, s[u][e]);  // a key that is not finite makes the score NaN, as in e4m3
    }
    __builtin_amdgcn_sched_barrier(0);
    u32x4 x[NW][2][2];
#pragma unroll
    for (int w = 0; w < NW; w++)
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int v = 0; v < 2; v++) x[w][u][v] = *(const u32x4*)(vt + (32 * w + m) * kKvBlock + 32 * u + 16 * h + 8 * v);
    __builtin_amdgcn_sched_barrier(0);
    mask(s, t.last);
    u32x4 pf[2][2];
    weigh(s, 1.f, 1.f, pf);
#pragma unroll
    for (int w = 0; w < NW; w++) {
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int v = 0; v < 2; v++) {
          some |= kv_fix16<DT>(x[w][u][v]);
          o[w] = Mma32<DT>::run(x[w][u][v], pf[u][v], o[w]);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (__any(some != 0)) {  // the queries that see a number that is not finite
    auto spoil = [&](int tile, auto load) {
#pragma unroll
      for (int w = 0; w < NW; w++) {
        f32x16 z = zeros();
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int v = 0; v < 2; v++) {
            const int key = tile * kKvBlock + 32 * u + 16 * h + 8 * v;
            u32x4 one;
#pragma unroll
            for (int e = 0; e < 4; e++) one[e] = (seen(key + 2 * e) ? F::kOne : 0u) | (seen(key + 2 * e + 1) ? F::kOne << 16 : 0u);
            z = Mma32<DT>::run(load(32 * w + m, 32 * u + 16 * h + 8 * v), one, z);
          }
#pragma unroll
        for (int e = 0; e < 16; e++) o[w][e] = z[e] > 0.f ? NAN : o[w][e];
      }
    };
    for (tile = t.tile_lo + 2 * split + kh; tile <= end8; tile += step)
      if (seen_tile(tile))
        spoil(tile, [&](int d, int key) { return kv_bad8<DT>((const uint8_t*)(v8 + (size_t)tile * kVecs) + d * kKvBlock + key); });
    if (tail) spoil(t.last, [&](int d, int key) { return kv_bad16<DT>(p.c.vt + ((size_t)pair * D + d) * kKvBlock + key); });
  }
  sum += __shfl_xor(sum, 32, kWave);
  // the other half of the keys
  __shared__ float s_top[2][32], s_sum[2][32];
  f32x4* s_o = (f32x4*)s_kv[rw][0][0];  // all tiles have been read: [D / 8][lane] of each wave
  if (kh == 1) {
#pragma unroll
    for (int w = 0; w < NW; w++)
#pragma unroll
      for (int a = 0; a < 4; a++) s_o[(4 * w + a) * kWave + lane] = f32x4{o[w][4 * a], o[w][4 * a + 1], o[w][4 * a + 2], o[w][4 * a + 3]};
    if (h == 0) {
      s_top[rw][m] = top;
      s_sum[rw][m] = sum;
    }
  }
  lds_barrier();
  if (kh == 1) return;
  {
    const float other = s_top[rw][m], now = fmaxf(top, other), f = __builtin_amdgcn_exp2f(top - now), g = __builtin_amdgcn_exp2f(other - now);
    sum = fmaf(g, s_sum[rw][m], f * sum);
    top = now;
#pragma unroll
    for (int w = 0; w < NW; w++)
#pragma unroll
      for (int a = 0; a < 4; a++) {
        const f32x4 x = s_o[(4 * w + a) * kWave + lane];
#pragma unroll
        for (int e = 0; e < 4; e++) o[w][4 * a + e] = fmaf(g, x[e], f * o[w][4 * a + e]);
      }
  }
  if (mine >= rows) return;
  if (t.active == 1) {
    const bool dead = mine / p.group >= n;
    const float f = 1.f / sum;
    uint16_t* out = kv_out_row(p, pair, mine, D);
#pragma unroll
    for (int w = 0; w < NW; w++)
#pragma unroll
      for (int a = 0; a < 4; a++) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = dead ? 0.f : o[w][4 * a + e] * f;
        *(u32x2*)(out + 32 * w + 8 * a + 4 * h) = u32x2{DT::pack(x[0], x[1]), DT::pack(x[2], x[3])};
      }
  } else {
    const size_t at = ((size_t)pair * p.splits + split) * rows + mine;
#pragma unroll
    for (int w = 0; w < NW; w++)
#pragma unroll
      for (int a = 0; a < 4; a++) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = o[w][4 * a + e];
        *(f32x4*)(p.part + at * D + 32 * w + 8 * a + 4 * h) = x;
      }
    if (h == 0) {
      float* ml = p.part + (size_t)p.pairs * p.splits * rows * D + 2 * at;
      ml[0] = top;
      ml[1] = sum;
    }
  }
}

// The splits' results, in a fixed order: 4 us, the launch and two trips to memory.  ALONE: a workgroup per (pair, row), whose groups of D / 4 lanes take
// every so manieth split and are joined in LDS.  Otherwise, for few splits, a row per group.  Rows whose cache was one split's are done already.  ROWS and UNIT are the
// attention kernel's.
template <class DT, int D, int ROWS, int UNIT, bool ALONE>
__global__ __launch_bounds__(256) void kv8_join_kernel(KvAttnArgs p) {
  constexpr int L = D / 4, G = 256 / L;
  const int grp = threadIdx.x / L, d = threadIdx.x % L * 4;
  const int rows = p.T * p.group, item = ALONE ? blockIdx.x : blockIdx.x * G + grp, pair = item / rows, r = item - pair * rows;
  if (pair >= p.pairs) return;
  int start, n;
  KvTiles t;
  if (!kv_span(p.span, pair / p.c.heads, p.T, start, n) || !kv_tiles<ROWS, UNIT>(p, r / ROWS * ROWS, start, n, t) || t.active == 1) return;
  const size_t at = (size_t)pair * p.splits * rows + r;
  const float* ml = p.part + (size_t)p.pairs * p.splits * rows * D + 2 * at;
  const float* part = p.part + at * D + d;
  float top = -FLT_MAX, den = 0.f;
  f32x4 num = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = ALONE ? grp : 0; s < t.active; s += ALONE ? G : 1) {
    const float mx = ml[2 * (size_t)s * rows], sm = ml[2 * (size_t)s * rows + 1];
    const f32x4 x = *(const f32x4*)(part + (size_t)s * rows * D);
    const float now = fmaxf(top, mx), keep = __builtin_amdgcn_exp2f(top - now), f = __builtin_amdgcn_exp2f(mx - now);
#pragma unroll
    for (int e = 0; e < 4; e++) num[e] = fmaf(f, x[e], num[e] * keep);
    den = fmaf(f, sm, den * keep);
    top = now;
  }
  if constexpr (ALONE) {
    __shared__ __align__(16) float s_o[G][D];
    __shared__ float s_top[G], s_sum[G];
    *(f32x4*)&s_o[grp][d] = num;
    if (d == 0) {
      s_top[grp] = top;
      s_sum[grp] = den;
    }
    __syncthreads();
    if (grp != 0) return;
    float most = s_top[0];
#pragma unroll
    for (int i = 1; i < G; i++) most = fmaxf(most, s_top[i]);
    num = f32x4{0.f, 0.f, 0.f, 0.f};
    den = 0.f;
#pragma unroll
    for (int i = 0; i < G; i++) {
      const float f = __builtin_amdgcn_exp2f(s_top[i] - most);
      const f32x4 x = *(const f32x4*)&s_o[i][d];
#pragma unroll
      for (int e = 0; e < 4; e++) num[e] = fmaf(f, x[e], num[e]);
      den = fmaf(f, s_sum[i], den);
    }
  }
  const bool dead = r / p.group >= n;
#pragma unroll
  for (int e = 0; e < 4; e++) num[e] = dead ? 0.f : num[e] / den;
  *(u32x2*)(kv_out_row(p, pair, r, D) + d) = u32x2{DT::pack(num[0], num[1]), DT::pack(num[2], num[3])};
}

}  // namespace cats
