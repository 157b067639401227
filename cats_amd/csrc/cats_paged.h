// A cache of pages, packed sequences, and attention over both (16-bit models).
//
// Tokens of a call are packed: sequence s has the tokens offsets[s] .. offsets[s + 1] - 1, at the positions start[s] onwards.  Nobody on the host knows how
// long any of them is, so a launch is sized by what N tokens of B sequences need at most, and workgroups find their sequence in `offsets`.
//   pages (pages, kv_heads, page, D)     token p of sequence s: page table[s][p / page], place p % page
#pragma once
#include "cats_kv8.h"

namespace cats {

// The last of the n entries 0 .. n - 1 whose base is at most x, base(0) taken to be: 64 candidates a trip to memory.  Bases ascend; where they do not,
// the result is some entry.  Uniform over the wave.
template <class B>
__device__ __forceinline__ int find_last(int n, long long x, B base) {
  const int lane = threadIdx.x & (kWave - 1);
  int lo = 0;
  while (n > 1) {
    const int step = (n + kWave - 1) / kWave;
    const bool in = (long long)lane * step < n;
    const uint64_t below = __ballot(in && base(lo + (in ? lane * step : 0)) <= x);
    const int last = below ? 63 - __builtin_clzll(below) : 0;
    lo += last * step;
    n = min(step, n - last * step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

struct Packed {
  const int64_t* offsets;  // B + 1
  int B, N;
};
__device__ __forceinline__ int packed_at(const Packed& p, int s) {
  const long long o = p.offsets[s];
  return (int)(o < 0 ? 0 : o > p.N ? p.N : o);
}
// The sequence of token t, -1 if it is nobody's.
__device__ __forceinline__ int packed_row(const Packed& p, int t) {
  const int s = find_last(p.B + 1, t, [&](int i) { return (long long)packed_at(p, i); });
  return s == p.B || packed_at(p, s) > t || packed_at(p, s + 1) <= t ? -1 : s;
}

struct Pool {
  uint16_t* k;
  uint16_t* v;
  const int32_t* table;
  long long table_stride;
  int heads, page_log, pages, width;
};

// ---- storing ----------------------------------------------------------------------------------------------------------------------

struct PagedAppendArgs {
  const uint16_t* q;  // (N, heads, D) in elements: strides of a token and a head
  const uint16_t* k;
  const uint16_t* v;
  long long q_tok, q_head, k_tok, k_head, v_tok, v_head;
  uint16_t* q_out;  // (N, heads, D)
  Packed seq;
  const int64_t* start;
  const void* cos;  // (positions, rot)
  const void* sin;
  int rot, positions;
  Pool pool;
  int heads, per;  // per: tokens of a workgroup, at most kAppendTokens
};

// x' = x cos + rot(x) sin in 32 bits, rounded once; v as it is.  Bound by memory: every number is read once and written once (8 prompts of 32 heads over 32 and 2000 tokens,
// 630 MB, 144 us, 4.4 TB/s, where a copy of 1 GiB reaches 5.1; stores past the caches gave the same, and the next token's loads before this one's stores 145).
// A head of a token is D / 16 units of two vectors: of what is rotated elements 8 u .. + 7 and those rot / 2 behind, of the rest sixteen in order, so that a thread has
// both halves of what it turns.  A thread has one unit of a workgroup's tokens: up to eight where there are many, so that finding their places is paid once, and one where
// there are few (1 token 5.5 us, 64 tokens 5.4, which is a launch).
constexpr int kAppendTokens = 8;
template <class DT, int D, bool WIDE>  // WIDE: rotary tables in float
__global__ __launch_bounds__(512) void paged_append_kernel(PagedAppendArgs p) {
  constexpr int U = D / 16;
  __shared__ long long s_place[kAppendTokens];  // element of the pool's head 0; -1: not stored
  __shared__ int s_pos[kAppendTokens];          // -1: bad, -2: nobody's
  const int t0 = blockIdx.x * p.per, n = min(p.per, p.seq.N - t0);
  for (int i = threadIdx.x / kWave; i < n; i += blockDim.x / kWave) {
    const int s = packed_row(p.seq, t0 + i);
    if (threadIdx.x % kWave == 0) {
      long long place = -1;
      int pos = -2;
      if (s >= 0) {
        const long long at = p.start[s] + (t0 + i - packed_at(p.seq, s));
        pos = -1;
        if (at >= 0 && at < (long long)p.pool.width << p.pool.page_log && (p.rot == 0 || at < p.positions)) {
          const int page = p.pool.table[s * p.pool.table_stride + (at >> p.pool.page_log)];
          if (page >= 0 && page < p.pool.pages) {
            place = ((((long long)page * p.pool.heads) << p.pool.page_log) + (at & ((1 << p.pool.page_log) - 1))) * D;
            pos = (int)at;
          }
        }
      }
      s_place[i] = place;
      s_pos[i] = pos;
    }
  }
  __syncthreads();
  const int units = (p.heads + 2 * p.pool.heads) * U, unit = blockIdx.y * blockDim.x + threadIdx.x;
  if (unit >= units) return;
  const int head = unit / U, u = unit % U, kh = head - p.heads, vh = kh - p.pool.heads;
  const bool is_q = kh < 0, is_v = vh >= 0, turned = !is_v && 16 * u < p.rot;
  const int d0 = turned ? 8 * u : 16 * u, d1 = turned ? 8 * u + p.rot / 2 : 16 * u + 8;
  const uint16_t* from = is_q ? p.q + head * p.q_head : is_v ? p.v + vh * p.v_head : p.k + kh * p.k_head;
  const long long step = is_q ? p.q_tok : is_v ? p.v_tok : p.k_tok;
  uint16_t* to = is_q ? p.q_out + (long long)head * D : (is_v ? p.pool.v : p.pool.k) + ((long long)(is_v ? vh : kh) << p.pool.page_log) * D;
  for (int i = 0; i < n; i++) {
    const int t = t0 + i, pos = s_pos[i];
    if (pos < 0) {
      if (is_q) {
        const uint32_t w = pos == -2 ? 0u : DT::fromf(NAN) * 0x10001u;
        uint16_t* out = to + (long long)t * p.heads * D;
        *(u32x4*)(out + d0) = u32x4{w, w, w, w};
        *(u32x4*)(out + d1) = u32x4{w, w, w, w};
      }
      continue;
    }
    u32x4 a = load_stream((const u32x4*)(from + t * step + d0)), b = load_stream((const u32x4*)(from + t * step + d1));
    if (turned) {
      float c0[8], c1[8], s0[8], s1[8];
      const long long at = (long long)pos * p.rot;
      auto row = [&](const void* table, int d, float* f) {
        if constexpr (WIDE) {
          const f32x4 x = *(const f32x4*)((const float*)table + at + d), y = *(const f32x4*)((const float*)table + at + d + 4);
#pragma unroll
          for (int e = 0; e < 4; e++) f[e] = x[e], f[4 + e] = y[e];
        } else {
          const u32x4 x = *(const u32x4*)((const uint16_t*)table + at + d);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const uint32_t w = x[e];
            f[2 * e] = DT::tof((uint16_t)w), f[2 * e + 1] = DT::tof((uint16_t)(w >> 16));
          }
        }
      };
      row(p.cos, d0, c0);
      row(p.cos, d1, c1);
      row(p.sin, d0, s0);
      row(p.sin, d1, s1);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const uint32_t wa = a[e], wb = b[e];
        const float al = DT::tof((uint16_t)wa), ah = DT::tof((uint16_t)(wa >> 16)), bl = DT::tof((uint16_t)wb), bh = DT::tof((uint16_t)(wb >> 16));
        a[e] = DT::pack(fmaf(al, c0[2 * e], -bl * s0[2 * e]), fmaf(ah, c0[2 * e + 1], -bh * s0[2 * e + 1]));
        b[e] = DT::pack(fmaf(bl, c1[2 * e], al * s1[2 * e]), fmaf(bh, c1[2 * e + 1], ah * s1[2 * e + 1]));
      }
    }
    uint16_t* out = to + (is_q ? (long long)t * p.heads * D : s_place[i]);
    *(u32x4*)(out + d0) = a;
    *(u32x4*)(out + d1) = b;
  }
}

}  // namespace cats
