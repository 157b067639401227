// Attention of packed tokens over keys and values of the call, or of pages (16-bit models).
#pragma once
#include "cats_paged.h"

namespace cats {

struct PackedAttnArgs {
  const uint16_t* q;  // (N, heads, D) in elements: strides of a token and a head
  long long q_tok, q_head;
  uint16_t* out;      // (N, heads, D)
  Packed seq;
  // pages
  const int64_t* start;
  Pool pool;
  const int64_t* shared;
  int shared_step, members;  // sequences of a group
  // or keys and values of the call
  const uint16_t* k;  // (M, kv_heads, D)
  const uint16_t* v;
  long long k_tok, k_head, v_tok, v_head;
  Packed keys;
  float scale;        // log2(e) * the softmax's scale
  int kv_heads, group;  // group: query heads of a cached head
  int window;         // keys that a query sees, at most; 0: all
  int slots;
};

// Row r of a (sequence, cached head) pair is head r % group of token r / group, and a workgroup has up to ROWS of them.  Which ones it finds by its slot: set i has the
// slots from  first token of it * group / ROWS + i  on, which is room enough for any lengths.  Set 0 are the tokens before the first sequence, set i sequence i - 1,
// and the last one the tokens behind the last; a call has packed_slots() of them.
inline int packed_slots(int N, int sets, int group, int rows) { return (int)((long long)N * group / rows) + sets; }
struct PackedRows {
  int set, tok0, n, r0;  // n: tokens of the set; r0: the workgroup's first row of it
  long long word;        // what the caller asked for of the set
};
// start_of(i): first token of set i (i = sets: N); word(i): something of set i that is worth a trip to memory beside it.
template <int ROWS, class S, class W>
__device__ __forceinline__ PackedRows packed_rows(int sets, int slot, int group, S start_of, W word) {
  const int lane = threadIdx.x & (kWave - 1);
  int lo = 0, n = sets;
  auto base = [&](int i, int tok) { return (long long)tok * group / ROWS + i; };
  while (n >= kWave) {
    const int step = (n + kWave - 1) / kWave;
    const bool in = lane * step < n;
    const int i = lo + (in ? lane * step : 0);
    const uint64_t below = __ballot(in && base(i, start_of(i)) <= slot);
    const int last = below ? 63 - __builtin_clzll(below) : 0;
    lo += last * step;
    n = min(step, n - last * step);
  }
  const int i = lo + min(lane, n), tok = start_of(i);  // one more than the candidates: where the last of them ends
  const long long w = word(min(i, sets - 1));
  const uint64_t below = __ballot(lane < n && base(i, tok) <= slot);
  const int last = below ? 63 - __builtin_clzll(below) : 0;
  PackedRows r;
  r.set = lo + last;
  r.tok0 = __builtin_amdgcn_readlane(tok, last);
  r.n = max(0, __builtin_amdgcn_readlane(tok, last + 1) - r.tok0);
  const long long first = slot - base(r.set, r.tok0);
  r.r0 = first < 0 || first > INT_MAX / ROWS ? INT_MAX : (int)first * ROWS;
  r.word = (long long)((unsigned)__builtin_amdgcn_readlane((int)w, last) | (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(w >> 32), last) << 32);
  return r;
}

template <class T>
__device__ __forceinline__ T load_uniform(const T* p) {  // through the scalar cache: what nothing writes during the launch
  return *(const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

// Pages that sequence s, whose first new token is at `start`, reads through the first one of its group: those that lie wholly within what is shared.
__device__ __forceinline__ int shared_pages(const PackedAttnArgs& p, int s, int start) {
  const long long n = load_uniform(p.shared + s / p.members * p.shared_step);
  return (int)(n < 0 ? 0 : n > start ? start : n) >> p.pool.page_log;
}

__device__ __forceinline__ uint16_t* packed_out(const PackedAttnArgs& p, int tok0, int c, int r, int D) {
  const int t = r / p.group;
  return p.out + ((long long)(tok0 + t) * p.kv_heads * p.group + c * p.group + (r - t * p.group)) * D;
}
// Rows r0 .. r0 + count - 1 of `rows` all alike.
template <int D>
__device__ __forceinline__ void packed_fill(const PackedAttnArgs& p, int tok0, int c, int r0, int count, int rows, uint32_t w) {
  for (int i = threadIdx.x; i < count * (D / 8); i += blockDim.x) {
    const int r = r0 + i / (D / 8);
    if (r < rows) ((u32x4*)packed_out(p, tok0, c, r, D))[i % (D / 8)] = u32x4{w, w, w, w};
  }
}

// Four tokens of sixteen elements in LDS turned round: lane i of each sixteen gives the place of elements 4 (i % 4) .. + 3 of token i / 4, and gets the four tokens of
// element i.
__device__ __forceinline__ u32x2 read_turned(const char* at) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at));
}

// Many tokens: 128 rows of queries a workgroup, 32 a wave, over tiles of 64 keys that come into LDS straight from memory, the next one while the weights of
// this one are computed.
//   S^T = K . Q^T   v_mfma_f32_32x32x16; tile u, row 8 a + 4 h + i of the result: token 32 u + 8 a + 4 h + i, in lanes of half h = lane / 32; columns are queries
//   O^T += V^T . P  operand of step v (16 tokens): tokens 16 v + 4 h + (0 .. 3) and 8 behind them, those whose weights the lane has; V comes turned round out of LDS
// Rows of LDS are 16-byte pieces, exchanged within a row so that lanes that read together find different banks.
constexpr int kTileKeys = 64, kTileRows = 128;
template <int D> __device__ __forceinline__ constexpr int tile_swap_k(int t) {
  return D >= 128 ? t & 15 : D == 64 ? t >> 1 & 7 : t >> 2 & 3;
}
template <int D> __device__ __forceinline__ constexpr int tile_swap_v(int t) {
  return D >= 128 ? (t & 3) * 4 : D == 64 ? (t >> 1 & 1) * 4 : 0;
}
template <class DT, int D, bool PAGED>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void packed_attn_tiles_kernel(PackedAttnArgs p) {
  constexpr int ROWS = kTileRows, C = D / 16, NW = D / 32, PK = D / 8, kVecs = kTileKeys * PK;
  constexpr int LOADS = PK / 4, STEP = kWave / PK;  // a wave's loads of a tile of keys (16 tokens), and tokens a load
  typedef Kv<DT> F;
  __shared__ u32x4 s_kv[2][2][kVecs];  // [buffer][keys, values]
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 31, h = lane >> 5;
  const int c = blockIdx.x % p.kv_heads, slot = p.slots - 1 - blockIdx.x / p.kv_heads;
  const int B = p.seq.B;
  const PackedRows at = packed_rows<ROWS>(B + 2, slot, p.group, [&](int i) { return i == 0 ? 0 : i > B + 1 ? p.seq.N : packed_at(p.seq, i - 1); },
                                          [&](int i) -> long long {
                                            const int s = min(max(i - 1, 0), B - 1);
                                            if constexpr (PAGED) return p.start[s];
                                            return (long long)packed_at(p.keys, s) << 32 | packed_at(p.keys, s + 1);
                                          });
  const int s = at.set - 1, n = at.n, rows = n * p.group, r0 = at.r0, tok0 = at.tok0;
  if (r0 >= rows) return;
  const bool live = s >= 0 && s < B;
  int pos0 = 0;  // position of the sequence's first query
  const int32_t *table = nullptr, *common = nullptr;  // entries of pages, and of the first `alike` of them, which a group shares
  int alike = 0;
  const uint16_t *k_base, *v_base;
  bool ok = true;
  if constexpr (PAGED) {
    ok = at.word >= 0 && at.word <= ((long long)p.pool.width << p.pool.page_log) - n;
    pos0 = ok ? (int)at.word : 0;
    table = common = p.pool.table + s * p.pool.table_stride;
    if (p.shared && live) {
      alike = shared_pages(p, s, pos0);
      common = p.pool.table + s / p.members * p.members * p.pool.table_stride;
    }
    k_base = p.pool.k + ((long long)c << p.pool.page_log) * D;
    v_base = p.pool.v + ((long long)c << p.pool.page_log) * D;
  } else {
    const int key0 = (int)(at.word >> 32), key1 = (int)at.word;
    pos0 = key1 - key0 - n;
    k_base = p.k + key0 * p.k_tok + c * p.k_head;
    v_base = p.v + key0 * p.v_tok + c * p.v_head;
  }
  const int end = pos0 + n;  // keys
  const int pos_lo = pos0 + r0 / p.group, pos_hi = pos0 + (min(r0 + ROWS, rows) - 1) / p.group;
  if (!live || !ok || pos_hi < 0) return packed_fill<D>(p, tok0, c, r0, ROWS, rows, live && !ok ? DT::fromf(NAN) * 0x10001u : 0u);
  const int tile_lo = p.window ? max(0, pos_lo - p.window + 1) / kTileKeys : 0, tile_hi = pos_hi / kTileKeys;

  const int mine = r0 + 32 * wave + m, row = min(mine, rows - 1), tok = row / p.group, pos = pos0 + tok;
  const int first = p.window ? pos - p.window : -1;  // the query sees first + 1 .. pos
  const int hi_pos = pos0 + min(r0 + 32 * wave + 31, rows - 1) / p.group, lo_pos = pos0 + min(r0 + 32 * wave, rows - 1) / p.group;
  u32x4 qf[C];
  {
    const uint16_t* q = p.q + (tok0 + tok) * p.q_tok + (c * p.group + row - tok * p.group) * p.q_head;
#pragma unroll
    for (int i = 0; i < C; i++) qf[i] = *(const u32x4*)(q + 16 * i + 8 * h);
  }

  // A wave brings sixteen tokens of a tile.  Lane l of load j writes piece 64 j + l of them and reads what belongs there; what is exchanged goes by bits of the
  // token, so load j differs from load 0 by constants, and reads of LDS differ by constants too.
  const unsigned t_lane = lane / PK;
  unsigned k_piece = ((lane % PK) ^ tile_swap_k<D>(t_lane)) * 16, v_piece = ((lane % PK) ^ tile_swap_v<D>(t_lane)) * 16;
  unsigned k_at = (m * PK + (h ^ tile_swap_k<D>(m))) * 16;
  unsigned v_at = ((4 * h + (m >> 2 & 3)) * PK + ((2 * (m >> 4) + (m >> 1 & 1)) ^ tile_swap_v<D>(m >> 2 & 3))) * 16 + 8 * (m & 1);
  asm volatile("" : "+v"(k_at), "+v"(v_at));
  const unsigned k_row = PAGED ? D * 2 : (unsigned)p.k_tok * 2, v_row = PAGED ? D * 2 : (unsigned)p.v_tok * 2;  // bytes
  unsigned none = 0, none1 = 0;  // bit i: tokens 16 i .. + 15 of the tile, and of the next one, have no page
  auto bring = [&](int tile, int buf) {
    u32x4 *kt = s_kv[buf][0] + 16 * wave * PK, *vt = s_kv[buf][1] + 16 * wave * PK;
    unsigned kp = k_piece, vp = v_piece;
    asm volatile("" : "+v"(kp), "+v"(vp));  // not a register for every load over the loop
    auto load = [&](const char* from, unsigned lane_at, u32x4* to) {
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + (size_t)lane_at), (__attribute__((address_space(3))) void*)to, 16, 0, 0);
    };
    auto loads = [&](const char* kf, const char* vf) {
#pragma unroll
      for (int j = 0; j < LOADS; j++) {
        load(kf + (size_t)j * STEP * k_row, t_lane * k_row + (kp ^ (16u * tile_swap_k<D>(STEP * j))), kt + j * kWave);
        load(vf + (size_t)j * STEP * v_row, t_lane * v_row + (vp ^ (16u * tile_swap_v<D>(STEP * j))), vt + j * kWave);
      }
    };
    const int t0 = tile * kTileKeys + 16 * wave;
    if constexpr (PAGED) {
      const int most = (end - 1) >> p.pool.page_log;
      int mine = 0;
      none1 = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int page = min((tile * kTileKeys + 16 * i) >> p.pool.page_log, most), id = load_uniform((page < alike ? common : table) + page);
        const bool in = (unsigned)id < (unsigned)p.pool.pages;
        none1 |= in ? 0u : 1u << i;
        if (i == wave) mine = in ? id : 0;
      }
      const long long place = ((((long long)mine * p.pool.heads) << p.pool.page_log) + (t0 & ((1 << p.pool.page_log) - 1))) * D;
      loads((const char*)(k_base + place), (const char*)(v_base + place));
    } else if (t0 + 16 <= end) {
      loads((const char*)(k_base + t0 * p.k_tok), (const char*)(v_base + t0 * p.v_tok));
    } else {  // tokens behind the last one are that one again
#pragma unroll
      for (int j = 0; j < LOADS; j++) {
        const long long t = min(t0 + (int)t_lane + STEP * j, end - 1);
        load((const char*)(k_base + t * p.k_tok), kp ^ (16u * tile_swap_k<D>(STEP * j)), kt + j * kWave);
        load((const char*)(v_base + t * p.v_tok), vp ^ (16u * tile_swap_v<D>(STEP * j)), vt + j * kWave);
      }
    }
  };

  float top = -FLT_MAX, sum = 0.f;
  bool far = false;  // whether some query's scores are
  f32x16 o[NW];
  auto zeros = [] {
    f32x16 z;
#pragma unroll
    for (int e = 0; e < 16; e++) z[e] = 0.f;
    return z;
  };
  // weights of a tile from its scores, as operands
  auto weigh = [&](f32x16 (&s)[2], u32x4 (&pf)[4]) {
    float mx = s[0][0];
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int e = 0; e < 16; e++) mx = fmaxf(mx, s[u][e]);
    mx = max_mod32(mx);
    const float now = fmaxf(top, kv_scaled(mx, p.scale));
    if (__any(now > top + F::SLACK)) {
      const float keep = __builtin_amdgcn_exp2f(top - now);
      sum *= keep;
#pragma unroll
      for (int w = 0; w < NW; w++) o[w] *= keep;
      top = now;
      far = __any(kv_far(top));
    }
    float off = F::HEAD - F::SLACK - top;
    if (far) {
      const float ref = fmaxf(mx, -FLT_MAX);
      off = fminf(kv_scaled(mx, p.scale) - top, F::SLACK) + F::HEAD - F::SLACK;
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
        s[u][e] = __builtin_amdgcn_exp2f(fmaf(s[u][e], p.scale, off));
        add += s[u][e];
      }
#pragma unroll
      for (int v = 0; v < 2; v++)
#pragma unroll
        for (int e = 0; e < 4; e++) pf[2 * u + v][e] = DT::pack(s[u][8 * v + 2 * e], s[u][8 * v + 2 * e + 1]);
    }
    sum += add;
  };
  // whether the query sees a key: all of the tile's, in turn
  auto each_seen = [&](int tile, auto f) {
    const int most = pos - tile * kTileKeys - 4 * h, least = max(most, -kTileKeys) - (p.window ? p.window : INT_MAX / 2);
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const int t = 32 * u + 8 * (e / 4) + e % 4;
        f(u, e, t <= most && t > least);
      }
  };
  // A masked weight is 0, but 0 times a NaN is not.  So where a sum is not finite at the end, the tiles are gone over again: once with numbers of V that are not
  // finite set to 0, and once to count, for each element, those that a query sees.
  enum { PLAIN, CLEAN, COUNT };
  // one tile; PART: some query of the wave does not see all of it
  auto take = [&](auto PART, auto AGAIN, int mode, int tile, int buf, auto behind) {
    f32x16 s[2] = {zeros(), zeros()};
    const char *kt = (const char*)s_kv[buf][0], *vt = (const char*)s_kv[buf][1];
#pragma unroll
    for (int i = 0; i < C; i++)
#pragma unroll
      for (int u = 0; u < 2; u++) s[u] = Mma32<DT>::run(*(const u32x4*)(kt + (k_at ^ 32u * i) + 32 * u * PK * 16), qf[i], s[u]);
    // All values are asked for before the next tile, which a read of LDS behind its loads would wait for.  (Heads of 256 elements do not have the registers.)
    constexpr bool ASK = D <= 128;
    auto values = [&](int w, int v) {
      const u32x2 lo = read_turned(vt + (v_at ^ 64u * w) + 16 * v * PK * 16), hi = read_turned(vt + (v_at ^ 64u * w) + (16 * v + 8) * PK * 16);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    u32x4 x[ASK ? 4 * NW : 1];
    if constexpr (ASK) {
#pragma unroll
      for (int i = 0; i < 4 * NW; i++) x[i] = values(i % NW, i / NW);
      __builtin_amdgcn_sched_barrier(0);
      behind();
      __builtin_amdgcn_sched_barrier(0);
    }
    if (PAGED && none) {
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int e = 0; e < 16; e++)
          if (none >> (2 * u + e / 8) & 1) s[u][e] = NAN;
    }
    if constexpr (PART) each_seen(tile, [&](int u, int e, bool seen) { s[u][e] = seen ? s[u][e] : -INFINITY; });
    u32x4 pf[4];
    if (!AGAIN || mode == CLEAN) {
      weigh(s, pf);
    }
    if constexpr (AGAIN) {
      if (mode == COUNT) {
        each_seen(tile, [&](int u, int e, bool seen) { s[u][e] = seen ? 1.f : 0.f; });
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) pf[i][e] = DT::pack(s[i / 2][8 * (i % 2) + 2 * e], s[i / 2][8 * (i % 2) + 2 * e + 1]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4 * NW; i++) {
      u32x4 y = ASK ? x[ASK ? i : 0] : values(i % NW, i / NW);
      if constexpr (AGAIN) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t bad = kv_nan16<DT>(y[e]);
          y[e] = mode == COUNT ? bad * F::kOne : y[e] & ~(bad * 0xffffu);
        }
      }
      o[i % NW] = Mma32<DT>::run(y, pf[i / NW], o[i % NW]);
    }
    if constexpr (!ASK) behind();
  };

  // tiles that a window cuts, tiles that all of the workgroup's queries see, tiles that hold some of their own keys
  const int cut = p.window && pos_hi >= p.window ? (pos_hi - p.window) / kTileKeys : -1, own = (pos_lo + 1) / kTileKeys;  // last and first of them
  auto sweep = [&](auto AGAIN, int mode) {
#pragma unroll
    for (int w = 0; w < NW; w++) o[w] = zeros();
    int tile = tile_lo, buf = 0;
    bring(tile, 0);
    auto arrive = [&] {
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): in LDS
      none = none1;
      lds_barrier();
    };
    arrive();
    auto run = [&](auto PART, int to) {
      for (; tile <= to; tile++, buf ^= 1) {
        take(PART, AGAIN, mode, tile, buf, [&] { bring(min(tile + 1, tile_hi), buf ^ 1); });
        arrive();
      }
    };
    if constexpr (AGAIN) {
      run(std::true_type(), tile_hi);
    } else {
      run(std::true_type(), min(cut, tile_hi));
      run(std::false_type(), min(own - 1, tile_hi));
      run(std::true_type(), tile_hi);
    }
  };
  auto store = [&](auto value) {
    if (mine >= rows) return;
    uint16_t* out = packed_out(p, tok0, c, mine, D);
#pragma unroll
    for (int w = 0; w < NW; w++)
#pragma unroll
      for (int a = 0; a < 4; a++) value(out + 32 * w + 8 * a + 4 * h, w, a);
  };
  sweep(std::false_type(), PLAIN);
  float odd = 0.f;
#pragma unroll
  for (int w = 0; w < NW; w++)
#pragma unroll
    for (int e = 0; e < 16; e++) odd = fmaf(o[w][e], 0.f, odd);
  const bool again = __syncthreads_or(odd != 0.f);  // NaN is
  if (again) {
    top = -FLT_MAX, sum = 0.f, far = false;
    sweep(std::true_type(), CLEAN);
  }
  sum += __shfl_xor(sum, 32, kWave);
  const float f = pos < 0 ? 0.f : 1.f / sum;
  store([&](uint16_t* out, int w, int a) {
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = pos < 0 ? 0.f : o[w][4 * a + e] * f;
    *(u32x2*)out = u32x2{DT::pack(x[0], x[1]), DT::pack(x[2], x[3])};
  });
  if (again) {
    sweep(std::true_type(), COUNT);
    store([&](uint16_t* out, int w, int a) {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (o[w][4 * a + e] > 0.f) out[e] = DT::fromf(NAN);
    });
  }
}

}  // namespace cats
