// Attention of packed tokens over keys and values of the call, or of pages (16-bit models).
#pragma once
#include "cats_paged.h"

namespace cats {

// n / d for n below 2^31, by a product: 2^(31 + shift) / d rounded up has 32 bits, and is near enough for 31 of n.
struct Divisor {
  unsigned mul;
  int shift;
  __device__ __forceinline__ int operator()(int n) const { return (int)(__umulhi((unsigned)n << 1, mul) >> shift); }
};
inline Divisor divisor(int d) {
  int shift = 0;
  while ((1ll << shift) < d) shift++;
  return {(unsigned)(((1ull << (31 + shift)) + d - 1) / d), shift};
}

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
  int cus;
  int slots;          // of the launch
  // Keys that are split: what the splits give is in `part`: [split][token, head][D] sums and, behind them, [split][token, head][2] largest exponent and sum of
  // weights.  The first group_splits are of the keys that a group of sequences shares, the others of a sequence's own.
  float* part;
  int splits, group_splits;
  int group_blocks;  // of the launch, without kv_heads: those of shared keys, which come first
  Divisor by_group, by_heads, by_members, by_splits, by_group_splits;  // group, kv_heads ..
};

// Row r of a (sequence, cached head) pair is head r % group of token r / group, and a workgroup has up to ROWS of them.  Which ones it finds by its slot: set 0 are the
// tokens before the first sequence, set i sequence i - 1, and the last one the tokens behind the last.  Up to 255 of them, their slots come one
// behind the other and those that nobody needs behind them all; else set i has those from  first token of it * group / ROWS + i  on.  packed_slots() are enough
// for any lengths.  (With gaps everywhere the workgroups that have work are spread unevenly over the CUs: a step of 32 sequences took 88 us for 72.)
inline int packed_slots(int N, int sets, int group, int rows) { return (int)((long long)N * group / rows) + sets; }
constexpr int kPackedScan = 4;  // sets that a lane has, at most
struct PackedRows {
  int set, tok0, n, r0;  // n: tokens of the set; r0: the workgroup's first row of it
  long long word;        // what the caller asked for of the set
};
__device__ __forceinline__ int sum_up_to(int v) {  // of the lanes up to this one
  auto step = [&](auto ctrl, auto rows) { v += __builtin_amdgcn_update_dpp(0, v, decltype(ctrl)::value, decltype(rows)::value, 0xf, false); };
  step(std::integral_constant<int, 0x111>(), std::integral_constant<int, 0xf>());  // row_shr
  step(std::integral_constant<int, 0x112>(), std::integral_constant<int, 0xf>());
  step(std::integral_constant<int, 0x114>(), std::integral_constant<int, 0xf>());
  step(std::integral_constant<int, 0x118>(), std::integral_constant<int, 0xf>());
  step(std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>());  // row_bcast:15
  step(std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xc>());  // row_bcast:31
  return v;
}
// slot_of(n): the workgroup's slot, of n that may have work.  start_of(i): first token of set i (i = sets: N); word(i): something of set i that is worth a trip to memory
// beside it.
template <int ROWS, class O, class S, class W>
__device__ __forceinline__ PackedRows packed_rows(int sets, int slots, int group, O slot_of, S start_of, W word) {
  const int lane = threadIdx.x & (kWave - 1);
  PackedRows r;
  long long w, first;
  int last;
  auto scan = [&](auto chunks) {
    constexpr int C = decltype(chunks)::value;
    int tok[C], n[C], upto[C], all = 0;
    long long words[C];
#pragma unroll
    for (int i = 0; i < C; i++) {
      tok[i] = n[i] = words[i] = 0;
      if (i == 0 || i * kWave < sets) {
        const int set = i * kWave + lane;
        tok[i] = start_of(min(set, sets));
        n[i] = max(0, start_of(min(set + 1, sets)) - tok[i]);
        words[i] = word(min(set, sets - 1));
      }
    }
#pragma unroll
    for (int i = 0; i < C; i++) {
      upto[i] = all;
      if (i == 0 || i * kWave < sets) {
        upto[i] += sum_up_to((n[i] * group + ROWS - 1) / ROWS);
        all = __builtin_amdgcn_readlane(upto[i], kWave - 1);
      }
    }
    const int slot = slot_of(all);
    int at = 0, toks = 0, ns = 0, before = 0;  // of the chunk that it is in, which the last one is that begins at or before it
    w = 0, last = 0;
#pragma unroll
    for (int i = C - 1; i >= 0; i--) {
      const uint64_t above = __ballot(upto[i] > slot);
      if (above) {
        last = __builtin_ctzll(above), at = i, toks = tok[i], ns = n[i], w = words[i];
        before = __builtin_amdgcn_readlane(upto[i], last) - (__builtin_amdgcn_readlane(n[i], last) * group + ROWS - 1) / ROWS;
      }
    }
    r.set = at * kWave + last;
    r.tok0 = __builtin_amdgcn_readlane(toks, last);
    r.n = __builtin_amdgcn_readlane(ns, last);
    first = slot < all ? slot - before : INT_MAX;
  };
  if (sets < kWave) {
    scan(std::integral_constant<int, 1>());
  } else if (sets < kPackedScan * kWave) {
    scan(std::integral_constant<int, kPackedScan>());
  } else {
    const int slot = slot_of(slots);
    int lo = 0, n = sets;
    auto base = [&](int i, int tok) { return (long long)tok * group / ROWS + i; };
    while (n >= kWave) {
      const int step = (n + kWave - 1) / kWave;
      const bool in = lane * step < n;
      const int i = lo + (in ? lane * step : 0);
      const uint64_t below = __ballot(in && base(i, start_of(i)) <= slot);
      const int at = below ? 63 - __builtin_clzll(below) : 0;
      lo += at * step;
      n = min(step, n - at * step);
    }
    const int i = lo + min(lane, n), tok = start_of(i);  // one more than the candidates: where the last of them ends
    w = word(min(i, sets - 1));
    const uint64_t below = __ballot(lane < n && base(i, tok) <= slot);
    last = below ? 63 - __builtin_clzll(below) : 0;
    r.set = lo + last;
    r.tok0 = __builtin_amdgcn_readlane(tok, last);
    r.n = max(0, __builtin_amdgcn_readlane(tok, last + 1) - r.tok0);
    first = slot - base(r.set, r.tok0);
  }
  for (int* i : {&r.set, &r.tok0, &r.n, &last}) *i = __builtin_amdgcn_readfirstlane(*i);  // (the compiler does not see that these are the same in all lanes)
  r.r0 = __builtin_amdgcn_readfirstlane(first < 0 || first > INT_MAX / ROWS ? INT_MAX : (int)first * ROWS);
  r.word = (long long)((unsigned)__builtin_amdgcn_readlane((int)w, last) | (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(w >> 32), last) << 32);
  return r;
}

template <class T>
__device__ __forceinline__ T load_uniform(const T* p) {  // through the scalar cache: what nothing writes during the launch
  return *(const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

// Pages that sequence s, whose first new token is at `start`, reads through the first one of its group: those that lie wholly within what is shared.
__device__ __forceinline__ int shared_pages(const PackedAttnArgs& p, int s, int start) {
  const long long n = load_uniform(p.shared + p.by_members(s) * p.shared_step);
  return (int)(n < 0 ? 0 : n > start ? start : n) >> p.pool.page_log;
}

__device__ __forceinline__ uint16_t* packed_out(const PackedAttnArgs& p, int tok0, int c, int r, int D) {
  const int t = p.by_group(r);
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

// A workgroup's share of attention whose keys are split: up to ROWS rows of a sequence over a part of its own keys, or of a group of sequences over a part of those that
// they share.
struct PackedPart {
  int set, tok0, n, r0, rows, here;  // tokens of the set; the first row, all of the set and those here
  bool common, live, ok;
  int split, splits;
  int s0, alike, start0;  // first sequence; of own keys: pages that come before them, which its group shares, and the first position
  long long at;           // in units of rows, where its results go in `part`
};
__device__ __forceinline__ long long packed_all_rows(const PackedAttnArgs& p) { return (long long)p.seq.N * p.kv_heads * p.group; }
template <int ROWS>
__device__ __forceinline__ PackedPart packed_part(const PackedAttnArgs& p, int block) {
  PackedPart s;
  const int B = p.seq.B, N = p.seq.N;
  s.common = block < p.group_blocks;
  if (!s.common) block -= p.group_blocks;
  s.splits = s.common ? p.group_splits : p.splits;
  const int slot = s.common ? p.by_group_splits(block) : p.by_splits(block), members = s.common ? p.members : 1, sets = (s.common ? p.by_members(B) : B) + 2;
  s.split = block - slot * s.splits;
  const PackedRows at = packed_rows<ROWS>(sets, INT_MAX, p.group, [&](int) { return slot; }, [&](int i) { return i == 0 ? 0 : i == sets ? N : packed_at(p.seq, (i - 1) * members); },
                                          [&](int i) -> long long { return p.start[min(max(i - 1, 0) * members, B - 1)]; });
  s.set = at.set, s.tok0 = at.tok0, s.n = at.n, s.r0 = at.r0;
  s.rows = at.n * p.group, s.here = min(ROWS, s.rows - at.r0);
  s.live = at.set >= 1 && at.set < sets - 1;
  s.s0 = s.live ? (at.set - 1) * members : 0;
  s.at = ((s.common ? 0 : p.group_splits) + s.split) * packed_all_rows(p);
  s.ok = true;
  s.alike = s.start0 = 0;
  if (!s.common && s.live) {
    s.ok = at.word >= 0 && at.word <= ((long long)p.pool.width << p.pool.page_log) - at.n;
    s.start0 = s.ok ? (int)at.word : 0;
    if (p.shared) s.alike = shared_pages(p, s.s0, s.start0);
  }
  return s;
}
__device__ __forceinline__ long long packed_row_at(const PackedAttnArgs& p, const PackedPart& s, int c, int r) {  // of (token, head)
  const int t = p.by_group(r);
  return (long long)(s.tok0 + t) * p.kv_heads * p.group + c * p.group + (r - t * p.group);
}
__device__ __forceinline__ float* packed_part_ml(const PackedAttnArgs& p, int D) { return p.part + (p.splits + p.group_splits) * packed_all_rows(p) * D; }
// Rows that see none of these keys, or (sum NaN) are of a sequence whose tokens do not lie in its pages.
template <class DT, int D>
__device__ __forceinline__ void packed_nothing(const PackedAttnArgs& p, const PackedPart& s, int c, float sum) {
  if (p.splits + p.group_splits == 1) return packed_fill<D>(p, s.tok0, c, s.r0, s.here, s.rows, sum == 0.f ? 0u : DT::fromf(NAN) * 0x10001u);
  if ((int)threadIdx.x < s.here) {
    float* ml = packed_part_ml(p, D) + 2 * (s.at + packed_row_at(p, s, c, s.r0 + threadIdx.x));
    ml[0] = -FLT_MAX;
    ml[1] = sum;
  }
}
// Keys lo .. hi that row r sees of these.
struct PackedKeys {
  int lo, hi;
};
__device__ __forceinline__ PackedKeys packed_keys(const PackedAttnArgs& p, const PackedPart& s, int r) {
  const int t = s.tok0 + p.by_group(r);
  if (!s.common) {
    const int pos = s.start0 + t - s.tok0;
    return {max(p.group_splits ? s.alike << p.pool.page_log : 0, p.window ? pos - p.window + 1 : 0), pos};
  }
  // the sequence among the group's: a token each, or looked for
  int b = s.s0 + min(t - s.tok0, p.members - 1);
  if (!__all(packed_at(p.seq, b) <= t && t < packed_at(p.seq, b + 1))) {
    int e = s.s0 + p.members;
    b = s.s0;
    for (int n = p.members; n > 1; n = (n + 1) / 2) {
      const int mid = (b + e) / 2;
      const bool in = mid > b && packed_at(p.seq, mid) <= t;
      b = in ? mid : b;
      e = in ? e : max(mid, b + 1);
    }
  }
  const long long start = p.start[b], room = (long long)p.pool.width << p.pool.page_log;
  const int first = packed_at(p.seq, b), n = packed_at(p.seq, b + 1) - first;
  if (!(start >= 0 && start <= room - n)) return {0, -1};
  const long long shared = p.shared[(s.set - 1) * p.shared_step];
  const int pos = (int)start + t - first, pages = (int)max(0ll, min(shared, start)) >> p.pool.page_log;
  return {p.window ? max(0, pos - p.window + 1) : 0, (pages << p.pool.page_log) - 1};
}
// Of all rows r0 .. r0 + ROWS - 1 that are here: the first key that any sees and the last one, and those that all see.
struct PackedBounds {
  int lo, hi, all_lo, all_hi;
};
__device__ __forceinline__ int least_of(int v) {
  auto step = [&](auto ctrl) { v = min(v, __builtin_amdgcn_update_dpp(v, v, decltype(ctrl)::value, 0xf, 0xf, false)); };
  step(std::integral_constant<int, 0xB1>());  // as in wave_sum
  step(std::integral_constant<int, 0x4E>());
  step(std::integral_constant<int, 0x141>());
  step(std::integral_constant<int, 0x140>());
  return min(min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)), min(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
template <int ROWS>
__device__ __forceinline__ PackedBounds packed_bounds(const PackedAttnArgs& p, const PackedPart& s) {
  if (!s.common) {  // both ends ascend with the row
    const PackedKeys a = packed_keys(p, s, s.r0), z = packed_keys(p, s, s.r0 + s.here - 1);
    return {__builtin_amdgcn_readfirstlane(a.lo), __builtin_amdgcn_readfirstlane(z.hi), __builtin_amdgcn_readfirstlane(z.lo), __builtin_amdgcn_readfirstlane(a.hi)};
  }
  int lo = INT_MAX, hi = -1, all_lo = 0, all_hi = INT_MAX;
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int i = 0; i < ROWS; i += kWave) {
    const PackedKeys k = packed_keys(p, s, s.r0 + min(lane + i, s.here - 1));
    if (k.lo <= k.hi) lo = min(lo, k.lo), hi = max(hi, k.hi);
    all_lo = max(all_lo, k.lo), all_hi = min(all_hi, k.hi);
  }
  return {least_of(lo), -least_of(-hi), -least_of(-all_lo), least_of(all_hi)};
}

// Where tokens of pages come from, sixteen at a time, which no page ends within.  Those outside lo .. hi, which nobody sees, are the nearest ones once more: their
// entries may be anything, and so may the places behind a sequence's last token.
struct PageRun {
  int from, id;  // first token that is read, and its entry
};
struct PageRows {
  const int32_t* table;
  const int32_t* common;  // of the first `alike` pages
  int alike, lo, hi;
};
__device__ __forceinline__ PageRows page_rows(const PackedAttnArgs& p, int s, int alike, int lo, int hi) {  // of sequence s
  const int32_t* table = p.pool.table + s * p.pool.table_stride;
  return {table, alike ? p.pool.table + p.by_members(s) * p.members * p.pool.table_stride : table, alike, lo, hi};
}
__device__ __forceinline__ PageRun page_run(const Pool& pool, const PageRows& rows, int t) {
  const int from = min(max(t, rows.lo & ~15), rows.hi & ~15), page = from >> pool.page_log;
  return {from, load_uniform((page < rows.alike ? rows.common : rows.table) + page)};
}
__device__ __forceinline__ bool page_none(const Pool& pool, const PageRun& run) { return (unsigned)run.id >= (unsigned)pool.pages; }
__device__ __forceinline__ long long page_place(const Pool& pool, const PageRun& run) {  // token of the pool's head 0
  return ((long long)(page_none(pool, run) ? 0 : run.id) * pool.heads << pool.page_log) + (run.from & ((1 << pool.page_log) - 1));
}

// Four tokens of sixteen elements in LDS turned round: lane i of each sixteen gives the place of elements 4 (i % 4) .. + 3 of token i / 4, and gets the four tokens of
// element i.
__device__ __forceinline__ u32x2 read_turned(const char* at) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at));
}

// Many tokens: 128 rows of queries a workgroup, 32 a wave, over tiles of 64 keys that come into LDS straight from memory.
//   S^T = K . Q^T   v_mfma_f32_32x32x16; tile u, row 8 a + 4 h + i of the result: token 32 u + 8 a + 4 h + i, in lanes of half h = lane / 32; columns are queries
//   O^T += V^T . P  operand of step v (16 tokens): tokens 16 v + 4 h + (0 .. 3) and 8 behind them, those whose weights the lane has; V comes turned round out of LDS
// Weights are rounded to the model's type, which the second product's operands have; scores, the largest of them, sums of weights (of the unrounded ones) and of values are 32
// bits.  The output is then off by 2.1e-3 to 2.3e-3 in bf16 and 2.7e-4 in fp16 (root of the mean square, relative), where weights in 32 bits and the output's own rounding give
// 1.6e-3 to 1.7e-3 and 2.0e-4.  Below 2^-21 of the largest, fp16 weights (which begin at 2^(HEAD - SLACK)) are steps of 2^-31 of it.
// So weights never leave their lane, and each number of a tile is read once out of LDS for 32 rows.  Rows of LDS are 16-byte pieces, exchanged within a row so that lanes
// that read together find different banks (no conflicts are counted).
// Bound by the matrix cores' and the vector units' power and issue: a tile and wave are 32 matrix and 150 other instructions, the weights of half a tile beside the products
// of the half before and the scores of the half behind.  8192 tokens of 32 heads over 8 in bf16 take 483 to 515 us (card by card), 1.07 to 1.14 PFLOP/s, where a product of
// 8192^3 reaches 1.25; with weights, scores and products one behind the other it was 536, with these side by side in whole tiles 515.  Two workgroups a CU (256 registers,
// 64 KiB of LDS): one alone needs 1.0 to 1.3 us a tile and two together 1.95, so what their first loads (4 us) and ends (2 to 3 us) take is hidden where there are
// enough of them: 2048 tokens of 32 heads, 512 workgroups of 2 to 32 tiles, take 47 to 50 us where the tiles alone are 33.
// Results leave sixteen bytes a lane, which two lanes put together (eight bytes each: 64 prompts of 128 tokens 52.2 us for 43.7).
// Tried: a ring of half tiles with a barrier for each (1.3 us a tile); operands read four ahead (no gain); all sequences' longest first (16 prompts to 1500 no gain, and
// 16 of 512 88 us for 65: more keys at once than a part of the chip's second cache holds).
constexpr int kTileKeys = 64, kTileRows = 128;
template <class DT> struct Limit { static constexpr float SUM = 0x1p15f; };  // 2^HEAD
template <> struct Limit<BF16> { static constexpr float SUM = 0x1p-32f; };

// A pointer that is the same in all lanes, as one that the compiler knows to be.
__device__ __forceinline__ const char* uniform(const void* p) {
  const uint64_t a = (uint64_t)p;
  return (const char*)((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(a >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)a));
}
// 1 KiB from memory straight into LDS, sixteen bytes a lane, in the lanes' order from `to` on.  As an instruction of its own and not the builtin: behind that one every read of LDS
// would wait for memory, whatever it reads.  It has no result in a register; who reads what it brings waits for vmcnt(0) first.
__device__ __forceinline__ void load_lds(const char* from, unsigned lane_at, const void* to) {
  const unsigned lds = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)to);
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // that nobody keeps m0 for us is what the list is to say
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %0" ::"s"(from), "s"(lds), "v"(lane_at) : "memory", "m0");
#pragma clang diagnostic pop
}
template <int D> __device__ __forceinline__ constexpr int tile_swap_k(int t) {
  return D >= 128 ? t & 15 : D == 64 ? t >> 1 & 7 : t >> 2 & 3;
}
template <int D> __device__ __forceinline__ constexpr int tile_swap_v(int t) {
  return D >= 128 ? (t & 3) * 4 : D == 64 ? (t >> 1 & 1) * 4 : 0;
}
// PROMPT: keys and values of the call.  PAGES: of pages.  SPLIT: of pages, a part of them (see PackedPart).
enum PackedMode { PROMPT, PAGES, SPLIT };
constexpr int kSplitTiles = 4;  // of a part, at least
constexpr int packed_tiles_waves(int D) { return D == 256 ? 1 : 2; }
template <int D> struct TilesLds {
  u32x4 kv[2][2][kTileKeys * D / 8];  // [buffer][keys, values]
};
template <class DT, int D, PackedMode MODE>
__device__ __forceinline__ void packed_attn_tiles(const PackedAttnArgs& p, TilesLds<D>& lds) {
  constexpr bool PAGED = MODE != PROMPT;
  constexpr int ROWS = kTileRows, C = D / 16, NW = D / 32, PK = D / 8;
  constexpr int LOADS = PK / 4, STEP = kWave / PK;  // a wave's loads of a tile of keys (16 tokens), and tokens a load
  typedef Kv<DT> F;
  auto& s_kv = lds.kv;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 31, h = lane >> 5;
  int c, rows, r0, tok0, tile_lo, tile_hi, all_lo, all_hi;  // the keys all_lo .. all_hi are seen by all queries
  PageRows pages = {};
  PackedKeys seen;                                          // by the lane's query
  const uint16_t *k_base, *v_base;
  PackedPart part;
  if constexpr (MODE == SPLIT) {
    const int block = p.by_heads(blockIdx.x);
    c = blockIdx.x - block * p.kv_heads;
    part = packed_part<ROWS>(p, block);
    rows = part.rows, r0 = part.r0, tok0 = part.tok0;
    if (part.here <= 0) return;
    if (!part.live || !part.ok) return packed_nothing<DT, D>(p, part, c, part.live ? NAN : 0.f);
    const PackedBounds ends = packed_bounds<ROWS>(p, part);
    const int first = ends.lo / kTileKeys, count = ends.hi / kTileKeys - first + 1, per = max(kSplitTiles, (part.common ? p.by_group_splits : p.by_splits)(count + part.splits - 1));
    tile_lo = first + part.split * per;
    tile_hi = min(tile_lo + per, first + count) - 1;
    if (ends.hi < 0 || tile_lo > tile_hi) return packed_nothing<DT, D>(p, part, c, 0.f);
    pages = page_rows(p, part.s0, part.alike, ends.lo, ends.hi);
    all_lo = ends.all_lo, all_hi = ends.all_hi;
  } else {
    // The last slots first, which have the most keys of a sequence.  Where a CU has two workgroups at once, the second ones come the other way round, so that those
    // with the most keys are beside those with the fewest.
    const int B = p.seq.B;
    const PackedRows at = packed_rows<ROWS>(
        B + 2, p.slots, p.group,
        [&](int slots) {
          const int all = slots * p.kv_heads, at = blockIdx.x, turn = at >= p.cus && at < all && all <= 2 * p.cus ? all - 1 - (at - p.cus) : at, order = p.by_heads(turn);
          c = turn - order * p.kv_heads;
          return order < slots ? slots - 1 - order : order;
        },
        [&](int i) { return i == 0 ? 0 : i > B + 1 ? p.seq.N : packed_at(p.seq, i - 1); },
        [&](int i) -> long long {
          const int s = min(max(i - 1, 0), B - 1);
          if constexpr (PAGED) return p.start[s];
          return (long long)packed_at(p.keys, s) << 32 | packed_at(p.keys, s + 1);
        });
    const int seq = at.set - 1, n = at.n;
    rows = n * p.group, r0 = at.r0, tok0 = at.tok0;
    if (r0 >= rows) return;
    const bool live = seq >= 0 && seq < B;
    int pos0;  // position of the sequence's first query
    bool ok = true;
    if constexpr (PAGED) {
      ok = at.word >= 0 && at.word <= ((long long)p.pool.width << p.pool.page_log) - n;
      pos0 = ok ? (int)at.word : 0;
    } else {
      const int key0 = (int)(at.word >> 32), key1 = (int)at.word;
      pos0 = key1 - key0 - n;
      k_base = p.k + key0 * p.k_tok + c * p.k_head;
      v_base = p.v + key0 * p.v_tok + c * p.v_head;
    }
    const int pos_lo = pos0 + p.by_group(r0), pos_hi = pos0 + p.by_group(min(r0 + ROWS, rows) - 1);
    if (!live || !ok || pos_hi < 0) return packed_fill<D>(p, tok0, c, r0, ROWS, rows, live && !ok ? DT::fromf(NAN) * 0x10001u : 0u);
    const int lo = p.window ? max(0, pos_lo - p.window + 1) : 0;
    if constexpr (PAGED) pages = page_rows(p, seq, p.shared ? shared_pages(p, seq, pos0) : 0, lo, pos_hi);
    tile_lo = lo / kTileKeys, tile_hi = pos_hi / kTileKeys;
    all_lo = p.window ? pos_hi - p.window + 1 : 0, all_hi = pos_lo;
    seen.hi = pos0;
  }
  if constexpr (PAGED) {
    k_base = p.pool.k + ((long long)c << p.pool.page_log) * D;
    v_base = p.pool.v + ((long long)c << p.pool.page_log) * D;
  }
  for (int* w : {&tile_lo, &tile_hi, &all_lo, &all_hi, &pages.lo, &pages.hi, &pages.alike}) *w = __builtin_amdgcn_readfirstlane(*w);
  const int mine = r0 + 32 * wave + m, row = min(mine, rows - 1), tok = p.by_group(row);
  if constexpr (MODE == SPLIT) {
    seen = packed_keys(p, part, row);
  } else {
    seen.hi += tok;
    seen.lo = p.window ? seen.hi - p.window + 1 : 0;
  }
  const int end = MODE == PROMPT ? all_hi - p.by_group(r0) + p.by_group(rows) : 0;  // keys of the call
  u32x4 qf[C];
  {
    const uint16_t* q = p.q + (tok0 + tok) * p.q_tok + (c * p.group + row - tok * p.group) * p.q_head;
#pragma unroll
    for (int i = 0; i < C; i++) qf[i] = *(const u32x4*)(q + 16 * i + 8 * h);
  }

  // A wave brings sixteen tokens of a tile.  Lane l of load j writes piece 64 j + l of them and reads what belongs there; what is exchanged goes by bits of the
  // token, so load j differs from load 0 by constants, and reads of LDS differ by constants too.
  unsigned k_at = (m * PK + (h ^ tile_swap_k<D>(m))) * 16;
  unsigned v_at = ((4 * h + (m >> 2 & 3)) * PK + ((2 * (m >> 4) + (m >> 1 & 1)) ^ tile_swap_v<D>(m >> 2 & 3))) * 16 + 8 * (m & 1);
  asm volatile("" : "+v"(k_at), "+v"(v_at));
  const unsigned k_row = PAGED ? D * 2 : (unsigned)p.k_tok * 2, v_row = PAGED ? D * 2 : (unsigned)p.v_tok * 2;  // bytes
  // Where the wave's sixteen tokens of a tile come from.  Entries of pages are asked for a tile ahead of that.
  struct Place {
    long long at;   // element of the keys and (PAGED) of the values, of the head
    int last;       // of the sixteen, the last that may be read: tokens behind it are that one again
    unsigned none;  // bit i: tokens 16 i .. + 15 of the tile have no page
  };
  PageRun runs[4] = {};
  auto ask = [&](int tile) {
    if constexpr (PAGED) {
#pragma unroll
      for (int i = 0; i < 4; i++) runs[i] = page_run(p.pool, pages, tile * kTileKeys + 16 * i);
    }
  };
  auto place_of = [&](int tile) -> Place {  // PAGED: of the tile that was asked for
    if constexpr (PAGED) {
      PageRun mine = runs[0];
      unsigned none = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        none |= page_none(p.pool, runs[i]) ? 1u << i : 0u;
        if (i == wave) mine = runs[i];
      }
      return {page_place(p.pool, mine) * D, pages.hi - mine.from, none};
    } else {
      const int from = min(tile * kTileKeys + 16 * wave, end - 1);
      return {from, end - 1 - from, 0u};
    }
  };
  // where the lanes read, in bytes from the first of the sixteen tokens on; last: the last token that is read
  auto lanes = [&](bool values, int last, unsigned (&to)[LOADS]) {
    int l = lane;
    asm volatile("" : "+v"(l));  // nothing that follows from it has a register over the loop
    const int t = l / PK, piece = (l % PK) ^ (values ? tile_swap_v<D>(t) : tile_swap_k<D>(t));
#pragma unroll
    for (int j = 0; j < LOADS; j++)
      to[j] = min(t + STEP * j, last) * (values ? v_row : k_row) + 16u * (piece ^ (values ? tile_swap_v<D>(STEP * j) : tile_swap_k<D>(STEP * j)));
  };
  unsigned k_lanes[LOADS], v_lanes[LOADS];
  auto all_lanes = [&] {
    lanes(false, 15, k_lanes);
    lanes(true, 15, v_lanes);
#pragma unroll
    for (int j = 0; j < LOADS; j++) asm volatile("" : "+v"(k_lanes[j]), "+v"(v_lanes[j]));
  };
  all_lanes();
  // Where a tile's keys or values are; behind one whose tokens end, none is read whose tokens do not.
  auto aim = [&](const Place& pl, bool values) {
    const int last = __builtin_amdgcn_readfirstlane(pl.last);
    if (__builtin_expect(last < 15, 0)) lanes(values, last, values ? v_lanes : k_lanes);
    return uniform((values ? v_base : k_base) + (PAGED ? pl.at : pl.at * (values ? p.v_tok : p.k_tok)));
  };
  auto bring = [&](const Place& pl, bool values, u32x4* to) {
    const char* from = aim(pl, values);
#pragma unroll
    for (int j = 0; j < LOADS; j++) load_lds(from, values ? v_lanes[j] : k_lanes[j], to + 16 * wave * PK + j * kWave);
  };

  float top = -FLT_MAX, sum = 0.f;
  bool far = false;  // whether some query's scores are
  f32x16 o[NW];
  // Weights of half a tile from its scores, as operands: 2^(HEAD - SLACK) times what they are relative to `top`, which was the largest score when it was last looked
  // at.  It is looked at again where a lane's weights add up to more than 2^HEAD.
  auto weights = [&](const f32x16& s, float off, u32x4 (&pf)[2]) {
    float add = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float a = __builtin_amdgcn_exp2f(fmaf(s[2 * j], p.scale, off)), b = __builtin_amdgcn_exp2f(fmaf(s[2 * j + 1], p.scale, off));
      add += a;
      add += b;
      pf[j / 4][j % 4] = DT::pack(a, b);
    }
    return add;
  };
  auto settle = [&](f32x16& s, u32x4 (&pf)[2], float add) {  // of the weights that are in pf now; what o holds is of keys before
    // (the same in all lanes: where the compiler doubts that, it keeps o twice)
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(__any(add > (far ? -1.f : Limit<DT>::SUM)) ? 1 : 0), 0)) {
      float mx = s[0];
#pragma unroll
      for (int e = 0; e < 16; e++) mx = fmaxf(mx, s[e]);
      mx = max_mod32(mx);
      const float at = kv_scaled(mx, p.scale), now = fmaxf(top, at), keep = __builtin_amdgcn_exp2f(top - now);
      sum *= keep;
#pragma unroll
      for (int w = 0; w < NW; w++) o[w] *= keep;
      top = now;
      far = __any(kv_far(top));
      float off = F::HEAD - F::SLACK - top;
      if (far) {
        const float ref = fmaxf(mx, -FLT_MAX);
        off = fminf(at - top, F::SLACK) + F::HEAD - F::SLACK;
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] -= ref;
      }
      add = weights(s, off, pf);
    }
    sum += add;
  };
  // tiles that a window cuts, tiles that all of the workgroup's queries see, tiles that hold some of their own keys
  const int cut = all_lo > 0 ? (all_lo - 1) / kTileKeys : -1, own = all_hi < 0 ? 0 : (all_hi + 1) / kTileKeys;  // last and first of them
  // half u of a tile: what replaces scores of keys that the query does not see, those behind it and those that a window hides, and of places that are no page's
  auto mask = [&](f32x16& s, int tile, int u, unsigned none, float hidden) {
    if (PAGED && __builtin_expect(none != 0, 0)) {
#pragma unroll
      for (int e = 0; e < 16; e++)
        if (none >> (2 * u + e / 8) & 1) s[e] = NAN;
    }
    const int key0 = tile * kTileKeys + 32 * u + 4 * h, most = seen.hi - key0, least = seen.lo - key0;
    if (tile >= own) {
#pragma unroll
      for (int e = 0; e < 16; e++) s[e] = 8 * (e / 4) + e % 4 <= most ? s[e] : hidden;
    }
    if (tile <= cut) {
#pragma unroll
      for (int e = 0; e < 16; e++) s[e] = 8 * (e / 4) + e % 4 >= least ? s[e] : hidden;
    }
  };
  // operands of half a tile, in the order of the products
  auto key = [&](const u32x4* keys, int i) { return *(const u32x4*)((const char*)keys + (k_at ^ 32u * i)); };
  auto value = [&](const u32x4* values, int i) {
    const char* at = (const char*)values + (v_at ^ 64u * (i % NW)) + 16 * (i / NW) * PK * 16;
    const u32x2 lo = read_turned(at), hi = read_turned(at + 8 * PK * 16);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  auto clear = [&] {
#pragma unroll
    for (int w = 0; w < NW; w++)
#pragma unroll
      for (int e = 0; e < 16; e++) o[w][e] = 0.f;
  };
  auto zeros = [] {
    f32x16 z;
#pragma unroll
    for (int e = 0; e < 16; e++) z[e] = 0.f;
    return z;
  };
  auto arrive = [&] {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): in LDS
    lds_barrier();
  };
  // The weights of half a tile from its scores `now`, beside the products of the half before, whose weights are `before`, and the scores of the half behind: of each an
  // eighth in turn, operands read two ahead, the argument of an exponential one.  Matrix cores and the rest of a SIMD then work at once.  load(i): the i-th of 2 LOADS
  // loads into LDS, which take their time to be issued.
  auto turn_of = [&](auto VALUES, auto KEYS, f32x16& now, f32x16& behind, const u32x4 (&before)[2], u32x4 (&pf)[2], const u32x4* values, const u32x4* keys, auto load) {
    constexpr int N = 2 * NW, STEPS = N > 8 ? N : 8;
    const float off = F::HEAD - F::SLACK - top;
    u32x4 x[3], y[3];
    f32x2v arg[2], w[2];
    float add = 0.f;
    auto argument = [&](int j) { arg[j & 1] = f32x2v{fmaf(now[2 * j], p.scale, off), fmaf(now[2 * j + 1], p.scale, off)}; };
    auto finish = [&](int j) {
      add += w[j & 1][0];
      add += w[j & 1][1];
      pf[j / 4][j % 4] = DT::pack(w[j & 1][0], w[j & 1][1]);
    };
#pragma unroll
    for (int i = 0; i < 2; i++) {
      if constexpr (KEYS) y[i] = key(keys, i);
      if constexpr (VALUES) x[i] = value(values, i);
    }
    if constexpr (KEYS) behind = zeros();
    argument(0);
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
      __builtin_amdgcn_sched_barrier(0);
      if (i * N % STEPS == 0) {
        const int k = i * N / STEPS;
        if constexpr (KEYS) {
          behind = Mma32<DT>::run(y[k % 3], qf[k], behind);
          if (k + 2 < N) y[(k + 2) % 3] = key(keys, k + 2);
        }
        if constexpr (VALUES) {
          o[k % NW] = Mma32<DT>::run(x[k % 3], before[k / NW], o[k % NW]);
          if (k + 2 < N) x[(k + 2) % 3] = value(values, k + 2);
        }
      }
      if (i * 2 * LOADS % STEPS == 0) load(i * 2 * LOADS / STEPS);
      if (i * 8 % STEPS == 0) {
        const int j = i * 8 / STEPS;
        w[j & 1] = f32x2v{__builtin_amdgcn_exp2f(arg[j & 1][0]), __builtin_amdgcn_exp2f(arg[j & 1][1])};
        if (j + 1 < 8) argument(j + 1);
        if (j > 0) finish(j - 1);
      }
    }
    finish(7);
#pragma unroll
    for (int i = 0; i < 2; i++) asm volatile("" : "+v"(pf[i]));  // here, and not where it is known that they are wanted
    __builtin_amdgcn_sched_barrier(0);
    settle(now, pf, add);
  };
  const std::true_type yes;
  const std::false_type no;

  // Halves in turn, 0 and 1 of a tile.  Between them, when all waves have read the one half, the keys of the tile behind the next come, and the values of the next.
  clear();
  f32x16 s0, s1;
  u32x4 p0[2], p1[2];
  Place at0, at1, at2;  // of the tile, and of the two behind it
  int tile = tile_lo, buf = 0;
  constexpr int HALF = 32 * PK;
  ask(tile);
  at0 = place_of(tile);
  bring(at0, false, s_kv[0][0]);
  bring(at0, true, s_kv[0][1]);
  ask(tile + 1);
  at1 = place_of(tile + 1);
  bring(at1, false, s_kv[1][0]);
  ask(tile + 2);
  arrive();
  s0 = zeros();
#pragma unroll
  for (int i = 0; i < C; i++) s0 = Mma32<DT>::run(key(s_kv[0][0], i), qf[i], s0);
  auto masked = [&](f32x16& s, int tile, int u, unsigned none) {
    if (__builtin_expect(tile >= own || tile <= cut || none, 0)) mask(s, tile, u, none, -INFINITY);
  };
  masked(s0, tile, 0, at0.none);
  const auto nothing = [](int) {};
  turn_of(no, yes, s0, s1, p1, p0, nullptr, s_kv[0][0] + HALF, nothing);
  for (; tile < tile_hi; tile++, buf ^= 1) {
    at2 = place_of(tile + 2);
    arrive();
    const char *v_from = aim(at1, true), *k_from = aim(at2, false);
    ask(tile + 3);
    masked(s1, tile, 1, at0.none);
    turn_of(yes, yes, s1, s0, p0, p1, s_kv[buf][1], s_kv[buf ^ 1][0], [&](int i) {
      if (i < LOADS) load_lds(v_from, v_lanes[i], s_kv[buf ^ 1][1] + 16 * wave * PK + i * kWave);
      else load_lds(k_from, k_lanes[i - LOADS], s_kv[buf][0] + 16 * wave * PK + (i - LOADS) * kWave);
    });
    masked(s0, tile + 1, 0, at1.none);
    turn_of(yes, yes, s0, s1, p1, p0, s_kv[buf][1] + HALF, s_kv[buf ^ 1][0] + HALF, nothing);
    at0 = at1, at1 = at2;
  }
  arrive();
  masked(s1, tile, 1, at0.none);
  turn_of(yes, no, s1, s0, p0, p1, s_kv[buf][1], nullptr, nothing);
#pragma unroll
  for (int i = 0; i < 2 * NW; i++) o[i % NW] = Mma32<DT>::run(value(s_kv[buf][1] + HALF, i), p1[i / NW], o[i % NW]);

  // A masked weight is 0, but 0 times a NaN is not.  So where a sum is not finite now, the tiles are gone over again: once with numbers of V that are not finite set
  // to 0, and once to count, for each element, those that a query sees.
  auto again = [&](bool count) {
    clear();
    for (int tile = tile_lo; tile <= tile_hi; tile++) {
      ask(tile);
      const Place at = place_of(tile);
      lds_barrier();
      if (tile == tile_lo) all_lanes();
      bring(at, false, s_kv[0][0]);
      bring(at, true, s_kv[0][1]);
      arrive();
      for (int u = 0; u < 2; u++) {
        s0 = zeros();
#pragma unroll
        for (int i = 0; i < C; i++) s0 = Mma32<DT>::run(key(s_kv[0][0] + u * HALF, i), qf[i], s0);
        mask(s0, tile, u, at.none, -INFINITY);
        if (count) {
#pragma unroll
          for (int e = 0; e < 16; e++) s0[e] = 1.f;
          mask(s0, tile, u, 0, 0.f);
#pragma unroll
          for (int j = 0; j < 8; j++) p0[j / 4][j % 4] = DT::pack(s0[2 * j], s0[2 * j + 1]);
        } else {
          settle(s0, p0, weights(s0, F::HEAD - F::SLACK - top, p0));
        }
#pragma unroll
        for (int i = 0; i < 2 * NW; i++) {
          u32x4 y = value(s_kv[0][1] + u * HALF, i);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const uint32_t bad = kv_nan16<DT>(y[e]);
            y[e] = count ? bad * F::kOne : y[e] & ~(bad * 0xffffu);
          }
          o[i % NW] = Mma32<DT>::run(y, p0[i / NW], o[i % NW]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  };
  auto store = [&](auto write) {  // four elements in order
    if (mine >= rows) return;
    long long to;
    if constexpr (MODE == SPLIT) to = (part.at + packed_row_at(p, part, c, mine)) * D;
    else to = packed_out(p, tok0, c, mine, D) - p.out;
#pragma unroll
    for (int w = 0; w < NW; w++)
#pragma unroll
      for (int a = 0; a < 4; a++) write(to + 32 * w + 8 * a + 4 * h, w, a);
  };
  float odd = 0.f;
#pragma unroll
  for (int w = 0; w < NW; w++)
#pragma unroll
    for (int e = 0; e < 16; e++) odd = fmaf(o[w][e], 0.f, odd);
  const bool bad = __syncthreads_or(odd != 0.f);  // NaN is
  if (bad) {
    top = -FLT_MAX, sum = 0.f, far = false;
    again(false);
  }
  sum += __shfl_xor(sum, 32, kWave);
  if constexpr (MODE == SPLIT) {
    store([&](long long to, int w, int a) { *(f32x4*)(p.part + to) = f32x4{o[w][4 * a], o[w][4 * a + 1], o[w][4 * a + 2], o[w][4 * a + 3]}; });
    if (h == 0 && mine < rows) {
      float* ml = packed_part_ml(p, D) + 2 * (part.at + packed_row_at(p, part, c, mine));
      ml[0] = top;  // as it is: at 2^27 and beyond 32 bits hold no top + SLACK.  Weights of 2^(HEAD - SLACK) are relative to it
      ml[1] = sum;
    }
  } else {
    const float f = sum == 0.f ? 0.f : 1.f / sum;  // no key, or none that weighs anything
    const long long to = packed_out(p, tok0, c, min(mine, rows - 1), D) - p.out + 8 * h;
#pragma unroll
    for (int w = 0; w < NW; w++)
#pragma unroll
      for (int a = 0; a < 4; a += 2) {  // the halves of the wave exchange what they have of eights a and a + 1, and each writes one of them
        u32x4 x;
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const auto r = __builtin_amdgcn_permlane32_swap(DT::pack(o[w][4 * a + 2 * e] * f, o[w][4 * a + 2 * e + 1] * f),
                                                          DT::pack(o[w][4 * a + 4 + 2 * e] * f, o[w][4 * a + 5 + 2 * e] * f), false, false);
          x[e] = r[0], x[2 + e] = r[1];
        }
        if (mine < rows) *(u32x4*)(p.out + to + 32 * w + 8 * a) = x;
      }
  }
  if (bad) {
    again(true);
    store([&](long long to, int w, int a) {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (o[w][4 * a + e] > 0.f) {
          if constexpr (MODE == SPLIT) p.part[to + e] = NAN;
          else p.out[to + e] = DT::fromf(NAN);
        }
    });
  }
}

// Few tokens: up to sixteen rows of queries a workgroup, which are an operand of v_mfma_f32_16x16x32, and keys split over workgroups.  In one launch those of the keys that a group
// of sequences shares, whose rows are the tokens of all of them, and those of a sequence's own keys.
//   S^T = K . Q^T   tile i, row 4 g + e of the result: token 16 i + 4 g + e, in lanes of group g = lane / 16; columns are queries
//   O^T += V^T . P  operand of 32 tokens: tokens 4 g .. + 3 and 16 + 4 g .. + 3, those whose weights the lane has; V comes turned round out of LDS
// Weights are rounded as above; they begin at 2^HEAD, so fp16 ones are steps of 2^-39 below 2^-29 of the largest (1.8e-3 for 1.7e-3 in bf16, 2.3e-4 for 2.1e-4 in fp16).
// Each wave has 32 keys of its own at a time and waits for nobody: keys come as operands, values into LDS of the wave's own.  What the waves give is joined in LDS at the end.
// Bound by memory: 32 rows of 32 heads over 8 behind 4096 tokens, 537 MB, take 86.5 us, 6.2 TB/s; with lengths to 4096 (407 MB) 72.5, 4.6 of them the join's.  Three workgroups a
// CU for heads of 128, which their registers allow (with keys by way of LDS there were two: 78 us).  More than 16 rows would need the matrix cores' other form: see above.
constexpr int kStepKeys = 32, kStepRows = 16;
template <int D> __device__ __forceinline__ constexpr int step_swap_v(int t) {
  return D >= 128 ? (t & 7) * 2 : D == 64 ? (t >> 1 & 3) * 2 : (t >> 2 & 1) * 2;
}
constexpr int packed_step_waves(int D) { return D == 256 ? 2 : D == 128 ? 3 : 4; }
template <int D> struct StepLds {
  union {
    u32x4 v[4][kStepKeys * D / 8];  // of each wave
    float joined[4][kStepRows][D + 4];
  };
  float top[4][kStepRows], sum[4][kStepRows];
};
// BESIDE: parts of packed_attn_tiles are joined with these, whose weights are 2^SLACK times as large: what goes to the join is scaled by 2^-SLACK, which is exact.
template <class DT, int D, bool BESIDE>
__device__ __forceinline__ void packed_attn_step(const PackedAttnArgs& p, StepLds<D>& lds) {
  constexpr int C = D / 32, NU = D / 16, PK = D / 8, STEP = kWave / PK, W = 4, LOADS = PK / 4;
  typedef Kv<DT> F;
  static_assert(F::SLACK == 8.f);
  constexpr float UNIT = BESIDE ? 0x1p-8f : 1.f;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, g = lane >> 4;
  const int block = p.by_heads(blockIdx.x), c = blockIdx.x - block * p.kv_heads;
  const PackedPart part = packed_part<kStepRows>(p, block);
  const int r0 = part.r0, here = part.here, tok0 = part.tok0;
  if (here <= 0) return;
  if (!part.live || !part.ok) return packed_nothing<DT, D>(p, part, c, part.live ? NAN : 0.f);
  const PackedBounds ends = packed_bounds<kStepRows>(p, part);
  const int tile_lo = ends.lo / kStepKeys, tile_hi = ends.hi / kStepKeys, active = min(part.splits, (tile_hi - tile_lo + W) / W), split = part.split;
  if (ends.hi < 0 || split >= active) return packed_nothing<DT, D>(p, part, c, 0.f);
  const PageRows pages = page_rows(p, part.s0, part.alike, ends.lo, ends.hi);
  const int row = r0 + min(m, here - 1);
  const PackedKeys k = packed_keys(p, part, row);
  u32x4 qf[C];
  {
    const int t = p.by_group(row);
    const uint16_t* q = p.q + (tok0 + t) * p.q_tok + (c * p.group + row - t * p.group) * p.q_head;
#pragma unroll
    for (int i = 0; i < C; i++) qf[i] = *(const u32x4*)(q + 32 * i + 8 * g);
  }
  const unsigned t_lane = lane / PK;
  unsigned v_at = ((4 * g + (m >> 2)) * PK + ((m >> 1 & 1) ^ step_swap_v<D>(4 * (g & 1) + (m >> 2)))) * 16 + 8 * (m & 1);
  asm volatile("" : "+v"(v_at));
  const uint16_t* k_base = p.pool.k + ((long long)c << p.pool.page_log) * D;
  const uint16_t* v_base = p.pool.v + ((long long)c << p.pool.page_log) * D;
  // Sixteen tokens into LDS; lane l of load j writes piece 64 j + l of them and reads what belongs there.
  auto lane_at = [&](int j, int last) {
    const unsigned t = t_lane + STEP * j, piece = (lane % PK) ^ step_swap_v<D>(t);
    return min((int)t, last) * (2 * D) + piece * 16;
  };

  float top = -FLT_MAX, sum = 0.f;
  bool far = false;
  f32x4 o[NU];
  auto weigh = [&](f32x4 (&s)[2]) {
    float mx = s[0][0];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) mx = fmaxf(mx, s[i][e]);
    mx = max_mod16(mx);
    const float now = fmaxf(top, kv_scaled(mx, p.scale));
    if (__any(now > top)) {
      const float keep = __builtin_amdgcn_exp2f(top - now);
      sum *= keep;
#pragma unroll
      for (int u = 0; u < NU; u++) o[u] *= keep;
      top = now;
      far = __any(kv_far(top));
    }
    float off = F::HEAD - top;
    if (far) {
      const float ref = fmaxf(mx, -FLT_MAX);
      off = fminf(kv_scaled(mx, p.scale) - top, 0.f) + F::HEAD;
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[i][e] -= ref;
    }
    float add = 0.f;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        s[i][e] = __builtin_amdgcn_exp2f(fmaf(s[i][e], p.scale, off));
        add += s[i][e];
      }
    sum += add;
  };
  enum { PLAIN, CLEAN, COUNT };  // gone over again as above
  // a tile; `behind` once its keys have been used
  auto take = [&](auto AGAIN, int mode, int tile, unsigned none, const u32x4* vt, u32x4 (&kk)[2][C], auto behind) {
    const int key0 = tile * kStepKeys;
    f32x4 s[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < C; j++) s[i] = Mma<DT>::run(kk[i][j], qf[j], s[i]);
    }
    __builtin_amdgcn_sched_barrier(0);
    behind();
    __builtin_amdgcn_sched_barrier(0);
    if (__builtin_expect(none != 0, 0)) {
#pragma unroll
      for (int i = 0; i < 2; i++)
        if (none >> i & 1) s[i] = f32x4{NAN, NAN, NAN, NAN};
    }
    auto seen = [&](int i, int e) {
      const int key = key0 + 16 * i + 4 * g + e;
      return key >= k.lo && key <= k.hi;
    };
    if (key0 < ends.all_lo || key0 + kStepKeys - 1 > ends.all_hi) {
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[i][e] = seen(i, e) ? s[i][e] : -INFINITY;
    }
    if (!AGAIN || mode == CLEAN) weigh(s);
    if constexpr (AGAIN) {
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[i][e] = mode == COUNT ? (seen(i, e) ? 1.f : 0.f) : s[i][e];
    }
    const u32x4 pf = u32x4{DT::pack(s[0][0], s[0][1]), DT::pack(s[0][2], s[0][3]), DT::pack(s[1][0], s[1][1]), DT::pack(s[1][2], s[1][3])};
    constexpr int AHEAD = NU < 4 ? NU : 4;  // operands are read four ahead
    u32x4 x[AHEAD];
    auto value = [&](int u) {
      const u32x2 lo = read_turned((const char*)vt + (v_at ^ 32u * u)), hi = read_turned((const char*)vt + (v_at ^ 32u * u) + 16 * PK * 16);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
#pragma unroll
    for (int u = 0; u < AHEAD; u++) x[u] = value(u);
#pragma unroll
    for (int u = 0; u < NU; u++) {
      __builtin_amdgcn_sched_barrier(0);
      u32x4 v = x[u % AHEAD];
      if (u + AHEAD < NU) x[u % AHEAD] = value(u + AHEAD);
      if constexpr (AGAIN) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t bad = kv_nan16<DT>(v[e]);
          v[e] = mode == COUNT ? bad * F::kOne : v[e] & ~(bad * 0xffffu);
        }
      }
      o[u] = Mma<DT>::run(v, pf, o[u]);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto sweep = [&](auto AGAIN, int mode) {
#pragma unroll
    for (int u = 0; u < NU; u++) o[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    PageRun runs[2];
    auto ask = [&](int tile) {
#pragma unroll
      for (int i = 0; i < 2; i++) runs[i] = page_run(p.pool, pages, min(tile, tile_hi) * kStepKeys + 16 * i);
    };
    const int step = active * W;
    int tile = tile_lo + split * W + wave;
    u32x4 kk[2][C];
    u32x4* vt = lds.v[wave];
    auto fetch_k = [&] {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const char* from = uniform(k_base + page_place(p.pool, runs[i]) * D);
#pragma unroll
        for (int j = 0; j < C; j++) kk[i][j] = load_stream((const u32x4*)(from + (size_t)((unsigned)(m * 2 * D + 16 * g) + 64u * j)));
      }
    };
    auto bring_v = [&] {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const char* from = uniform(v_base + page_place(p.pool, runs[i]) * D);
#pragma unroll
        for (int j = 0; j < LOADS; j++)
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + (size_t)lane_at(j, pages.hi - runs[i].from)),
                                           (__attribute__((address_space(3))) void*)(vt + 16 * i * PK + j * kWave), 16, 0, 2);
      }
    };
    ask(tile);
    if (tile <= tile_hi) {
      fetch_k();
      bring_v();
    }
    while (tile <= tile_hi) {
      const unsigned none = (unsigned)page_none(p.pool, runs[0]) | (unsigned)page_none(p.pool, runs[1]) << 1;
      const bool more = tile + step <= tile_hi;
      ask(tile + step);
      take(AGAIN, mode, tile, none, vt, kk, [&] {
        if (more) fetch_k();
      });
      tile += step;
      if (more) bring_v();
    }
  };
  sweep(std::false_type(), PLAIN);
  float odd = 0.f;
#pragma unroll
  for (int u = 0; u < NU; u++)
#pragma unroll
    for (int e = 0; e < 4; e++) odd = fmaf(o[u][e], 0.f, odd);
  const bool again = __syncthreads_or(odd != 0.f);
  if (again) {
    top = -FLT_MAX, sum = 0.f, far = false;
    sweep(std::true_type(), CLEAN);
    __syncthreads();
  }
  sum += __shfl_xor(sum, 16, kWave);
  sum += __shfl_xor(sum, 32, kWave);

  // the waves' results, and where the tiles have been gone over again, what is to be put there instead
  auto join = [&](bool count) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NU; u++) *(f32x4*)&lds.joined[wave][m][16 * u + 4 * g] = o[u];
    if (!count && g == 0) {
      lds.top[wave][m] = top;
      lds.sum[wave][m] = sum;
    }
    __syncthreads();
    for (int i = tid; i < here * (D / 4); i += 256) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      float mx = lds.top[0][r];
#pragma unroll
      for (int w = 1; w < W; w++) mx = fmaxf(mx, lds.top[w][r]);
      f32x4 num = f32x4{0.f, 0.f, 0.f, 0.f};
      float den = 0.f;
#pragma unroll
      for (int w = 0; w < W; w++) {
        const float f = count ? 1.f : __builtin_amdgcn_exp2f(lds.top[w][r] - mx) * UNIT;
        const f32x4 x = *(const f32x4*)&lds.joined[w][r][d];
#pragma unroll
        for (int e = 0; e < 4; e++) num[e] = fmaf(f, x[e], num[e]);
        den = fmaf(f, lds.sum[w][r], den);
      }
      const long long to = packed_row_at(p, part, c, r0 + r);
      const bool whole = p.splits + p.group_splits == 1;
      if (count) {  // not finite where something has been counted
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (num[e] > 0.f) {
            if (whole) p.out[to * D + d + e] = DT::fromf(NAN);
            else p.part[(part.at + to) * D + d + e] = NAN;
          }
      } else if (whole) {
        const float f = den == 0.f ? 0.f : 1.f / den;
        *(u32x2*)(p.out + to * D + d) = u32x2{DT::pack(num[0] * f, num[1] * f), DT::pack(num[2] * f, num[3] * f)};
      } else {
        *(f32x4*)(p.part + (part.at + to) * D + d) = num;
        if (d == 0) {
          float* ml = packed_part_ml(p, D) + 2 * (part.at + to);
          ml[0] = mx;
          ml[1] = den;
        }
      }
    }
  };
  join(false);
  if (again) {
    __syncthreads();
    sweep(std::true_type(), COUNT);
    join(true);
  }
}

template <class DT, int D, PackedMode MODE>
__global__ __launch_bounds__(256, packed_tiles_waves(D)) void packed_attn_tiles_kernel(PackedAttnArgs p) {
  __shared__ TilesLds<D> lds;
  packed_attn_tiles<DT, D, MODE>(p, lds);
}
template <class DT, int D>
__global__ __launch_bounds__(256, packed_step_waves(D)) void packed_attn_step_kernel(PackedAttnArgs p) {
  __shared__ StepLds<D> lds;
  packed_attn_step<DT, D, false>(p, lds);
}
// Many rows behind keys that they share, and few with keys of their own: the first wait for the matrix cores, the others for memory, so they run side by side (64 rows
// behind 16384 tokens they share and 500 each: 45 us, in two launches 58, with the shared ones in parts of 16 rows 54).
template <class DT, int D>
__global__ __launch_bounds__(256, packed_tiles_waves(D)) void packed_attn_both_kernel(PackedAttnArgs p) {
  __shared__ union {
    TilesLds<D> tiles;
    StepLds<D> step;
  } lds;
  if (p.by_heads(blockIdx.x) < p.group_blocks) packed_attn_tiles<DT, D, SPLIT>(p, lds.tiles);
  else packed_attn_step<DT, D, true>(p, lds.step);
}

// The splits' results, in a fixed order: part s counts sum_s = sum of 2^(score - top_s), and num / sum = (sum of 2^(top_s - top) num_s) / (sum of 2^(top_s - top) sum_s).  A launch
// of its own behind the other, 3 to 4.6 us for two parts of 1024 rows, and 5.4 for 17 of 2048, which would be one wave's loop over them.  ALONE: a workgroup a row, for more than
// eight parts, else a wave a row; groups of D / 4 lanes take every so manieth.
template <class DT, int D, bool ALONE>
__global__ __launch_bounds__(256) void packed_join_kernel(PackedAttnArgs p) {
  constexpr int L = D / 4, G = (ALONE ? 256 : kWave) / L;
  const int tid = ALONE ? threadIdx.x : threadIdx.x & (kWave - 1), grp = tid / L, d = tid % L * 4, n = p.splits + p.group_splits;
  const long long all = (long long)p.seq.N * p.kv_heads * p.group, r = ALONE ? blockIdx.x : (long long)blockIdx.x * 4 + threadIdx.x / kWave;
  if (r >= all) return;
  const float* ml = p.part + n * all * D + 2 * r;
  const float* part = p.part + r * D + d;
  float top = -FLT_MAX, den = 0.f;
  f32x4 num = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = grp; s < n; s += G) {
    const float mx = ml[2 * s * all], sm = ml[2 * s * all + 1];
    f32x4 x = *(const f32x4*)(part + s * all * D);
    if (sm == 0.f) x = f32x4{0.f, 0.f, 0.f, 0.f};  // nothing has been written
    const float now = fmaxf(top, mx), keep = __builtin_amdgcn_exp2f(top - now), f = __builtin_amdgcn_exp2f(mx - now);
#pragma unroll
    for (int e = 0; e < 4; e++) num[e] = fmaf(f, x[e], num[e] * keep);
    den = fmaf(f, sm, den * keep);
    top = now;
  }
#pragma unroll
  for (int i = L; i < kWave; i <<= 1) {
    const float mx = __shfl_xor(top, i, kWave), now = fmaxf(top, mx), keep = __builtin_amdgcn_exp2f(top - now), f = __builtin_amdgcn_exp2f(mx - now);
#pragma unroll
    for (int e = 0; e < 4; e++) num[e] = fmaf(f, __shfl_xor(num[e], i, kWave), num[e] * keep);
    den = fmaf(f, __shfl_xor(den, i, kWave), den * keep);
    top = now;
  }
  if constexpr (ALONE) {
    constexpr int W = 4;
    __shared__ __align__(16) float s_o[W][D];
    __shared__ float s_top[W], s_sum[W];
    const int wave = threadIdx.x / kWave;
    if ((threadIdx.x & (kWave - 1)) < L) {
      *(f32x4*)&s_o[wave][d] = num;
      if (d == 0) {
        s_top[wave] = top;
        s_sum[wave] = den;
      }
    }
    __syncthreads();
    if (threadIdx.x >= L) return;
    float most = s_top[0];
#pragma unroll
    for (int i = 1; i < W; i++) most = fmaxf(most, s_top[i]);
    num = f32x4{0.f, 0.f, 0.f, 0.f};
    den = 0.f;
#pragma unroll
    for (int i = 0; i < W; i++) {
      const float f = __builtin_amdgcn_exp2f(s_top[i] - most);
      const f32x4 x = *(const f32x4*)&s_o[i][d];
#pragma unroll
      for (int e = 0; e < 4; e++) num[e] = fmaf(f, x[e], num[e]);
      den = fmaf(f, s_sum[i], den);
    }
  } else if (grp != 0) {
    return;
  }
  const float f = den == 0.f ? 0.f : 1.f / den;
  *(u32x2*)(p.out + r * D + d) = u32x2{DT::pack(num[0] * f, num[1] * f), DT::pack(num[2] * f, num[3] * f)};
}

}  // namespace cats
