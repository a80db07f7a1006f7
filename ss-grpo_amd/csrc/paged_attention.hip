// Attention of new tokens over a paged cache (fg_paged.h): N new tokens per sequence (tree nodes with ancestor masks, or a
// causal chain; one token is a chain of one) attend to the committed tokens [0, seq_len[b]) of their cache row and to the new
// ones, which lie behind them (flashgrpo/decoding/tree_attention.py:6-67 and the attention it feeds).
//
//   out[q] = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale log2(e) q . k_j - m),  m the running maximum, one pass over the keys
//
// A row that sees no key is 0. The G = q heads / kv heads rows of a node share every K and V row that is read. Times of more than 32
// rows of a kv head are those of one bf16 part of P, unless two are named (paged_attn_kernel).
#include "fg_paged.h"

#include <algorithm>
#include <type_traits>

namespace {

using fg::kPageBF16;
using fg::kPageE4M3;
using fg::Pages;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;
typedef __attribute__((address_space(4))) int32_t const_i32;  // read by the scalar unit

struct PagedAttn {
  Pages pages;
  const void* q;  // [B, N, Hq, D] bf16
  void* out;
  const int32_t* seq_len;
  const int32_t* new_len;
  const int32_t* row_map;
  const uint64_t* anc;
  int64_t anc_stride;
  int batch, N, Hq;
  float scale;
  int slots;   // parts that the sequences' keys may be cut into together (a kv head's, of a row tile); 0: none is cut
  int most;    // parts of one sequence at most
  float* o_part;    // [slots][N, Hq, D]
  float2* ml_part;  // [slots][N, Hq]
  int2* shares;     // [B] a sequence's first slot and its parts
};

constexpr float kRescaleSlack = 8.0f;  // log2 units
constexpr float kLog2e = 1.44269504088896341f;
constexpr int kMinPartKeys = 256;      // a sequence has at most one part for each so many keys that it begins
constexpr int kCUs = 256;
constexpr int kThreads = 512;          // of a workgroup of the attention kernels; sequences that are put in order
constexpr int kMaxCut = 64;            // sequences that are cut: a lane each
constexpr int kStreamWaves = 8;        // of a workgroup of the stream kernel

FG_DEVICE int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }
FG_DEVICE int c_row32(int i, int lane) { return (i >> 2) * 8 + (lane >> 5) * 4 + (i & 3); }

// Bits j < n of a 64-bit mask.
FG_DEVICE uint64_t low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : ((1ull << n) - 1ull); }
// Keys first .. first + 63, sh = seq_len - first: prefix keys (j < sh) and the new tokens whose bit is set.
FG_DEVICE uint64_t seen_mask(int sh, uint64_t bits) {
  const uint64_t fresh = sh >= 64 ? 0ull : sh >= 0 ? (bits << sh) : sh <= -64 ? 0ull : (bits >> -sh);
  return low_bits(sh) | fresh;
}

FG_DEVICE float xor32_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
FG_DEVICE float xor32_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// What a sequence's rows may see, from its device-side lengths: nothing where they make no sense.
struct Span {
  int committed, fresh, row;  // committed tokens, new tokens, cache row
};
FG_DEVICE Span span_of(const PagedAttn& a, int b) {
  const int cap = a.pages.capacity();
  Span s;
  s.row = a.row_map ? a.row_map[b] : b;
  s.fresh = a.new_len ? min(max(a.new_len[b], 0), a.N) : a.N;
  s.committed = a.seq_len[b];
  if ((unsigned)s.row >= (unsigned)a.pages.table_rows || s.committed < 0) s.row = -1;
  s.committed = min(max(s.committed, 0), cap);
  return s;
}
FG_DEVICE int keys_of(const PagedAttn& a, const Span& s) {
  return s.row < 0 ? 0 : min(s.committed + s.fresh, a.pages.capacity());
}
// What a workgroup does: a sequence's keys [begin, end), and the slot of its partial result. b < 0: nothing.
struct Work {
  Span seq;
  int b, begin, end, slot;
};

// Sums over the lanes up to each: row shifts, then the last lane of each row and of the lower half to those behind.
template <typename T>
FG_DEVICE T scan_add(T x) {
#define FG_MOVED(ctrl, rows) \
  __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), ctrl, rows, 0xf, false))
  x += FG_MOVED(0x111, 0xf);
  x += FG_MOVED(0x112, 0xf);
  x += FG_MOVED(0x114, 0xf);
  x += FG_MOVED(0x118, 0xf);
  x += FG_MOVED(0x142, 0xa);
  x += FG_MOVED(0x143, 0xc);
#undef FG_MOVED
  return x;
}

// Which part of which sequence is slot idx, from lengths that only the device knows. A sequence of k keys gets
// 1 + floor((k - 1) f) parts of equal length, f the same for all: 1 / kMinPartKeys, or as large as the slots allow (all of them
// over all keys, else five steps of bisection down to slots - batch, with which the parts always fit). So the order of a sequence's
// sums follows from the other sequences' lengths too, where the slots do not suffice. Every wave works that out for itself, a lane a sequence;
// the first workgroup leaves the shares for the kernel that joins the parts. (A token over 65536 keys beside seven over 1000,
// at 8B: 44 us, with the same number of parts for each sequence 102; 3 verify rounds of 29 over 1096 to 4096 at 14B: 31 and 40.
// What it costs: 0.3 us of 9.6 for a few tokens over short lengths.)
template <int TILE>
FG_DEVICE Work cut_work(const PagedAttn& a, int idx) {
  const int lane = threadIdx.x & 63;
  const Span s = span_of(a, min(lane, a.batch - 1));
  const int keys = lane < a.batch && s.fresh ? keys_of(a, s) : 0;
  const float sums = scan_add((float)keys);
  const float sum = fmaxf(__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, sums), 63)), 1.0f);
  int n, upto;  // a lane's parts, and the parts up to it
  auto fits = [&](float f) __attribute__((always_inline)) {
    n = keys ? min(1 + (int)((float)(keys - 1) * f), a.most) : 0;
    upto = scan_add(n);
    return __builtin_amdgcn_readlane(upto, 63) <= a.slots;
  };
  float high = fminf((float)a.slots / sum, 1.0f / kMinPartKeys), low = fminf((float)(a.slots - a.batch) / sum, high);
  if (!fits(high)) {
    for (int step = 0; step < 5; ++step) {
      const float f = 0.5f * (low + high);
      const bool ok = fits(f);
      high = ok ? high : f;
      low = ok ? f : low;
    }
    if (!fits(low)) fits(low * (1.0f - 1e-4f));  // (one part more by rounding)
  }
  if (blockIdx.x == 0 && threadIdx.x < 64 && lane < a.batch) a.shares[lane] = make_int2(upto - n, n);
  const uint64_t it = __ballot((unsigned)(idx - (upto - n)) < (unsigned)n);
  if (!it) return {{0, 0, -1}, -1, 0, 0, 0};
  const int b = __builtin_ctzll(it);
  auto of = [&](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(x, b); };
  const int all = of(keys), parts = of(n), p = idx - of(upto - n);
  const int part = ((all + parts - 1) / parts + TILE - 1) & ~(TILE - 1);
  const int begin = (int)min((int64_t)p * part, (int64_t)all);
  return {{of(s.committed), of(s.fresh), of(s.row)}, b, begin, (int)min((int64_t)begin + part, (int64_t)all), idx};
}

// The largest lane's value, in lane 63.
FG_DEVICE int scan_max(int x) {
#define FG_MOVED(ctrl, rows) __builtin_amdgcn_update_dpp(x, x, ctrl, rows, 0xf, false)
  x = max(x, FG_MOVED(0x111, 0xf));
  x = max(x, FG_MOVED(0x112, 0xf));
  x = max(x, FG_MOVED(0x114, 0xf));
  x = max(x, FG_MOVED(0x118, 0xf));
  x = max(x, FG_MOVED(0x142, 0xa));
  x = max(x, FG_MOVED(0x143, 0xc));
#undef FG_MOVED
  return x;
}

// The idx-th sequence, long ones first: up to twice as many workgroups as CUs go in that order, so that no long one begins when
// the others end. Sequences are sorted into eight classes by length, a thread a sequence, by ballots; within a class they keep
// their order. 64 tokens over 1096 to 4096 keys at 8B 71 -> 66 us, 128 verify rounds of 29 over 548 to 2048 at 7B 131 -> 112, 4 x
// 1024 tokens 106 -> 100; equal lengths lose 0.5 to 1 us. More workgroups even out by themselves: 128 tokens over 2096 to 4096 at
// 14B, 1024 of them, take 153.5 us unsorted and 157.5 sorted, 256 over 200 to 2000 at 8B 118 and 126. (A sequence's rank by
// comparing it with each other one: 151 in the last case.)
struct Order {
  int4 spans[kThreads];
  uint64_t members[8][kThreads / 64];  // of a class among a wave's sequences
  int top[kThreads / 64];
};
FG_DEVICE Work ordered_work(const PagedAttn& a, int idx, Order& at) {
  static_assert(kThreads == 512 && 2 * kCUs <= kThreads, "eight waves and classes: a lane each; a thread a sequence");
  const int i = threadIdx.x, lane = i & 63, wave = i >> 6;
  int keys = -1;
  if (i < a.batch) {
    const Span s = span_of(a, i);
    keys = s.fresh ? keys_of(a, s) : 0;
    at.spans[i] = make_int4(s.committed, s.fresh, s.row, keys);
  }
  const int top = scan_max(keys);
  if (lane == 63) at.top[wave] = top;
  __syncthreads();
  const int4 x = *(const int4*)at.top, y = *(const int4*)(at.top + 4);
  const float most = (float)(max(max(max(x.x, x.y), max(x.z, x.w)), max(max(y.x, y.y), max(y.z, y.w))) + 1);
  const int its = keys < 0 ? 8 : 7 - min((int)((float)keys * (8.0f / most)), 7);
  uint64_t mine = 0;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const uint64_t m = __ballot(its == c);
    mine = lane == c ? m : mine;
  }
  if (lane < 8) at.members[lane][wave] = mine;
  __syncthreads();
  const uint64_t m = (&at.members[0][0])[lane];
  const int count = __popcll(m), upto = scan_add(count);
  const int l = __builtin_ctzll(__ballot((unsigned)(idx - (upto - count)) < (unsigned)count));
  const int rest = idx - __builtin_amdgcn_readlane(upto - count, l);
  const uint64_t one = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(m >> 32), l) << 32 |
                       (uint32_t)__builtin_amdgcn_readlane((int)m, l);
  const int b = l % 8 * 64 + __builtin_ctzll(__ballot((one >> lane & 1) && __popcll(one & low_bits(lane)) == rest));
  const int4 s = at.spans[b];
  return {{s.x, s.y, s.z}, b, 0, s.w, 0};
}

// The work of workgroup idx of a kv head and row tile (the same in all its threads). A workgroup has kThreads
// threads.
template <int TILE>
FG_DEVICE Work work_of(const PagedAttn& a, int idx, Order& order) {
  if (a.slots) return cut_work<TILE>(a, idx);
  if (gridDim.x > kCUs && gridDim.x <= 2 * kCUs) return ordered_work(a, idx, order);
  const Span s = span_of(a, idx);
  return {s, idx, 0, keys_of(a, s), 0};
}

// 16 e4m3 codes times 2^(s - 127) as bf16: exact, and NaN for s = 255 (a float scale of infinity makes the conversion answer
// NaN for every code, zero included).
FG_DEVICE void expand16(u32x4 w, uint32_t s, u32x4& lo, u32x4& hi) {
  const float f = __uint_as_float(s << 23);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    lo[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], f, false));
    lo[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], f, true));
    hi[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[2 + i], f, false));
    hi[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[2 + i], f, true));
  }
}

// bf16 values that are not finite have all exponent bits: as 15-bit numbers they are 0x7f80 or more.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
FG_DEVICE uint32_t max_u16x2(uint32_t x, uint32_t y) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, x), __builtin_bit_cast(u16x2, y)));
}
FG_DEVICE uint32_t largest_u16(u32x4 w) {  // by halves
  constexpr uint32_t m = 0x7fff7fffu;
  return max_u16x2(max_u16x2(w[0] & m, w[1] & m), max_u16x2(w[2] & m, w[3] & m));
}
FG_DEVICE bool not_finite(u32x4 w) {
  const uint32_t x = largest_u16(w);
  return (x & 0xffffu) >= 0x7f80u || x >= 0x7f800000u;
}
// Eight of them with 0 in the place of those that are not finite.
FG_DEVICE u32x4 finite_part(u32x4 w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = w[i] & 0x7fff7fffu;
    w[i] &= ((x & 0xffffu) >= 0x7f80u ? 0u : 0xffffu) | (x >= 0x7f800000u ? 0u : 0xffff0000u);
  }
  return w;
}

// One element of V as a float.
template <int FMT, int D>
FG_DEVICE float v_element(const Pages& pg, int page, int r, int d) {
  const uint8_t* base = pg.v + pg.at(page);
  if constexpr (FMT == kPageBF16) return fg::bf16_to_f32(((const uint16_t*)base)[(int64_t)r * D + d]);
  const auto x = __builtin_amdgcn_cvt_pk_f32_fp8((int)base[(int64_t)r * D + d], false);
  return x[0] * fg::mx_scale(pg.vs[pg.scales_at(page) + (int64_t)r * (D / fg::kMxBlock) + d / fg::kMxBlock]);
}

// Infinities and NaN of V. The loops keep them at 0 where not every row sees them (the new tokens' tiles), since p = 0 times
// them would be NaN, and in bf16 everywhere where P has a lower part, which is 0 or negative too and would make NaN of infinities.
// Here, once, they are added for the rows that see them: p > 0 times an infinity or a NaN is that. `add(page, row, token)` is
// called for each such token in [from, end).
template <int FMT, int D, typename F>
FG_DEVICE void each_unusual(const Pages& pg, const const_i32* trow, int hkv, int lane, int from, int end, F add) {
  constexpr int PER = D / 64;  // elements of a lane
  for (int key = from; key < end; ++key) {
    const int page = trow[key >> pg.log2_page];
    if ((unsigned)page >= (unsigned)pg.pages) continue;
    const int row = pg.row_in_page(hkv, key);
    bool bad = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) bad |= !(fabsf(v_element<FMT, D>(pg, page, row, lane * PER + i)) < INFINITY);
    if (__any(bad)) add(page, row, key);
  }
}

FG_DEVICE void wave_barrier() {  // a wave's LDS operations are done in order; this keeps the compiler's in theirs
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// More than 32 rows of a kv head. A workgroup takes 32 RW query rows of one (sequence, kv head, part of the keys), row r being
// head r % G of node r / G, in KW groups of RW waves. Tiles of KB keys go to the groups in turn. A group's threads fetch a
// tile's K and V rows into registers, 16 bytes each, two tiles ahead; every load of a wave is a consecutive 1 KB of at most 16
// tokens, which lie in one page, so that pages are looked up by the scalar unit. Codes are expanded to bf16 (exactly) on their
// way to one of two LDS stages, while the tile in the other is multiplied; one barrier per tile. S^T = K Q^T puts a query into
// a lane: the softmax needs one exchange with the other half-wave, and P^T goes from the accumulators straight into O^T += V^T
// P^T. The groups merge their (m, l, O) at the end through LDS, the parts of the keys by a second kernel.
//
// PARTS 2: P in two bf16 parts (hi + lo, p but for 2^-18 of it), so that the products with V are made twice and nothing but the
// output's own rounding is left, 1.7e-3 from 64 bits. 1, for callers who ask for it: rounded to bf16 once (2^-9 of each weight in the
// mean, the error of the bf16 output again: 2.3e-3), the sum that of the rounded weights, as in the contiguous cache's attention.
//
// What bounds it: products, reads of fragments, exponentials and expansion, which a SIMD's two waves overlap in part. 64 rounds
// of 29 nodes over 2048 keys at 7B (203 of 256 rows) take 93 us with two parts, 74 with one; the products of the padded rows alone
// would take 86 and 57 at the 1215 TFLOP/s of a large product. Of the 74, 67 are left without fetching and expanding, 63 without
// the barrier too, 57 without reading the fragments. 4 x 1024 tokens at 8B: 122 and 100 us.
// Slower, with one part: two workgroups of four waves per CU (85 us), halves of the waves a phase apart (83), 32-key steps with the next
// fragments read ahead (81), tiles of 128 keys (87); 3 or 4 tiles in flight took the same. With two: all of P before V (93 to 97),
// 16 keys at a time (95).
//
// SHARED, for five or six 32-row blocks: waves w and w + 4 sit on one SIMD, so that a fifth block doubles the time of a tile.
// Two waves take 32 keys each of every tile for such a block instead, and join their results at the end (32 verify rounds of 29
// over 3096 to 4096 keys at 14B, 145 rows, with one part of P: 124 -> 116 us, on bf16 pages 128 -> 124). Steps of 32 keys cost rows
// that are not shared 2 to 5 % (203 rows 77.3 -> 79.3, 4 x 1024 tokens 101 -> 106).
template <int FMT, int D, int RW, int KW, int KB, bool SHARED, int PARTS>
__global__ void __launch_bounds__(RW * KW * 64, 2) paged_attn_kernel(PagedAttn a, int m_tiles) {
  constexpr int T = RW * 64, ROWS = RW * 32;
  constexpr int CPK = D * fg::page_elem_bytes<FMT> / 16;  // 16-byte pieces of a K or V row
  constexpr int NU = KB * CPK / T, KPW = 64 / CPK;        // pieces of a tile's K (and of its V) per thread; keys of a load
  constexpr int CHUNKS = FMT == kPageBF16 ? 1 : 2;        // 16-byte chunks that a piece is as bf16
  constexpr int KROW = D * 2 + 16, VROW = D * 2, BLOCKS = D / fg::kMxBlock;
  constexpr int ND = D / 32, NS = D / 16;
  static_assert(KB * CPK % T == 0 && NU >= 1 && NU <= 32 && KPW <= 16 && KB <= 64 && (!SHARED || (RW == 8 && KB == 64)), "pieces");
  constexpr int TILE = KB * (KROW + VROW);
  constexpr int MERGE = KW > 1 ? RW * KW * 32 * ((D + 4) * 4 + 8) : SHARED ? RW * 32 * (D * 4 + 16) : 0;
  __shared__ __attribute__((aligned(16))) unsigned char lds[KW * 2 * TILE > MERGE ? KW * 2 * TILE : MERGE];
  __shared__ uint64_t no_page[3][KW];  // a tile's keys without a page
  __shared__ int gone_any[3][KW];      // whether there are any
  __shared__ int odd_from, odd_to;     // the tokens among which V was kept at 0 where it is not finite

  const Pages& pg = a.pages;
  static_assert(KW * T == kThreads, "threads of work_of");
  __shared__ __attribute__((aligned(16))) Order order;
  int unit = blockIdx.x / m_tiles, mt = blockIdx.x % m_tiles;
  if (gridDim.x > kCUs) {
    // The row tiles of a unit on one XCD (workgroups go to the eight in turn), those with the most keys first: 4 x 1024 tokens
    // 110.5 -> 105 us, 8 x 512 at 7B's heads 225 -> 214.
    const int whole = gridDim.x / m_tiles & ~7u, turn = blockIdx.x / 8;
    if ((int)(blockIdx.x / m_tiles) < whole) unit = turn / m_tiles * 8 + blockIdx.x % 8, mt = turn % m_tiles;
    mt = m_tiles - 1 - mt;
  }
  const int hkv = unit % pg.kv_heads;
  const Work work = work_of<KB>(a, unit / pg.kv_heads, order);
  const int b = scalar(work.b);
  if (b < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5, l32 = lane & 31;
  const int rw = wave % RW, kw = wave / RW;
  const int G = a.Hq / pg.kv_heads;
  const Span seq = {scalar(work.seq.committed), scalar(work.seq.fresh), scalar(work.seq.row)};
  const int M = G * seq.fresh;
  if (mt * ROWS >= M) return;  // rows behind the sequence's new tokens stay as they are
  const int last = a.anc ? seq.fresh : (min((mt + 1) * ROWS, M) - 1) / G + 1;  // a chain's rows see no later token
  const int begin = scalar(work.begin), end = max(begin, min(scalar(work.end), seq.committed + last));
  const int s0 = seq.committed, clear = a.anc ? s0 : s0 + mt * ROWS / G + 1;  // every row sees the keys before `clear`
  const const_i32* trow = (const const_i32*)(uintptr_t)(pg.table + (int64_t)max(seq.row, 0) * pg.table_stride);
  unsigned char* const group = lds + kw * 2 * TILE;

  struct Loads {
    u32x4 kp[NU], vp[NU];
    uint32_t ksc[NU], vsc[NU], paged;  // paged: bit u, the tokens of load u have a page
  };
  constexpr int DEPTH = 2;  // tiles in flight
  Loads ring[DEPTH];
  const uint32_t head_row = (uint32_t)hkv << pg.log2_page, slot_mask = (1u << pg.log2_page) - 1u;
  const uint32_t sc_lane = (uint32_t)(lane / CPK * BLOCKS + lane % CPK / 2);
  // Page numbers are looked up a turn before they are needed, in front of its barrier: scalar loads come back in any order, so
  // that a wait for LDS reads waits for one that is under way as well.
  int page_of[NU];
  auto lookup = [&](int key0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NU; ++u) page_of[u] = trow[min(key0 + (u * RW + rw) * KPW, end - 1) >> pg.log2_page];
  };
  auto fetch = [&](int key0, Loads& x) __attribute__((always_inline)) {
    x.paged = 0;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      // Behind the part's end, and without a page, rows that exist are read and not used.
      const int key = min(key0 + (u * RW + rw) * KPW, end - 1), found = page_of[u];
      const bool ok = (unsigned)found < (unsigned)pg.pages;
      x.paged |= (uint32_t)ok << u;
      const uint32_t row = head_row + ((uint32_t)key & slot_mask & ~(uint32_t)(KPW - 1));
      const uint64_t at = pg.at(ok ? found : 0) + row * (CPK * 16);
      x.kp[u] = *(const u32x4*)(pg.k + at + (uint32_t)lane * 16);
      x.vp[u] = *(const u32x4*)(pg.v + at + (uint32_t)lane * 16);
      if constexpr (FMT == kPageE4M3) {
        const uint64_t sat = pg.scales_at(ok ? found : 0) + row * BLOCKS;
        x.ksc[u] = (pg.ks + sat)[sc_lane];
        x.vsc[u] = (pg.vs + sat)[sc_lane];
      }
    }
  };
  const int tiles = (end - begin + KB - 1) / KB;  // group kw takes tiles kw, kw + KW, ..
  const int turns = (tiles + KW - 1) / KW, mine = (tiles - kw + KW - 1) / KW;  // (the barriers are the workgroup's)
  auto key_of = [&](int t) { return begin + (t * KW + kw) * KB; };
  if (tiles) {
#pragma unroll
    for (int x = 0; x < DEPTH; ++x) {
      lookup(key_of(x));
      fetch(key_of(x), ring[x]);
    }
    lookup(key_of(DEPTH));
  }

  // A wave's 32-row block, and which of its sharers this is.
  int block = rw, share = 0, sharers = 1;
  if constexpr (SHARED) {
    const int half = rw >> 2, in = rw & 3, blocks = min(max((M - mt * ROWS + 31) / 32 - 4 * half, 0), 4);
    if (blocks == 1 || blocks == 2) share = in / blocks, sharers = 2, block = share < 2 ? 4 * half + in % blocks : RW;
  }
  const int row0 = block < RW ? mt * ROWS + block * 32 : M, r = row0 + l32;
  const bool row_ok = r < M;
  const int qn = row_ok ? r / G : 0, qh = hkv * G + (row_ok ? r % G : 0);
  const uint64_t anc = (row_ok && a.anc) ? a.anc[(int64_t)b * a.anc_stride + qn] : 0ull;
  const uint64_t bits = anc & low_bits(seq.fresh);
  bf16x8 qf[NS];
  {
    const uint16_t* qrow = (const uint16_t*)a.q + (((int64_t)b * a.N + qn) * a.Hq + qh) * D;
#pragma unroll
    for (int s = 0; s < NS; ++s)
      qf[s] = __builtin_bit_cast(bf16x8, row_ok ? *(const u32x4*)(qrow + s * 16 + g * 8) : u32x4(0));
  }
  floatx16 o[ND];
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;
  const float sl2 = a.scale * kLog2e;

  const uint32_t k_lane = (uint32_t)(l32 * KROW + g * 16);
  // V^T fragments by transposed reads: lane 16 gq + i addresses key 4 (gq / 2) + i / 4 and d 32 db + 16 (gq % 2) + 4 (i % 4),
  // and receives keys 4 (lane / 32) + j (and 8 + ..) of d = 32 db + lane % 32. V's 16-byte chunks are swizzled by their key,
  // so that the 4 keys of a 16-lane read meet different banks.
  auto v_swizzle = [](int key) { return D == 128 ? 4 * (key & 3) : 4 * ((key >> 1) & 1); };
  uint32_t v_lane[ND];
  {
    const int gq = lane >> 4, i = lane & 15, key = 4 * (gq >> 1) + (i >> 2);
    const int low = 2 * (gq & 1) + ((i & 3) >> 1);
#pragma unroll
    for (int db = 0; db < ND; ++db)
      v_lane[db] = (uint32_t)(KB * KROW + key * VROW + (((4 * db + low) ^ v_swizzle(key)) * 16) + 8 * (i & 1));
  }

  // V is 0 behind the part's end and without a page and, in the tiles that reach the new tokens (bf16 and two parts of P: in all),
  // where it is not finite; K's rows there may be anything, their scores are masked.
  uint32_t k_put[NU], v_put[NU];  // where this thread's pieces go
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    const int j = (u * RW + rw) * KPW + lane / CPK, c = lane % CPK;
    k_put[u] = (uint32_t)(j * KROW + c * CHUNKS * 16);
    v_put[u] = (uint32_t)(KB * KROW + j * VROW + ((c * CHUNKS) ^ v_swizzle(j)) * 16);
  }
  auto put = [&](int key0, int buf, int slot, Loads& x) __attribute__((always_inline)) {
    unsigned char* const at = group + buf * TILE;
    bool look = key0 + KB > end || x.paged != (1u << NU) - 1u;  // the last tiles, and the rare ones
    if constexpr (FMT == kPageE4M3 || PARTS == 1) {
      look |= key0 + KB > clear;
    } else {
      uint32_t most = 0;
#pragma unroll
      for (int u = 0; u < NU; ++u) most = max_u16x2(most, largest_u16(x.vp[u]));
      look |= __any((most & 0xffffu) >= 0x7f80u || most >= 0x7f800000u);
    }
    if (look) {
      uint64_t gone = 0;
      bool odd = false;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int j0 = (u * RW + rw) * KPW;
        const bool ok = ((x.paged >> u) & 1u) && key0 + j0 + lane / CPK < end;
        const bool bad = ok && (key0 + KB > clear || (FMT == kPageBF16 && PARTS == 2)) && (FMT == kPageE4M3 ? x.vsc[u] == 255u : not_finite(x.vp[u]));
        odd |= bad;
        if (!((x.paged >> u) & 1u)) gone |= low_bits(KPW) << j0;
        if (bad || !ok) x.vp[u] = FMT == kPageE4M3 || !ok ? u32x4(0) : finite_part(x.vp[u]);  // (e4m3: all of a block's 32)
        if (FMT == kPageE4M3 && (bad || !ok)) x.vsc[u] = 127u;
      }
      if (__any(odd) && lane == 0) {
        atomicMin(&odd_from, key0);
        atomicMax(&odd_to, min(key0 + KB, end));
      }
      if (gone && lane == 0) {
        atomicOr((unsigned long long*)&no_page[slot][kw], gone);
        gone_any[slot][kw] = 1;
      }
    }
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      if constexpr (FMT == kPageE4M3) {
        u32x4 lo, hi;
        expand16(x.kp[u], x.ksc[u], lo, hi);
        *(u32x4*)(at + k_put[u]) = lo;
        *(u32x4*)(at + k_put[u] + 16) = hi;
        expand16(x.vp[u], x.vsc[u], lo, hi);
        *(u32x4*)(at + v_put[u]) = lo;
        *(u32x4*)(at + v_put[u] + 16) = hi;
      } else {
        *(u32x4*)(at + k_put[u]) = x.kp[u];
        *(u32x4*)(at + v_put[u]) = x.vp[u];
      }
    }
  };

  // Keys first .. first + 32 nb - 1, which lie `from` keys into the tile.
  auto compute = [&](auto nb, int first, int from, int buf, int slot) __attribute__((always_inline)) {
    constexpr int NB = decltype(nb)::value, KEYS = 32 * NB;
    const unsigned char* const at = group + buf * TILE + from * KROW;
    const unsigned char* const v_base = group + buf * TILE + from * VROW;
    const int is_gone = __builtin_amdgcn_readfirstlane(gone_any[slot][kw]);
    bf16x8 fr[NB * NS];
    // all K fragments before the first MFMA (one LDS latency)
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int s = 0; s < NS; ++s) fr[kb * NS + s] = *(const bf16x8*)(at + k_lane + kb * 32 * KROW + s * 32);
    floatx16 sc[NB];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[kb][i] = 0.0f;
#pragma unroll
      for (int s = 0; s < NS; ++s)
        sc[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[kb * NS + s], qf[s], sc[kb], 0, 0, 0);
    }
    if (first + KEYS > clear || first + KEYS > end || is_gone) {
      uint64_t sees = (a.anc ? seen_mask(s0 - first, bits) : low_bits(s0 + qn + 1 - first)) & low_bits(end - first);
      if (is_gone) sees &= ~(no_page[slot][kw] >> from);
      const uint64_t mine = sees >> (g * 4);
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool ok = (mine >> (kb * 32 + c_row32(i, 0))) & 1ull;
          sc[kb][i] = ok ? sc[kb][i] : -INFINITY;
        }
    }
    float tmax = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) tmax = fmaxf(tmax, sc[kb][i]);
    const float m_new = fmaxf(m_run, xor32_max(tmax) * sl2);
    // The reference maximum moves only where some lane's grew by more than 2^kRescaleSlack.
    if (__any(m_new > m_run + kRescaleSlack)) {
      const float m_sub = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_sub);
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
      m_run = m_new;
    }
    const float m_sub = m_run == -INFINITY ? 0.0f : m_run;
    if constexpr (PARTS == 2) {
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        bf16x8 hi[2], lo[2];  // p = hi + lo but for 2^-18 of it
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          uint32_t ph[4], pl[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[kb][ks * 8 + 2 * j], sl2, -m_sub));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[kb][ks * 8 + 2 * j + 1], sl2, -m_sub));
            l_run += p0 + p1;
            ph[j] = fg::pack_bf16x2(p0, p1);
            pl[j] = fg::pack_bf16x2(p0 - __uint_as_float(ph[j] << 16), p1 - __uint_as_float(ph[j] & 0xffff0000u));
          }
          hi[ks] = __builtin_bit_cast(bf16x8, u32x4{ph[0], ph[1], ph[2], ph[3]});
          lo[ks] = __builtin_bit_cast(bf16x8, u32x4{pl[0], pl[1], pl[2], pl[3]});
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int db = 0; db < ND; ++db) {
            const unsigned char* p0 = v_base + v_lane[db] + (2 * kb + ks) * 16 * VROW;
            const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)p0);
            const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p0 + 8 * VROW));
            const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
            o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, hi[ks], o[db], 0, 0, 0);
            o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, lo[ks], o[db], 0, 0, 0);
          }
      }
    } else {
      float psum = l_run;
      bf16x8 pf[NB][2];
      const bf16x2 ones2 = __builtin_bit_cast(bf16x2, 0x3f803f80u);
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          uint32_t packed[4];
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[kb][ks * 8 + j], sl2, -m_sub));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[kb][ks * 8 + j + 1], sl2, -m_sub));
            packed[j / 2] = fg::pack_bf16x2(p0, p1);
            psum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, packed[j / 2]), ones2, psum, false);
          }
          pf[kb][ks] = __builtin_bit_cast(bf16x8, u32x4{packed[0], packed[1], packed[2], packed[3]});
        }
      l_run = psum;
#pragma unroll
      for (int ks = 0; ks < 2 * NB; ++ks)
#pragma unroll
        for (int db = 0; db < ND; ++db) {
          const unsigned char* p0 = v_base + v_lane[db] + ks * 16 * VROW;
          const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)p0);
          const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p0 + 8 * VROW));
          const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
          o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[ks >> 1][ks & 1], o[db], 0, 0, 0);
        }
    }
  };

  if (tid < 3 * KW) (&no_page[0][0])[tid] = 0, (&gone_any[0][0])[tid] = 0;
  if (tid == 0) odd_from = end, odd_to = 0;
  __syncthreads();
  if (tiles) {
    if (mine > 0) put(key_of(0), 0, 0, ring[0]);
    fetch(key_of(DEPTH), ring[0]);
    lookup(key_of(DEPTH + 1));
  }
  __syncthreads();
  int slot = 0;
  auto turn = [&](int t, Loads& x) __attribute__((always_inline)) {
    const int next = slot == 2 ? 0 : slot + 1;
    if (t + 1 < mine) put(key_of(t + 1), (t + 1) & 1, next, x);
    fetch(key_of(t + 1 + DEPTH), x);
    if (t < mine && row0 < M) {
      if constexpr (!SHARED) {
        compute(std::integral_constant<int, KB / 32>(), key_of(t), 0, t & 1, slot);
      } else {
        if (share == 0) compute(std::integral_constant<int, 1>(), key_of(t), 0, t & 1, slot);
        if (sharers == 1 || share) compute(std::integral_constant<int, 1>(), key_of(t) + 32, 32, t & 1, slot);
      }
    }
    // the bits of tile t - 1 become those of tile t + 2, which are written behind the next barrier
    const int old = next == 2 ? 0 : next + 1;
    if (tid < KW) no_page[old][tid] = 0, gone_any[old][tid] = 0;
    lookup(key_of(t + 2 + DEPTH));
    __syncthreads();
    slot = next;
  };
  for (int t = 0; t < turns;) {
    turn(t++, ring[1]);
    if (t == turns) break;
    turn(t++, ring[0]);
  }
  const int unusual = scalar(odd_from), until = scalar(odd_to);
  if (unusual < until && row0 < M)
    each_unusual<FMT, D>(pg, trow, hkv, lane, unusual, until, [&](int page, int row, int key) {
      // (the waves that met the key: the others' m may be -inf)
      if (KW > 1 ? (key - begin) / KB % KW != kw : (key - begin) % KB * sharers / KB != share) return;
      const bool sees = key < s0 || (a.anc ? (bits >> (key - s0)) & 1ull : key - s0 <= qn);
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = v_element<FMT, D>(pg, page, row, db * 32 + c_row32(i, lane));
          if (sees && !(fabsf(x) < INFINITY)) o[db][i] += x;
        }
    });

  if constexpr (SHARED) {
    // a shared block's waves to its first one: lanes hold the same rows and dims
    float* const om = (float*)lds + wave * 64 * (D / 2) + lane * 4;
    float2* const ml = (float2*)(lds + RW * 64 * (D / 2) * 4);
    if (share) {
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *(float4*)(om + (db * 4 + i / 4) * 256) = make_float4(o[db][i], o[db][i + 1], o[db][i + 2], o[db][i + 3]);
      ml[tid] = make_float2(m_run, l_run);
    }
    __syncthreads();
    if (share || row0 >= M) return;
    if (sharers == 2) {
      const int there = min((M - mt * ROWS + 31) / 32 - 4 * (rw >> 2), 2);  // waves on
      const float2 its = ml[tid + there * 64];
      const float m_new = fmaxf(m_run, its.x), m_sub = m_new == -INFINITY ? 0.0f : m_new;
      const float mine = __builtin_amdgcn_exp2f(m_run - m_sub), other = __builtin_amdgcn_exp2f(its.x - m_sub);
      m_run = m_new;
      l_run = l_run * mine + its.y * other;
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 v = *(const float4*)(om + there * 64 * (D / 2) + (db * 4 + i / 4) * 256);
          o[db][i] = o[db][i] * mine + v.x * other;
          o[db][i + 1] = o[db][i + 1] * mine + v.y * other;
          o[db][i + 2] = o[db][i + 2] * mine + v.z * other;
          o[db][i + 3] = o[db][i + 3] * mine + v.w * other;
        }
    }
  }
  float l = xor32_sum(l_run);
  if constexpr (KW > 1) {
    // merge the key waves' results: O and (m, l) of 32 rows each
    float* om = (float*)lds;
    float2* ml = (float2*)(lds + RW * KW * 32 * (D + 4) * 4);
    __syncthreads();
    {
      float* dst = om + (wave * 32 + l32) * (D + 4);
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *(float4*)(dst + db * 32 + c_row32(i, lane)) = make_float4(o[db][i], o[db][i + 1], o[db][i + 2], o[db][i + 3]);
      if (g == 0) ml[wave * 32 + l32] = make_float2(m_run, l);
    }
    __syncthreads();
    for (int e = tid; e < ROWS * (D / 4); e += T) {
      const int rr = e / (D / 4), d0 = e % (D / 4) * 4, gr = mt * ROWS + rr;
      if (gr >= M) break;
      float mx = -INFINITY, den = 0.0f, s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < KW; ++w) mx = fmaxf(mx, ml[(w * RW + rr / 32) * 32 + rr % 32].x);
      const float sub = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const int at = (w * RW + rr / 32) * 32 + rr % 32;
        const float f = __builtin_amdgcn_exp2f(ml[at].x - sub);
        const float4 x = *(const float4*)(om + at * (D + 4) + d0);
        den += f * ml[at].y;
        s[0] += f * x.x; s[1] += f * x.y; s[2] += f * x.z; s[3] += f * x.w;
      }
      const int64_t orow = ((int64_t)b * a.N + gr / G) * a.Hq + hkv * G + gr % G;
      if (a.slots) {
        const int64_t prow = orow + (int64_t)(scalar(work.slot) - b) * a.N * a.Hq;
        *(float4*)(a.o_part + prow * D + d0) = make_float4(s[0], s[1], s[2], s[3]);
        if (d0 == 0) a.ml_part[prow] = make_float2(mx, den);
      } else {
        const float inv = den == 0.0f ? 0.0f : 1.0f / den;
        *(uint2*)((uint16_t*)a.out + orow * D + d0) =
            make_uint2(fg::pack_bf16x2(s[0] * inv, s[1] * inv), fg::pack_bf16x2(s[2] * inv, s[3] * inv));
      }
    }
  } else {
    if (!row_ok) return;
    const int64_t orow = ((int64_t)b * a.N + qn) * a.Hq + qh;
    if (a.slots) {
      const int64_t prow = orow + (int64_t)(scalar(work.slot) - b) * a.N * a.Hq;
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *(float4*)(a.o_part + prow * D + db * 32 + c_row32(i, lane)) =
              make_float4(o[db][i], o[db][i + 1], o[db][i + 2], o[db][i + 3]);
      if (g == 0) a.ml_part[prow] = make_float2(m_run, l);
    } else {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *(uint2*)((uint16_t*)a.out + orow * D + db * 32 + c_row32(i, lane)) =
              make_uint2(fg::pack_bf16x2(o[db][i] * inv, o[db][i + 1] * inv),
                         fg::pack_bf16x2(o[db][i + 2] * inv, o[db][i + 3] * inv));
    }
  }
}

typedef float floatx4 __attribute__((ext_vector_type(4)));

FG_DEVICE float quad_max(float x) {  // over the four lanes of a query: lane, + 16, + 32, + 48
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return xor32_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
FG_DEVICE float quad_sum(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return xor32_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Few rows (single tokens; at most 16 NQ rows of a kv head): the pages are streamed past them. A workgroup of eight waves takes
// one (sequence, kv head, part of the keys), its waves 32-key tiles in turn, each with registers and LDS of its own, no barrier
// in the loop. S^T = K Q^T on 16 x 16 x 32 MFMAs: lane 16 gq + i holds key i of 16 and, of every 64 bytes of its row, the 16 at
// 16 gq; which d a k index stands for is free as long as Q follows, so K's rows go from memory through the expansion into the
// MFMA's registers and never see LDS. V is expanded into a tile of LDS and read transposed. P goes to V in two bf16 parts (hi +
// lo, p to 16 bits), which costs nothing: what bounds the kernel is the stream of codes. 64 tokens over 1096 to 4096 keys at
// 8B: 62 us, 5.5 TB/s; 2 over 131072 and 123140: 96 us, 5.6 TB/s (a large sum reads 6.0). The other kernel, which takes K
// through LDS too, took 98 us for the first. Four or twelve waves, and two tiles in flight, were no faster.
template <int FMT, int D>
struct StreamTile {  // a tile's loads: 32 keys
  static constexpr int kLoads = D * fg::page_elem_bytes<FMT> / 64;  // 16-byte loads of a lane per 16 keys
  u32x4 k[2][kLoads], v[2 * kLoads];
  uint32_t ks[2], vs[2 * kLoads];  // scales: of K's key all four, of a piece of V its own
  int there;                       // bit h: keys 16 h .. have a page
};

template <int FMT, int D, int NQ>
__global__ void __launch_bounds__(kStreamWaves * 64, 2) paged_stream_kernel(PagedAttn a) {
  constexpr int W = kStreamWaves;
  constexpr int ES = fg::page_elem_bytes<FMT>, CPK = D * ES / 16, VROW = D * 2;
  constexpr int NL = StreamTile<FMT, D>::kLoads, NS = D / 32, ND = D / 16, BLOCKS = D / fg::kMxBlock;
  constexpr int VTILE = 32 * VROW, OROW = D + 4;
  constexpr int MERGE = W * NQ * 16 * (OROW * 4 + 8);
  __shared__ __attribute__((aligned(16))) unsigned char lds[W * VTILE > MERGE ? W * VTILE : MERGE];
  const Pages& pg = a.pages;
  static_assert(W * 64 == kThreads, "threads of work_of");
  __shared__ __attribute__((aligned(16))) Order order;
  const int hkv = blockIdx.x % pg.kv_heads;
  const Work work = work_of<32>(a, blockIdx.x / pg.kv_heads, order);
  const int b = scalar(work.b);
  if (b < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), gq = lane >> 4, i16 = lane & 15;
  const int G = a.Hq / pg.kv_heads;
  const Span seq = {scalar(work.seq.committed), scalar(work.seq.fresh), scalar(work.seq.row)};
  const int M = G * seq.fresh;
  if (M == 0) return;
  const int begin = scalar(work.begin), end = scalar(work.end), s0 = seq.committed;
  const const_i32* trow = (const const_i32*)(uintptr_t)(pg.table + (int64_t)max(seq.row, 0) * pg.table_stride);
  unsigned char* const vt = lds + wave * VTILE;
  typedef StreamTile<FMT, D> Tile;

  // A head's rows within a page, and those of its scales.
  const uint32_t head_row = (uint32_t)hkv << pg.log2_page, slot_mask = (1u << pg.log2_page) - 1u;
  const uint32_t k_lane = (uint32_t)(i16 * (D * ES) + gq * 16);
  int page_of[2];  // of the next tile's two times 16 tokens: looked up a turn ahead
  auto lookup = [&](int key0) __attribute__((always_inline)) {
    page_of[0] = trow[min(key0, end - 1) >> pg.log2_page];
    page_of[1] = trow[min(key0 + 16, end - 1) >> pg.log2_page];
  };
  auto fetch = [&](int key0, Tile& t) __attribute__((always_inline)) {
    // Behind the part's end, and without a page, rows that exist are read and not used.
    t.there = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = min(key0 + 16 * h, end - 1), found = page_of[h];
      const bool ok = (unsigned)found < (unsigned)pg.pages;
      t.there |= (int)ok << h;
      const uint32_t row = head_row + ((uint32_t)key & slot_mask & ~15u);
      const uint64_t at = pg.at(ok ? found : 0) + row * (D * ES);
      const uint8_t* kr = pg.k + at;
      const uint8_t* vr = pg.v + at;
#pragma unroll
      for (int s = 0; s < NL; ++s) t.k[h][s] = *(const u32x4*)(kr + k_lane + s * 64);
#pragma unroll
      for (int s = 0; s < NL; ++s) t.v[h * NL + s] = *(const u32x4*)(vr + (uint32_t)lane * 16 + s * 1024);
      if constexpr (FMT == kPageE4M3) {
        const uint64_t sat = pg.scales_at(ok ? found : 0) + row * BLOCKS;
        const uint8_t* ks = pg.ks + sat;
        const uint8_t* vs = pg.vs + sat;
        t.ks[h] = BLOCKS == 4 ? *(const uint32_t*)(ks + i16 * 4) : *(const uint16_t*)(ks + i16 * 2);
#pragma unroll
        for (int s = 0; s < NL; ++s) t.vs[h * NL + s] = vs[s * (1024 / 32) + lane / 2];
      }
    }
  };
  const int tiles = (end - begin + 31) / 32, mine = (tiles - wave + W - 1) / W;
  auto key_of = [&](int t) { return begin + (t * W + wave) * 32; };
  Tile cur;
  if (mine > 0) {
    lookup(key_of(0));
    fetch(key_of(0), cur);
    lookup(key_of(1));
  }

  int qn[NQ], qh[NQ];
  bool row_ok[NQ];
  uint64_t bits[NQ];
  bf16x8 qf[NQ][NS];
#pragma unroll
  for (int c = 0; c < NQ; ++c) {
    const int r = c * 16 + i16;
    row_ok[c] = r < M;
    qn[c] = row_ok[c] ? r / G : 0;
    qh[c] = hkv * G + (row_ok[c] ? r % G : 0);
    bits[c] = row_ok[c] && a.anc ? a.anc[(int64_t)b * a.anc_stride + qn[c]] & low_bits(seq.fresh) : 0ull;
    const uint16_t* qrow = (const uint16_t*)a.q + (((int64_t)b * a.N + qn[c]) * a.Hq + qh[c]) * D;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      // the d of k-step s: e4m3: 8 of the 16 codes of load s / 2, bf16: the 8 elements of load s
      const int d = FMT == kPageE4M3 ? s / 2 * 64 + gq * 16 + s % 2 * 8 : s * 32 + gq * 8;
      qf[c][s] = __builtin_bit_cast(bf16x8, row_ok[c] ? *(const u32x4*)(qrow + d) : u32x4(0));
    }
  }
  floatx4 o[NQ][ND];
  float m_run[NQ], l_run[NQ];
#pragma unroll
  for (int c = 0; c < NQ; ++c) {
    m_run[c] = -INFINITY;
    l_run[c] = 0.0f;
#pragma unroll
    for (int db = 0; db < ND; ++db) o[c][db] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const float sl2 = a.scale * kLog2e;
  // V^T fragments (16 d x 32 keys): lane 16 gq + i addresses key 4 gq + i / 4 (+ 16) and d 16 db + 4 (i % 4), and receives keys
  // 4 gq + j (and 16 + ..) of d = 16 db + i: the keys of S^T's accumulators. Chunks of 16 bytes are swizzled by their key, so that
  // the four keys of a 16-lane read meet different banks.
  auto v_swizzle = [](int key) { return D == 128 ? 4 * (key & 3) : 4 * ((key >> 1) & 1); };
  const int v_key = 4 * gq + (i16 >> 2);
  const uint32_t v_at = (uint32_t)(v_key * VROW + 8 * (i16 & 1)), v_x = (uint32_t)v_swizzle(v_key), v_low = (i16 & 3) >> 1;

  int odd_from = end, odd_to = 0;  // the tokens among which V was kept at 0 where it is not finite
  for (int t = 0; t < mine; ++t) {
    const int first = key_of(t);
    // ---------------- V to LDS
    // As in put() above.
    bool look = first + 32 > end || cur.there != 3;
    if constexpr (FMT == kPageE4M3) {
      look |= first + 32 > s0;
    } else {
      uint32_t most = 0;
#pragma unroll
      for (int s = 0; s < 2 * NL; ++s) most = max_u16x2(most, largest_u16(cur.v[s]));
      look |= __any((most & 0xffffu) >= 0x7f80u || most >= 0x7f800000u);
    }
    if (look) {
      bool odd = false;
#pragma unroll
      for (int s = 0; s < 2 * NL; ++s) {
        const int j = s * (64 / CPK) + lane / CPK;
        const bool ok = first + j < end && ((cur.there >> (j >> 4)) & 1);
        const bool bad = ok && (FMT == kPageE4M3 ? first + 32 > s0 && cur.vs[s] == 255u : not_finite(cur.v[s]));
        odd |= bad;
        if (bad || !ok) cur.v[s] = FMT == kPageE4M3 || !ok ? u32x4(0) : finite_part(cur.v[s]);
        if (FMT == kPageE4M3 && (bad || !ok)) cur.vs[s] = 127u;
      }
      if (__any(odd)) odd_from = min(odd_from, first), odd_to = min(first + 32, end);
    }
#pragma unroll
    for (int s = 0; s < 2 * NL; ++s) {
      const int j = s * (64 / CPK) + lane / CPK, c = lane % CPK;
      if constexpr (FMT == kPageE4M3) {
        u32x4 lo, hi;
        expand16(cur.v[s], cur.vs[s], lo, hi);
        unsigned char* dst = vt + j * VROW + ((2 * c) ^ v_swizzle(j)) * 16;
        *(u32x4*)dst = lo;
        *(u32x4*)(dst + 16) = hi;
      } else {
        *(u32x4*)(vt + j * VROW + (c ^ v_swizzle(j)) * 16) = cur.v[s];
      }
    }
    // ---------------- S^T
    floatx4 sc[NQ][2];
#pragma unroll
    for (int c = 0; c < NQ; ++c) sc[c][0] = sc[c][1] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int s = 0; s < NL; ++s) {
        u32x4 part[2];
        if constexpr (FMT == kPageE4M3) {
          const uint32_t e = __builtin_amdgcn_ubfe(cur.ks[h], (uint32_t)(16 * s + 8 * (gq >> 1)), 8u);
          expand16(cur.k[h][s], e, part[0], part[1]);
#pragma unroll
          for (int c = 0; c < NQ; ++c)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              sc[c][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, part[x]), qf[c][2 * s + x], sc[c][h], 0, 0, 0);
        } else {
#pragma unroll
          for (int c = 0; c < NQ; ++c)
            sc[c][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, cur.k[h][s]), qf[c][s], sc[c][h], 0, 0, 0);
        }
      }
    const uint64_t gone = (cur.there & 1 ? 0ull : 0xffffull) | (cur.there & 2 ? 0ull : 0xffff0000ull);
    fetch(key_of(t + 1), cur);  // (past the last tile: rows that exist, not used)
    lookup(key_of(t + 2));
    // ---------------- softmax
    const bool masked = first + 32 > s0 || first + 32 > end || gone;
    bf16x8 hi[NQ], lo[NQ];
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
      if (masked) {
        const uint64_t sees = (a.anc ? seen_mask(s0 - first, bits[c]) : low_bits(s0 + qn[c] + 1 - first)) & low_bits(end - first) & ~gone;
        const uint64_t at = sees >> (4 * gq);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[c][h][i] = (at >> (16 * h + i)) & 1ull ? sc[c][h][i] : -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[c][h][i]);
      const float m_new = fmaxf(m_run[c], quad_max(top) * sl2);
      if (__any(m_new > m_run[c] + kRescaleSlack)) {
        const float alpha = __builtin_amdgcn_exp2f(m_run[c] - (m_new == -INFINITY ? 0.0f : m_new));
        l_run[c] *= alpha;
#pragma unroll
        for (int db = 0; db < ND; ++db)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[c][db][i] *= alpha;
        m_run[c] = m_new;
      }
      const float sub = m_run[c] == -INFINITY ? 0.0f : m_run[c];
      uint32_t ph[4], pl[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[c][x >> 1][2 * (x & 1)], sl2, -sub));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[c][x >> 1][2 * (x & 1) + 1], sl2, -sub));
        l_run[c] += p0 + p1;
        ph[x] = fg::pack_bf16x2(p0, p1);
        pl[x] = fg::pack_bf16x2(p0 - __uint_as_float(ph[x] << 16), p1 - __uint_as_float(ph[x] & 0xffff0000u));
      }
      hi[c] = __builtin_bit_cast(bf16x8, u32x4{ph[0], ph[1], ph[2], ph[3]});
      lo[c] = __builtin_bit_cast(bf16x8, u32x4{pl[0], pl[1], pl[2], pl[3]});
    }
    // ---------------- O^T += V^T P^T
    wave_barrier();
#pragma unroll
    for (int db = 0; db < ND; ++db) {
      const unsigned char* at = vt + v_at + (((2 * db + v_low) ^ v_x) * 16);
      const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at);
      const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 16 * VROW));
      const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int c = 0; c < NQ; ++c) {
        o[c][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, hi[c], o[c][db], 0, 0, 0);
        o[c][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, lo[c], o[c][db], 0, 0, 0);
      }
    }
    wave_barrier();
  }
  if (odd_from < odd_to)
    each_unusual<FMT, D>(pg, trow, hkv, lane, odd_from, odd_to, [&](int page, int row, int key) {
      if ((key - begin) / 32 % W != wave) return;  // (the wave that met the key: the others' m may be -inf)
#pragma unroll
      for (int c = 0; c < NQ; ++c) {
        const bool sees = key < s0 || (a.anc ? (bits[c] >> (key - s0)) & 1ull : key - s0 <= qn[c]);
#pragma unroll
        for (int db = 0; db < ND; ++db)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = v_element<FMT, D>(pg, page, row, 16 * db + 4 * gq + i);
            if (sees && !(fabsf(x) < INFINITY)) o[c][db][i] += x;
          }
      }
    });

  // ---------------- merge the waves
  float* om = (float*)lds;
  float2* ml = (float2*)(lds + W * NQ * 16 * OROW * 4);
  __syncthreads();
#pragma unroll
  for (int c = 0; c < NQ; ++c) {
    const int at = (wave * NQ + c) * 16 + i16;
#pragma unroll
    for (int db = 0; db < ND; ++db) *(floatx4*)(om + at * OROW + 16 * db + 4 * gq) = o[c][db];
    const float l = quad_sum(l_run[c]);
    if (gq == 0) ml[at] = make_float2(m_run[c], l);
  }
  __syncthreads();
  for (int e = tid; e < M * (D / 4); e += W * 64) {
    const int r = e / (D / 4), d0 = e % (D / 4) * 4;
    float mx = -INFINITY, den = 0.0f, s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < W; ++w) mx = fmaxf(mx, ml[w * NQ * 16 + r].x);
    const float sub = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int at = w * NQ * 16 + r;
      const float f = __builtin_amdgcn_exp2f(ml[at].x - sub);
      const float4 x = *(const float4*)(om + at * OROW + d0);
      den += f * ml[at].y;
      s[0] += f * x.x; s[1] += f * x.y; s[2] += f * x.z; s[3] += f * x.w;
    }
    const int64_t orow = ((int64_t)b * a.N + r / G) * a.Hq + hkv * G + r % G;
    if (a.slots) {
      const int64_t prow = orow + (int64_t)(scalar(work.slot) - b) * a.N * a.Hq;
      *(float4*)(a.o_part + prow * D + d0) = make_float4(s[0], s[1], s[2], s[3]);
      if (d0 == 0) a.ml_part[prow] = make_float2(mx, den);
    } else {
      const float inv = den == 0.0f ? 0.0f : 1.0f / den;
      *(uint2*)((uint16_t*)a.out + orow * D + d0) =
          make_uint2(fg::pack_bf16x2(s[0] * inv, s[1] * inv), fg::pack_bf16x2(s[2] * inv, s[3] * inv));
    }
  }
}

// The parts of a row: sum_p 2^(m_p - M) (O_p, l_p) over the parts that saw a key, a lane for 4 dims of a part. Up to D / 4
// parts: D / 4 threads a row. More (WIDE): a workgroup a row, 1024 / D parts side by side. A thread reads a part's (m, l), so
// that all of them take one round trip, and no load of O waits for another: 64 rows of 16 parts 4.8 us (one part after the
// other 26), 4992 rows of 2 parts 4.1 us.
template <int D, bool WIDE>
__global__ void __launch_bounds__(256) paged_combine_kernel(PagedAttn a) {
  constexpr int LANES = D / 4, SLOTS = WIDE ? 256 / LANES : 1, PER = 256 / (LANES * SLOTS), MOST = LANES * SLOTS;
  __shared__ float weight[PER][MOST], wave_at[8];
  __shared__ float4 sums[WIDE ? 256 : 1];
  const int ti = threadIdx.x % (LANES * SLOTS), in = threadIdx.x / (LANES * SLOTS), slot = ti / LANES, d0 = ti % LANES * 4;
  const int64_t rows = (int64_t)a.batch * a.N * a.Hq, step = (int64_t)a.N * a.Hq;
  const int64_t row = min((int64_t)blockIdx.x * PER + in, rows - 1);  // (behind the last row: it once more)
  const int n = (int)(row / a.Hq % a.N), b = (int)(row / step);
  const bool asked = n < (a.new_len ? min(max(a.new_len[b], 0), a.N) : a.N);
  const int2 share = a.shares[b];
  const int parts = asked ? share.y : 0;
  const int64_t first = share.x * step + row % step;
  const float2 ml = ti < parts ? a.ml_part[ti * step + first] : make_float2(-INFINITY, 0.0f);
  float mx = ml.x, den;
  if constexpr (WIDE) {
    mx = fg::wave_max(mx);
    if ((threadIdx.x & 63) == 0) wave_at[threadIdx.x >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(wave_at[0], wave_at[1]), fmaxf(wave_at[2], wave_at[3]));
  } else {
#pragma unroll
    for (int x = LANES / 2; x; x >>= 1) mx = fmaxf(mx, __shfl_xor(mx, x, 64));
  }
  const float w = ml.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml.x - (mx == -INFINITY ? 0.0f : mx));
  den = w * ml.y;
  weight[in][ti] = w;
  if constexpr (WIDE) {
    den = fg::wave_sum(den);
    if ((threadIdx.x & 63) == 0) wave_at[4 + (threadIdx.x >> 6)] = den;
    __syncthreads();
    den = wave_at[4] + wave_at[5] + wave_at[6] + wave_at[7];
  } else {
#pragma unroll
    for (int x = LANES / 2; x; x >>= 1) den += __shfl_xor(den, x, 64);
    __syncthreads();
  }
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int p0 = slot; p0 < parts; p0 += 4 * SLOTS) {
    float4 x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = *(const float4*)(a.o_part + (min(p0 + u * SLOTS, parts - 1) * step + first) * D + d0);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float f = p0 + u * SLOTS < parts ? weight[in][p0 + u * SLOTS] : 0.0f;
      if (f != 0.0f) o.x += f * x[u].x, o.y += f * x[u].y, o.z += f * x[u].z, o.w += f * x[u].w;
    }
  }
  if constexpr (WIDE) {
    sums[threadIdx.x] = o;
    __syncthreads();
    if (slot) return;
#pragma unroll
    for (int s = 1; s < SLOTS; ++s) {
      const float4 x = sums[threadIdx.x + s * LANES];
      o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
    }
  }
  if (!asked) return;
  const float inv = den == 0.0f ? 0.0f : 1.0f / den;
  *(uint2*)((uint16_t*)a.out + row * D + d0) =
      make_uint2(fg::pack_bf16x2(o.x * inv, o.y * inv), fg::pack_bf16x2(o.z * inv, o.w * inv));
}

struct Plan {
  int rw, kw, kb, slots;
  int rows() const { return rw * 32; }
  // Whether the kernel that joins the parts takes a workgroup for each row: where there are many parts (3 tokens of 10 parts 17.6
  // us, narrow 18.7), and few rows or too many parts for narrow ones (3 verify rounds of 10 parts, 3480 rows: 30.5 us, narrow 28.9).
  bool wide(int batch, int64_t rows) const { return slots > 8 * batch && (rows < 1024 || slots > 16 * batch); }
};

Plan plan_of(int batch, int num_nodes, int q_heads, int kv_heads, int head_dim, int64_t capacity) {
  const int64_t m = (int64_t)(q_heads / kv_heads) * num_nodes;
  // Eight waves, one workgroup per CU: row tiles side by side as far as there are rows, the rest of the waves on other keys (32
  // rounds of 29 at 8B, 116 rows: 55 us; a wave per 32 rows and no more, 61).
  Plan p;
  if (m <= 32) p = {1, kStreamWaves, 32, 0};
  else if (m <= 64) p = {2, 4, 32, 0};
  else if (m <= 128 || head_dim == 64) p = {4, 2, 64, 0};
  else p = {8, 1, 64, 0};
  const int64_t each = kv_heads * ((m + p.rows() - 1) / p.rows());  // workgroups of a sequence that is not cut
  // Parts where every sequence gets two at least (20 tokens over 2048 keys at 8B, 160 workgroups: whole 19.5 us, in 320 parts 28),
  // and no more workgroups than CUs, which would take two rounds (3 over 8192: 264 workgroups 22.5 us, 256 17.6). Few rows stay
  // whole in caches whose table is short, where the second launch costs more (one over 600 keys at 8B: 8.2 us whole, 10.5 in parts; 4
  // over 1000 at most: 11.4 and 10.3). Lengths are on the device: as few keys in a wide table are cut.
  if (batch <= kMaxCut && 2 * batch * each <= kCUs && (m > 32 || capacity >= 1024)) {
    const int64_t most = std::max<int64_t>(1, capacity / kMinPartKeys);
    p.slots = (int)std::min<int64_t>(kCUs / each, batch * most);
    if (p.slots < 2 * batch) p.slots = 0;
  }
  return p;
}

int64_t workspace_of(const Plan& p, int batch, int num_nodes, int q_heads, int head_dim) {
  return p.slots ? (int64_t)p.slots * num_nodes * q_heads * (head_dim * 4 + 8) + batch * 8ll : 0;
}

template <int FMT, int D, int PARTS>
void launch(const PagedAttn& a, const Plan& p, hipStream_t s) {
  const int64_t m = (int64_t)(a.Hq / a.pages.kv_heads) * a.N;
  const int m_tiles = (int)((m + p.rows() - 1) / p.rows());
  const dim3 grid((unsigned)((int64_t)(a.slots ? a.slots : a.batch) * a.pages.kv_heads * m_tiles)), block(p.rw * p.kw * 64);
  if (m <= 16)
    hipLaunchKernelGGL((paged_stream_kernel<FMT, D, 1>), grid, block, 0, s, a);
  else if (m <= 32)
    hipLaunchKernelGGL((paged_stream_kernel<FMT, D, 2>), grid, block, 0, s, a);
  else if (p.rw == 2)
    hipLaunchKernelGGL((paged_attn_kernel<FMT, D, 2, 4, 32, false, PARTS>), grid, block, 0, s, a, m_tiles);
  else if (D == 64 || p.rw == 4)
    hipLaunchKernelGGL((paged_attn_kernel<FMT, D, 4, 2, 64, false, PARTS>), grid, block, 0, s, a, m_tiles);
  else if (m <= 192)
    hipLaunchKernelGGL((paged_attn_kernel<FMT, 128, 8, 1, 64, true, PARTS>), grid, block, 0, s, a, m_tiles);
  else
    hipLaunchKernelGGL((paged_attn_kernel<FMT, 128, 8, 1, 64, false, PARTS>), grid, block, 0, s, a, m_tiles);
  if (a.slots) {
    const int64_t rows = (int64_t)a.batch * a.N * a.Hq;
    if (p.wide(a.batch, rows))
      hipLaunchKernelGGL((paged_combine_kernel<D, true>), dim3((unsigned)rows), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((paged_combine_kernel<D, false>), dim3((unsigned)((rows + 1024 / D - 1) / (1024 / D))), dim3(256), 0, s, a);
  }
}

bool sizes_ok(int batch, int num_nodes, int q_heads, int kv_heads, int head_dim) {
  return batch > 0 && num_nodes > 0 && num_nodes <= 8192 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 &&
         (head_dim == 64 || head_dim == 128) && (int64_t)batch * num_nodes < (1ll << 31) / q_heads;
}

template <int PARTS>
int attend(const char* what, const void* q, void* out, const fg_kv_pages* pages, int batch, int num_nodes, int q_heads,
           const int32_t* seq_len, const int32_t* new_len, const int32_t* row_map, const uint64_t* anc,
           int64_t anc_batch_stride, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  const std::string w(what);
  PagedAttn a;
  if (int rc = fg::pages_of(pages, what, a.pages)) return rc;
  FG_REQUIRE(q && out && seq_len, w + ": null pointer");
  FG_REQUIRE(!anc || num_nodes <= 64, w + ": num_nodes must be in [1, 64] with masks, [1, 8192] for a chain");
  FG_REQUIRE(sizes_ok(batch, num_nodes, q_heads, pages->kv_heads, pages->head_dim), w + ": bad shape");
  FG_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 7) == 0, w + ": q must start 16-byte aligned, out 8-byte");
  // Masked scores are minus infinity before they are scaled, and the largest score has to be the largest scaled one.
  FG_REQUIRE(scale > 0.0f && scale * kLog2e < INFINITY, w + ": scale must be positive and finite (times log2 e too)");
  a.q = q;
  a.out = out;
  a.seq_len = seq_len;
  a.new_len = new_len;
  a.row_map = row_map;
  a.anc = anc;
  a.anc_stride = anc_batch_stride;
  a.batch = batch;
  a.N = num_nodes;
  a.Hq = q_heads;
  a.scale = scale;
  Plan p = plan_of(batch, num_nodes, q_heads, pages->kv_heads, pages->head_dim, (int64_t)pages->table_width * pages->page_size);
  const int64_t need = workspace_of(p, batch, num_nodes, q_heads, pages->head_dim);
  if (need && (!workspace || workspace_bytes < (size_t)need || ((uintptr_t)workspace & 15))) p.slots = 0;
  const int64_t m = (int64_t)(q_heads / pages->kv_heads) * num_nodes;
  FG_REQUIRE((int64_t)batch * pages->kv_heads * ((m + p.rows() - 1) / p.rows()) < (1ll << 31),
             w + ": bad shape (too many workgroups)");
  a.slots = p.slots;
  a.most = p.wide(batch, (int64_t)batch * num_nodes * q_heads) ? 256 : pages->head_dim / 4;
  a.o_part = (float*)workspace;
  a.ml_part = (float2*)(a.o_part + (int64_t)p.slots * num_nodes * q_heads * pages->head_dim);
  a.shares = (int2*)(a.ml_part + (int64_t)p.slots * num_nodes * q_heads);
  hipStream_t s = (hipStream_t)stream;
  if (pages->format == kPageE4M3)
    pages->head_dim == 128 ? launch<kPageE4M3, 128, PARTS>(a, p, s) : launch<kPageE4M3, 64, PARTS>(a, p, s);
  else
    pages->head_dim == 128 ? launch<kPageBF16, 128, PARTS>(a, p, s) : launch<kPageBF16, 64, PARTS>(a, p, s);
  return fg::check_launch(what);
}

}  // namespace

extern "C" size_t fg_paged_attention_workspace(int batch, int num_nodes, int q_heads, int kv_heads, int head_dim,
                                               int capacity) {
  if (!sizes_ok(batch, num_nodes, q_heads, kv_heads, head_dim) || capacity <= 0) return 0;
  return (size_t)workspace_of(plan_of(batch, num_nodes, q_heads, kv_heads, head_dim, capacity), batch, num_nodes, q_heads, head_dim);
}

extern "C" int fg_paged_attention(const void* q, void* out, const fg_kv_pages* pages, int batch, int num_nodes,
                                  int q_heads, const int32_t* seq_len, const int32_t* new_len,
                                  const int32_t* row_map, const uint64_t* anc, int64_t anc_batch_stride,
                                  float scale, void* workspace, size_t workspace_bytes, void* stream) {
  return attend<2>("fg_paged_attention", q, out, pages, batch, num_nodes, q_heads, seq_len, new_len, row_map, anc,
                   anc_batch_stride, scale, workspace, workspace_bytes, stream);
}

extern "C" int fg_paged_attention_bf16_weights(const void* q, void* out, const fg_kv_pages* pages, int batch,
                                               int num_nodes, int q_heads, const int32_t* seq_len,
                                               const int32_t* new_len, const int32_t* row_map,
                                               const uint64_t* anc, int64_t anc_batch_stride, float scale,
                                               void* workspace, size_t workspace_bytes, void* stream) {
  return attend<1>("fg_paged_attention_bf16_weights", q, out, pages, batch, num_nodes, q_heads, seq_len, new_len, row_map,
                   anc, anc_batch_stride, scale, workspace, workspace_bytes, stream);
}
