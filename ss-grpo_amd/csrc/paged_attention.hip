// Attention of new tokens over a paged cache (fg_paged.h): N new tokens per sequence (tree nodes with ancestor masks, or a
// causal chain; one token is a chain of one) attend to the committed tokens [0, seq_len[b]) of their cache row and to the new
// ones, which lie behind them (flashgrpo/decoding/tree_attention.py:6-67 and the attention it feeds).
//
//   out[q] = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale log2(e) q . k_j - m),  m the running maximum, one pass over the keys
//
// A row that sees no key is 0. The G = q heads / kv heads rows of a node share every K and V row that is read.
#include "fg_paged.h"

#include <algorithm>

namespace {

using fg::kPageBF16;
using fg::kPageE4M3;
using fg::Pages;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

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
  int splits;  // parts that a sequence's keys may be cut into
  float* o_part;
  float2* ml_part;
};

constexpr float kRescaleSlack = 8.0f;  // log2 units
constexpr int kMinPartKeys = 256;      // a part of a sequence's keys is at least so long

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
// Parts of a sequence's keys, and a part's length (a multiple of `tile`).
FG_DEVICE int part_keys(int keys, int splits, int tile) {
  const int n = min(splits, max(1, (keys + kMinPartKeys - 1) / kMinPartKeys));
  return ((keys + n - 1) / n + tile - 1) / tile * tile;
}

// 16 e4m3 codes times 2^(s - 127) as bf16 (exact).
FG_DEVICE void expand16(uint4 w, uint32_t s, uint4& lo, uint4& hi) {
  const float f = __uint_as_float(s << 23);
  uint32_t r[8];
  const uint32_t c[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], f, false));
    r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], f, true));
  }
  lo = make_uint4(r[0], r[1], r[2], r[3]);
  hi = make_uint4(r[4], r[5], r[6], r[7]);
}

// Whether 16 bytes hold a value that is not finite: e4m3 code 0x7f (or 0xff), bf16 with all exponent bits set.
template <int FMT>
FG_DEVICE bool unusual(uint4 w) {
  const uint32_t keep = FMT == kPageE4M3 ? 0x7f7f7f7fu : 0x7f807f80u, one = FMT == kPageE4M3 ? 0x01010101u : 0x00800080u,
                 top = FMT == kPageE4M3 ? 0x80808080u : 0x80008000u;
  return (((w.x & keep) + one) | ((w.y & keep) + one) | ((w.z & keep) + one) | ((w.w & keep) + one)) & top;
}

// One element of V as a float.
template <int FMT, int D>
FG_DEVICE float v_element(const Pages& pg, int page, int r, int d) {
  const uint8_t* base = pg.v + page * pg.page_bytes;
  if constexpr (FMT == kPageBF16) return fg::bf16_to_f32(((const uint16_t*)base)[(int64_t)r * D + d]);
  const auto x = __builtin_amdgcn_cvt_pk_f32_fp8((int)base[(int64_t)r * D + d], false);
  return x[0] * fg::mx_scale(pg.vs[page * pg.scale_bytes + (int64_t)r * (D / fg::kMxBlock) + d / fg::kMxBlock]);
}

// A workgroup of RW x KW waves takes 32 RW query rows of one (sequence, kv head, part of the keys), row r being head r % G of
// node r / G. Tiles of KB KW keys go through LDS as bf16: every thread fetches 16-byte pieces of K and V rows, expands codes
// (exactly) and stores them. Wave (rw, kw) multiplies rows 32 rw .. with keys KB kw .. of each tile; S^T = K Q^T puts a query
// into a lane, so that the softmax needs one exchange with the other half-wave, and P^T goes from the accumulators straight
// into O^T += V^T P^T. The KW waves of a row tile merge their (m, l, O) at the end through LDS; parts are merged by a second
// kernel.
template <int FMT, int D, int RW, int KW, int KB>
__global__ void __launch_bounds__(RW * KW * 64, 2) paged_attn_kernel(PagedAttn a, int m_tiles) {
  constexpr int T = RW * KW * 64, KT = KB * KW, ROWS = RW * 32;
  constexpr int CPK = D * fg::page_elem_bytes<FMT> / 16;  // 16-byte pieces of a K or V row
  constexpr int PIECES = KT * CPK, NP = 2 * PIECES / T;   // pieces of a tile's K (and of its V), of both per thread
  constexpr int CHUNKS = FMT == kPageBF16 ? 1 : 2;        // 16-byte chunks that a piece is as bf16
  constexpr int KROW = D * 2 + 16, VROW = D * 2;
  constexpr int NB = KB / 32, ND = D / 32, NS = D / 16;
  static_assert(2 * PIECES % T == 0 && NP >= 1 && NP <= 32 && PIECES % 64 == 0, "pieces");
  constexpr int TILE = KT * (KROW + VROW);
  constexpr int MERGE = KW > 1 ? RW * KW * 32 * ((D + 4) * 4 + 8) : 0;
  __shared__ __attribute__((aligned(16))) unsigned char lds[TILE > MERGE ? TILE : MERGE];
  __shared__ uint64_t odd_keys[2][(KT + 63) / 64], no_page[2][(KT + 63) / 64];
  unsigned char* const kt = lds;
  unsigned char* const vt = lds + KT * KROW;

  const Pages& pg = a.pages;
  const int unit = blockIdx.x / m_tiles, mt = blockIdx.x % m_tiles;
  const int sp = unit % a.splits, hkv = unit / a.splits % pg.kv_heads, b = unit / (a.splits * pg.kv_heads);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5, l32 = lane & 31;
  const int rw = wave % RW, kw = wave / RW;
  const int G = a.Hq / pg.kv_heads;
  const Span seq = span_of(a, b);
  const int M = G * seq.fresh;
  if (mt * ROWS >= M) return;  // rows behind the sequence's new tokens stay as they are
  const int keys = keys_of(a, seq);
  const int part = part_keys(keys, a.splits, KT);
  const int last = a.anc ? seq.fresh : (min((mt + 1) * ROWS, M) - 1) / G + 1;  // a chain's rows see no later token
  const int begin = min(sp * part, keys);
  const int end = max(begin, min(min(begin + part, keys), seq.committed + last));
  const int s0 = seq.committed;
  const int32_t* trow = pg.table + (int64_t)max(seq.row, 0) * pg.table_stride;

  const int row0 = mt * ROWS + rw * 32, r = row0 + l32;
  const bool row_ok = r < M;
  const int qn = row_ok ? r / G : 0, qh = hkv * G + (row_ok ? r % G : 0);
  const uint64_t anc = (row_ok && a.anc) ? a.anc[(int64_t)b * a.anc_stride + qn] : 0ull;
  const uint64_t bits = anc & low_bits(seq.fresh);
  bf16x8 qf[NS];
  {
    const uint16_t* qrow = (const uint16_t*)a.q + (((int64_t)b * a.N + qn) * a.Hq + qh) * D;
#pragma unroll
    for (int s = 0; s < NS; ++s)
      qf[s] = __builtin_bit_cast(bf16x8, row_ok ? *(const uint4*)(qrow + s * 16 + g * 8) : make_uint4(0, 0, 0, 0));
  }
  floatx16 o[ND];
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;
  const float sl2 = a.scale * 1.44269504088896341f;
  const bf16x2 ones2 = __builtin_bit_cast(bf16x2, 0x3f803f80u);

  const uint32_t k_lane = (uint32_t)((kw * KB + l32) * KROW + g * 16);
  // V^T fragments by transposed reads, as laid out in v_chunk below: lane 16 gq + i addresses key 4 (gq / 2) + i / 4 and d
  // 32 db + 16 (gq % 2) + 4 (i % 4), and receives keys 4 (lane / 32) + j (and 8 + ..) of d = 32 db + lane % 32.
  auto v_swizzle = [](int key) { return D == 128 ? 4 * (key & 3) : 4 * ((key >> 1) & 1); };
  uint32_t v_lane[ND];
  {
    const int gq = lane >> 4, i = lane & 15, key = 4 * (gq >> 1) + (i >> 2);
    const int low = 2 * (gq & 1) + ((i & 3) >> 1);
#pragma unroll
    for (int db = 0; db < ND; ++db)
      v_lane[db] = (uint32_t)((kw * KB + key) * VROW + (((4 * db + low) ^ v_swizzle(key)) * 16) + 8 * (i & 1));
  }

  if (tid < 2 * ((KT + 63) / 64)) (&odd_keys[0][0])[tid] = 0, (&no_page[0][0])[tid] = 0;
  uint4 piece[NP];
  uint32_t scale[NP], held = 0;  // held: bit u, piece u's token is in the part and has a page
  auto fetch = [&](int key0) __attribute__((always_inline)) {
    held = 0;
#pragma unroll
    for (int u = 0; u < NP; ++u) {
      const int i = u * T + tid;
      const bool is_v = i >= PIECES;
      const int j = (is_v ? i - PIECES : i) / CPK, c = i % CPK;
      const int key = min(key0 + j, end - 1), page = pg.page(trow, key);  // loads are unconditional, from a place that exists
      held |= (uint32_t)(key0 + j < end && page >= 0) << u;
      const int64_t p = max(page, 0), row = pg.row_in_page(hkv, key);
      piece[u] = *(const uint4*)((is_v ? pg.v : pg.k) + p * pg.page_bytes + row * (CPK * 16) + c * 16);
      if constexpr (FMT == kPageE4M3) scale[u] = (is_v ? pg.vs : pg.ks)[p * pg.scale_bytes + row * (D / 32) + c / 2];
    }
  };
  // Rows behind the part's end are 0; so is V where it is not finite (its products with p = 0 must stay 0), which the tile's
  // odd_keys bits tell, and keys that have no page (no_page bits).
  auto put = [&](int key0, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NP; ++u) {
      const int i = u * T + tid;
      const bool is_v = i >= PIECES, ok = (held >> u) & 1u;
      const int j = (is_v ? i - PIECES : i) / CPK, c = i % CPK;
      uint4 w = piece[u];
      bool bad = false;
      if constexpr (FMT == kPageE4M3) bad = scale[u] == 255u;
      if (is_v) {
        bad |= unusual<FMT>(w);
        if (ok && bad) atomicOr((unsigned long long*)&odd_keys[slot][j >> 6], 1ull << (j & 63));
        if (bad) w = make_uint4(0, 0, 0, 0);
      } else if (!ok && c == 0 && key0 + j < end) {
        atomicOr((unsigned long long*)&no_page[slot][j >> 6], 1ull << (j & 63));
      }
      if (!ok) w = make_uint4(0, 0, 0, 0);
      unsigned char* dst = is_v ? vt + j * VROW : kt + j * KROW;
      const int c0 = is_v ? (c * CHUNKS) ^ v_swizzle(j) : c * CHUNKS;
      if constexpr (FMT == kPageE4M3) {
        uint4 lo, hi;
        expand16(w, bad || !ok ? 127u : scale[u], lo, hi);
        if (!is_v && ok && bad) lo = hi = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
        *(uint4*)(dst + c0 * 16) = lo;
        *(uint4*)(dst + c0 * 16 + 16) = hi;
      } else {
        *(uint4*)(dst + c0 * 16) = w;
      }
    }
  };

  auto compute = [&](int key0, int slot) __attribute__((always_inline)) {
    const int first = key0 + kw * KB;  // this wave's keys
    bf16x8 kf[NB * NS];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int s = 0; s < NS; ++s) kf[kb * NS + s] = *(const bf16x8*)(kt + k_lane + kb * 32 * KROW + s * 32);
    floatx16 sc[NB];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[kb][i] = 0.0f;
#pragma unroll
      for (int s = 0; s < NS; ++s)
        sc[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kb * NS + s], qf[s], sc[kb], 0, 0, 0);
    }
    uint64_t odd = odd_keys[slot][kw * KB / 64], gone = no_page[slot][kw * KB / 64];
    if (KB < 64) {
      odd = (odd >> (kw * KB % 64)) & low_bits(KB);
      gone = (gone >> (kw * KB % 64)) & low_bits(KB);
    }
    const uint64_t sees = a.anc ? seen_mask(s0 - first, bits) : low_bits(s0 + qn + 1 - first);
    const uint64_t allowed = sees & low_bits(end - first) & ~gone;
    if (first + KB > s0 || first + KB > end || gone) {
      const uint64_t mine = allowed >> (g * 4);
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
    float psum = l_run;
    bf16x8 pf[NB][2];
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
          // the sum is that of the rounded p, the ones that multiply V
          psum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, packed[j / 2]), ones2, psum, false);
        }
        pf[kb][ks] = __builtin_bit_cast(bf16x8, make_uint4(packed[0], packed[1], packed[2], packed[3]));
      }
    l_run = psum;
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const unsigned char* p0 = vt + v_lane[db] + (kb * 2 + ks) * 16 * VROW;
          const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)p0);
          const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p0 + 8 * VROW));
          const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
          o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[kb][ks], o[db], 0, 0, 0);
        }
    // Infinities and NaN of V reach only the rows that see their key.
    while (odd) {
      const int j = __builtin_ctzll(odd);
      odd &= odd - 1;
      if (!((allowed >> j) & 1ull)) continue;
      const int page = pg.page(trow, first + j), row = pg.row_in_page(hkv, first + j);
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = v_element<FMT, D>(pg, page, row, db * 32 + c_row32(i, lane));
          if (!(fabsf(x) < INFINITY)) o[db][i] += x;
        }
    }
  };

  __syncthreads();
  const int ntiles = (end - begin + KT - 1) / KT;
  for (int t = 0; t < ntiles; ++t) {
    const int key0 = begin + t * KT, slot = t & 1;
    fetch(key0);
    __syncthreads();  // every wave is done with the tile before
    put(key0, slot);
    if (tid < (KT + 63) / 64) odd_keys[slot ^ 1][tid] = 0, no_page[slot ^ 1][tid] = 0;
    __syncthreads();
    if (row0 < M) compute(key0, slot);
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
      if (a.splits > 1) {
        const int64_t prow = (int64_t)sp * a.batch * a.N * a.Hq + orow;
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
    if (a.splits > 1) {
      const int64_t prow = (int64_t)sp * a.batch * a.N * a.Hq + orow;
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

// The parts of a row, in order: D / 4 lanes per row, 4 dims each. Parts that saw no key (m = -inf) weigh nothing.
template <int D>
__global__ void __launch_bounds__(256) paged_combine_kernel(PagedAttn a, int tile) {
  constexpr int LANES = D / 4;
  const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int64_t rows = (int64_t)a.batch * a.N * a.Hq;
  if (row >= rows) return;
  const int n = (int)(row / a.Hq % a.N), b = (int)(row / a.Hq / a.N), d0 = threadIdx.x % LANES * 4;
  const Span seq = span_of(a, b);
  if (n >= seq.fresh) return;
  const int keys = keys_of(a, seq), part = part_keys(keys, a.splits, tile);
  const int parts = part > 0 ? min(a.splits, (keys + part - 1) / part) : 0;
  float mx = -INFINITY;
  for (int p = 0; p < parts; ++p) mx = fmaxf(mx, a.ml_part[p * rows + row].x);
  float den = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int p = 0; p < parts; ++p) {
    const float2 ml = a.ml_part[p * rows + row];
    if (ml.y == 0.0f) continue;
    const float w = __builtin_amdgcn_exp2f(ml.x - (mx == -INFINITY ? 0.0f : mx));
    const float4 x = *(const float4*)(a.o_part + (p * rows + row) * D + d0);
    den += w * ml.y;
    o[0] += w * x.x; o[1] += w * x.y; o[2] += w * x.z; o[3] += w * x.w;
  }
  const float inv = den == 0.0f ? 0.0f : 1.0f / den;
  *(uint2*)((uint16_t*)a.out + row * D + d0) =
      make_uint2(fg::pack_bf16x2(o[0] * inv, o[1] * inv), fg::pack_bf16x2(o[2] * inv, o[3] * inv));
}

struct Plan {
  int rw, kw, kb, splits;
  int rows() const { return rw * 32; }
  int tile() const { return kw * kb; }
};

Plan plan_of(int batch, int num_nodes, int q_heads, int kv_heads, int64_t capacity) {
  const int64_t m = (int64_t)(q_heads / kv_heads) * num_nodes;
  Plan p;
  if (m <= 32) p = {1, 4, 32, 1};
  else if (m <= 128) p = {4, 1, 64, 1};
  else p = {8, 1, 64, 1};
  const int64_t base = (int64_t)batch * kv_heads * ((m + p.rows() - 1) / p.rows());
  const int64_t target = 256 * (8 / (p.rw * p.kw));
  if (base < target) {
    const int64_t most = std::max<int64_t>(1, capacity / kMinPartKeys);
    p.splits = (int)std::min<int64_t>(std::min<int64_t>((target + base - 1) / base, most), 64);
  }
  return p;
}

int64_t workspace_of(const Plan& p, int batch, int num_nodes, int q_heads, int head_dim) {
  if (p.splits <= 1) return 0;
  return (int64_t)p.splits * batch * num_nodes * q_heads * (head_dim * 4 + 8);
}

template <int FMT, int D>
void launch(const PagedAttn& a, const Plan& p, hipStream_t s) {
  const int64_t m = (int64_t)(a.Hq / a.pages.kv_heads) * a.N;
  const int m_tiles = (int)((m + p.rows() - 1) / p.rows());
  const dim3 grid((unsigned)((int64_t)a.batch * a.pages.kv_heads * a.splits * m_tiles)), block(p.rw * p.kw * 64);
  if (p.rw == 1)
    hipLaunchKernelGGL((paged_attn_kernel<FMT, D, 1, 4, 32>), grid, block, 0, s, a, m_tiles);
  else if (p.rw == 4)
    hipLaunchKernelGGL((paged_attn_kernel<FMT, D, 4, 1, 64>), grid, block, 0, s, a, m_tiles);
  else
    hipLaunchKernelGGL((paged_attn_kernel<FMT, D, 8, 1, 64>), grid, block, 0, s, a, m_tiles);
  if (a.splits > 1) {
    const int64_t rows = (int64_t)a.batch * a.N * a.Hq;
    const int per = 256 / (D / 4);
    hipLaunchKernelGGL(paged_combine_kernel<D>, dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, s, a, p.tile());
  }
}

bool sizes_ok(int batch, int num_nodes, int q_heads, int kv_heads, int head_dim) {
  return batch > 0 && num_nodes > 0 && num_nodes <= 8192 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 &&
         (head_dim == 64 || head_dim == 128) && (int64_t)batch * num_nodes < (1ll << 31) / q_heads;
}

}  // namespace

extern "C" size_t fg_paged_attention_workspace(int batch, int num_nodes, int q_heads, int kv_heads, int head_dim,
                                               int capacity) {
  if (!sizes_ok(batch, num_nodes, q_heads, kv_heads, head_dim) || capacity <= 0) return 0;
  return (size_t)workspace_of(plan_of(batch, num_nodes, q_heads, kv_heads, capacity), batch, num_nodes, q_heads, head_dim);
}

extern "C" int fg_paged_attention(const void* q, void* out, const fg_kv_pages* pages, int batch, int num_nodes,
                                  int q_heads, const int32_t* seq_len, const int32_t* new_len, const int32_t* row_map,
                                  const uint64_t* anc, int64_t anc_batch_stride, float scale, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  PagedAttn a;
  if (int rc = fg::pages_of(pages, "fg_paged_attention", a.pages)) return rc;
  FG_REQUIRE(q && out && seq_len, "fg_paged_attention: null pointer");
  FG_REQUIRE(!anc || num_nodes <= 64, "fg_paged_attention: num_nodes must be in [1, 64] with masks, [1, 8192] for a chain");
  FG_REQUIRE(sizes_ok(batch, num_nodes, q_heads, pages->kv_heads, pages->head_dim), "fg_paged_attention: bad shape");
  FG_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 7) == 0, "fg_paged_attention: q must start 16-byte aligned, out 8-byte");
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
  Plan p = plan_of(batch, num_nodes, q_heads, pages->kv_heads, (int64_t)pages->table_width * pages->page_size);
  const int64_t need = workspace_of(p, batch, num_nodes, q_heads, pages->head_dim);
  if (need && (!workspace || workspace_bytes < (size_t)need || ((uintptr_t)workspace & 15))) p.splits = 1;
  const int64_t m = (int64_t)(q_heads / pages->kv_heads) * num_nodes;
  FG_REQUIRE((int64_t)batch * pages->kv_heads * p.splits * ((m + p.rows() - 1) / p.rows()) < (1ll << 31),
             "fg_paged_attention: bad shape (too many workgroups)");
  a.splits = p.splits;
  a.o_part = (float*)workspace;
  a.ml_part = (float2*)((char*)workspace + (int64_t)p.splits * batch * num_nodes * q_heads * pages->head_dim * 4);
  hipStream_t s = (hipStream_t)stream;
  if (pages->format == kPageE4M3)
    pages->head_dim == 128 ? launch<kPageE4M3, 128>(a, p, s) : launch<kPageE4M3, 64>(a, p, s);
  else
    pages->head_dim == 128 ? launch<kPageBF16, 128>(a, p, s) : launch<kPageBF16, 64>(a, p, s);
  return fg::check_launch("fg_paged_attention");
}
