// The paged KV cache (fg_paged.h) beside the attention that reads it: rotary positions with the K/V write into pages,
// which quantises as it writes, the values read back, and the accepted path's compaction. They stand where a contiguous
// cache has fg_rope_kv_write, its rows themselves and fg_kv_path_gather (flashgrpo/models/qwen_flashgrpo_wrapper.py:172-180,
// flashgrpo/decoding/kv_extraction.py:54-84).
#include "fg_paged.h"

namespace {

using fg::kPageBF16;
using fg::kPageE4M3;
using fg::Pages;

constexpr int kThreads = 256;

// Four consecutive bf16 as floats.
FG_DEVICE void load4(const void* p, int64_t i, float (&v)[4]) {
  const uint2 r = *(const uint2*)((const uint16_t*)p + i);
  v[0] = __uint_as_float(r.x << 16);
  v[1] = __uint_as_float(r.x & 0xffff0000u);
  v[2] = __uint_as_float(r.y << 16);
  v[3] = __uint_as_float(r.y & 0xffff0000u);
}
FG_DEVICE void store4(void* p, int64_t i, const float (&v)[4]) {
  *(uint2*)((uint16_t*)p + i) = make_uint2(fg::pack_bf16x2(v[0], v[1]), fg::pack_bf16x2(v[2], v[3]));
}

// A token's projected row: bf16, or the fp32 split-K parts of the projection summed in split order, plus the bias, rounded to
// bf16 as the projection's output would be.
template <bool PARTS>
struct Rows {
  const void* qkv;
  const float* part;
  int64_t part_stride;
  int splits;
  const void* bias;

  FG_DEVICE void get4(int64_t row, int col, float (&v)[4]) const {
    if constexpr (!PARTS) {
      load4(qkv, row + col, v);
    } else {
      const float* src = part + row + col;
      float4 a = *(const float4*)src;
      for (int s = 1; s < splits; ++s) {
        const float4 b = *(const float4*)(src + s * part_stride);
        a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
      }
      float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (bias) load4(bias, col, c);
      v[0] = fg::round_bf16(a.x + c[0]);
      v[1] = fg::round_bf16(a.y + c[1]);
      v[2] = fg::round_bf16(a.z + c[2]);
      v[3] = fg::round_bf16(a.w + c[3]);
    }
  }
};

struct WriteArgs {
  Pages pages;
  int64_t ld;
  int N, Hq;
  const int32_t* seq_len;
  const int32_t* pos_offset;
  int64_t pos_stride;
  const float* inv_freq;
  const int32_t* new_len;
  const int32_t* row_map;
  void* q_out;
  int32_t* err_flag;
};

FG_DEVICE uint32_t group8_max(uint32_t a) {  // over 8 neighbouring lanes
  a = max(a, (uint32_t)__shfl_xor((int)a, 1, 64));
  a = max(a, (uint32_t)__shfl_xor((int)a, 2, 64));
  return max(a, (uint32_t)__shfl_xor((int)a, 4, 64));
}

// Four values of a block whose largest magnitude's bits are `amax`: their e4m3 codes; the block's scale byte by `s`.
FG_DEVICE uint32_t quantize4(const float (&v)[4], uint32_t amax, uint32_t& s) {
  s = fg::mx_scale_byte<fg::kE4M3>(amax);
  const float inv = fg::mx_inverse_scale(s);
  int c = 0;
  c = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, c, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, c, true);
}
FG_DEVICE uint32_t amax4(const float (&v)[4]) {
  uint32_t a = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) a = max(a, __float_as_uint(v[j]) & 0x7fffffffu);
  return a;
}

// One workgroup per token: position seq_len[b] + pos_offset, slot seq_len[b] + n. bf16 pages get the values of
// fg_rope_kv_write (every product and sum rounded to bf16, cos and sin too). e4m3 pages: q is rotated in fp32 and rounded once; the
// angles are taken in 64 bits (of an angle of 10^5 radians fp32 keeps 2 decimals), and so is K's rotation (512 elements a
// token, hidden behind the row's loads), which is rounded to fp32 and quantised from there: codes are those of the 64-bit
// definition but where a value is within half an fp32 step of a tie, which it then falls on.
// Memory bounds it: 2944 tokens at 8B (66 MB) 16 us, 4.2 TB/s of the 4.9 that a large copy reaches; 64 x 29 at 7B (32 MB) 8.8 us;
// one token 2.7 us, its length, its page and its row one after the other.
template <int FMT, int D, bool PARTS>
__global__ void __launch_bounds__(kThreads) paged_write_kernel(WriteArgs a, Rows<PARTS> in) {
  constexpr int HALF = D / 2, QUADS = HALF / 4, BLOCKS = D / fg::kMxBlock;
  __shared__ double cs[HALF], sn[HALF];
  const int tok = blockIdx.x, b = tok / a.N, n = tok % a.N;
  if (a.new_len && n >= a.new_len[b]) return;
  const Pages& pg = a.pages;
  const int s = a.seq_len[b];
  const int cb = a.row_map ? a.row_map[b] : b;
  const int slot = (unsigned)s < (1u << 31) - 65536u ? s + n : -1;
  int page = -1;
  if ((unsigned)cb < (unsigned)pg.table_rows && slot >= 0 && slot < pg.capacity())
    page = pg.page(pg.table + (int64_t)cb * pg.table_stride, slot);
  if (page < 0 && threadIdx.x == 0 && a.err_flag) atomicOr(a.err_flag, 8);
  if (threadIdx.x < HALF) {
    const int off = a.pos_offset[(int64_t)b * a.pos_stride + n];
    const float f = a.inv_freq[threadIdx.x];
    if constexpr (FMT == kPageE4M3) {
      const double turns = (double)((int64_t)s + off) * (double)f * 0.15915494309189533577;  // / 2 pi
      double sv, cv;
      sincospi(2.0 * (turns - rint(turns)), &sv, &cv);
      cs[threadIdx.x] = cv;
      sn[threadIdx.x] = sv;
    } else {
      const float ang = (float)((int64_t)s + off) * f;
      cs[threadIdx.x] = fg::round_bf16(cosf(ang));
      sn[threadIdx.x] = fg::round_bf16(sinf(ang));
    }
  }
  __syncthreads();
  const int64_t row = (int64_t)tok * a.ld;
  const int Hq = a.Hq, Hkv = pg.kv_heads;
  // 4 pairs (i, i + d/2) of a q or k head per thread; the threads of a head are neighbours
  for (int e = threadIdx.x; e < (Hq + Hkv) * QUADS; e += kThreads) {
    const int h = e / QUADS, i0 = (e % QUADS) * 4;
    float x1[4], x2[4], y1[4], y2[4];
    in.get4(row, h * D + i0, x1);
    in.get4(row, h * D + i0 + HALF, x2);
    if (FMT == kPageE4M3 && h >= Hq) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double c = cs[i0 + j], v = sn[i0 + j];
        y1[j] = (float)((double)x1[j] * c - (double)x2[j] * v);
        y2[j] = (float)((double)x2[j] * c + (double)x1[j] * v);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma clang fp contract(off)
        const float c = (float)cs[i0 + j], v = (float)sn[i0 + j];
        if constexpr (FMT == kPageE4M3) {
          y1[j] = fmaf(x1[j], c, -(x2[j] * v));
          y2[j] = fmaf(x2[j], c, x1[j] * v);
        } else {
          y1[j] = fg::round_bf16(fg::round_bf16(x1[j] * c) - fg::round_bf16(x2[j] * v));
          y2[j] = fg::round_bf16(fg::round_bf16(x2[j] * c) + fg::round_bf16(x1[j] * v));
        }
      }
    }
    if (h < Hq) {
      const int64_t dst = ((int64_t)tok * Hq + h) * D;
      store4(a.q_out, dst + i0, y1);
      store4(a.q_out, dst + i0 + HALF, y2);
      continue;
    }
    const int r = pg.row_in_page(h - Hq, slot);
    if constexpr (FMT == kPageBF16) {
      if (page < 0) continue;
      uint16_t* dst = (uint16_t*)(pg.k + pg.at(page)) + (int64_t)r * D;
      store4(dst, i0, y1);
      store4(dst, i0 + HALF, y2);
    } else {
      uint32_t s1, s2;  // 8 lanes hold a block of either half
      const uint32_t c1 = quantize4(y1, group8_max(amax4(y1)), s1);
      const uint32_t c2 = quantize4(y2, group8_max(amax4(y2)), s2);
      if (page < 0) continue;
      uint8_t* dst = pg.k + pg.at(page) + (int64_t)r * D;
      *(uint32_t*)(dst + i0) = c1;
      *(uint32_t*)(dst + i0 + HALF) = c2;
      if (i0 % fg::kMxBlock == 0) {
        uint8_t* sc = pg.ks + pg.scales_at(page) + (int64_t)r * BLOCKS;
        sc[i0 / fg::kMxBlock] = (uint8_t)s1;
        sc[(i0 + HALF) / fg::kMxBlock] = (uint8_t)s2;
      }
    }
  }
  for (int e = threadIdx.x; e < Hkv * (D / 4); e += kThreads) {
    const int h = e / (D / 4), i0 = (e % (D / 4)) * 4;
    float x[4];
    in.get4(row, (Hq + Hkv + h) * D + i0, x);
    const int r = pg.row_in_page(h, slot);
    if constexpr (FMT == kPageBF16) {
      if (page >= 0) store4(pg.v + pg.at(page), (int64_t)r * D + i0, x);
    } else {
      uint32_t s1;
      const uint32_t c = quantize4(x, group8_max(amax4(x)), s1);
      if (page < 0) continue;
      *(uint32_t*)(pg.v + pg.at(page) + (int64_t)r * D + i0) = c;
      if (i0 % fg::kMxBlock == 0) pg.vs[pg.scales_at(page) + (int64_t)r * BLOCKS + i0 / fg::kMxBlock] = (uint8_t)s1;
    }
  }
}

// The values of 8 elements of a row; tokens without a page are 0. (4 x 1024 tokens at 8B, 25 MB: 7.3 to 9.4 us, 1.5 times what a copy's
// rate allows: 8-byte loads; a few tokens 2 us, the latency of the page and the row.)
template <int FMT, int D, int DT>
__global__ void __launch_bounds__(kThreads) paged_read_kernel(Pages pg, int batch, const int32_t* start, int count,
                                                              const int32_t* row_map, void* k_out, void* v_out) {
  constexpr int OCT = D / 8;
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t rows = (int64_t)batch * pg.kv_heads * count;
  if (id >= rows * OCT * 2) return;
  const bool is_v = id >= rows * OCT;
  const int64_t r = (is_v ? id - rows * OCT : id) / OCT;
  const int c = (int)(id % OCT) * 8;
  const int j = (int)(r % count), h = (int)(r / count % pg.kv_heads), b = (int)(r / count / pg.kv_heads);
  const int cb = row_map ? row_map[b] : b;
  const int64_t t = (start ? (int64_t)start[b] : 0) + j;
  int page = -1;
  if ((unsigned)cb < (unsigned)pg.table_rows && t >= 0 && t < pg.capacity())
    page = pg.page(pg.table + (int64_t)cb * pg.table_stride, (int)t);
  float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (page >= 0) {
    const int row = pg.row_in_page(h, (int)t);
    const uint8_t* base = (is_v ? pg.v : pg.k) + pg.at(page);
    if constexpr (FMT == kPageBF16) {
      fg::load8<fg::kBF16>(base, (int64_t)row * D + c, x);
    } else {
      const uint2 w = *(const uint2*)(base + (int64_t)row * D + c);
      const uint8_t* sc = (is_v ? pg.vs : pg.ks) + pg.scales_at(page);
      const float f = fg::mx_scale(sc[(int64_t)row * (D / fg::kMxBlock) + c / fg::kMxBlock]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t d = i ? w.y : w.x;
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)d, false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)d, true);
        x[4 * i] = lo[0] * f;
        x[4 * i + 1] = lo[1] * f;
        x[4 * i + 2] = hi[0] * f;
        x[4 * i + 3] = hi[1] * f;
      }
    }
  }
  fg::store8<DT>(is_v ? v_out : k_out, r * D + c, x);
}

// As kv_path_gather_kernel: a thread owns one column (16 bytes of codes, or the row's scales) of one (layer, K or V, sequence,
// kv head) and reads all its accepted rows before it writes any, so moves may overlap. Three dependent reads bound it, the path and
// lengths, the pages, the rows: 6.0 us for 64 rounds at 7B, 5.2 for 32 at 1.5B.
struct GatherArgs {
  Pages pages;
  int layers, batch, cols;  // cols: 16-byte columns of a row, and one more for its scales (e4m3)
  int64_t layer_bytes, scale_layer_bytes;
  const int32_t* seq_len;
  const int32_t* row_map;
  const int32_t* acc_nodes;
  int acc_stride;
  const int32_t* acc_len;
  int tree_nodes;
  int32_t* err_flag;
};

template <int FMT, int D, int MAXACC>
__global__ void __launch_bounds__(kThreads) paged_path_gather_kernel(GatherArgs a, int total) {
  constexpr int ROW = D * fg::page_elem_bytes<FMT>, BLOCKS = D / fg::kMxBlock;
  const int gid = blockIdx.x * kThreads + threadIdx.x;
  if (gid >= total) return;
  const Pages& pg = a.pages;
  const int col = gid % a.cols;
  int r = gid / a.cols;
  const int h = r % pg.kv_heads;
  r /= pg.kv_heads;
  const int b = r % a.batch, t = r / a.batch;  // t: 2 * layer + (V)
  const int n_acc = a.acc_len[b], s0 = a.seq_len[b], cb = a.row_map ? a.row_map[b] : b;
  const int32_t* nodes = a.acc_nodes + (int64_t)b * a.acc_stride;
  int nd[MAXACC];
#pragma unroll
  for (int j = 0; j < MAXACC; ++j) nd[j] = j < a.acc_stride ? nodes[j] : j;
  bool ok = n_acc >= 1 && n_acc <= a.acc_stride && n_acc <= a.tree_nodes && (unsigned)cb < (unsigned)pg.table_rows &&
            s0 >= 0 && s0 <= pg.capacity() - a.tree_nodes;
#pragma unroll
  for (int j = 0; j < MAXACC; ++j) {
    ok &= j >= n_acc || (nd[j] >= 0 && nd[j] < a.tree_nodes);
    nd[j] = j < n_acc ? nd[j] : j;
  }
  const int32_t* row = pg.table + (int64_t)cb * pg.table_stride;
  int from[MAXACC], to[MAXACC];
#pragma unroll
  for (int j = 0; j < MAXACC; ++j) {
    from[j] = to[j] = 0;
    if (ok && nd[j] != j) {
      from[j] = pg.page(row, s0 + nd[j]);
      to[j] = pg.page(row, s0 + j);
    }
  }
#pragma unroll
  for (int j = 0; j < MAXACC; ++j) ok &= from[j] >= 0 && to[j] >= 0;
  if (!ok) {
    if (t == 0 && h == 0 && col == 0 && a.err_flag) atomicOr(a.err_flag, 1);
    return;
  }
  const bool is_v = t & 1;
  if (FMT == kPageE4M3 && col == a.cols - 1) {
    uint8_t* base = (is_v ? pg.vs : pg.ks) + (int64_t)(t >> 1) * a.scale_layer_bytes;
    uint32_t v[MAXACC];
    typedef typename std::conditional<BLOCKS == 4, uint32_t, uint16_t>::type S;
#pragma unroll
    for (int j = 0; j < MAXACC; ++j)
      v[j] = nd[j] != j ? *(const S*)(base + pg.scales_at(from[j]) + pg.row_in_page(h, s0 + nd[j]) * BLOCKS) : 0u;
#pragma unroll
    for (int j = 0; j < MAXACC; ++j)
      if (nd[j] != j) *(S*)(base + pg.scales_at(to[j]) + pg.row_in_page(h, s0 + j) * BLOCKS) = (S)v[j];
    return;
  }
  uint8_t* base = (is_v ? pg.v : pg.k) + (int64_t)(t >> 1) * a.layer_bytes + col * 16;
  uint4 v[MAXACC];
#pragma unroll
  for (int j = 0; j < MAXACC; ++j)
    v[j] = nd[j] != j ? *(const uint4*)(base + pg.at(from[j]) + (int64_t)pg.row_in_page(h, s0 + nd[j]) * ROW)
                      : make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < MAXACC; ++j)
    if (nd[j] != j) *(uint4*)(base + pg.at(to[j]) + (int64_t)pg.row_in_page(h, s0 + j) * ROW) = v[j];
}

template <bool PARTS>
int launch_write(const char* what, const fg_kv_pages* pages, int batch, int num_nodes, int q_heads, int64_t ld,
                 const int32_t* seq_len, const int32_t* pos_offset, int64_t pos_batch_stride, const float* inv_freq,
                 const int32_t* new_len, const int32_t* row_map, void* q_out, int32_t* err_flag, Rows<PARTS> in,
                 void* stream) {
  const std::string w(what);
  WriteArgs a;
  if (int rc = fg::pages_of(pages, what, a.pages)) return rc;
  FG_REQUIRE(seq_len && pos_offset && inv_freq && q_out, w + ": null pointer");
  FG_REQUIRE(batch > 0 && num_nodes > 0 && num_nodes <= 8192 && q_heads > 0 && (int64_t)batch * num_nodes < (1ll << 31),
             w + ": bad shape");
  FG_REQUIRE((int64_t)(q_heads + 2 * (int64_t)pages->kv_heads) * pages->head_dim < (1ll << 30) &&
                 ld >= (int64_t)(q_heads + 2 * pages->kv_heads) * pages->head_dim && ld % 4 == 0,
             w + ": rows must be apart, their stride a multiple of 4");
  FG_REQUIRE(((uintptr_t)q_out & 7) == 0, w + ": q_out must start 8-byte aligned");
  a.ld = ld;
  a.N = num_nodes;
  a.Hq = q_heads;
  a.seq_len = seq_len;
  a.pos_offset = pos_offset;
  a.pos_stride = pos_batch_stride;
  a.inv_freq = inv_freq;
  a.new_len = new_len;
  a.row_map = row_map;
  a.q_out = q_out;
  a.err_flag = err_flag;
  const dim3 grid((unsigned)(batch * num_nodes)), block(kThreads);
  hipStream_t s = (hipStream_t)stream;
  if (pages->format == kPageE4M3) {
    if (pages->head_dim == 128)
      hipLaunchKernelGGL((paged_write_kernel<kPageE4M3, 128, PARTS>), grid, block, 0, s, a, in);
    else
      hipLaunchKernelGGL((paged_write_kernel<kPageE4M3, 64, PARTS>), grid, block, 0, s, a, in);
  } else {
    if (pages->head_dim == 128)
      hipLaunchKernelGGL((paged_write_kernel<kPageBF16, 128, PARTS>), grid, block, 0, s, a, in);
    else
      hipLaunchKernelGGL((paged_write_kernel<kPageBF16, 64, PARTS>), grid, block, 0, s, a, in);
  }
  return fg::check_launch(what);
}

}  // namespace

extern "C" int fg_rope_kv_write_paged(const void* qkv, int64_t ld_qkv, int batch, int num_nodes, int q_heads,
                                      const fg_kv_pages* pages, const int32_t* seq_len, const int32_t* pos_offset,
                                      int64_t pos_batch_stride, const float* inv_freq, const int32_t* new_len,
                                      const int32_t* row_map, void* q_out, int32_t* err_flag, void* stream) {
  FG_REQUIRE(qkv, "fg_rope_kv_write_paged: null pointer");
  FG_REQUIRE(((uintptr_t)qkv & 7) == 0, "fg_rope_kv_write_paged: qkv must start 8-byte aligned");
  return launch_write<false>("fg_rope_kv_write_paged", pages, batch, num_nodes, q_heads, ld_qkv, seq_len, pos_offset,
                             pos_batch_stride, inv_freq, new_len, row_map, q_out, err_flag,
                             Rows<false>{qkv, nullptr, 0, 0, nullptr}, stream);
}

extern "C" int fg_rope_kv_write_paged_parts(const float* part, int splits, const void* bias, int batch, int num_nodes,
                                            int q_heads, const fg_kv_pages* pages, const int32_t* seq_len,
                                            const int32_t* pos_offset, int64_t pos_batch_stride, const float* inv_freq,
                                            const int32_t* new_len, const int32_t* row_map, void* q_out,
                                            int32_t* err_flag, void* stream) {
  FG_REQUIRE(part && pages, "fg_rope_kv_write_paged_parts: null pointer");
  FG_REQUIRE(splits > 0 && ((uintptr_t)part & 15) == 0 && ((uintptr_t)bias & 7) == 0,
             "fg_rope_kv_write_paged_parts: splits must be positive, parts 16-byte and bias 8-byte aligned");
  const int64_t width = (int64_t)(q_heads + 2 * (int64_t)pages->kv_heads) * pages->head_dim;
  return launch_write<true>("fg_rope_kv_write_paged_parts", pages, batch, num_nodes, q_heads, width, seq_len, pos_offset,
                            pos_batch_stride, inv_freq, new_len, row_map, q_out, err_flag,
                            Rows<true>{nullptr, part, (int64_t)batch * num_nodes * width, splits, bias}, stream);
}

extern "C" int fg_kv_read_paged(const fg_kv_pages* pages, int batch, const int32_t* start, int count,
                                const int32_t* row_map, void* k_out, void* v_out, int dtype, void* stream) {
  Pages pg;
  if (int rc = fg::pages_of(pages, "fg_kv_read_paged", pg)) return rc;
  FG_REQUIRE(k_out && v_out, "fg_kv_read_paged: null pointer");
  FG_REQUIRE(batch > 0 && count > 0, "fg_kv_read_paged: bad shape");
  FG_REQUIRE(dtype == fg::kF32 || dtype == fg::kBF16, "fg_kv_read_paged: dtype");
  FG_REQUIRE(((uintptr_t)k_out & 15) == 0 && ((uintptr_t)v_out & 15) == 0, "fg_kv_read_paged: outputs must start 16-byte aligned");
  const int64_t items = (int64_t)batch * pages->kv_heads * count;
  FG_REQUIRE(items < (1ll << 40) && (items * (pages->head_dim / 8) * 2 + kThreads - 1) / kThreads < (1ll << 31),
             "fg_kv_read_paged: too many rows for one launch");
  const dim3 grid((unsigned)((items * (pages->head_dim / 8) * 2 + kThreads - 1) / kThreads)), block(kThreads);
  hipStream_t s = (hipStream_t)stream;
#define FG_READ(F, D, T) hipLaunchKernelGGL((paged_read_kernel<F, D, T>), grid, block, 0, s, pg, batch, start, count, row_map, k_out, v_out)
  if (pages->format == kPageE4M3) {
    if (pages->head_dim == 128) { if (dtype == fg::kF32) FG_READ(kPageE4M3, 128, fg::kF32); else FG_READ(kPageE4M3, 128, fg::kBF16); }
    else { if (dtype == fg::kF32) FG_READ(kPageE4M3, 64, fg::kF32); else FG_READ(kPageE4M3, 64, fg::kBF16); }
  } else {
    if (pages->head_dim == 128) { if (dtype == fg::kF32) FG_READ(kPageBF16, 128, fg::kF32); else FG_READ(kPageBF16, 128, fg::kBF16); }
    else { if (dtype == fg::kF32) FG_READ(kPageBF16, 64, fg::kF32); else FG_READ(kPageBF16, 64, fg::kBF16); }
  }
#undef FG_READ
  return fg::check_launch("fg_kv_read_paged");
}

extern "C" int fg_kv_path_gather_paged(const fg_kv_pages* pages, int layers, int64_t layer_stride,
                                       int64_t scale_layer_stride, int batch, const int32_t* seq_len,
                                       const int32_t* row_map, const int32_t* acc_nodes, int acc_stride,
                                       const int32_t* acc_len, int tree_nodes, int32_t* err_flag, void* stream) {
  GatherArgs a;
  if (int rc = fg::pages_of(pages, "fg_kv_path_gather_paged", a.pages)) return rc;
  FG_REQUIRE(seq_len && acc_nodes && acc_len, "fg_kv_path_gather_paged: null pointer");
  FG_REQUIRE(layers > 0 && batch > 0, "fg_kv_path_gather_paged: bad shape");
  FG_REQUIRE(acc_stride >= 1 && acc_stride <= 32 && tree_nodes >= 1 &&
                 tree_nodes <= pages->table_width * pages->page_size,
             "fg_kv_path_gather_paged: acc_stride must be in [1, 32] and the tree fit a row");
  const bool q8 = pages->format == kPageE4M3;
  const int row_bytes = pages->head_dim * (q8 ? 1 : 2);
  a.layer_bytes = layer_stride * (q8 ? 1 : 2);
  a.scale_layer_bytes = scale_layer_stride;
  FG_REQUIRE(layers == 1 || (layer_stride >= 0 && a.layer_bytes % 16 == 0 && scale_layer_stride >= 0 && scale_layer_stride % 4 == 0),
             "fg_kv_path_gather_paged: layers must start 16-byte aligned, their scales 4-byte");
  a.layers = layers;
  a.batch = batch;
  a.cols = row_bytes / 16 + (q8 ? 1 : 0);
  a.seq_len = seq_len;
  a.row_map = row_map;
  a.acc_nodes = acc_nodes;
  a.acc_stride = acc_stride;
  a.acc_len = acc_len;
  a.tree_nodes = tree_nodes;
  a.err_flag = err_flag;
  FG_REQUIRE((int64_t)2 * layers * batch < (1ll << 31) / pages->kv_heads, "fg_kv_path_gather_paged: too many rows for one launch");
  const int64_t total = (int64_t)2 * layers * batch * pages->kv_heads * a.cols;
  FG_REQUIRE(total < (1ll << 31) - kThreads, "fg_kv_path_gather_paged: too many rows for one launch");
  const dim3 grid((unsigned)((total + kThreads - 1) / kThreads)), block(kThreads);
  hipStream_t s = (hipStream_t)stream;
#define FG_GATHER(F, D)                                                                                          \
  do {                                                                                                           \
    if (acc_stride <= 8)                                                                                         \
      hipLaunchKernelGGL((paged_path_gather_kernel<F, D, 8>), grid, block, 0, s, a, (int)total);                 \
    else                                                                                                         \
      hipLaunchKernelGGL((paged_path_gather_kernel<F, D, 32>), grid, block, 0, s, a, (int)total);                \
  } while (0)
  if (q8 && pages->head_dim == 128) FG_GATHER(kPageE4M3, 128);
  else if (q8) FG_GATHER(kPageE4M3, 64);
  else if (pages->head_dim == 128) FG_GATHER(kPageBF16, 128);
  else FG_GATHER(kPageBF16, 64);
#undef FG_GATHER
  return fg::check_launch("fg_kv_path_gather_paged");
}
