// Products of MX rows (fg_mx.h) with 4-bit MX weights on the scaled matrix instructions of gfx950:
//
//   out[m, n] = bf16(sum_b Xx[m, b] Xw[n, b] sum_{k in block b} x[m, k] w[n, k]  (+ bias[n]) (+ residual[m, n]))
//   MX e4m3 of SiLU(g) * u,  g and u the first and second half of the product's columns     (fg_mx_gate_up_swiglu)
//
// x [rows, K] in e4m3 or e2m1, w [cols, K] in e2m1, fp32 sums. v_mfma_scale_f32_32x32x64_f8f6f4 multiplies codes of
// both formats as they are and applies each block's two scales itself, so nothing is decoded on the way: a byte of
// weights is two operands. It does 2048 (e4m3 x e2m1) or 4096 (e2m1 x e2m1) multiply-adds per clock and SIMD.
// Products of e2m1 codes are exact; with e4m3 codes the instruction aligns the products of a few neighbouring
// elements to their largest before it adds them in 32 bits, and bits under 2^-14 of that one are lost (measured:
// 1e-5 of the sum of magnitudes on random codes), a hundredth of the rounding that the bf16 output makes.
//
// Operand layout (lane l, r = l % 32, h = l / 32, 64 elements of K per instruction), found by exact comparison over
// random codes and scales: e2m1 lanes hold row r, elements 32h .. 32h + 31 (16 bytes); e4m3 lanes hold row r,
// elements 16h .. 16h + 15 and 32 + 16h .. 32 + 16h + 15; both take the scale of block h of row r from a byte of a
// register that the instruction selects. D: lane l holds column r of the second operand and rows 8g + 4h + 0..3 of
// the first in registers 4g .. 4g + 3. The weights are the first operand, so that a lane ends with four consecutive
// output columns of one row.
//
// Tiling: a workgroup of 4 waves per output tile of BM rows x BN weight rows. K advances 128 elements (one dword of
// scales per row) per step through an NS-stage ring in LDS that direct HBM->LDS loads fill: x rows of 128 (or 64)
// bytes, weight rows of 64, and the step's scale dwords of both, which lie side by side in memory. Chunks of 16
// bytes are XOR-swizzled by row so that the fragment reads of neighbouring rows hit distinct banks. A step is two
// sub-steps of 64 elements; a sub-step's fragment reads stand between the matrix instructions of the one before,
// and the loads of step t + NS between those of step t's second sub-step, after the step's one barrier.
#include "fg_mx.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef int intx8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kStep = fg::kMxStep;  // K per step
constexpr uint32_t kOutside = 0x80000000u;  // a buffer offset outside every descriptor: reads 0

enum Epilogue : int { kLinear = 0, kGateUp = 1, kParts = 2 };

template <int N>
FG_DEVICE void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt field is 6 bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
}
FG_DEVICE void wait_lgkmcnt0() { __builtin_amdgcn_s_waitcnt(0xF | (0x3 << 14) | (0x7 << 4)); }

// Wait until at most `steps` steps of this wave's loads (LPW each) are outstanding, for a wave-uniform steps in
// [0, MAXS] (immediates for s_waitcnt; larger values wait for MAXS).
template <int LPW, int MAXS>
FG_DEVICE void wait_steps(int steps) {
  if constexpr (MAXS >= 3) {
    if (steps >= 3) {
      wait_vmcnt<3 * LPW>();
      return;
    }
  }
  if constexpr (MAXS >= 2) {
    if (steps >= 2) {
      wait_vmcnt<2 * LPW>();
      return;
    }
  }
  if constexpr (MAXS >= 1) {
    if (steps >= 1) {
      wait_vmcnt<LPW>();
      return;
    }
  }
  wait_vmcnt<0>();
}

struct MxArgs {
  const uint8_t* x;    // codes [rows, xb]
  const uint32_t* xs;  // [steps][rows]
  const uint8_t* w;    // codes [wrows, wb]
  const uint32_t* ws;  // [steps][wrows]
  int xb, wb;          // bytes of a row of codes
  int rows, cols;      // output rows; output columns (gate_up: the intermediate size, half of wrows)
  int wrows;
  int steps, steps_per_split;
  int tiles_m, tiles_n, tiles, per_xcd;
  // kLinear
  const uint16_t* bias;
  const uint16_t* residual;
  int64_t ldr;
  uint16_t* out;
  int64_t ldo;
  int wide;  // out (and residual, bias) take 16-byte accesses at every 8th column
  // kGateUp
  uint8_t* codes;
  uint32_t* scales;
  // kParts
  float* part;  // [splits][rows][wrows]
};

FG_DEVICE float silu_mul(float g, float u) { return fg::silu_f32(g) * u; }

// One buffer's loads: rows of RB bytes per step, 1 KB per instruction and wave.
template <int RB>
struct RowLoads {
  static constexpr int kChunks = RB / 16, kRows = 1024 / RB;
  static FG_DEVICE int swizzle(int row) { return RB == 128 ? row & 7 : (row >> 1) & 3; }
  static FG_DEVICE int lane_row(int lane) { return lane / kChunks; }
  static FG_DEVICE int lane_chunk(int lane) { return (lane % kChunks) ^ swizzle(lane / kChunks); }
};

template <int FMT, int BM, int BN, int WAVES_M, int NS, int EPI>
__global__ void __launch_bounds__(256, 1) mx_gemm_kernel(MxArgs p) {
  constexpr int XB = FMT == fg::kE4M3 ? 128 : 64, WB = 64;  // bytes per row and step
  constexpr int WAVES_N = 4 / WAVES_M;
  constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N;
  constexpr int FM = WM / 32, FN = WN / 32;  // MFMA tiles per wave
  constexpr int X_BYTES = BM * XB, W_BYTES = BN * WB, SX_BYTES = (BM + 63) / 64 * 256, SW_BYTES = BN * 4;
  constexpr int STAGE = X_BYTES + W_BYTES + SX_BYTES + SW_BYTES;
  // loads per step over the four waves; a wave without one of its own repeats the last, so that all count alike
  constexpr int TX = X_BYTES / 1024, TW = W_BYTES / 1024, TS = (SX_BYTES + SW_BYTES) / 256;
  constexpr int LX = (TX + 3) / 4, LW = (TW + 3) / 4, LS = (TS + 3) / 4, LPW = LX + LW + LS;
  static_assert(FM >= 1 && FN >= 1 && TX * 1024 == X_BYTES && TW * 1024 == W_BYTES && BN % 64 == 0, "tile sizes");
  static_assert(EPI != kGateUp || FN % 2 == 0, "a wave holds gate and up of its columns");
  static_assert(NS >= 2 && (NS - 1) * LPW < 64, "vmcnt");
  constexpr int OUT_LD = WN + 4;  // floats per row of the epilogue's staging: 16-byte rows on distinct banks
  constexpr int EPI_BYTES = EPI == kLinear ? 4 * 32 * OUT_LD * 4 : 0;
  static_assert(NS * STAGE <= 160 * 1024 && EPI_BYTES <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(1024))) unsigned char smem[NS * STAGE > EPI_BYTES ? NS * STAGE : EPI_BYTES];

  // XCD-aware order: workgroup b runs on XCD b % 8; XCD x takes tiles x * per_xcd .. , which walk down the rows for
  // one (weight stripe, split) before the next: a stripe is read from HBM by one XCD and reused from its L2.
  const int xcd = blockIdx.x % 8, jj = blockIdx.x / 8;
  const int tile = xcd * p.per_xcd + jj;
  if (jj >= p.per_xcd || tile >= p.tiles) return;  // whole workgroup: before any barrier
  const int tm = tile % p.tiles_m, rest = tile / p.tiles_m;
  const int tn = rest % p.tiles_n, split = rest / p.tiles_n;
  const int m0 = tm * BM;
  const int n0 = tn * (EPI == kGateUp ? BN / 2 : BN);  // first output column
  const int ks0 = split * p.steps_per_split;
  const int nk = min(p.steps - ks0, p.steps_per_split);  // >= 1: the host makes every split non-empty
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WAVES_M, wn = wave / WAVES_M;

  // Row j of the tile's weight block is weight row n0 + j; for gate_up, whose waves own WN/2 gate rows followed by
  // the WN/2 up rows of the same columns, n0 + (j / WN) * (WN / 2) + j % WN, the up ones `cols` further.
  auto weight_row = [&](int j) __attribute__((always_inline)) {
    if constexpr (EPI == kGateUp) {
      const int c = j % WN, o = n0 + (j / WN) * (WN / 2) + c % (WN / 2);
      return min(o, p.cols - 1) + (c >= WN / 2 ? p.cols : 0);
    } else {
      return min(n0 + j, p.wrows - 1);
    }
  };
  // Descriptors over the rows of this tile (x; rows behind the last repeat it) and over whole matrices.
  auto rsrc = [&](const void* base, int64_t bytes) __attribute__((always_inline)) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, (int)(bytes < 0x7fffffff ? bytes : 0x7fffffff),
                                             0x00020000);
  };
  const int64_t w_first = EPI == kGateUp ? 0 : (int64_t)n0 * p.wb;
  const __amdgpu_buffer_rsrc_t xrs = rsrc(p.x + (int64_t)m0 * p.xb, (int64_t)(p.rows - m0) * p.xb);
  const __amdgpu_buffer_rsrc_t wrs = rsrc(p.w + w_first, (int64_t)p.wrows * p.wb - w_first);
  const __amdgpu_buffer_rsrc_t xsrs = rsrc(p.xs, (int64_t)p.steps * p.rows * 4);
  const __amdgpu_buffer_rsrc_t wsrs = rsrc(p.ws, (int64_t)p.steps * p.wrows * 4);

  using XL = RowLoads<XB>;
  using WL = RowLoads<WB>;
  uint32_t xoff[LX], woff[LW], soff[LS];
#pragma unroll
  for (int u = 0; u < LX; ++u) {
    const int r = min(wave * LX + u, TX - 1) * XL::kRows + XL::lane_row(lane);
    xoff[u] = (uint32_t)min(r, p.rows - 1 - m0) * p.xb + XL::lane_chunk(lane) * 16;
  }
#pragma unroll
  for (int u = 0; u < LW; ++u) {
    const int r = min(wave * LW + u, TW - 1) * WL::kRows + WL::lane_row(lane);
    woff[u] = (uint32_t)((int64_t)weight_row(r) * p.wb - w_first) + WL::lane_chunk(lane) * 16;
  }
#pragma unroll
  for (int u = 0; u < LS; ++u) {
    const int q = min(wave * LS + u, TS - 1);
    const int j = q * 64 + lane - SX_BYTES / 4;
    soff[u] = (uint32_t)(q < SX_BYTES / 256 ? min(m0 + q * 64 + lane, p.rows - 1) : weight_row(j)) * 4;
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)smem;
  // The last step of a K that is no multiple of 128: chunks behind the row's end read 0.
  const int last = p.steps - 1 - ks0;
  const uint32_t xmask = XL::lane_chunk(lane) * 16 >= p.xb - (p.steps - 1) * XB ? kOutside : 0u;
  const uint32_t wmask = WL::lane_chunk(lane) * 16 >= p.wb - (p.steps - 1) * WB ? kOutside : 0u;

  // One HBM->LDS load of step ks of this split into ring slot `slot`: 1 KB of codes, or 64 dwords of scales. M0
  // holds the LDS address; the s_nop covers the M0-write -> LDS-DMA hazard.
  auto issue = [&](int ks, int slot, int q) __attribute__((always_inline)) {
    const uint32_t sbase = lds0 + slot * STAGE;
    if (q < LX) {
      const uint32_t m0v = sbase + min(wave * LX + q, TX - 1) * 1024, k = (uint32_t)(ks0 + ks) * XB;
      const uint32_t off = xoff[q] | (ks == last ? xmask : 0u);
      asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(off), "s"(xrs), "s"(k), "{m0}"(m0v)
                   : "memory");
    } else if (q < LX + LW) {
      const uint32_t m0v = sbase + X_BYTES + min(wave * LW + q - LX, TW - 1) * 1024, k = (uint32_t)(ks0 + ks) * WB;
      const uint32_t off = woff[q - LX] | (ks == last ? wmask : 0u);
      asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(off), "s"(wrs), "s"(k), "{m0}"(m0v)
                   : "memory");
    } else {
      const int e = min(wave * LS + q - LX - LW, TS - 1);
      const uint32_t m0v = sbase + X_BYTES + W_BYTES + e * 256;
      if (e < SX_BYTES / 256) {
        const uint32_t k = (uint32_t)(ks0 + ks) * p.rows * 4;
        asm volatile("s_nop 4\n\tbuffer_load_dword %0, %1, %2 offen lds" ::"v"(soff[q - LX - LW]), "s"(xsrs), "s"(k),
                     "{m0}"(m0v)
                     : "memory");
      } else {
        const uint32_t k = (uint32_t)(ks0 + ks) * p.wrows * 4;
        asm volatile("s_nop 4\n\tbuffer_load_dword %0, %1, %2 offen lds" ::"v"(soff[q - LX - LW]), "s"(wsrs), "s"(k),
                     "{m0}"(m0v)
                     : "memory");
      }
    }
  };

  floatx16 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int k = 0; k < FM; ++k)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][k][v] = 0.0f;
  intx8 fx[2][FM], fw[2][FN];
  int sx[2][FM], sw[2][FN];  // a row's scales of one step, its own half's first block in byte 0, second in byte 2
  const int xswz = XL::swizzle(l32), wswz = WL::swizzle(l32);
  auto read = [&](int slot, int s, int buf) __attribute__((always_inline)) {
    const unsigned char* st = smem + slot * STAGE;
#pragma unroll
    for (int f = 0; f < FM; ++f) {
      const unsigned char* row = st + (wm * WM + f * 32 + l32) * XB;
      if constexpr (FMT == fg::kE4M3) {
        const int4 lo = *(const int4*)(row + ((4 * s + half) ^ xswz) * 16);
        const int4 hi = *(const int4*)(row + ((4 * s + 2 + half) ^ xswz) * 16);
        fx[buf][f] = intx8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      } else {
        const int4 lo = *(const int4*)(row + ((2 * s + half) ^ xswz) * 16);
        fx[buf][f] = intx8{lo.x, lo.y, lo.z, lo.w, 0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int f = 0; f < FN; ++f) {
      const int4 lo = *(const int4*)(st + X_BYTES + (wn * WN + f * 32 + l32) * WB + ((2 * s + half) ^ wswz) * 16);
      fw[buf][f] = intx8{lo.x, lo.y, lo.z, lo.w, 0, 0, 0, 0};
    }
  };
  auto read_scales = [&](int slot, int buf) __attribute__((always_inline)) {
    const uint32_t* sc = (const uint32_t*)(smem + slot * STAGE + X_BYTES + W_BYTES);
#pragma unroll
    for (int f = 0; f < FM; ++f) sx[buf][f] = (int)(sc[wm * WM + f * 32 + l32] >> (8 * half));
#pragma unroll
    for (int f = 0; f < FN; ++f) sw[buf][f] = (int)(sc[SX_BYTES / 4 + wn * WN + f * 32 + l32] >> (8 * half));
  };
  constexpr int kBF = FMT == fg::kE4M3 ? 0 : 4;  // the instruction's code of x's format; 4 is e2m1
#define FG_MX_MFMA(i, k, buf, sel, sb)                                                                              \
  acc[i][k] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fw[buf][i], fx[buf][k], acc[i][k], 4, kBF, sel,       \
                                                              sw[sb][i], sel, sx[sb][k])

  // Prologue: steps 0 .. min(NS, nk) - 1 in flight, wait for step 0.
  const int first = min(NS, nk);
#pragma unroll
  for (int h = 0; h < NS; ++h)
    if (h < first) {
#pragma unroll
      for (int q = 0; q < LPW; ++q) issue(h, h, q);
    }
  wait_steps<LPW, NS - 1>(first - 1);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  read(0, 0, 0);
  read_scales(0, 0);

  // Step t in slot t % NS, which takes step t + NS once consumed; sb: which of the two scale registers it uses.
  auto step = [&](int t, int slot, int next, auto sbc, auto with_load) __attribute__((always_inline)) {
    constexpr int sb = decltype(sbc)::value;
    constexpr bool load = decltype(with_load)::value;
    read(slot, 1, 1);
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int k = 0; k < FM; ++k) FG_MX_MFMA(i, k, 0, 0, sb);
    __builtin_amdgcn_sched_barrier(0);
    wait_lgkmcnt0();  // this wave's reads of the slot are done
    // step t + 1 has landed for this wave; t + 2 .. min(t + NS - 1, nk - 1) may still load
    if constexpr (load)
      wait_vmcnt<(NS - 2) * LPW>();
    else
      wait_steps<LPW, NS - 2>(min(NS - 2, nk - 2 - t));
    __builtin_amdgcn_s_barrier();  // ... and for every wave, and no wave still reads slot t
    __builtin_amdgcn_sched_barrier(0);
    if (t + 1 < nk) {
      read(next, 0, 0);
      read_scales(next, 1 - sb);
    }
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int k = 0; k < FM; ++k) {
        FG_MX_MFMA(i, k, 1, 2, sb);
        if constexpr (load) {
          if (i * FM + k < LPW) {
            __builtin_amdgcn_sched_barrier(0);
            issue(t + NS, slot, i * FM + k);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    if constexpr (load) {
#pragma unroll
      for (int q = FM * FN; q < LPW; ++q) issue(t + NS, slot, q);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  int t = 0, slot = 0;
  auto advance = [&](auto sbc, auto with_load) __attribute__((always_inline)) {
    const int next = slot + 1 == NS ? 0 : slot + 1;
    step(t, slot, next, sbc, with_load);
    slot = next;
    ++t;
  };
  using S0 = std::integral_constant<int, 0>;
  using S1 = std::integral_constant<int, 1>;
  // two steps per round, as the scale registers alternate; the tail has no more loads to issue
  while (t + 1 + NS < nk) {
    advance(S0{}, std::true_type{});
    advance(S1{}, std::true_type{});
  }
  if (t + NS < nk) {
    advance(S0{}, std::true_type{});
    while (t < nk) {
      advance(S1{}, std::false_type{});
      if (t < nk) advance(S0{}, std::false_type{});
    }
  } else {
    while (t < nk) {
      advance(S0{}, std::false_type{});
      if (t < nk) advance(S1{}, std::false_type{});
    }
  }
  wait_vmcnt<0>();  // no load still writes LDS when the workgroup ends
#undef FG_MX_MFMA

  // Epilogue: acc[i][k] lane l holds output row m0 + wm * WM + k * 32 + l % 32 and the columns wn * WN + i * 32 + 8g +
  // 4 * half + 0..3 of the tile in elements 4g .. 4g + 3.
  if constexpr (EPI == kParts) {
    float* dst = p.part + (int64_t)split * p.rows * p.wrows;
#pragma unroll
    for (int k = 0; k < FM; ++k) {
      const int m = m0 + wm * WM + k * 32 + l32;
      if (m >= p.rows) continue;
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int n = n0 + wn * WN + i * 32 + 8 * g + 4 * half;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < p.wrows) dst[(int64_t)m * p.wrows + n + e] = acc[i][k][4 * g + e];
        }
    }
  } else if constexpr (EPI == kGateUp) {
    const int out_steps = (p.cols + kStep - 1) / kStep;
#pragma unroll
    for (int k = 0; k < FM; ++k) {
      const int m = m0 + wm * WM + k * 32 + l32;
#pragma unroll
      for (int i = 0; i < FN / 2; ++i) {
        float v[16];
        uint32_t a = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          v[e] = silu_mul(acc[i][k][e], acc[i + FN / 2][k][e]);
          a = max(a, __float_as_uint(v[e]) & 0x7fffffffu);
        }
        a = max(a, (uint32_t)__shfl_xor((int)a, 32, 64));
        const uint32_t s = fg::mx_scale_byte<fg::kE4M3>(a);
        const float inv = fg::mx_inverse_scale(s);
        const int c = n0 + wn * (WN / 2) + i * 32;  // the block's first output column
        if (m >= p.rows || c >= p.cols) continue;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = s == 255u ? 0.0f : v[4 * g + e] * inv;
          int q = 0;
          q = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], q, false);
          q = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], q, true);
          *(int*)(p.codes + (int64_t)m * p.cols + c + 8 * g + 4 * half) = q;
        }
        if (half == 0) {
          uint8_t* sc = (uint8_t*)(p.scales + (int64_t)(c / kStep) * p.rows + m);
          const int b = (c / 32) & 3;
          sc[b] = (uint8_t)s;
          if (c + 32 >= p.cols) {  // the last block also writes the zeros behind it
            for (int e = b + 1; e < 4; ++e) sc[e] = 0;
          }
        }
      }
    }
    (void)out_steps;
  } else {
    __syncthreads();  // no wave still reads the ring: each stages 32 of its rows at a time in it
    float* stage = (float*)smem + wave * 32 * OUT_LD;
    constexpr int LANES = WN / 8;          // lanes per row when reading back, 8 columns each
    constexpr int ROWS = 64 / LANES;       // rows per pass
    const int rr = lane / LANES, cc = (lane % LANES) * 8;
    const int n = n0 + wn * WN + cc;
    float bv[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) bv[e] = p.bias && n + e < p.wrows ? fg::bf16_to_f32(p.bias[n + e]) : 0.0f;
#pragma unroll
    for (int k = 0; k < FM; ++k) {
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(float4*)(stage + l32 * OUT_LD + i * 32 + 8 * g + 4 * half) =
              make_float4(acc[i][k][4 * g], acc[i][k][4 * g + 1], acc[i][k][4 * g + 2], acc[i][k][4 * g + 3]);
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += ROWS) {
        const int m = m0 + wm * WM + k * 32 + r0 + rr;
        const float4 a = *(const float4*)(stage + (r0 + rr) * OUT_LD + cc);
        const float4 b = *(const float4*)(stage + (r0 + rr) * OUT_LD + cc + 4);
        float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        if (m >= p.rows || n >= p.wrows) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += bv[e];
        uint16_t* dst = p.out + (int64_t)m * p.ldo + n;
        const uint16_t* res = p.residual ? p.residual + (int64_t)m * p.ldr + n : nullptr;
        if (p.wide && n + 8 <= p.wrows) {
          if (res) {
            float rv[8];
            fg::load8<fg::kBF16>(res, 0, rv);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += rv[e];
          }
          fg::store8<fg::kBF16>(dst, 0, v);
        } else {
          for (int e = 0; e < 8 && n + e < p.wrows; ++e)
            dst[e] = fg::f32_to_bf16(v[e] + (res ? fg::bf16_to_f32(res[e]) : 0.0f));
        }
      }
    }
  }
}

template <int FMT, int BM, int BN, int WAVES_M, int NS, int EPI>
void launch(MxArgs p, int splits, hipStream_t s) {
  constexpr int kOutCols = EPI == kGateUp ? BN / 2 : BN;
  p.tiles_m = (p.rows + BM - 1) / BM;
  p.tiles_n = ((EPI == kGateUp ? p.cols : p.wrows) + kOutCols - 1) / kOutCols;
  p.tiles = p.tiles_m * p.tiles_n * splits;
  p.per_xcd = (p.tiles + 7) / 8;
  hipLaunchKernelGGL((mx_gemm_kernel<FMT, BM, BN, WAVES_M, NS, EPI>), dim3(8 * p.per_xcd), dim3(256), 0, s, p);
}

int check(const char* what, const void* x_codes, const void* x_scales, int x_format, const void* w_codes,
          const void* w_scales, int rows, int64_t wrows, int hidden) {
  const std::string f(what);
  FG_REQUIRE(x_codes && x_scales && w_codes && w_scales, f + ": null pointer");
  FG_REQUIRE(x_format == fg::kE4M3 || x_format == fg::kE2M1, f + ": bad format");
  FG_REQUIRE(rows > 0 && rows <= (1 << 22) && wrows > 0 && wrows <= (1 << 22) && hidden > 0 && hidden <= (1 << 20),
             f + ": bad shape");
  FG_REQUIRE(hidden % fg::kMxBlock == 0, f + ": hidden must be a multiple of 32");
  FG_REQUIRE((((uintptr_t)x_codes | (uintptr_t)w_codes) & 15) == 0 && (((uintptr_t)x_scales | (uintptr_t)w_scales) & 3) == 0,
             f + ": codes must be 16-byte aligned, scales 4-byte aligned");
  const int64_t steps = (hidden + kStep - 1) / kStep;
  // 32-bit offsets within one operand
  FG_REQUIRE(wrows * hidden / 2 < (1ll << 31) && steps * wrows * 4 < (1ll << 31) && steps * rows * 4 < (1ll << 31),
             f + ": operands must be smaller than 2 GiB");
  return 0;
}

}  // namespace

extern "C" {

int fg_mx_linear(const void* x_codes, const void* x_scales, int x_format, const void* w_codes, const void* w_scales,
                 int rows, int cols, int hidden, const void* bias, const void* residual, int64_t ldr, void* out,
                 int64_t ldo, void* stream) {
  if (int rc = check("fg_mx_linear", x_codes, x_scales, x_format, w_codes, w_scales, rows, cols, hidden)) return rc;
  FG_REQUIRE(out, "fg_mx_linear: null pointer");
  FG_REQUIRE(ldo >= cols && (!residual || ldr >= cols), "fg_mx_linear: bad row strides");
  FG_REQUIRE((((uintptr_t)out | (uintptr_t)bias | (uintptr_t)residual) & 1) == 0, "fg_mx_linear: outputs must be 2-byte aligned");
  MxArgs p{};
  p.x = (const uint8_t*)x_codes;
  p.xs = (const uint32_t*)x_scales;
  p.w = (const uint8_t*)w_codes;
  p.ws = (const uint32_t*)w_scales;
  p.xb = x_format == fg::kE4M3 ? hidden : hidden / 2;
  p.wb = hidden / 2;
  p.rows = rows;
  p.cols = cols;
  p.wrows = cols;
  p.steps = (hidden + kStep - 1) / kStep;
  p.steps_per_split = p.steps;
  p.bias = (const uint16_t*)bias;
  p.residual = (const uint16_t*)residual;
  p.ldr = ldr;
  p.out = (uint16_t*)out;
  p.ldo = ldo;
  p.wide = ldo % 8 == 0 && ((uintptr_t)out & 15) == 0 && (!residual || (ldr % 8 == 0 && ((uintptr_t)residual & 15) == 0));
  hipStream_t s = (hipStream_t)stream;
  if (x_format == fg::kE4M3)
    launch<fg::kE4M3, 128, 128, 2, 4, kLinear>(p, 1, s);
  else
    launch<fg::kE2M1, 128, 128, 2, 4, kLinear>(p, 1, s);
  return fg::check_launch("fg_mx_linear");
}

int fg_mx_gate_up_swiglu(const void* x_codes, const void* x_scales, int x_format, const void* w_codes,
                         const void* w_scales, int rows, int inter, int hidden, void* codes, void* scales,
                         void* stream) {
  if (int rc = check("fg_mx_gate_up_swiglu", x_codes, x_scales, x_format, w_codes, w_scales, rows, 2 * (int64_t)inter, hidden))
    return rc;
  FG_REQUIRE(codes && scales, "fg_mx_gate_up_swiglu: null pointer");
  FG_REQUIRE(inter % fg::kMxBlock == 0, "fg_mx_gate_up_swiglu: inter must be a multiple of 32");
  FG_REQUIRE(((uintptr_t)codes & 15) == 0 && ((uintptr_t)scales & 3) == 0,
             "fg_mx_gate_up_swiglu: codes must be 16-byte aligned, scales 4-byte aligned");
  MxArgs p{};
  p.x = (const uint8_t*)x_codes;
  p.xs = (const uint32_t*)x_scales;
  p.w = (const uint8_t*)w_codes;
  p.ws = (const uint32_t*)w_scales;
  p.xb = x_format == fg::kE4M3 ? hidden : hidden / 2;
  p.wb = hidden / 2;
  p.rows = rows;
  p.cols = inter;
  p.wrows = 2 * inter;
  p.steps = (hidden + kStep - 1) / kStep;
  p.steps_per_split = p.steps;
  p.codes = (uint8_t*)codes;
  p.scales = (uint32_t*)scales;
  hipStream_t s = (hipStream_t)stream;
  if (x_format == fg::kE4M3)
    launch<fg::kE4M3, 128, 128, 2, 4, kGateUp>(p, 1, s);
  else
    launch<fg::kE2M1, 128, 128, 2, 4, kGateUp>(p, 1, s);
  return fg::check_launch("fg_mx_gate_up_swiglu");
}

}  // extern "C"
