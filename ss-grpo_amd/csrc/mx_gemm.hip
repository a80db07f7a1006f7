// Products of MX rows (fg_mx.h) with 4-bit MX weights on the scaled matrix instructions of gfx950:
//
//   out[m, n] = bf16(sum_b Xx[m, b] Xw[n, b] sum_{k in block b} x[m, k] w[n, k]  (+ bias[n]) (+ residual[m, n]))
//   MX e4m3 of SiLU(g) * u,  g and u the first and second half of the product's columns     (fg_mx_gate_up_swiglu)
//
// x [rows, K] in e4m3 or e2m1, w [cols, K] in e2m1, fp32 sums. v_mfma_scale_f32_32x32x64_f8f6f4 multiplies codes of
// both formats as they are and applies each block's two scales itself, so nothing is decoded on the way: a byte of
// weights is two operands. It does 1024 (e4m3 x e2m1) or 2048 (e2m1 x e2m1) multiply-adds per clock and SIMD.
// Products of e2m1 codes are exact; with e4m3 codes the instruction adds the products of eight neighbouring elements
// cut (towards zero) to multiples of 2^-13 of 2^e, e the largest sum of the two factors' exponents among them, and carries
// 24 bits from there on (found by comparison; 1e-5 of the sum of magnitudes on random codes). That is a hundredth of the
// rounding that a bf16 output makes, so the products with one (kLinear) take it. Codes of 8 bits show it: one in 1,000 to
// 2,000 goes to its neighbour, 1.5e-3 to 1.8e-3 of the output. The gate/up product therefore multiplies e4m3 rows' codes in
// two parts of fewer bits (take_low), of whose products the instruction loses nothing, at twice the matrix instructions
// (1856 rows at 7B 340 us, in one part 196; 416 rows at 1.5B 23.6 and 16.9; 64 rows at 7B 31 and 28; one token at 8B 14.4
// and 13.9).
//
// Operand layout (lane l, r = l % 32, h = l / 32, 64 elements of K per instruction), found by exact comparison over
// random codes and scales: e2m1 lanes hold row r, elements 32h .. 32h + 31 (16 bytes); e4m3 lanes hold row r,
// elements 16h .. 16h + 15 and 32 + 16h .. 32 + 16h + 15; both take the scale of block h of row r from a byte of a
// register that the instruction selects. D: lane l holds column r of the second operand and rows 8g + 4h + 0..3 of
// the first in registers 4g .. 4g + 3. The weights are the first operand, so that a lane ends with four consecutive
// output columns of one row.
//
// Tiling: a workgroup of 4 or 8 waves (1 for the smallest) per output tile of BM rows x BN weight rows. K advances 128
// elements (one dword of scales per row) per step through an NS-stage ring in LDS that direct HBM->LDS loads fill: x rows
// of 128 (or 64) bytes, weight rows of 64, and the step's scale dwords of both, which lie side by side in memory. Chunks
// of 16 bytes are XOR-swizzled by row so that the fragment reads of neighbouring rows hit distinct banks. A step is two
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
  float* part;  // [splits][rows][ldp], ldp the weight rows rounded up to a multiple of 4
  int splits, ldp;
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

// Bytes of one ring stage: codes of x and w, scale dwords of x (rounded up to a load of 64) and w.
constexpr int stage_bytes(int fmt, int bm, int bn) {
  return bm * (fmt == fg::kE4M3 ? 128 : 64) + bn * 64 + (bm + 63) / 64 * 256 + bn * 4;
}

// Takes the e4m3 codes of magnitude below 4 (up to 0x47) out of x, zeros in their places, and returns them. The products
// of either part with e2m1 codes are multiples of 2^-13 of the largest power of two that their factors' exponents add up to
// (2^-2 beside 2^10, and 2^-10 beside 2^3), so the matrix instruction loses nothing of them. Bit 7 of a magnitude plus 0x38
// tells the parts apart; v_perm_b32's selectors 8 .. 11 make a byte of it (bit 15, 31, 47 or 63 of the pair of dwords).
FG_DEVICE intx8 take_low(intx8& x) {
  intx8 low;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t v = (uint32_t)x[j], t = (v & 0x7f7f7f7fu) + 0x38383838u;
    const uint32_t high = v & __builtin_amdgcn_perm(t, t << 8, 0x0b090a08u);
    low[j] = (int)(v ^ high);
    x[j] = (int)high;
  }
  return low;
}

template <int FMT, int BM, int BN, int WAVES_M, int WAVES_N, int NS, int EPI, int PARTS>
__global__ void __launch_bounds__(64 * WAVES_M * WAVES_N, NS * stage_bytes(FMT, BM, BN) <= 40 * 1024   ? 4
                                                          : NS * stage_bytes(FMT, BM, BN) <= 80 * 1024 ? 2
                                                                                                       : 1)
    mx_gemm_kernel(MxArgs p) {
  constexpr int XB = FMT == fg::kE4M3 ? 128 : 64, WB = 64;  // bytes per row and step
  constexpr int WAVES = WAVES_M * WAVES_N;
  constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N;
  constexpr int FM = WM / 32, FN = WN / 32;  // MFMA tiles per wave
  constexpr int X_BYTES = BM * XB, W_BYTES = BN * WB, SX_BYTES = (BM + 63) / 64 * 256, SW_BYTES = BN * 4;
  constexpr int STAGE = X_BYTES + W_BYTES + SX_BYTES + SW_BYTES;
  static_assert(STAGE == stage_bytes(FMT, BM, BN), "stage");
  // loads per step over the waves; a wave without one of its own repeats the last, so that all count alike
  constexpr int TX = X_BYTES / 1024, TW = W_BYTES / 1024, TS = (SX_BYTES + SW_BYTES) / 256;
  constexpr int LX = (TX + WAVES - 1) / WAVES, LW = (TW + WAVES - 1) / WAVES, LS = (TS + WAVES - 1) / WAVES;
  constexpr int LPW = LX + LW + LS;
  static_assert(FM >= 1 && FN >= 1 && TX * 1024 == X_BYTES && TW * 1024 == W_BYTES && BN % 64 == 0, "tile sizes");
  static_assert(EPI != kGateUp || FN % 2 == 0, "a wave holds gate and up of its columns");
  static_assert(NS >= 2 && (NS - 1) * LPW < 64, "vmcnt");
  constexpr int OUT_LD = WN + 4;  // floats per row of the epilogue's staging: 16-byte rows on distinct banks
  constexpr int EPI_BYTES = EPI == kLinear ? WAVES * 32 * OUT_LD * 4 + BN * 4 : 0;
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

  using XL = RowLoads<XB>;
  using WL = RowLoads<WB>;
  uint32_t xoff[LX], woff[LW], soff[LS];
  // scales: each load of a wave is of x rows or of weight rows throughout, chosen here and not by a branch between
  // the matrix instructions, which would part them from the loads they are to cover
  __amdgpu_buffer_rsrc_t srs[LS];
  uint32_t sstep[LS];
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
    const bool of_x = q < SX_BYTES / 256;
    soff[u] = (uint32_t)(of_x ? min(m0 + q * 64 + lane, p.rows - 1) : weight_row(j)) * 4;
    sstep[u] = (uint32_t)(of_x ? p.rows : p.wrows) * 4;
    srs[u] = rsrc(of_x ? p.xs : p.ws, (int64_t)p.steps * sstep[u]);
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
      const int e = q - LX - LW;
      const uint32_t m0v = sbase + X_BYTES + W_BYTES + min(wave * LS + e, TS - 1) * 256;
      const uint32_t k = (uint32_t)(ks0 + ks) * sstep[e];
      asm volatile("s_nop 4\n\tbuffer_load_dword %0, %1, %2 offen lds" ::"v"(soff[e]), "s"(srs[e]), "s"(k), "{m0}"(m0v)
                   : "memory");
    }
  };

  float bias_v = 0.0f;  // of the tile's column tid, on its way while the sums are made
  if constexpr (EPI == kLinear) {
    static_assert(64 * WAVES >= BN, "a thread per column");
    if (p.bias && tid < BN && n0 + tid < p.wrows) bias_v = fg::bf16_to_f32(p.bias[n0 + tid]);
  }
  floatx16 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int k = 0; k < FM; ++k)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][k][v] = 0.0f;
  constexpr int XR = FMT == fg::kE4M3 ? 2 : 1;  // 16-byte reads per fragment of x
  int4 fx[2][FM][XR], fw[2][FN];
  // a row's scale dword of this step, its own half's first block in byte 0 and second in byte 2; as read for the next
  uint32_t sx[FM], sw[FN], nx[FM], nw[FN];
  const int xswz = XL::swizzle(l32), wswz = WL::swizzle(l32);
  constexpr int kReads = FM * XR + FN, kScaleReads = FM + FN;
  // One of the LDS reads of sub-step s of a slot; those from kReads on are the step's scales.
  auto read = [&](int slot, int s, int buf, int q) __attribute__((always_inline)) {
    const unsigned char* st = smem + slot * STAGE;
    if (q < FM * XR) {
      const int f = q / XR, h = q % XR;
      const int chunk = FMT == fg::kE4M3 ? 4 * s + 2 * h + half : 2 * s + half;
      fx[buf][f][h] = *(const int4*)(st + (wm * WM + f * 32 + l32) * XB + (chunk ^ xswz) * 16);
    } else if (q < kReads) {
      const int f = q - FM * XR;
      fw[buf][f] = *(const int4*)(st + X_BYTES + (wn * WN + f * 32 + l32) * WB + ((2 * s + half) ^ wswz) * 16);
    } else {
      const uint32_t* sc = (const uint32_t*)(st + X_BYTES + W_BYTES);
      const int f = q - kReads;
      if (f < FM) nx[f] = sc[wm * WM + f * 32 + l32];
      else nw[f - FM] = sc[SX_BYTES / 4 + wn * WN + (f - FM) * 32 + l32];
    }
  };
  auto take_scales = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < FM; ++f) sx[f] = nx[f] >> (8 * half);
#pragma unroll
    for (int f = 0; f < FN; ++f) sw[f] = nw[f] >> (8 * half);
  };
  auto x_frag = [&](int buf, int f) __attribute__((always_inline)) {
    const int4 lo = fx[buf][f][0];
    if constexpr (XR == 2) {
      const int4 hi = fx[buf][f][1];
      return intx8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    } else {
      return intx8{lo.x, lo.y, lo.z, lo.w, 0, 0, 0, 0};
    }
  };
  auto w_frag = [&](int buf, int f) __attribute__((always_inline)) {
    const int4 lo = fw[buf][f];
    return intx8{lo.x, lo.y, lo.z, lo.w, 0, 0, 0, 0};
  };
  constexpr int kBF = FMT == fg::kE4M3 ? 0 : 4;  // the instruction's code of x's format; 4 is e2m1
  intx8 low[FM];  // (PARTS 2) the part of a sub-step's x that is taken out of fx
  auto part_frag = [&](int buf, int f) __attribute__((always_inline)) {
    if constexpr (PARTS == 2) {
      intx8 x = x_frag(buf, f);
      low[f] = take_low(x);
      fx[buf][f][0] = make_int4(x[0], x[1], x[2], x[3]);
      fx[buf][f][XR - 1] = make_int4(x[4], x[5], x[6], x[7]);
    }
  };
  // matrix instruction j of a sub-step's FM * FN * PARTS, those of the low parts first
#define FG_MX_MFMA(j, buf, sel)                                                                                     \
  do {                                                                                                              \
    constexpr int NM_ = FM * FN;                                                                                    \
    const int i_ = (j) % NM_ / FM, k_ = (j) % FM;                                                                   \
    if ((j) < FM) part_frag(buf, k_);                                                                               \
    const intx8 x_ = PARTS == 2 && (j) < NM_ ? low[k_] : x_frag(buf, k_);                                           \
    acc[i_][k_] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w_frag(buf, i_), x_, acc[i_][k_], 4, kBF, sel,     \
                                                                  (int)sw[i_], sel, (int)sx[k_]);                    \
  } while (0)

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
#pragma unroll
  for (int q = 0; q < kReads + kScaleReads; ++q) read(0, 0, 0, q);
  take_scales();

  // Step t in slot t % NS, which takes step t + NS once consumed.
  int slot = 0;
  auto step = [&](int t, auto with_load, auto with_math) __attribute__((always_inline)) {
    constexpr bool load = decltype(with_load)::value;
    constexpr bool math = decltype(with_math)::value;
    const int next = slot + 1 == NS ? 0 : slot + 1;
    constexpr int NM = FM * FN, NJ = NM * PARTS;
    constexpr int R1 = (kReads + NJ - 1) / NJ, R2 = (kReads + kScaleReads + NJ - 1) / NJ;  // reads per MFMA, at least
    // First sub-step: the second's fragments are read between its matrix instructions.
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if constexpr (math) {
        FG_MX_MFMA(j, 0, 0);
#pragma unroll
        for (int q = j * R1; q < (j + 1) * R1; ++q)
          if (q < kReads) read(slot, 1, 1, q);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    wait_lgkmcnt0();  // this wave's reads of the slot are done
    // step t + 1 has landed for this wave; t + 2 .. min(t + NS - 1, nk - 1) may still load
    if constexpr (load)
      wait_vmcnt<(NS - 2) * LPW>();
    else
      wait_steps<LPW, NS - 2>(min(NS - 2, nk - 2 - t));
    __builtin_amdgcn_s_barrier();  // ... and for every wave, and no wave still reads slot t
    __builtin_amdgcn_sched_barrier(0);
    // Second sub-step: the next step's first fragments and scales are read, and the loads of step t + NS issued.
    // (Behind the last step the ring holds nothing newer, and what is read is not used.)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if constexpr (math) {
        FG_MX_MFMA(j, 1, 2);
#pragma unroll
        for (int q = j * R2; q < (j + 1) * R2; ++q)
          if (q < kReads + kScaleReads) read(next, 0, 0, q);
      }
      if constexpr (load) {
        if (j < LPW) issue(t + NS, slot, j);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (load) {
#pragma unroll
      for (int q = NJ; q < LPW; ++q) issue(t + NS, slot, q);
    }
    if constexpr (math) take_scales();
    __builtin_amdgcn_sched_barrier(0);
    slot = next;
  };
  auto steps = [&](auto with_math) __attribute__((always_inline)) {
    int t = 0;
    for (; t + NS < nk; ++t) step(t, std::true_type{}, with_math);  // NS - 1 steps in flight at each wait
    for (; t < nk; ++t) step(t, std::false_type{}, with_math);      // the tail: no more loads to issue
  };
  // A wave whose rows are all behind the last one loads its share and multiplies nothing: the card's power, which
  // bounds large products, goes to the others.
  if (m0 + wm * WM < p.rows)
    steps(std::true_type{});
  else
    steps(std::false_type{});
  wait_vmcnt<0>();  // no load still writes LDS when the workgroup ends
#undef FG_MX_MFMA

  // Epilogue: acc[i][k] lane l holds output row m0 + wm * WM + k * 32 + l % 32 and the columns wn * WN + i * 32 + 8g +
  // 4 * half + 0..3 of the tile in elements 4g .. 4g + 3.
  if constexpr (EPI == kParts) {
    float* dst = p.part + (int64_t)split * p.rows * p.ldp;
#pragma unroll
    for (int k = 0; k < FM; ++k) {
      const int m = m0 + wm * WM + k * 32 + l32;
      if (m >= p.rows) continue;
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int n = n0 + wn * WN + i * 32 + 8 * g + 4 * half;
          if (n < p.ldp)  // whole groups of four: what lies behind the last column is never read
            *(float4*)(dst + (int64_t)m * p.ldp + n) =
                make_float4(acc[i][k][4 * g], acc[i][k][4 * g + 1], acc[i][k][4 * g + 2], acc[i][k][4 * g + 3]);
        }
    }
  } else if constexpr (EPI == kGateUp) {
    // Each wave's codes go out through LDS, its rows of WN / 2 bytes as 16-byte chunks side by side (stored from the
    // accumulators, four bytes of 32 rows at a time: 1.5 us more per 256 x 256 tile).
    __syncthreads();  // no wave still reads the ring
    constexpr int OB = WN / 2, CH = OB / 16;  // bytes and chunks of an output row
    unsigned char* stage = smem + wave * WM * OB;
    auto place = [&](int r, int q) __attribute__((always_inline)) { return r * OB + ((q ^ ((r >> 1) & (CH - 1))) * 16); };
    const int cw = n0 + wn * OB;  // the wave's first output column
    if (m0 + wm * WM >= p.rows || cw >= p.cols) return;
#pragma unroll
    for (int k = 0; k < FM; ++k) {
      const int r = k * 32 + l32, m = m0 + wm * WM + r;
      uint32_t bytes = 0;  // the scales of the wave's blocks
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
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          int q = 0;
          q = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * g] * inv, v[4 * g + 1] * inv, q, false);
          q = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * g + 2] * inv, v[4 * g + 3] * inv, q, true);
          *(int*)(stage + place(r, i * 2 + g / 2) + (g % 2) * 8 + half * 4) = q;
        }
        if (cw + i * 32 < p.cols) bytes |= s << (8 * i);  // zeros behind the last block
      }
      if (half == 0 && m < p.rows) {
        uint8_t* sc = (uint8_t*)(p.scales + (int64_t)(cw / kStep) * p.rows + m) + ((cw / 32) & 3);
        if constexpr (FN / 2 == 2) *(uint16_t*)sc = (uint16_t)bytes;
        else *sc = (uint8_t)bytes;
        if (cw + OB >= p.cols)  // the last wave of the row also writes the zeros behind its blocks
          for (int e = ((cw / 32) & 3) + FN / 2; e < 4; ++e) sc[e - ((cw / 32) & 3)] = 0;
      }
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int it = 0; it < WM * CH / 64; ++it) {
      const int r = it * (64 / CH) + lane / CH, q = lane % CH;
      const int m = m0 + wm * WM + r, c = cw + q * 16;
      const uint4 v = *(const uint4*)(stage + place(r, q));
      if (m < p.rows && c < p.cols) *(uint4*)(p.codes + (int64_t)m * p.cols + c) = v;
    }
  } else {
    __syncthreads();  // no wave still reads the ring: each stages 32 of its rows at a time in it
    float* stage = (float*)smem + wave * 32 * OUT_LD;
    float* s_bias = (float*)smem + WAVES * 32 * OUT_LD;
    if (tid < BN) s_bias[tid] = bias_v;
    __syncthreads();
    s_bias += wn * WN;
    const int nb = n0 + wn * WN, cols = min(WN, p.wrows - nb);  // the wave's first column, how many it has
    // One copy of the code behind the accumulators' stores for all k: a workgroup runs it once, and instructions that
    // have to be fetched cost more than those of a loop.
#pragma clang loop unroll(disable)
    for (int k = 0; k < FM; ++k) {
      const int mk = m0 + wm * WM + k * 32;
      if (mk >= p.rows || cols <= 0) break;
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int kk = 0; kk < FM; ++kk)
        if (kk == k) {
#pragma unroll
          for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g)
              *(float4*)(stage + l32 * OUT_LD + i * 32 + 8 * g + 4 * half) =
                  make_float4(acc[i][kk][4 * g], acc[i][kk][4 * g + 1], acc[i][kk][4 * g + 2], acc[i][kk][4 * g + 3]);
        }
      __builtin_amdgcn_wave_barrier();
      if (p.wide) {  // 8 columns per lane
        constexpr int PER = WN / 8, AT_ONCE = 64 / PER;  // lanes per row, rows per pass
        const int c = (lane % PER) * 8, r = lane / PER;
        if (c >= cols) continue;
#pragma unroll 4
        for (int r0 = 0; r0 < 32; r0 += AT_ONCE) {
          const int m = mk + r0 + r;
          if (m >= p.rows) continue;
          float v[8], bv[8], rv[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
          fg::load8<fg::kF32>(stage + (r0 + r) * OUT_LD + c, 0, v);
          fg::load8<fg::kF32>(s_bias + c, 0, bv);
          uint16_t* dst = p.out + (int64_t)m * p.ldo + nb + c;
          const uint16_t* res = p.residual + (int64_t)m * p.ldr + nb + c;
          if (c + 8 <= cols) {
            if (p.residual) fg::load8<fg::kBF16>(res, 0, rv);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = v[e] + bv[e] + rv[e];
            fg::store8<fg::kBF16>(dst, 0, v);
          } else {
            for (int e = 0; c + e < cols; ++e)
              dst[e] = fg::f32_to_bf16(stage[(r0 + r) * OUT_LD + c + e] + s_bias[c + e] +
                                       (p.residual ? fg::bf16_to_f32(res[e]) : 0.0f));
          }
        }
      } else {
        // Rows that start anywhere: a column per lane, one row at a time (its address is the wave's), eight rows' loads in
        // flight. (Pairs of columns in the row's aligned dwords took more instructions than they saved stores.)
#pragma unroll
        for (int c0 = 0; c0 < WN; c0 += 64) {
          const int c = c0 + lane;
          if (c >= cols) continue;
          const float bias = s_bias[c];
#pragma clang loop unroll(disable)
          for (int r0 = 0; r0 < 32 && mk + r0 < p.rows; r0 += 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = stage[(r0 + u) * OUT_LD + c] + bias;
            if (p.residual) {
#pragma unroll
              for (int u = 0; u < 8; ++u)
                v[u] += fg::bf16_to_f32((p.residual + (int64_t)min(mk + r0 + u, p.rows - 1) * p.ldr + nb)[c]);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u)
              if (mk + r0 + u < p.rows)
                (p.out + (int64_t)(mk + r0 + u) * p.ldo + nb)[c] = (uint16_t)fg::pack_bf16x2(v[u], 0.0f);
          }
        }
      }
    }
  }
}

// Few rows (up to 16 MT): the weights are streamed once, straight into registers, and the rows are read beside them. A
// workgroup takes NT tiles of 16 weight rows (gate_up: 32 gate and 32 up rows, one block of 32 output columns) and its
// waves take every waves-th step of 128 elements, so that together they read each row's bytes in order; v_mfma_scale_
// f32_16x16x128_f8f6f4 multiplies a step (lane l: row l % 16; e2m1 elements 32 (l / 16) .. + 31, e4m3 elements
// 16 (l / 16) .. + 15 and 64 further; scale of block l / 16 from a byte of its register; D: column l % 16 of the second
// operand, rows 4 (l / 16) + 0..3 of the first) for each of MT tiles of 16 rows. The waves' sums meet in LDS, added in
// wave order.
// There are no loads to wait for but the weights and (from L2) the rows, so the loop only keeps U steps of them in
// flight per wave; long reductions over few columns take more waves per workgroup instead of a second launch.
constexpr int kStreamLd = 20;  // floats per x row and tile in LDS: 16-byte stores on distinct banks
constexpr int kStreamLds = 64 * 1024;

constexpr int stream_waves(int nt) { return nt == 1 ? 12 : 8; }  // at most

template <int FMT, int NT, int MT, int U, int EPI>
__global__ void __launch_bounds__(64 * stream_waves(NT)) mx_stream_kernel(MxArgs p) {
  typedef float floatx4 __attribute__((ext_vector_type(4)));
  constexpr int XR = FMT == fg::kE4M3 ? 2 : 1, XB = FMT == fg::kE4M3 ? 128 : 64;
  constexpr int kBF = FMT == fg::kE4M3 ? 0 : 4;
  static_assert(EPI != kGateUp || NT == 4, "gate_up: two tiles of gate rows and two of up rows");
  extern __shared__ __attribute__((aligned(16))) float red[];  // [MT][waves][NT][16 x rows][16 weight rows]
  constexpr int RLD = kStreamLd;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
  const int n0 = blockIdx.x * (EPI == kGateUp ? 32 : NT * 16);

  uint32_t wrow[NT];  // offsets: the weight, and so few rows, are under 2 GiB
  uint32_t wscale[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    int n = n0 + (EPI == kGateUp ? (i & 1) * 16 : i * 16) + r;
    n = min(n, (EPI == kGateUp ? p.cols : p.wrows) - 1) + (EPI == kGateUp && i >= 2 ? p.cols : 0);
    wrow[i] = (uint32_t)n * p.wb;
    wscale[i] = n;
  }
  uint32_t xrow[MT], xm[MT];
#pragma unroll
  for (int k = 0; k < MT; ++k) {
    xm[k] = (uint32_t)min(k * 16 + r, p.rows - 1);
    xrow[k] = xm[k] * p.xb;
  }

  floatx4 acc[MT][NT];
#pragma unroll
  for (int k = 0; k < MT; ++k)
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[k][i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  int4 wv[U][NT], xv[U][MT][XR];
  uint32_t ws[U][NT], xs[U][MT];
  // A step's loads; chunks behind the rows' end (the last step of a K that is no multiple of 128) read the row's
  // first bytes and count as zeros.
  auto load = [&](int u, int t) __attribute__((always_inline)) {
    const uint32_t wo = t * 64 + g * 16;
    const bool w_in = wo < (uint32_t)p.wb;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int4 v = *(const int4*)(p.w + (wrow[i] + (w_in ? wo : 0)));
      wv[u][i] = w_in ? v : make_int4(0, 0, 0, 0);
      ws[u][i] = p.ws[(uint32_t)t * p.wrows + wscale[i]];
    }
#pragma unroll
    for (int k = 0; k < MT; ++k) {
#pragma unroll
      for (int h = 0; h < XR; ++h) {
        const uint32_t xo = t * XB + g * 16 + h * 64;
        const bool x_in = xo < (uint32_t)p.xb;
        const int4 v = *(const int4*)(p.x + (xrow[k] + (x_in ? xo : 0)));
        xv[u][k][h] = x_in ? v : make_int4(0, 0, 0, 0);
      }
      xs[u][k] = p.xs[(uint32_t)t * p.rows + xm[k]];
    }
  };
  auto multiply_part = [&](int u, int k, const intx8& x) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const intx8 w = intx8{wv[u][i].x, wv[u][i].y, wv[u][i].z, wv[u][i].w, 0, 0, 0, 0};
      acc[k][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, acc[k][i], 4, kBF, 0,
                                                                   (int)(ws[u][i] >> (8 * g)), 0, (int)(xs[u][k] >> (8 * g)));
    }
  };
  auto multiply = [&](int u) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < MT; ++k) {
      const int4 lo = xv[u][k][0];
      intx8 x = intx8{lo.x, lo.y, lo.z, lo.w, 0, 0, 0, 0};
      if constexpr (XR == 2) {
        const int4 hi = xv[u][k][1];
        x[4] = hi.x; x[5] = hi.y; x[6] = hi.z; x[7] = hi.w;
      }
      if constexpr (EPI == kGateUp && FMT == fg::kE4M3) multiply_part(u, k, take_low(x));
      multiply_part(u, k, x);
    }
  };
  int t = wave;
  for (; t + (U - 1) * waves < p.steps; t += U * waves) {
#pragma unroll
    for (int u = 0; u < U; ++u) load(u, t + u * waves);
#pragma unroll
    for (int u = 0; u < U; ++u) multiply(u);
  }
  for (; t < p.steps; t += waves) {
    load(0, t);
    multiply(0);
  }

#pragma unroll
  for (int k = 0; k < MT; ++k)
#pragma unroll
    for (int i = 0; i < NT; ++i)  // x row r, weight rows 4g .. 4g + 3
      *(floatx4*)(red + (((k * waves + wave) * NT + i) * 16 + r) * RLD + 4 * g) = acc[k][i];
  __syncthreads();
  auto sum = [&](int i, int row, int c) __attribute__((always_inline)) {
    float v = 0.0f;
    for (int w = 0; w < waves; ++w) v += red[((((row >> 4) * waves + w) * NT + i) * 16 + (row & 15)) * RLD + c];
    return v;
  };
  if constexpr (EPI == kGateUp) {
    for (int e = tid; e < ((p.rows * 32 + 63) & ~63); e += blockDim.x) {  // whole waves
      const int row = min(e >> 5, p.rows - 1), c = e & 31;
      const float v = silu_mul(sum(c >> 4, row, c & 15), sum(2 + (c >> 4), row, c & 15));
      uint32_t a = __float_as_uint(v) & 0x7fffffffu;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) a = max(a, (uint32_t)__shfl_xor((int)a, o, 64));
      const uint32_t s = fg::mx_scale_byte<fg::kE4M3>(a);
      const float y = s == 255u ? 0.0f : v * fg::mx_inverse_scale(s);
      if ((e >> 5) >= p.rows) continue;
      p.codes[(int64_t)row * p.cols + n0 + c] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false);
      if (c == 0) {
        uint8_t* sc = (uint8_t*)(p.scales + (int64_t)(n0 / kStep) * p.rows + row);
        const int b = (n0 / 32) & 3;
        sc[b] = (uint8_t)s;
        if (n0 + 32 >= p.cols)  // the last block also writes the zeros behind it
          for (int q = b + 1; q < 4; ++q) sc[q] = 0;
      }
    }
  } else {
    for (int e = tid; e < p.rows * NT * 16; e += blockDim.x) {
      const int row = e / (NT * 16), c = e - row * (NT * 16), n = n0 + c;
      if (n >= p.wrows) continue;
      float v = sum(c >> 4, row, c & 15);
      if (p.bias) v += fg::bf16_to_f32(p.bias[n]);
      if (p.residual) v += fg::bf16_to_f32(p.residual[(int64_t)row * p.ldr + n]);
      p.out[(int64_t)row * p.ldo + n] = fg::f32_to_bf16(v);
    }
  }
}

// The sums of a split product, added in split order, with what the epilogue of an unsplit one does: four columns per
// thread, or (gate_up) eight, sixteen threads to a dword of scales.
__global__ void __launch_bounds__(256) mx_finish_linear_kernel(MxArgs p) {
  const int groups = p.ldp / 4;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = e / groups;
  if (row >= p.rows) return;
  const int n = (int)(e - row * groups) * 4;
  const float* src = p.part + row * p.ldp + n;
  const int64_t stride = (int64_t)p.rows * p.ldp;
  float4 a = *(const float4*)src;
#pragma unroll 4
  for (int s = 1; s < p.splits; ++s) {  // (several loads in flight)
    const float4 b = *(const float4*)(src + s * stride);
    a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
  }
  const float v[4] = {a.x, a.y, a.z, a.w};
  uint16_t* dst = p.out + row * p.ldo + n;
  const uint16_t* res = p.residual ? p.residual + row * p.ldr + n : nullptr;
  float o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    o[j] = v[j];
    if (n + j < p.wrows) {
      if (p.bias) o[j] += fg::bf16_to_f32(p.bias[n + j]);
      if (res) o[j] += fg::bf16_to_f32(res[j]);
    }
  }
  if (p.wide && n + 4 <= p.wrows) {
    *(uint2*)dst = make_uint2(fg::pack_bf16x2(o[0], o[1]), fg::pack_bf16x2(o[2], o[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < p.wrows) dst[j] = fg::f32_to_bf16(o[j]);
  }
}

__global__ void __launch_bounds__(256) mx_finish_gate_up_kernel(MxArgs p) {
  const int out_steps = (p.cols + kStep - 1) / kStep;
  const int64_t g = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);  // (row, step) of these 16 threads
  const int l = threadIdx.x & 15;
  const int64_t row = g / out_steps;
  const int step = (int)(g - row * out_steps), n = step * kStep + l * 8;
  const bool row_ok = row < p.rows, valid = row_ok && n < p.cols;
  float v[8];
  if (valid) {
    const int64_t stride = (int64_t)p.rows * p.ldp;
    float gt[8], up[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) gt[j] = up[j] = 0.0f;
#pragma unroll 2
    for (int s = 0; s < p.splits; ++s) {
      const float* src = p.part + s * stride + row * p.ldp + n;
      float a[8], b[8];
      fg::load8<fg::kF32>(src, 0, a);
      fg::load8<fg::kF32>(src + p.cols, 0, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        gt[j] += a[j];
        up[j] += b[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = silu_mul(gt[j], up[j]);
  }
  fg::mx_store_step<fg::kE4M3>(v, valid, l, p.codes + row * p.cols + n, p.scales + (int64_t)step * p.rows + row, row_ok);
}

// ------------------------------------------------------------------ which kernel
struct Cost {
  float step_us;   // one step of one workgroup, a CU to itself
  float tile_us;   // what a workgroup takes beside its steps: filling the ring, the epilogue
  float pflops;    // what the whole card sustains with it: power bounds it, and smaller tiles move more bytes per product
  float pair;      // where two workgroups or more fit a CU: what each of many takes of a lone one's time (0: one fits)
  float least;     // and what more than 256 of them take at least, in lone ones' times
};
struct Tile {
  int bm, bn, wave_rows, stages;  // rows and weight rows of a workgroup, rows of a wave, steps in the ring
  float e2m1;  // what a step takes of `once` with e2m1 rows
  Cost once;   // with e4m3 rows
  Cost parts;  // with e4m3 rows in two parts (gate_up)
};
// Fitted to times of every tile and many splits with rows of both formats over some 1900 sizes, 1 .. 8192 rows x 64 ..
// 152000 columns x 160 .. 19000. Over 860 others what the estimates pick is 1.3 % behind the fastest in the geometric
// mean, 35 % at worst. `parts` was fitted to 3600 sizes of the gate/up and the four model sizes that this repository names
// with 1 .. 4096 rows (0.4 % behind, 8 % at worst); over 1950 others 0.6 % and 32 %.
constexpr Tile kTiles[] = {
    {64, 128, 32, 4, 1.02f, {0.329f, 2.42f, 1.63f, 0.762f, 2.95f}, {0.588f, 3.07f, 1.61f, 0.832f, 1.4f}},
    {128, 128, 64, 3, 0.922f, {0.424f, 4.49f, 2.08f, 0.906f, 2.47f}, {0.909f, 5.39f, 2.08f, 0.906f, 2.49f}},
    {128, 256, 64, 4, 0.881f, {0.68f, 4.36f, 2.73f, 0, 0}, {1.4f, 3.49f, 2.75f, 0, 0}},
    {192, 256, 96, 3, 0.946f, {0.787f, 5.48f, 2.8f, 0, 0}, {2.11f, 4.76f, 2.81f, 0, 0}},
    {256, 256, 64, 3, 0.725f, {1.08f, 5.61f, 2.77f, 0, 0}, {2.03f, 7.99f, 2.74f, 0, 0}},
    // up to 32 rows by more columns than the first tile has a CU for: the weights' loads spread over all of them (37888 x
    // 3584, 32 rows: 22.0 us, the first tile 25.0 and the last 26.0, in two parts 22.4, 25.9 and 33; 28672 x 4096, 224 of the
    // first tile: both 17.4)
    {32, 64, 32, 4, 0.962f, {0.434f, 1.85f, 0.703f, 0.627f, 1.08f}, {0.709f, 1.98f, 0.701f, 0.372f, 1.09f}},
    {128, 256, 64, 2, 1.2f, {1.02f, 3.06f, 2.06f, 0.749f, 2.21f}, {1.16f, 3.27f, 1.84f, 0.735f, 1.95f}},
    {64, 128, 32, 2, 1.03f, {0.328f, 1.97f, 0.96f, 0.381f, 1.89f}, {0.46f, 1.93f, 1.17f, 0.389f, 1.84f}},
};
constexpr int kTileCount = 8, kUnsplit = 5, kMaxSplits = 16;  // from kUnsplit on: never split

struct Plan {
  int tile;    // of kTiles; -1: the stream of few rows
  int splits;
};

constexpr float kReadRate = 5.5e6f;  // bytes per us that the weights are read at

// Estimated microseconds of a plan: whole rounds of 256 workgroups (where more than one fit a CU, the share that each
// takes, and not under what a first full round of them was found to take), not under what the card sustains in matrix work
// (1.44 times as much where both operands are e2m1) or in bytes; the output's bytes on top where nothing else runs
// meanwhile. A split product writes and reads its fp32 sums instead and takes a second launch. (A call of few rows waits for
// these lines on the host, so what does not depend on the split is computed once per tile.)
struct TileCost {
  const Cost& t;
  int steps;
  int64_t tiles;
  float step, flops, in, out, sums;
  TileCost(const Tile& tile, bool gate_up, int fmt, int rows, int wrows, int ksteps)
      : t(gate_up && fmt == fg::kE4M3 ? tile.parts : tile.once), steps(ksteps) {
    const int tiles_n = (wrows + tile.bn - 1) / tile.bn;
    tiles = (int64_t)((rows + tile.bm - 1) / tile.bm) * tiles_n;
    const bool e4m3 = fmt == fg::kE4M3;
    step = t.step_us * (e4m3 ? 1.0f : tile.e2m1);
    // waves without a row multiply nothing
    const float active = (float)((rows + tile.wave_rows - 1) / tile.wave_rows) * tile.wave_rows;
    flops = 2.0f * active * tiles_n * tile.bn * steps * kStep / (t.pflops * (e4m3 ? 1e9f : 1.44e9f));
    in = ((float)wrows * steps * 68 + (float)rows * steps * (e4m3 ? 132 : 68)) / kReadRate;
    out = (float)rows * wrows * (gate_up ? 0.5f : 2.0f) / kReadRate;
    sums = (float)rows * wrows * 4 * 2;
  }
  float us(int splits, int per_split) const {
    const int64_t n = tiles * splits;
    const bool beside = t.pair > 0 && n > 256;
    const float rounds = beside ? std::max(t.least, t.pair * n / 256) : (float)((n + 255) / 256);
    const float work = rounds * per_split * step, ends = rounds * t.tile_us, o = splits > 1 ? 0.0f : out;
    const float bytes = sums * splits, parts = splits == 1 ? 0.0f : 3.74f + bytes / (bytes < 16e6f ? 4.3e6f : 5.34e6f);
    if (beside) return 2.0f + std::max(work + ends, std::max(flops, in + o)) + parts;
    return 2.0f + std::max(work, std::max(flops, in)) + ends + o + parts;
  }
};

// The stream of few rows: tiles of 16 weight rows per workgroup as many as leave a workgroup per CU, up to four (the rows
// are read again for each workgroup, which costs little for up to four of them: two tiles then), and up to 64, 32 and 16
// rows with one, two and four tiles: beyond, the rows' bytes from L2 cost more than a tile's loads into LDS (4096 x 4096,
// 32 rows: 7.7 against 10.1 us, 64 rows 12.2 against 12.3; 8192 x 4096, 32 rows: 8.9 against 11.3).
int stream_tiles(bool gate_up, int rows, int wrows) {
  return gate_up ? 4 : wrows <= 4096 ? 1 : wrows <= 8192 || rows <= 4 ? 2 : 4;
}
int stream_rows(int nt) { return 64 / nt; }

// Estimated microseconds: a workgroup's steps (the weights' loads or the rows', whichever takes longer; with more
// workgroups than CUs both), not under the weights' bytes.
float stream_us(int nt, int fmt, int rows, int wrows, int steps) {
  const float load = (float)((wrows + 16 * nt - 1) / (16 * nt)) / 256;
  const float x = rows * (fmt == fg::kE4M3 ? 3e-3f : 1.5e-3f), w = nt == 1 ? 0.054f : nt == 2 ? 0.085f : 0.163f;
  const float step = load <= 1 ? std::max(w, 0.054f + x) : (w + x) * std::max(load, 2.36f);
  return std::max(2.45f + 6 * x + steps * step, 2.0f + (float)wrows * steps * 68 / kReadRate);
}

Plan make_plan(bool gate_up, int fmt, int rows, int wrows, int steps, bool may_split) {
  Plan best{0, 1};
  float least = 1e30f;
  for (int c = 0; c < kTileCount; ++c) {
    const TileCost cost(kTiles[c], gate_up, fmt, rows, wrows, steps);
    // One workgroup of the last tile's two stages per CU cannot cover a long reduction's loads (against the first tile, up
    // to 8 steps 0.95 .. 1.05 of its time, 9 to 12 steps 1.2, 41 and more 1.6).
    if (c == kTileCount - 1 && steps > 8 && cost.tiles <= 256) continue;
    // No splits of less than three steps, of the last tiles (two stages keep too little in flight, and few columns leave the
    // smallest nothing to spread) or of what fills the card four times.
    // With rows in two parts the second and third tiles are taken in splits only: whole, the second was the fastest at 3 of
    // 5500 sizes, by 6 % at most, and the third at none.
    const int fewest = (c == 1 || c == 2) && gate_up && fmt == fg::kE4M3 ? 2 : 1;
    const int most = !may_split || c >= kUnsplit || cost.tiles > 1024 ? 1 : std::max(1, std::min(kMaxSplits, steps / 3));
    for (int s = fewest; s <= most; ++s) {
      const int per = (steps + s - 1) / s;
      if ((steps + per - 1) / per != s) continue;  // one split would be empty
      const float us = cost.us(s, per);
      if (us < least) {
        least = us;
        best = Plan{c, s};
      }
    }
  }
  const int nt = stream_tiles(gate_up, rows, wrows);
  if (rows <= stream_rows(nt) && stream_us(nt, fmt, rows, wrows, steps) <= least) return Plan{-1, 1};
  return best;
}

size_t parts_bytes(const Plan& plan, int rows, int wrows) {
  return plan.splits > 1 ? (size_t)plan.splits * rows * ((wrows + 3) & ~3) * 4 : 0;
}

// ------------------------------------------------------------------ launches
template <int FMT, int BM, int BN, int WAVES_M, int WAVES_N, int NS, int EPI, int PARTS>
void launch(MxArgs p, int splits, hipStream_t s) {
  constexpr int kOutCols = EPI == kGateUp ? BN / 2 : BN;
  p.tiles_m = (p.rows + BM - 1) / BM;
  p.tiles_n = ((EPI == kGateUp ? p.cols : p.wrows) + kOutCols - 1) / kOutCols;
  p.tiles = p.tiles_m * p.tiles_n * splits;
  p.per_xcd = (p.tiles + 7) / 8;
  hipLaunchKernelGGL((mx_gemm_kernel<FMT, BM, BN, WAVES_M, WAVES_N, NS, EPI, PARTS>), dim3(8 * p.per_xcd),
                     dim3(64 * WAVES_M * WAVES_N), 0, s, p);
}

// kTiles[TILE] with its waves.
template <int TILE, int WAVES_M, int WAVES_N, int FMT, int EPI, int PARTS>
void launch_one(const MxArgs& p, int splits, hipStream_t s) {
  constexpr Tile t = kTiles[TILE];
  static_assert(t.bm == WAVES_M * t.wave_rows, "waves");
  launch<FMT, t.bm, t.bn, WAVES_M, WAVES_N, t.stages, EPI, PARTS>(p, splits, s);
}

template <int FMT, int EPI, int PARTS>
void launch_tile(const MxArgs& p, const Plan& plan, hipStream_t s) {
  constexpr bool kWhole = EPI != kGateUp || PARTS == 1;  // (make_plan: those two in splits only)
  switch (plan.tile) {
    case 0: launch_one<0, 2, 2, FMT, EPI, PARTS>(p, plan.splits, s); break;
    case 1:
      if constexpr (kWhole) launch_one<1, 2, 2, FMT, EPI, PARTS>(p, plan.splits, s);
      break;
    case 2:
      if constexpr (kWhole) launch_one<2, 2, 4, FMT, EPI, PARTS>(p, plan.splits, s);
      break;
    case 3: launch_one<3, 2, 4, FMT, EPI, PARTS>(p, plan.splits, s); break;
    case 4: launch_one<4, 4, 2, FMT, EPI, PARTS>(p, plan.splits, s); break;
    default:
      if constexpr (EPI != kParts) {
        if (plan.tile == 5) launch_one<5, 1, 1, FMT, EPI, PARTS>(p, 1, s);
        else if (plan.tile == 6) launch_one<6, 2, 2, FMT, EPI, PARTS>(p, 1, s);
        else launch_one<7, 2, 2, FMT, EPI, PARTS>(p, 1, s);
      }
  }
}

// Tiles of 16 rows that the stream holds, and its waves: eight per workgroup, twelve where a wave would have more than a
// dozen steps and columns are few.
int stream_row_tiles(int nt, int rows) { return nt == 1 && rows > 32 ? 4 : nt <= 2 && rows > 16 ? 2 : 1; }
int stream_wave_count(int nt, int steps) { return nt == 1 && steps >= 96 ? 12 : std::max(1, std::min(8, steps)); }

template <int FMT, int NT, int MT, int EPI>
void launch_stream_rows(const MxArgs& p, int waves, hipStream_t s) {
  const int per = EPI == kGateUp ? 32 : NT * 16, cols = EPI == kGateUp ? p.cols : p.wrows;
  // One step per wave in flight with x in two parts (8B gate/up of one row: 14.4 us, two steps' registers 16.8; not in
  // parts 13.9), else two.
  constexpr int U = EPI == kGateUp || MT > 1 ? 1 : 2;
  static_assert(stream_waves(NT) * MT * NT * 16 * kStreamLd * 4 <= kStreamLds, "LDS");
  hipLaunchKernelGGL((mx_stream_kernel<FMT, NT, MT, U, EPI>), dim3((cols + per - 1) / per), dim3(64 * waves),
                     MT * waves * NT * 16 * kStreamLd * 4, s, p);
}
template <int FMT, int NT, int EPI>
void launch_stream(const MxArgs& p, hipStream_t s) {
  const int waves = stream_wave_count(NT, p.steps), mt = stream_row_tiles(NT, p.rows);
  if constexpr (NT == 1)
    if (mt == 4) return launch_stream_rows<FMT, NT, 4, EPI>(p, waves, s);
  if constexpr (NT <= 2)
    if (mt == 2) return launch_stream_rows<FMT, NT, 2, EPI>(p, waves, s);
  launch_stream_rows<FMT, NT, 1, EPI>(p, waves, s);
}

template <int FMT, int EPI>
void run_format(MxArgs p, const Plan& plan, hipStream_t s) {
  constexpr int PARTS = EPI == kGateUp && FMT == fg::kE4M3 ? 2 : 1;
  if (plan.tile < 0) {
    if constexpr (EPI == kGateUp) {
      launch_stream<FMT, 4, EPI>(p, s);
    } else {
      switch (stream_tiles(false, p.rows, p.wrows)) {
        case 1: launch_stream<FMT, 1, EPI>(p, s); break;
        case 2: launch_stream<FMT, 2, EPI>(p, s); break;
        default: launch_stream<FMT, 4, EPI>(p, s);
      }
    }
    return;
  }
  if (plan.splits == 1) {
    launch_tile<FMT, EPI, PARTS>(p, plan, s);
    return;
  }
  launch_tile<FMT, kParts, PARTS>(p, plan, s);
  if constexpr (EPI == kGateUp) {
    const int64_t groups = (int64_t)p.rows * ((p.cols + kStep - 1) / kStep);
    hipLaunchKernelGGL(mx_finish_gate_up_kernel, dim3((unsigned)((groups + 15) / 16)), dim3(256), 0, s, p);
  } else {
    const int64_t n = (int64_t)p.rows * (p.ldp / 4);
    hipLaunchKernelGGL(mx_finish_linear_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p);
  }
}

template <int EPI>
void run(MxArgs p, int x_format, void* workspace, size_t workspace_bytes, hipStream_t s) {
  p.steps = (p.wb * 2 + kStep - 1) / kStep;
  Plan plan = make_plan(EPI == kGateUp, x_format, p.rows, p.wrows, p.steps, true);
  if (plan.splits > 1 && (!workspace || workspace_bytes < parts_bytes(plan, p.rows, p.wrows)))
    plan = make_plan(EPI == kGateUp, x_format, p.rows, p.wrows, p.steps, false);
  p.splits = plan.splits;
  p.steps_per_split = (p.steps + plan.splits - 1) / plan.splits;
  p.part = (float*)workspace;
  p.ldp = (p.wrows + 3) & ~3;
  if (x_format == fg::kE4M3)
    run_format<fg::kE4M3, EPI>(p, plan, s);
  else
    run_format<fg::kE2M1, EPI>(p, plan, s);
}

// Row counts whose grids (up to 512 threads for each 128 x 256 tile, 256 for each 64 x 128, 64 for each 32 x 64) stay under
// 2^32 threads.
bool sizes_ok(int rows, int64_t wrows, int hidden) {
  return rows > 0 && rows <= (1 << 22) && wrows > 0 && wrows <= (1 << 22) && hidden > 0 && hidden <= (1 << 20) &&
         (int64_t)((rows + 63) / 64) * ((wrows + 127) / 128) < (1 << 23);
}

int check(const char* what, const void* x_codes, const void* x_scales, int x_format, const void* w_codes,
          const void* w_scales, int rows, int64_t wrows, int hidden) {
  const std::string f(what);
  FG_REQUIRE(x_codes && x_scales && w_codes && w_scales, f + ": null pointer");
  FG_REQUIRE(x_format == fg::kE4M3 || x_format == fg::kE2M1, f + ": bad format");
  FG_REQUIRE(sizes_ok(rows, wrows, hidden), f + ": bad shape");
  FG_REQUIRE(hidden % fg::kMxBlock == 0, f + ": hidden must be a multiple of 32");
  FG_REQUIRE((((uintptr_t)x_codes | (uintptr_t)w_codes) & 15) == 0 && (((uintptr_t)x_scales | (uintptr_t)w_scales) & 3) == 0,
             f + ": codes must be 16-byte aligned, scales 4-byte aligned");
  const int64_t steps = (hidden + kStep - 1) / kStep;
  // 32-bit offsets within the weights and the scales, and up to a step of codes behind them (which reads as 0)
  FG_REQUIRE(wrows * hidden / 2 <= (1ll << 31) - 256 && steps * wrows * 4 < (1ll << 31) && steps * rows * 4 < (1ll << 31),
             f + ": the weight and the scales must be smaller than 2 GiB each");
  return 0;
}

}  // namespace

extern "C" {

size_t fg_mx_linear_workspace(int rows, int cols, int hidden, int x_format) {
  if (!sizes_ok(rows, cols, hidden)) return 0;
  return parts_bytes(make_plan(false, x_format, rows, cols, (hidden + kStep - 1) / kStep, true), rows, cols);
}

int fg_mx_linear(const void* x_codes, const void* x_scales, int x_format, const void* w_codes, const void* w_scales,
                 int rows, int cols, int hidden, const void* bias, const void* residual, int64_t ldr, void* out,
                 int64_t ldo, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check("fg_mx_linear", x_codes, x_scales, x_format, w_codes, w_scales, rows, cols, hidden)) return rc;
  FG_REQUIRE(out, "fg_mx_linear: null pointer");
  FG_REQUIRE(ldo >= cols && (!residual || ldr >= cols), "fg_mx_linear: bad row strides");
  FG_REQUIRE((((uintptr_t)out | (uintptr_t)bias | (uintptr_t)residual) & 1) == 0, "fg_mx_linear: outputs must be 2-byte aligned");
  FG_REQUIRE(((uintptr_t)workspace & 15) == 0, "fg_mx_linear: workspace must be 16-byte aligned");
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
  p.bias = (const uint16_t*)bias;
  p.residual = (const uint16_t*)residual;
  p.ldr = ldr;
  p.out = (uint16_t*)out;
  p.ldo = ldo;
  p.wide = ldo % 8 == 0 && ((uintptr_t)out & 15) == 0 && (!residual || (ldr % 8 == 0 && ((uintptr_t)residual & 15) == 0));
  run<kLinear>(p, x_format, workspace, workspace_bytes, (hipStream_t)stream);
  return fg::check_launch("fg_mx_linear");
}

size_t fg_mx_gate_up_swiglu_workspace(int rows, int inter, int hidden, int x_format) {
  if (!sizes_ok(rows, 2 * (int64_t)inter, hidden)) return 0;
  return parts_bytes(make_plan(true, x_format, rows, 2 * inter, (hidden + kStep - 1) / kStep, true), rows, 2 * inter);
}

int fg_mx_gate_up_swiglu(const void* x_codes, const void* x_scales, int x_format, const void* w_codes,
                         const void* w_scales, int rows, int inter, int hidden, void* codes, void* scales,
                         void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check("fg_mx_gate_up_swiglu", x_codes, x_scales, x_format, w_codes, w_scales, rows, 2 * (int64_t)inter, hidden))
    return rc;
  FG_REQUIRE(codes && scales, "fg_mx_gate_up_swiglu: null pointer");
  FG_REQUIRE(inter % fg::kMxBlock == 0, "fg_mx_gate_up_swiglu: inter must be a multiple of 32");
  FG_REQUIRE(((uintptr_t)codes & 15) == 0 && ((uintptr_t)scales & 3) == 0,
             "fg_mx_gate_up_swiglu: codes must be 16-byte aligned, scales 4-byte aligned");
  FG_REQUIRE(((uintptr_t)workspace & 15) == 0, "fg_mx_gate_up_swiglu: workspace must be 16-byte aligned");
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
  p.codes = (uint8_t*)codes;
  p.scales = (uint32_t*)scales;
  run<kGateUp>(p, x_format, workspace, workspace_bytes, (hipStream_t)stream);
  return fg::check_launch("fg_mx_gate_up_swiglu");
}

int fg_mx_plan(int gate_up, int rows, int cols, int hidden, int x_format, int plan[4]) {
  const int64_t wrows = (gate_up ? 2 : 1) * (int64_t)cols;
  FG_REQUIRE(plan, "fg_mx_plan: null pointer");
  FG_REQUIRE(x_format == fg::kE4M3 || x_format == fg::kE2M1, "fg_mx_plan: bad format");
  FG_REQUIRE(sizes_ok(rows, wrows, hidden) && hidden % fg::kMxBlock == 0, "fg_mx_plan: bad shape");
  const int steps = (hidden + kStep - 1) / kStep;
  const Plan p = make_plan(gate_up, x_format, rows, (int)wrows, steps, true);
  if (p.tile < 0) {
    const int nt = stream_tiles(gate_up, rows, (int)wrows);
    plan[0] = 16 * stream_row_tiles(nt, rows);
    plan[1] = 16 * nt;
    plan[2] = 0;
    plan[3] = stream_wave_count(nt, steps);
  } else {
    plan[0] = kTiles[p.tile].bm;
    plan[1] = kTiles[p.tile].bn;
    plan[2] = kTiles[p.tile].stages;
    plan[3] = p.splits;
  }
  return 0;
}

}  // extern "C"
