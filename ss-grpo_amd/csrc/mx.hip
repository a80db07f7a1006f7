// Microscaled rows (fg_mx.h): quantisation, the values they stand for, and the RMSNorm whose output is MX e4m3.
//
// All three move each element once and are bound by HBM: a row is read as 16-byte (bf16) or 32-byte (fp32) pieces of
// eight elements per lane, four lanes hold a block, sixteen a dword of scales.
#include "fg_mx.h"

namespace {

// A workgroup takes 16 rows x 512 columns, a wave four of the rows: each load instruction reads 1 KB of one row, and
// all four are issued before the first is used. 16 rows, because the scale dwords of a step are neighbours along the
// rows: the workgroup's make 64 bytes.
constexpr int kTileRows = 16, kWaveRows = 4, kTileSteps = 4;

template <int DT, int FMT>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const void* __restrict__ x, int64_t ldx, int rows, int cols,
                                                          int steps, int step_tiles, uint8_t* __restrict__ codes,
                                                          uint32_t* __restrict__ scales) {
  const int rt = blockIdx.x / step_tiles, st = blockIdx.x - rt * step_tiles;
  const int lane = threadIdx.x & 63, l = lane & 15;
  const int row0 = rt * kTileRows + (threadIdx.x >> 6) * kWaveRows;
  const int step = st * kTileSteps + (lane >> 4), col = step * fg::kMxStep + l * 8;
  float v[kWaveRows][8];
#pragma unroll
  for (int u = 0; u < kWaveRows; ++u) {
    if (row0 + u < rows && col < cols) {
      fg::load8<DT>(x, (int64_t)(row0 + u) * ldx + col, v[u]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[u][j] = 0.0f;
    }
  }
#pragma unroll
  for (int u = 0; u < kWaveRows; ++u) {
    const int row = row0 + u;
    if (row >= rows) break;  // for the whole wave
    const int64_t at = (int64_t)row * cols + col;
    fg::mx_store_step<FMT>(v[u], col < cols, l, codes + (FMT == fg::kE4M3 ? at : at / 2),
                           scales + (int64_t)step * rows + row, step < steps);
  }
}

template <int DT, int FMT>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales, int rows, int cols,
                                                            int step_tiles, void* __restrict__ out, int64_t ldo) {
  const int rt = blockIdx.x / step_tiles, st = blockIdx.x - rt * step_tiles;
  const int lane = threadIdx.x & 63, l = lane & 15;
  const int row0 = rt * kTileRows + (threadIdx.x >> 6) * kWaveRows;
  const int step = st * kTileSteps + (lane >> 4), col = step * fg::kMxStep + l * 8;
  if (col >= cols) return;
  uint2 c[kWaveRows];
  uint32_t s[kWaveRows];
#pragma unroll
  for (int u = 0; u < kWaveRows; ++u) {
    c[u] = make_uint2(0u, 0u);
    s[u] = 0;
    if (row0 + u < rows) {
      const int64_t at = (int64_t)(row0 + u) * cols + col;
      if constexpr (FMT == fg::kE4M3)
        c[u] = *(const uint2*)(codes + at);
      else
        c[u].x = *(const uint32_t*)(codes + at / 2);
      s[u] = scales[((int64_t)step * rows + row0 + u) * 4 + (l >> 2)];
    }
  }
#pragma unroll
  for (int u = 0; u < kWaveRows; ++u) {
    const int row = row0 + u;
    if (row >= rows) break;
    float v[8];
    if constexpr (FMT == fg::kE4M3) {
      const fg::f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(c[u].x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(c[u].x, true);
      const fg::f32x2_t d = __builtin_amdgcn_cvt_pk_f32_fp8(c[u].y, false), e = __builtin_amdgcn_cvt_pk_f32_fp8(c[u].y, true);
      v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
      v[4] = d.x; v[5] = d.y; v[6] = e.x; v[7] = e.y;
    } else {
      const fg::f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u].x, 1.0f, 0);
      const fg::f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u].x, 1.0f, 1);
      const fg::f32x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u].x, 1.0f, 2);
      const fg::f32x2_t e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u].x, 1.0f, 3);
      v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
      v[4] = d.x; v[5] = d.y; v[6] = e.x; v[7] = e.y;
    }
    const float f = fg::mx_scale(s[u]);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= f;
    fg::store8<DT>(out, (int64_t)row * ldo + col, v);
  }
}

// (hi + lo) as the float next to it towards zero, with the last bit set where the float is not the value ("round to
// odd"), for hi the value's nearest float: a later rounding to fewer bits then gives what rounding the value at once
// would give, ties included. Zeros, infinities and NaN stay.
FG_DEVICE float round_odd(float hi, float lo) {
  uint32_t b = __float_as_uint(hi);
  if (lo != 0.0f && (b & 0x7fffffffu) - 1u < 0x7f7fffffu) b = (b - ((b ^ __float_as_uint(lo)) >> 31)) | 1u;
  return __uint_as_float(b);
}

// The sum over the wave's 64 lanes, in every lane: six additions of what the data-parallel moves bring (within rows
// of 16 lanes, then from row to row), where shuffles through LDS would put six round trips in front of the norm.
template <int CTRL, int ROWS>
FG_DEVICE double moved(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, true);
  return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}
FG_DEVICE double wave_sum(double v) {
  v += moved<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8: lane 15 of each row has the row's sum
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);  // row_bcast 15 into rows 1 and 3, row_bcast 31 into rows 2 and 3
  v += moved<0x143, 0xc>(v);
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 63);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
  return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}

// s = x + delta (rounded to the row type, written to sum), y = s * rsqrt(mean(s^2) + eps) * w, MX e4m3 of y. One
// workgroup per row, eight columns per thread and chunk; the row stays in registers between the two passes. An 8-bit
// code has a rounding border every 1/8 of a value, and with plain 32-bit arithmetic one value in a million falls on
// another side of it than the definition's. So the squares are summed in 64 bits (bf16's are exact there, and so is
// their sum to 2^-50), and where a product is so near a tie that its two roundings decide (by the 19 bits at its end, 5
// of whose 2^19 values are: one wave in 205 per chunk of its 512 products, so one in 100 over 2048 columns), it is taken
// again with the rounding errors of both multiplications, which fused multiply-adds give exactly. For 1856 rows of 3584
// with an addend, 46.8 MB: 12.7 us (3.7 TB/s; 5.3 for 8192 x 4096); with every product in 64 bits and the sums shuffled
// through LDS 15.4. Without an addend bf16 rows move half the bytes under the same conversions and 64-bit multiply-adds,
// which bound them then: 8.2 us for 1856 x 3584 (2.5 TB/s), 14.7 for 4096 x 4096 (3.5), 104 for 37,888 x 3584 (4.0).
// fp32 rows: 42.5 us for 8192 x 5120 (5.0).
//
// PARTS: delta is a projection's split-K parts, fp32 [splits][rows][H], added in split order and rounded to bf16.
template <int DT, int CHUNKS, bool PARTS>
__global__ void __launch_bounds__(512) rmsnorm_mx_kernel(const void* x, int64_t ldx, const void* delta, int splits,
                                                         const void* __restrict__ w, void* sum, int rows,
                                                         int H, double inv_h, float eps, uint8_t* __restrict__ codes,
                                                         uint32_t* __restrict__ scales) {
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, nch = H / 8, threads = blockDim.x;
  __shared__ double red[8];
  float v[CHUNKS][8];
  double ss = 0.0;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int ch = tid + c * threads;
    if (ch < nch) {
      fg::load8<DT>(x, row * ldx + ch * 8, v[c]);
      if (PARTS || delta) {
        float d[8];
        if constexpr (PARTS) {
          const float* part = (const float*)delta + row * H + ch * 8;
          fg::load8<fg::kF32>(part, 0, d);
#pragma unroll 4
          for (int s = 1; s < splits; ++s) {
            float e[8];
            fg::load8<fg::kF32>(part + s * ((int64_t)rows * H), 0, e);
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] += e[j];
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) d[j] = fg::round_bf16(d[j]);
        } else {
          fg::load8<DT>(delta, row * H + ch * 8, d);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c][j] = DT == fg::kBF16 ? fg::round_bf16(v[c][j] + d[j]) : v[c][j] + d[j];
        fg::store8<DT>(sum, row * ldx + ch * 8, v[c]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fma((double)v[c][j], (double)v[c][j], ss);
    }
  }
  ss = wave_sum(ss);
  if ((tid & 63) == 0) red[tid >> 6] = ss;
  __syncthreads();
  ss = 0.0;
  for (int i = 0; i < threads / 64; ++i) ss += red[i];
  double rs = rsqrt(ss * inv_h + (double)eps);
  if (!(rs > 0x1p-64 && rs < 0x1p64)) {  // fp32 rows near the type's ends: both factors where 32 bits hold them in full
    const float f = rs < 1.0 ? 0x1p-64f : 0x1p64f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c][j] *= f;
    rs /= (double)f;
  }
  const float rs_hi = (float)rs, rs_lo = (float)(rs - (double)rs_hi);
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int ch = tid + c * threads;
    float wv[8], y[8];
    const bool valid = ch < nch;
    if (valid) {
      fg::load8<DT>(w, ch * 8, wv);
      uint32_t low = ~0u;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = v[c][j] * rs_hi * wv[j];
        low = min(low, (__float_as_uint(y[j]) + 2u) << 13);
      }
      if (low <= 4u << 13) {  // within two units of its last place of a multiple of 2^19 of them
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float t = v[c][j] * rs_hi;
          const float tl = __builtin_fmaf(v[c][j], rs_lo, __builtin_fmaf(v[c][j], rs_hi, -t));
          const float r = __builtin_fmaf(tl, wv[j], __builtin_fmaf(t, wv[j], -y[j]));  // what y[j] lacks
          const float hi = y[j] + r;
          y[j] = round_odd(hi, r - (hi - y[j]));
        }
      }
    }
    fg::mx_store_step<fg::kE4M3>(y, valid, ch & 15, codes + row * H + ch * 8,
                                 scales + (int64_t)(ch / 16) * rows + row, (ch & ~15) < nch);
  }
}

template <int DT, bool PARTS>
void launch_norm(const void* x, int64_t ldx, const void* delta, int splits, const void* w, void* sum, int rows, int H,
                 float eps, void* codes, void* scales, void* stream) {
  // one chunk per thread up to 256 threads, then two (one chunk and 448 threads, 1856 rows of 3584 without an
  // addend: 8.5 against 8.0 us)
  const int nch = H / 8, chunks = nch <= 256 ? 1 : 2;
  const dim3 g(rows), b(((nch + chunks - 1) / chunks + 63) / 64 * 64);
  const double inv_h = 1.0 / H;
  hipStream_t s = (hipStream_t)stream;
  uint8_t* c = (uint8_t*)codes;
  uint32_t* sc = (uint32_t*)scales;
  if (chunks == 1)
    hipLaunchKernelGGL((rmsnorm_mx_kernel<DT, 1, PARTS>), g, b, 0, s, x, ldx, delta, splits, w, sum, rows, H, inv_h, eps, c, sc);
  else
    hipLaunchKernelGGL((rmsnorm_mx_kernel<DT, 2, PARTS>), g, b, 0, s, x, ldx, delta, splits, w, sum, rows, H, inv_h, eps, c, sc);
}

int64_t tiles_of(int64_t rows, int64_t cols, int* steps, int* step_tiles) {
  *steps = (int)((cols + fg::kMxStep - 1) / fg::kMxStep);
  *step_tiles = (*steps + kTileSteps - 1) / kTileSteps;
  return (rows + kTileRows - 1) / kTileRows * *step_tiles;
}
constexpr int64_t kMaxThreads = (1ll << 32) - 1;  // of a launch

}  // namespace

extern "C" {

int fg_mx_quantize(const void* x, int dtype, int64_t ldx, int rows, int cols, int format, void* codes, void* scales,
                   void* stream) {
  FG_REQUIRE(x && codes && scales, "fg_mx_quantize: null pointer");
  FG_REQUIRE(dtype == fg::kF32 || dtype == fg::kBF16, "fg_mx_quantize: bad dtype");
  FG_REQUIRE(format == fg::kE4M3 || format == fg::kE2M1, "fg_mx_quantize: bad format");
  FG_REQUIRE(rows > 0 && cols > 0 && ldx >= cols, "fg_mx_quantize: bad shape");
  FG_REQUIRE(cols % fg::kMxBlock == 0, "fg_mx_quantize: columns must be a multiple of 32");
  FG_REQUIRE(ldx % 8 == 0 && (((uintptr_t)x | (uintptr_t)codes) & 15) == 0 && ((uintptr_t)scales & 3) == 0,
             "fg_mx_quantize: rows must start 16-byte aligned, scales 4-byte aligned");
  int steps, st;
  const int64_t tiles = tiles_of(rows, cols, &steps, &st);
  FG_REQUIRE(tiles * 256 <= kMaxThreads, "fg_mx_quantize: bad shape (too many rows for one call)");
  hipStream_t s = (hipStream_t)stream;
  const dim3 g((unsigned)tiles), b(256);
  uint8_t* c = (uint8_t*)codes;
  uint32_t* sc = (uint32_t*)scales;
  if (dtype == fg::kBF16 && format == fg::kE4M3)
    hipLaunchKernelGGL((mx_quantize_kernel<fg::kBF16, fg::kE4M3>), g, b, 0, s, x, ldx, rows, cols, steps, st, c, sc);
  else if (dtype == fg::kBF16)
    hipLaunchKernelGGL((mx_quantize_kernel<fg::kBF16, fg::kE2M1>), g, b, 0, s, x, ldx, rows, cols, steps, st, c, sc);
  else if (format == fg::kE4M3)
    hipLaunchKernelGGL((mx_quantize_kernel<fg::kF32, fg::kE4M3>), g, b, 0, s, x, ldx, rows, cols, steps, st, c, sc);
  else
    hipLaunchKernelGGL((mx_quantize_kernel<fg::kF32, fg::kE2M1>), g, b, 0, s, x, ldx, rows, cols, steps, st, c, sc);
  return fg::check_launch("fg_mx_quantize");
}

int fg_mx_dequantize(const void* codes, const void* scales, int format, int rows, int cols, void* out, int dtype,
                     int64_t ldo, void* stream) {
  FG_REQUIRE(codes && scales && out, "fg_mx_dequantize: null pointer");
  FG_REQUIRE(dtype == fg::kF32 || dtype == fg::kBF16, "fg_mx_dequantize: bad dtype");
  FG_REQUIRE(format == fg::kE4M3 || format == fg::kE2M1, "fg_mx_dequantize: bad format");
  FG_REQUIRE(rows > 0 && cols > 0 && ldo >= cols, "fg_mx_dequantize: bad shape");
  FG_REQUIRE(cols % fg::kMxBlock == 0, "fg_mx_dequantize: columns must be a multiple of 32");
  FG_REQUIRE(ldo % 8 == 0 && (((uintptr_t)out | (uintptr_t)codes) & 15) == 0 && ((uintptr_t)scales & 3) == 0,
             "fg_mx_dequantize: rows must start 16-byte aligned, scales 4-byte aligned");
  int steps, st;
  const int64_t tiles = tiles_of(rows, cols, &steps, &st);
  FG_REQUIRE(tiles * 256 <= kMaxThreads, "fg_mx_dequantize: bad shape (too many rows for one call)");
  hipStream_t s = (hipStream_t)stream;
  const dim3 g((unsigned)tiles), b(256);
  const uint8_t *c = (const uint8_t*)codes, *sc = (const uint8_t*)scales;
  if (dtype == fg::kBF16 && format == fg::kE4M3)
    hipLaunchKernelGGL((mx_dequantize_kernel<fg::kBF16, fg::kE4M3>), g, b, 0, s, c, sc, rows, cols, st, out, ldo);
  else if (dtype == fg::kBF16)
    hipLaunchKernelGGL((mx_dequantize_kernel<fg::kBF16, fg::kE2M1>), g, b, 0, s, c, sc, rows, cols, st, out, ldo);
  else if (format == fg::kE4M3)
    hipLaunchKernelGGL((mx_dequantize_kernel<fg::kF32, fg::kE4M3>), g, b, 0, s, c, sc, rows, cols, st, out, ldo);
  else
    hipLaunchKernelGGL((mx_dequantize_kernel<fg::kF32, fg::kE2M1>), g, b, 0, s, c, sc, rows, cols, st, out, ldo);
  return fg::check_launch("fg_mx_dequantize");
}

int fg_rmsnorm_mx(const void* x, const void* delta, const void* weight, void* sum, int dtype, int rows, int hidden,
                  float eps, void* codes, void* scales, void* stream) {
  FG_REQUIRE(x && weight && codes && scales && (!delta || sum), "fg_rmsnorm_mx: null pointer");
  FG_REQUIRE(dtype == fg::kF32 || dtype == fg::kBF16, "fg_rmsnorm_mx: bad dtype");
  FG_REQUIRE(rows > 0 && hidden > 0, "fg_rmsnorm_mx: bad shape");
  FG_REQUIRE(hidden % fg::kMxBlock == 0 && hidden <= 8192,
             "fg_rmsnorm_mx: hidden must be a multiple of 32, at most 8192");
  FG_REQUIRE((int64_t)rows * 512 <= kMaxThreads, "fg_rmsnorm_mx: bad shape (too many rows for one call)");
  FG_REQUIRE((((uintptr_t)x | (uintptr_t)delta | (uintptr_t)weight | (uintptr_t)sum | (uintptr_t)codes) & 15) == 0 &&
                 ((uintptr_t)scales & 3) == 0,
             "fg_rmsnorm_mx: rows must start 16-byte aligned, scales 4-byte aligned");
  if (dtype == fg::kBF16)
    launch_norm<fg::kBF16, false>(x, hidden, delta, 0, weight, sum, rows, hidden, eps, codes, scales, stream);
  else
    launch_norm<fg::kF32, false>(x, hidden, delta, 0, weight, sum, rows, hidden, eps, codes, scales, stream);
  return fg::check_launch("fg_rmsnorm_mx");
}

int fg_residual_rmsnorm_mx_parts(const float* part, int splits, int rows, int hidden, void* x, int64_t ldx,
                                 const void* weight, float eps, void* codes, void* scales, void* stream) {
  FG_REQUIRE(part && x && weight && codes && scales, "fg_residual_rmsnorm_mx_parts: null pointer");
  FG_REQUIRE(rows > 0 && splits >= 1 && hidden > 0, "fg_residual_rmsnorm_mx_parts: bad shape");
  FG_REQUIRE(hidden % fg::kMxBlock == 0 && hidden <= 8192,
             "fg_residual_rmsnorm_mx_parts: hidden must be a multiple of 32, at most 8192");
  FG_REQUIRE(ldx >= hidden && ldx % 8 == 0,
             "fg_residual_rmsnorm_mx_parts: the row stride must be a multiple of 8, at least hidden");
  FG_REQUIRE((int64_t)rows * 512 <= kMaxThreads, "fg_residual_rmsnorm_mx_parts: bad shape (too many rows for one call)");
  FG_REQUIRE((((uintptr_t)part | (uintptr_t)x | (uintptr_t)weight | (uintptr_t)codes) & 15) == 0 && ((uintptr_t)scales & 3) == 0,
             "fg_residual_rmsnorm_mx_parts: rows must start 16-byte aligned, scales 4-byte aligned");
  launch_norm<fg::kBF16, true>(x, ldx, part, splits, weight, x, rows, hidden, eps, codes, scales, stream);
  return fg::check_launch("fg_residual_rmsnorm_mx_parts");
}

}  // extern "C"
