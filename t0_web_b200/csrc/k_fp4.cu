// k_fp4.cu -- quantisation, expansion and products of 4-bit microscaled
// matrices (layout: t0b.h, t0b_fp4).
#include <cuda_bf16.h>

#include "common.cuh"
#include "t0b_internal.h"

namespace {

enum : int { TY_F32 = 0, TY_F16 = 1, TY_BF16 = 30 };  // ggml type ids

template <int TY>
struct Plain;
template <>
struct Plain<TY_F32> {
  using T = float;
  T0B_DEV static float get(float v) { return v; }
  T0B_DEV static float put(float v) { return v; }
};
template <>
struct Plain<TY_F16> {
  using T = __half;
  T0B_DEV static float get(__half v) { return __half2float(v); }
  T0B_DEV static __half put(float v) { return __float2half_rn(v); }
};
template <>
struct Plain<TY_BF16> {
  using T = __nv_bfloat16;
  T0B_DEV static float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  T0B_DEV static __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

// ------------------------------------------------------------- the format
T0B_DEV size_t code_pitch(int k) { return (size_t)((k + 31) / 32) * 16; }
// byte of row r, block b in the scale tiles; kt = tiles along k
T0B_DEV size_t scale_at(int r, int b, int kt) {
  return ((size_t)(r >> 7) * kt + (b >> 2)) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (b & 3);
}
// Four values, already divided by their scale, to 4 bits each (first value
// lowest): rounded to nearest, ties to the even index, at most 6.
T0B_DEV uint32_t codes4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n .reg .b8 lo, hi;\n .reg .b16 w;\n cvt.rn.satfinite.e2m1x2.f32 lo, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 hi, %4, "
      "%3;\n mov.b16 w, {lo, hi};\n cvt.u32.u16 %0, w;\n}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
// f32 >= 0 to an unsigned 4-exponent, 3-mantissa bit float: nearest, ties to
// even, at most 448.
T0B_DEV uint32_t e4m3_of(float v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
  return r & 0xFF;
}
T0B_DEV float e4m3_value(uint32_t b) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)b));
  return __half2float(__ushort_as_half((uint16_t)h2));
}
T0B_DEV float scale_value(int blk, uint32_t byte) {
  if (blk == 16) return e4m3_value(byte);
  return byte == 255 ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float(byte ? byte << 23 : 1u << 22);
}
T0B_DEV float code_value(uint32_t c) {
  const uint32_t m = c & 7;
  const float v = m < 2 ? 0.5f * m : __uint_as_float(((126 + (m >> 1)) << 23) | ((m & 1) << 22));
  return c & 8 ? -v : v;
}

// ------------------------------------------------------------ quantisation
// One thread per block of values.
template <int TY>
__global__ void fp4_quantize_kernel(const typename Plain<TY>::T *x, int64_t ldx, Fp4Mat q) {
  const int kt = (q.k + 4 * q.blk - 1) / (4 * q.blk), nb = kt * 4;
  const size_t id = blockIdx.x * (size_t)blockDim.x + threadIdx.x;
  const int r = (int)(id / nb), b = (int)(id % nb);
  if (r >= (q.rows + 127) / 128 * 128) return;
  uint8_t *sc = q.scales + scale_at(r, b, kt);
  const int k0 = b * q.blk;
  if (r >= q.rows || k0 >= q.k) {
    *sc = 0;
    // the second half of a 32-value group whose last block is missing
    if (r < q.rows && (size_t)k0 / 2 < code_pitch(q.k))
      for (int i = 0; i < q.blk / 2; ++i) q.codes[r * code_pitch(q.k) + k0 / 2 + i] = 0;
    return;
  }
  float v[32];
  uint32_t amax = 0;
  for (int i = 0; i < q.blk; ++i) {
    v[i] = k0 + i < q.k ? Plain<TY>::get(x[r * ldx + k0 + i]) : 0.0f;
    amax = max(amax, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  }
  uint32_t byte;
  float d;  // the block's scale
  if (q.blk == 32) {
    byte = amax >= 0x7F800000u ? 255u : max(amax >> 23, 2u) - 2u;
    d = __uint_as_float(byte ? byte << 23 : 1u << 22);
  } else {
    byte = amax >= 0x7F800000u ? 127u : e4m3_of(__fdiv_rn(__uint_as_float(amax), 6.0f * q.ts));
    d = e4m3_value(byte) * q.ts;
  }
  *sc = (uint8_t)byte;
  uint8_t *c = q.codes + r * code_pitch(q.k) + k0 / 2;
  for (int i = 0; i < q.blk; i += 4) {
    float u[4];
    for (int j = 0; j < 4; ++j) u[j] = byte == 0 && q.blk == 16 ? 0.0f : fminf(fmaxf(__fdiv_rn(v[i + j], d), -6.0f), 6.0f);
    const uint32_t w = codes4(u[0], u[1], u[2], u[3]);
    c[i / 2] = (uint8_t)w;
    c[i / 2 + 1] = (uint8_t)(w >> 8);
  }
}

template <int TY>
__global__ void fp4_dequantize_kernel(Fp4Mat q, typename Plain<TY>::T *y, int64_t ldy) {
  const int kt = (q.k + 4 * q.blk - 1) / (4 * q.blk);
  const size_t id = blockIdx.x * (size_t)blockDim.x + threadIdx.x;
  const int64_t r = id / q.k;
  const int k = (int)(id % q.k);
  if (r >= q.rows) return;
  const uint32_t c = q.codes[r * code_pitch(q.k) + k / 2] >> (k % 2 * 4) & 15;
  const float s = scale_value(q.blk, q.scales[scale_at((int)r, k / q.blk, kt)]);
  y[r * ldy + k] = Plain<TY>::put(code_value(c) * s * q.ts);
}

// One value per lane, 32 consecutive columns c0 .. c0 + 31 of row r (zeros
// behind the matrix) to 4 bits: the block's largest magnitude by shuffles.
// Every lane of the warp calls it; c0 is a multiple of 32.
T0B_DEV void quantize_lanes(const Fp4Mat &q, int r, int c0, float v) {
  const int lane = threadIdx.x & 31;
  const int kt = (q.k + 4 * q.blk - 1) / (4 * q.blk);
  uint32_t amax = r < q.rows ? __float_as_uint(v) & 0x7FFFFFFFu : 0;
  for (int o = q.blk / 2; o; o >>= 1) amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
  uint32_t byte;
  float d;
  if (q.blk == 32) {
    byte = amax >= 0x7F800000u ? 255u : max(amax >> 23, 2u) - 2u;
    d = __uint_as_float(byte ? byte << 23 : 1u << 22);
  } else {
    byte = amax >= 0x7F800000u ? 127u : e4m3_of(__fdiv_rn(__uint_as_float(amax), 6.0f * q.ts));
    d = e4m3_value(byte) * q.ts;
  }
  const int b = (c0 + lane) / q.blk;
  if (b < 4 * kt && lane % q.blk == 0) q.scales[scale_at(r, b, kt)] = r < q.rows && b * q.blk < q.k ? (uint8_t)byte : 0;
  float u = byte == 0 && q.blk == 16 ? 0.0f : fminf(fmaxf(__fdiv_rn(v, d), -6.0f), 6.0f);
  const float u1 = __shfl_down_sync(0xFFFFFFFFu, u, 1);
  if (r < q.rows && lane % 2 == 0 && (size_t)c0 / 2 < code_pitch(q.k))
    q.codes[r * code_pitch(q.k) + (c0 + lane) / 2] = (uint8_t)codes4(u, u1, 0.0f, 0.0f);
}

// ----------------------------------------------------------------- product
T0B_DEV float mat_at(const Fp4Mat &q, int r, int k, int kt) {
  const uint32_t c = q.codes[r * code_pitch(q.k) + k / 2] >> (k % 2 * 4) & 15;
  return code_value(c) * scale_value(q.blk, q.scales[scale_at(r, k / q.blk, kt)]);
}

// One 32 x 32 tile of the result per CTA, one thread per value; with GLU two
// sums per thread.
template <int TY, bool GLU>
__global__ void fp4_gemm_kernel(Fp4Mat w, Fp4Mat x, Fp4Out out, int n) {
  __shared__ float xs[32][33], ws[32][33], us[32][33];
  const int tx = threadIdx.x, ty = threadIdx.y;
  const int r = blockIdx.y * 32 + ty, c = blockIdx.x * 32 + tx;
  const int kt = (w.k + 4 * w.blk - 1) / (4 * w.blk);
  float acc = 0.0f, acu = 0.0f;
  for (int k0 = 0; k0 < w.k; k0 += 32) {
    const bool kin = k0 + tx < w.k;
    const int wr = blockIdx.x * 32 + ty;
    xs[ty][tx] = kin && r < x.rows ? mat_at(x, r, k0 + tx, kt) : 0.0f;
    ws[ty][tx] = kin && wr < n ? mat_at(w, wr, k0 + tx, kt) : 0.0f;
    if (GLU) us[ty][tx] = kin && wr < n ? mat_at(w, wr + n, k0 + tx, kt) : 0.0f;
    __syncthreads();
    for (int k = 0; k < 32; ++k) {
      acc = fmaf(xs[ty][k], ws[tx][k], acc);
      if (GLU) acu = fmaf(xs[ty][k], us[tx][k], acu);
    }
    __syncthreads();
  }
  const bool live = r < x.rows && c < n;
  if (!live && !out.quant) return;
  acc = acc * (w.ts * x.ts) + (live && out.bias ? out.bias[c] : 0.0f);
  if (GLU) {
    acu = acu * (w.ts * x.ts) + (live && out.bias ? out.bias[c + n] : 0.0f);
    acc = acc / (1.0f + expf(-acc)) * acu;
  }
  if (out.quant) {
    quantize_lanes(out.q, r, blockIdx.x * 32, live ? acc : 0.0f);
    return;
  }
  reinterpret_cast<typename Plain<TY>::T *>(out.y)[r * out.ld + c] = Plain<TY>::put(acc);
}

template <typename... P, typename... A>
cudaError_t launch(void (*k)(P...), dim3 grid, dim3 block, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = st;
  return cudaLaunchKernelEx(&cfg, k, args...);
}

}  // namespace

cudaError_t t0b_launch_fp4_quantize(int x_type, const void *x, int64_t ldx, const Fp4Mat &q, cudaStream_t st) {
  const size_t n = (size_t)((q.rows + 127) / 128 * 128) * ((q.k + 4 * q.blk - 1) / (4 * q.blk) * 4);
  const dim3 grid((unsigned)((n + 127) / 128));
  if (x_type == TY_F32) return launch(fp4_quantize_kernel<TY_F32>, grid, 128, st, (const float *)x, ldx, q);
  if (x_type == TY_F16) return launch(fp4_quantize_kernel<TY_F16>, grid, 128, st, (const __half *)x, ldx, q);
  return launch(fp4_quantize_kernel<TY_BF16>, grid, 128, st, (const __nv_bfloat16 *)x, ldx, q);
}

cudaError_t t0b_launch_fp4_dequantize(const Fp4Mat &q, int y_type, void *y, int64_t ldy, cudaStream_t st) {
  const dim3 grid((unsigned)(((size_t)q.rows * q.k + 127) / 128));
  if (y_type == TY_F32) return launch(fp4_dequantize_kernel<TY_F32>, grid, 128, st, q, (float *)y, ldy);
  if (y_type == TY_F16) return launch(fp4_dequantize_kernel<TY_F16>, grid, 128, st, q, (__half *)y, ldy);
  return launch(fp4_dequantize_kernel<TY_BF16>, grid, 128, st, q, (__nv_bfloat16 *)y, ldy);
}

template <int TY>
static cudaError_t gemm_ty(const Fp4Mat &w, const Fp4Mat &x, const Fp4Out &out, cudaStream_t st) {
  const int n = out.glu ? w.rows / 2 : w.rows;
  // a 4-bit result: the scale tiles' rows and blocks behind the matrix too
  const int cols = out.quant ? (n + 4 * w.blk - 1) / (4 * w.blk) * 4 * w.blk : n;
  const int rows = out.quant ? (x.rows + 127) / 128 * 128 : x.rows;
  const dim3 grid((cols + 31) / 32, (rows + 31) / 32), block(32, 32);
  return out.glu ? launch(fp4_gemm_kernel<TY, true>, grid, block, st, w, x, out, n)
                 : launch(fp4_gemm_kernel<TY, false>, grid, block, st, w, x, out, n);
}

cudaError_t t0b_launch_fp4_gemm(const Fp4Mat &w, const Fp4Mat &x, const Fp4Out &out, int *err, cudaStream_t st) {
  (void)err;
  if (out.type == TY_F32) return gemm_ty<TY_F32>(w, x, out, st);
  if (out.type == TY_F16) return gemm_ty<TY_F16>(w, x, out, st);
  return gemm_ty<TY_BF16>(w, x, out, st);
}
