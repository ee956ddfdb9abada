// k_fp4.cu -- quantisation, expansion and products of 4-bit microscaled
// matrices (layout and formulas: t0b.h, t0b_fp4).
//
// Three kinds of kernel:
//   fp4_quantize / fp4_dequantize_kernel   one pass over memory
//   fp4_gemm_pair_kernel    products with tiles enough for the SM pairs
//   fp4_gemm_split_kernel   the others: few tokens, few tiles
// Both products use the block-scaled tensor-core instruction, which applies
// the blocks' scales inside the product (K = 64 values a step, f32 sums), so
// 4-bit operands go from memory to the tensor cores as they are.  Both start
// as programmatic dependents of the previous kernel on the stream.
#include <cuda_bf16.h>

#include <map>
#include <mutex>

#include "common.cuh"
#include "fp4_plan.h"
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

// N values that are read or written as one word: aligned to it, wherever they lie.
template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack {
  T v[N];
};
static_assert(alignof(Pack<float, 8>) >= alignof(uint4) && alignof(Pack<__half, 8>) >= alignof(uint4) &&
                  alignof(Pack<__half, 2>) >= alignof(uint32_t) && alignof(Pack<__nv_bfloat16, 2>) >= alignof(uint32_t),
              "packs are read as words");

// ------------------------------------------------------------- the format
T0B_DEV size_t code_pitch(int k) { return (size_t)((k + 31) / 32) * 16; }
// byte of row r, block b in the scale tiles; kt = tiles along k
T0B_DEV size_t scale_at(int r, int b, int kt) {
  return ((size_t)(r >> 7) * kt + (b >> 2)) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (b & 3);
}
// Eight values, already divided by their scale, to 4 bits each (first value
// lowest): rounded to nearest, ties to the even index, at most 6.
T0B_DEV uint32_t codes8(const float *v) {
  uint32_t r;
  asm("{\n .reg .b8 a, b, c, d;\n cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n mov.b32 %0, {a, b, c, d};\n}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
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
template <bool NV>
T0B_DEV float scale_value(uint32_t byte) {
  if constexpr (NV) return e4m3_value(byte);
  return byte == 255 ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float(byte ? byte << 23 : 1u << 22);
}
// Eight codes (first value lowest) to their values without scale.
T0B_DEV void values8(uint32_t w, float *v) {
  uint32_t h[4];
  asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
      " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// Pairs of f32, two lanes of one instruction.
struct F2 {
  uint64_t v;
  T0B_DEV F2(uint64_t x) : v(x) {}
  T0B_DEV F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  T0B_DEV void get(float &a, float &b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
T0B_DEV F2 fma2(F2 a, F2 b, F2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}
T0B_DEV F2 mul2(F2 a, F2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a.v), "l"(b.v));
  return d;
}

// The largest of a and two magnitudes; keeps a NaN (as bits above infinity's).
T0B_DEV float absmax(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}
template <int N>
T0B_DEV float absmax_of(const float *v) {
  float t = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i += 2) t = absmax(t, v[i], v[i + 1]);
  return t;
}
// A block's scale byte and the division by its scale, from the bits of its
// largest magnitude (infinities and NaNs compare above every finite value).
// Every rounding to 4 bits is decided as by the exact quotient.  MX: the
// product with 1 / d is exact.  NV: d has four significant bits; 1 / d is held
// as hi + lo to about 2^-41 (hi is below it by at most 5.5 units of 2^-23, and
// one correction leaves the square of that), and u = fma(x, hi, x lo) is the
// quotient so nearly that every border is decided rightly: a quotient on a
// border is representable and comes out as itself, one that is not differs
// from the border by at least 1.06 half ulps, a margin of some 2^-29.  lo >= 0:
// the sign of a zero and of an overflow stays.
template <bool NV>
struct BlockScale {
  uint32_t byte;
  float hi, lo;
  T0B_DEV BlockScale(uint32_t amax, const Fp4Mat &q) {
    if constexpr (!NV) {
      byte = amax >= 0x7F800000u ? 255u : max(amax >> 23, 2u) - 2u;
      hi = __uint_as_float((254u - min(byte, 252u)) << 23);
      lo = 0.0f;
    } else {
      const float a = __uint_as_float(amax);
      byte = e4m3_of(fmaf(a, q.r6_hi, a * q.r6_lo));  // a / (6 tensor_scale), the same way
      if (amax >= 0x7F800000u) byte = 127u;
      const float d = e4m3_value(min(byte, 126u)) * q.ts;  // finite: zeros stay zeros in a block of scale NaN too
      float r;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
      hi = byte ? __uint_as_float(__float_as_uint(r) - 4u) : 0.0f;  // below 1 / d
      lo = fmaf(-hi, d, 1.0f) * hi;
    }
  }
};

// Eight values of a block to a word of codes.
template <bool NV>
T0B_DEV uint32_t quantize8(const BlockScale<NV> &s, const float *v) {
  float u[8];
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const F2 x(v[j], v[j + 1]), hi(s.hi, s.hi);
    if constexpr (NV)
      fma2(x, hi, mul2(x, F2(s.lo, s.lo))).get(u[j], u[j + 1]);
    else
      mul2(x, hi).get(u[j], u[j + 1]);
  }
  const uint32_t w = codes8(u);
  return NV && s.byte == 0 ? 0u : w;  // a scale of zero: no signs either
}

// One value of a block to a code, the same way.
template <bool NV>
T0B_DEV uint32_t quantize1(const BlockScale<NV> &s, float v) {
  const float u = NV ? fmaf(v, s.hi, __fmul_rn(v, s.lo)) : v * s.hi;
  uint32_t r;
  asm("{\n .reg .b8 a;\n cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n mov.b32 %0, {a, a, a, a};\n}" : "=r"(r) : "f"(u), "f"(0.0f));
  return NV && s.byte == 0 ? 0u : r & 15;
}

// ------------------------------------------------------------ quantisation
// A lane takes 8 consecutive values of a row, a warp 256 (or, for short rows,
// one scale tile's 64 or 128 of adjacent rows), each of the rows r, r + 32,
// r + 64 and r + 96, whose scale words lie side by side in a scale tile: four
// loads are in flight per lane, and a tile's 16 bytes of scales are written
// together.  A block spans two (NV) or four lanes; its largest magnitude is
// joined by shuffles, the scale words by a 4 x 4 byte transposition.
// Bound by HBM: 65,536 x 1024 bf16 in 31.9 us (MX) and 32.1 us (NV), 170 MB =
// 5.3 TB/s; f32 6.2 TB/s.  One thread per block took 535 us for this
// and the way back.
constexpr int QT_WARPS = 8;
constexpr int QT_CHUNKS = 4;  // 65,536 x 1024 bf16: 39 us with 1, 35 with 2, 32 with 4 and 8

// 8 values from x[k0 ..] as they lie in memory, zeros from k on; `align`: the
// rows start on this many bytes (16 or more, 8, 4, 2).
template <int TY>
struct Raw8 {
  using T = typename Plain<TY>::T;
  uint4 w[sizeof(T) / 2];
  T0B_DEV void load(const T *x, int k0, int k, int align) {
    x += k0;
    if (align >= 16 && k0 + 8 <= k) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4 *>(x)[i];
    } else if (align == 8 && k0 + 8 <= k) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        const uint2 a = reinterpret_cast<const uint2 *>(x)[2 * i], b = reinterpret_cast<const uint2 *>(x)[2 * i + 1];
        w[i] = make_uint4(a.x, a.y, b.x, b.y);
      }
    } else if (align == 4 && k0 + 8 <= k) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        const uint32_t *p = reinterpret_cast<const uint32_t *>(x) + 4 * i;
        w[i] = make_uint4(p[0], p[1], p[2], p[3]);
      }
    } else {
      Pack<T, 8> e;
#pragma unroll
      for (int i = 0; i < 8; ++i) e.v[i] = k0 + i < k ? x[i] : Plain<TY>::put(0.0f);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4 *>(&e)[i];
    }
  }
  T0B_DEV void zero() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  // The same for the 256 values of a warp, x[c0 ..], of f32 rows that are not
  // aligned: the lanes load neighbouring values, and turn() hands each lane
  // its 8 through shared memory (256 values of the warp's own).  65,536 x 1001
  // 55 us, 71 us with 8 loads of 4 bytes a lane.  (For 16-bit rows the turn
  // costs more than it saves: 67 to 89 us against 59.)
  T0B_DEV void load_turned(const T *x, int c0, int k) {
    const int lane = threadIdx.x & 31, n = k - c0;
    uint32_t *word = reinterpret_cast<uint32_t *>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) word[i] = lane + 32 * i < n ? __float_as_uint(x[c0 + lane + 32 * i]) : 0u;
  }
  T0B_DEV void turn(uint32_t *sm) {
    const int lane = threadIdx.x & 31;
    const uint32_t *word = reinterpret_cast<const uint32_t *>(w);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) sm[lane + 32 * i] = word[i];
    __syncwarp();
    w[0] = reinterpret_cast<const uint4 *>(sm)[2 * lane];
    w[1] = reinterpret_cast<const uint4 *>(sm)[2 * lane + 1];
  }
  T0B_DEV void get(float *v) const {
    const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = Plain<TY>::get(e[i]);
  }
};

// LPR: lanes along a row, 8 (one NV scale tile), 16 or 32.
// A warp goes through `chunks` such pieces along its rows and fetches the next
// one before it works on the present one.
// TURN: f32 rows that are not aligned (LPR 32), see Raw8::load_turned.
template <int TY, bool NV, int LPR, bool TURN>
__global__ void __launch_bounds__(32 * QT_WARPS)
    fp4_quantize_kernel(const typename Plain<TY>::T *x, int64_t ldx, Fp4Mat q, int align, int chunks) {
  constexpr int BLK = NV ? 16 : 32, LB = BLK / 8;  // lanes of a block
  constexpr int RPW = 32 / LPR;                    // adjacent rows of a warp
  const int kt = (q.k + 4 * BLK - 1) / (4 * BLK);
  const int lane = threadIdx.x & 31;
  const int r0 = blockIdx.x * (QT_WARPS * RPW) + (threadIdx.x >> 5) * RPW + lane / LPR;  // counts 32 rows of each group
  const int group = r0 >> 5, r = group * 128 + (r0 & 31);
  int k0 = (blockIdx.y * chunks * LPR + lane % LPR) * 8;
  const int live = min(4, (q.rows - r + 31) / 32);  // of this lane's four rows
  const size_t pitch = code_pitch(q.k);
  const typename Plain<TY>::T *row = x + r * ldx;
  uint8_t *codes = q.codes + r * pitch + k0 / 2;
  const int t0 = k0 / (4 * BLK), b = lane / LB % 4;
  uint8_t *scales = q.scales + ((size_t)group * kt + t0) * 512 + (r & 31) * 16 + 4 * b;
  const uint32_t sel1 = b & 1 ? 0x3715 : 0x6240, sel2 = b & 2 ? 0x3276 : 0x5410;
  const bool writes_scales = lane % LB == 0 && group < (q.rows + 127) / 128;
  __shared__ __align__(16) uint32_t turned[TURN ? QT_WARPS : 1][TURN ? 256 : 4];
  pdl_wait();
  pdl_launch_dependents();
  Raw8<TY> next[4];
  auto fetch = [&](int k) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i >= live) {
        next[i].zero();
      } else {
        if constexpr (TURN)
          next[i].load_turned(row + 32 * i * ldx, k - 8 * lane, q.k);
        else
          next[i].load(row + 32 * i * ldx, k, q.k, align);
      }
  };
  fetch(k0);
  for (int c = 0; c < chunks; ++c) {
    Raw8<TY> raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = next[i];
    if (c + 1 < chunks) fetch(k0 + 8 * LPR);
    const int rows = k0 / 2 < (int)pitch ? live : 0;
    uint32_t sc = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v[8];
      if constexpr (TURN) raw[i].turn(turned[threadIdx.x >> 5]);
      raw[i].get(v);
      float top = absmax_of<8>(v);
#pragma unroll
      for (int o = 1; o < LB; o *= 2) top = absmax(top, __shfl_xor_sync(0xFFFFFFFFu, top, o), 0.0f);
      const BlockScale<NV> s(__float_as_uint(top), q);
      sc |= s.byte << (8 * i);
      if (i < rows) *reinterpret_cast<uint32_t *>(codes + 32 * i * pitch) = quantize8<NV>(s, v);
    }
    // sc: one block of four rows; the tile's words are four blocks of one row
    sc = __byte_perm(sc, __shfl_xor_sync(0xFFFFFFFFu, sc, LB), sel1);
    sc = __byte_perm(sc, __shfl_xor_sync(0xFFFFFFFFu, sc, 2 * LB), sel2);
    if (writes_scales && k0 < 4 * BLK * kt) *reinterpret_cast<uint32_t *>(scales) = sc;
    k0 += 8 * LPR;
    codes += 4 * LPR;
    scales += 512 * (8 * LPR / (4 * BLK));
  }
}

// ----------------------------------------------------------- the other way
// The same division of work: 4 bytes of codes to 8 values a lane, the scale
// words of four rows in one 16-byte load.  8 values of a lane go out at once
// where rows are aligned to them (the largest: 32 bytes, so that no sector is
// written in halves).  A tensor scale that is no power of two rounds once in
// f32 before the result's type.  Bound by HBM: 65,536 x 1024 bf16 in 30.2 us,
// 5.6 TB/s; rows that are not aligned (65,536 x 1001 f16) 51 us, written
// value by value 181 us.
template <int TY>
T0B_DEV void store8(typename Plain<TY>::T *y, int k0, int k, bool vec, const float *v) {
  using T = typename Plain<TY>::T;
  Pack<T, 8> t;
#pragma unroll
  for (int i = 0; i < 8; ++i) t.v[i] = Plain<TY>::put(v[i]);
  if (vec && k0 + 8 <= k) {
    if constexpr (TY == TY_F32)
      asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(y + k0), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                   "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                   : "memory");
    else
      *reinterpret_cast<uint4 *>(y + k0) = *reinterpret_cast<const uint4 *>(&t);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k0 + i < k) y[k0 + i] = t.v[i];
  }
}
// A warp's 256 values of a row that is not aligned, columns c0 .. of k, turned
// in shared memory so that the lanes write neighbouring 4-byte words (two
// 16-bit values; single ones at the ends).
template <int TY>
T0B_DEV void store_unaligned(typename Plain<TY>::T *y, int c0, int k, typename Plain<TY>::T *sm, const float *v) {
  using T = typename Plain<TY>::T;
  const int lane = threadIdx.x & 31, n = min(256, k - c0);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) sm[lane * 8 + i] = Plain<TY>::put(v[i]);
  __syncwarp();
  y += c0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < n) y[lane + 32 * i] = sm[lane + 32 * i];
  } else {
    const int odd = (int)((uintptr_t)y >> 1 & 1);
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      const int e = 2 * (lane + 32 * i) - odd;  // values e, e + 1 share a word
      if (e >= n || e > 255) break;
      if (e >= 0 && e + 1 < n) {
        const Pack<T, 2> t{{sm[e], sm[e + 1]}};
        *reinterpret_cast<uint32_t *>(y + e) = *reinterpret_cast<const uint32_t *>(&t);
      } else {
        y[e < 0 ? 0 : e] = sm[e < 0 ? 0 : e];
      }
    }
  }
}

template <int TY, bool NV, int LPR>
__global__ void __launch_bounds__(32 * QT_WARPS) fp4_dequantize_kernel(Fp4Mat q, typename Plain<TY>::T *y, int64_t ldy, bool vec) {
  constexpr int BLK = NV ? 16 : 32, LB = BLK / 8, RPW = 32 / LPR;
  const int kt = (q.k + 4 * BLK - 1) / (4 * BLK);
  const int lane = threadIdx.x & 31;
  const int r0 = blockIdx.x * (QT_WARPS * RPW) + (threadIdx.x >> 5) * RPW + lane / LPR;
  const int group = r0 >> 5, r = group * 128 + (r0 & 31);
  const int k0 = (blockIdx.y * LPR + lane % LPR) * 8;
  pdl_wait();
  pdl_launch_dependents();
  // rows that are not aligned are written by the whole warp
  const bool turn = LPR == 32 && !vec;
  if ((k0 >= q.k && !turn) || r >= q.rows) return;
  __shared__ typename Plain<TY>::T turned[QT_WARPS][LPR == 32 ? 256 : 1];
  const bool in = k0 < q.k;
  uint4 s4 = make_uint4(0, 0, 0, 0);
  if (in) s4 = *reinterpret_cast<const uint4 *>(q.scales + ((size_t)group * kt + k0 / (4 * BLK)) * 512 + (r & 31) * 16);
  const uint32_t sw[4] = {s4.x, s4.y, s4.z, s4.w};
  uint32_t w[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (r + 32 * i < q.rows && in) w[i] = *reinterpret_cast<const uint32_t *>(q.codes + (r + 32 * i) * code_pitch(q.k) + k0 / 2);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (r + 32 * i >= q.rows) break;
    const float s = scale_value<NV>(sw[i] >> (8 * (lane / LB % 4)) & 255);
    float v[8];
    values8(w[i], v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = NV ? v[j] * s * q.ts : v[j] * s;
    if (turn)
      store_unaligned<TY>(y + (r + 32 * i) * ldy, blockIdx.y * 256, q.k, turned[threadIdx.x >> 5], v);
    else
      store8<TY>(y + (r + 32 * i) * ldy, k0, q.k, vec, v);
  }
}

// ----------------------------------------------------------------- product
// silu(g) * u.  1 / (1 + exp(-g)) with exp as 2^-t, t = g log2(e) carried to
// twice the precision (the rounding error of t would otherwise grow with g);
// above 126 the sigmoid is 1 to the last bit, and the clamp keeps the
// correction finite.
constexpr float LOG2E = 1.44269504f, LOG2E_LO = 1.92596299e-8f, LN2 = 0.693147181f;
T0B_DEV float ex2_approx(float t) {
  float p;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(t));
  return p;
}
T0B_DEV float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
T0B_DEV float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
// Below SILU_TAIL 1 / (1 + exp(-g)) is exp(g) to 2^-125, and soon no normal
// number; its product with u may be one all the same.  exp(g) = 2^n 2^r, and
// the powers of two are multiplied in one after the other, so that only the
// result is rounded where it leaves the range.  From -208 on it is zero for
// every u.
constexpr float SILU_TAIL = 87.0f;
T0B_DEV float silu_mul_tail(float g, float u) {
  const float c = fmaxf(g, -208.0f) + (g - g);  // -infinity: NaN, as -infinity / (1 + exp(infinity))
  const float n = rintf(c * LOG2E);             // -300 .. -125
  const float r = fmaf(c, LOG2E_LO, fmaf(c, LOG2E, -n));
  const float v = __fmul_rn(__fmul_rn(__fmul_rn(c, ex2_approx(r)), pow2(-120)), u);
  const int e = (int)n + 120, half = e / 2;
  return __fmul_rn(__fmul_rn(v, pow2(half)), pow2(e - half));
}
// For g >= -SILU_TAIL (or NaN).
T0B_DEV float silu_mul_body(float g, float u) {
  const float c = fminf(g, 126.0f);
  const float t = __fmul_rn(c, LOG2E);
  const float f = fmaf(fmaf(c, -LOG2E_LO, fmaf(c, -LOG2E, t)), LN2, 1.0f);
  return __fmul_rn(__fmul_rn(g, rcp_approx(fmaf(ex2_approx(-t), f, 1.0f))), u);
}
T0B_DEV float silu_mul(float g, float u) { return g < -SILU_TAIL ? silu_mul_tail(g, u) : silu_mul_body(g, u); }
// The body on pairs, for g below 2^20 (no clamp: the correction stays near 1
// there), with the same results.
T0B_DEV F2 silu_mul2(F2 g, F2 u) {
  const F2 t = mul2(g, F2(LOG2E, LOG2E));
  const F2 e = fma2(g, F2(-LOG2E_LO, -LOG2E_LO), fma2(g, F2(-LOG2E, -LOG2E), t));
  const F2 f = fma2(e, F2(LN2, LN2), F2(1.0f, 1.0f));
  float t0, t1, d0, d1;
  t.get(t0, t1);
  fma2(F2(ex2_approx(-t0), ex2_approx(-t1)), f, F2(1.0f, 1.0f)).get(d0, d1);
  return mul2(mul2(g, F2(rcp_approx(d0), rcp_approx(d1))), u);
}

// 32 accumulator columns of this thread's lane; the values may be used after
// tmem_ld_wait on them.
T0B_DEV void tmem_ld32(uint32_t addr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
T0B_DEV void tmem_ld_wait(uint32_t *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])::"memory");
}
// 16 accumulator columns of this thread's lane; used after the wait on them.
T0B_DEV void tmem_ld16(uint32_t addr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
T0B_DEV void tmem_ld_wait16(uint32_t *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15])::"memory");
}
T0B_DEV void tma_load_3d_pair(void *dst, const void *tmap, uint32_t bar_cl, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, "
      "%5}], [%2];" ::"r"(smem_u32(dst)),
      "l"((uint64_t)tmap), "r"(bar_cl), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// Shared-memory descriptor of a K-major tile of 128-byte rows (256 4-bit
// values) with the 128-byte swizzle: 8-row atoms of 1024 bytes.
T0B_DEV uint64_t sw128_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024u >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
// A 512-byte scale tile (32 rows of 16 bytes, no swizzle), for tcgen05.cp.
T0B_DEV uint64_t scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(128u >> 4) << 32 | (uint64_t)1 << 46;
}
// Copies a scale tile into four TMEM columns, the 32 rows repeated in the four
// lane quarters, in both CTAs of a pair (each from its own shared memory).
T0B_DEV void scale_cp_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// Instruction descriptor of the block-scaled 4-bit product: e2m1 A and B
// (format 1), scales as unsigned e4m3 (NV) or powers of two, M x N, K-major.
template <bool NV>
__host__ __device__ constexpr uint32_t idesc_fp4(int M, int N) {
  return 1u << 7 | 1u << 10 | (uint32_t)(N >> 3) << 17 | (NV ? 0u : 1u) << 23 | (uint32_t)(M >> 4) << 24;
}
// Which bytes of the scale words a K = 64 step uses (blocks of 32: two of the
// four, so steps alternate; blocks of 16: all four).
T0B_DEV uint32_t idesc_scale_id(uint32_t id) { return id << 4 | id << 29; }
template <bool NV>
T0B_DEV void umma_fp4_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t acc) {
  if constexpr (NV)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
        : "memory");
}

// One lane of a converged warp, known to the compiler as such: what it issues
// keeps its operands in uniform registers.  (Chosen by `lane == 0`, the MMA
// warp issued an 8192 x 8192 x 8192 product's instructions in 360 us instead
// of 193; loops and waits stay with the whole warp.)
T0B_DEV bool elect_one() {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(ok));
  return ok != 0;
}

// Arguments of the product kernels beside the tensor maps.
struct Fp4Args {
  int M, n, K;     // tokens, result columns (a gated product's F), values
  int kt;          // scale tiles along K
  float alpha;     // product of the tensor scales
  const float *bias;
  void *y;
  int64_t ld;
  Fp4Mat q;        // the 4-bit result, where the kernel quantises it
  int up_row;      // gated: first up row (F)
  int n_tiles_n, n_tiles;
  bool vec;        // rows of y can be written in 16-byte pieces
  int *err;
};

// The product on CTA pairs (cta_group::2): 256 tokens x 256 weight rows a
// tile, one M = 256, N = 256, K = 64 block-scaled MMA over both CTAs'
// tiles of codes per step; CTA r holds tokens 128 r .. of the tile and weight
// rows 128 r .. (gated: CTA 0 gate rows, CTA 1 the matching up rows), and the
// scales of its tokens and of all 256 weight rows.  256 columns of tensor
// memory hold the sums, the others a set of scales per stage (tcgen05.cp), so
// a set is not written before its stage's MMAs are done.  The epilogue holds a
// tile's sums in registers and gives the columns back before it does anything
// else; it works while the next tile is multiplied.
// Bound by the tensor cores and, in a long run, by the power limit: 8192 x
// 8192 x 8192 MX 170 to 177 us, NV 176 to 188 us in a graph of ten, by the card
// (6.5 to 5.8 PFLOP/s; 192 and 199 us as single launches after a pause); short K by the
// epilogue: 65,536 x 1024 x 1024 to f32 54 us (268 MB written), gated and
// quantised 32,768 x 4096 x 1024 MX 131 to 134 us, NV 145 to 149 us.  There no
// unit is full (XU 47 %, tensor pipe 42 %, issue 0.44 a cycle): the 16 epilogue
// warps start on one barrier and go through loads, exp and reciprocal, and
// quantisation in step, and the next tile waits for the one accumulator.
// Measured and not kept: three accumulators of 128 columns in turn (equal,
// NV 9 % slower: the MMA warp issues twice the MMAs); the scale copies by
// another warp (8 % slower: one more hop a stage); token tiles fastest (equal).
constexpr int PAIR_EPI_WARPS = 16;
constexpr int PAIR_THREADS = 128 + 32 * PAIR_EPI_WARPS;
// Registers per thread (setmaxnreg): the kernel is launched with PAIR_REGS and
// its warpgroups divide them; the host refuses a build with another count.
constexpr int PAIR_REGS = 96, PAIR_REGS_LOW = 32, PAIR_REGS_EPI = 112;
static_assert(PAIR_REGS_LOW * 128 + PAIR_REGS_EPI * 32 * PAIR_EPI_WARPS <= PAIR_REGS * PAIR_THREADS, "registers over the launch's");

template <bool NV, bool ROT>
struct PairCfg {
  static constexpr int AT = NV ? 4 : 2;                    // scale tiles of a 256-value stage
  static constexpr uint32_t CODES = 128 * 128;             // one operand's codes of a stage
  static constexpr uint32_t SC = AT * 512;                 // 128 rows' scales of a stage
  static constexpr uint32_t STAGE = 2 * CODES + (ROT ? 5 : 3) * SC;
  static constexpr int NS = NV && ROT ? 4 : 5;             // stages
  static constexpr uint32_t OFF_A = 0, OFF_B = CODES, OFF_SA = 2 * CODES, OFF_SB = OFF_SA + SC, OFF_RAW = OFF_SB + 2 * SC;
  static constexpr uint32_t OFF_STG = NS * STAGE;          // 32 rows x 64 bytes per epilogue warp
  static constexpr uint32_t OFF_BIAS = OFF_STG + PAIR_EPI_WARPS * 2048;  // 64 floats per epilogue warp
  static constexpr uint32_t OFF_BAR = OFF_BIAS + PAIR_EPI_WARPS * 256, USED = OFF_BAR + 256;
  // and up to 1024 bytes to align the start, which is aligned already as far as it goes
  static constexpr uint32_t SMEM = USED + 1024 < 232448 ? USED + 1024 : 232448;
  static constexpr uint32_t SFC = AT * 12;                 // TMEM columns of a stage's scales
  static_assert(256 + NS * SFC <= 512, "accumulator and scales in TMEM");
  static_assert(STAGE % 1024 == 0 && USED <= 232448, "shared memory");
};

// 32 consecutive values of row r, columns c0 .. (a multiple of 32), to 4 bits;
// values behind the matrix are taken as zero and its padding is written.
template <bool NV>
T0B_DEV void store_quant32(const Fp4Mat &q, int r, int c0, float *v) {
  constexpr int BLK = NV ? 16 : 32, NB = 32 / BLK;
  const int kt = (q.k + 4 * BLK - 1) / (4 * BLK);
  if (r >= (q.rows + 127) / 128 * 128 || c0 >= kt * 4 * BLK) return;
  if (r >= q.rows || c0 + 32 > q.k) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (r >= q.rows || c0 + j >= q.k) v[j] = 0.0f;
  }
  uint32_t w[4], sc = 0;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const BlockScale<NV> s(__float_as_uint(absmax_of<BLK>(v + b * BLK)), q);
    sc |= s.byte << (8 * b);
#pragma unroll
    for (int i = 0; i < BLK / 8; ++i) w[b * BLK / 8 + i] = quantize8<NV>(s, v + b * BLK + 8 * i);
  }
  uint8_t *ps = q.scales + scale_at(r, c0 / BLK, kt);
  if (NV)
    *reinterpret_cast<uint16_t *>(ps) = (uint16_t)sc;
  else
    *ps = (uint8_t)sc;
  if (r < q.rows && c0 < q.k) *reinterpret_cast<uint4 *>(q.codes + r * code_pitch(q.k) + c0 / 2) = make_uint4(w[0], w[1], w[2], w[3]);
}

// 32 rows x 64 bytes of the result, one row per lane, columns c0 .. : through
// the warp's staging buffer (64-byte swizzle) and out by a TMA store.  A TMA
// store ends a row on a 16-byte boundary, not at the tensor's last column: the
// 64 bytes that hold the end of rows of another width are written value by
// value, as nothing behind the last column may be touched.
template <int TY>
T0B_DEV void store_rows(const Fp4Args &p, const void *tm_y, uint8_t *stg, int row0, int c0, const float *v) {
  using T = typename Plain<TY>::T;
  constexpr int W = 64 / sizeof(T);
  if (c0 + W > p.n && p.n % (16 / (int)sizeof(T))) {
    const int row = row0 + (threadIdx.x & 31);
    T *y = reinterpret_cast<T *>(p.y) + row * p.ld + c0;
#pragma unroll
    for (int j = 0; j < W; ++j)
      if (row < p.M && c0 + j < p.n) y[j] = Plain<TY>::put(v[j]);
    return;
  }
  const int lane = threadIdx.x & 31;
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  __syncwarp();  // the buffer has been read
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    constexpr int PER = 16 / sizeof(T);
    Pack<T, PER> t;
#pragma unroll
    for (int j = 0; j < PER; ++j) t.v[j] = Plain<TY>::put(v[i * PER + j]);
    *reinterpret_cast<uint4 *>(stg + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) = *reinterpret_cast<const uint4 *>(&t);
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    if (row0 < p.M && c0 < p.n && T0B_CHECK_TMA(c0, (int)sizeof(T), row0, p.err)) tma_store_2d(tm_y, stg, c0, row0);
    bulk_commit();
  }
}

// The same where the result's rows are not 16-byte aligned: the four warps h of
// a lane quarter bring their 64 bytes a row together in the quarter's 8 KB
// (16-byte pieces swizzled by the row), and each writes 8 of the 32 rows, 256
// bytes of a row at a time: the sectors at both ends are written in part, and
// that is what unaligned rows cost.  32,768 x 4001 x 1024 to bf16 116 us, to
// f32 189 us; with 64 bytes of a row at a time 214 and 309 us.  In aligned rows:
// bf16 86 us (4008 values apart) to 70 us (4032 apart: 128 bytes), f32 97 to
// 101 us.
T0B_DEV void quarter_sync(int q) { asm volatile("bar.sync %0, 128;" ::"r"(2 + q) : "memory"); }
template <int TY>
T0B_DEV void store_rows_unaligned(const Fp4Args &p, uint8_t *quarter, int q, int h, int row0, int c0, const float *v) {
  using T = typename Plain<TY>::T;
  constexpr int W = 256 / sizeof(T), PER = 16 / sizeof(T);  // columns of the four warps
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    Pack<T, PER> t;
#pragma unroll
    for (int j = 0; j < PER; ++j) t.v[j] = Plain<TY>::put(v[i * PER + j]);
    *reinterpret_cast<uint4 *>(quarter + lane * 256 + (((4 * h + i) ^ (lane & 15)) << 4)) = *reinterpret_cast<const uint4 *>(&t);
  }
  quarter_sync(q);
  const int first = c0 - W / 4 * h, n = p.n - first;
  const int rows = min(8, p.M - row0 - 8 * h);
  T *y = reinterpret_cast<T *>(p.y) + (int64_t)(row0 + 8 * h) * p.ld + first + lane;
  constexpr int B = 2 * sizeof(T);  // rows at a time
#pragma unroll 1
  for (int r0 = 0; r0 < rows; r0 += B) {
    T t[B][W / 32];
#pragma unroll
    for (int r = 0; r < B; ++r)
#pragma unroll
      for (int i = 0; i < W / 32; ++i) {
        const int c = lane + 32 * i, row = 8 * h + r0 + r;
        t[r][i] = *reinterpret_cast<const T *>(quarter + row * 256 + (((c / PER) ^ (row & 15)) << 4) + c % PER * (int)sizeof(T));
      }
#pragma unroll
    for (int r = 0; r < B; ++r, y += p.ld)
      if (r0 + r < rows)
#pragma unroll
        for (int i = 0; i < W / 32; ++i)
          if (lane + 32 * i < n) y[32 * i] = t[r][i];
  }
  quarter_sync(q);
}

// The scale tiles hold 128 rows from a multiple of 128 on; the up rows of a
// gated tile start at F + f0, `off` rows into one.  Moves the scales of 128
// rows from two row groups' tiles to their place in one (one warp, every lane
// of which has waited for the tiles), ready for the async proxy.
template <int AT>
T0B_DEV void move_scales(uint8_t *to, const uint8_t *from, int off) {
  const int lane = threadIdx.x & 31;
  uint32_t *dst = reinterpret_cast<uint32_t *>(to);
  const uint32_t *raw = reinterpret_cast<const uint32_t *>(from);
#pragma unroll
  for (int a = 0; a < AT; ++a)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = off + 32 * j + lane;
      dst[a * 128 + lane * 4 + j] = raw[(r >> 7) * (AT * 128) + a * 128 + (r & 31) * 4 + ((r >> 5) & 3)];
    }
  fence_proxy_async_smem();
  __syncwarp();
}

// TY: result type, or -1 for the 4-bit result of a gated product.
template <bool NV, bool GLU, bool ROT, int TY>
__global__ void __launch_bounds__(PAIR_THREADS, 1)
    fp4_gemm_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                         const __grid_constant__ CUtensorMap tm_xs, const __grid_constant__ CUtensorMap tm_ws,
                         const __grid_constant__ CUtensorMap tm_y, Fp4Args p) {
  using C = PairCfg<NV, ROT>;
  constexpr int AT = C::AT, NS = C::NS;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t *smem = smem_raw + (base - smem_u32(smem_raw));
  if (cluster_size() != 2 || base - smem_u32(smem_raw) > C::SMEM - C::USED) {
    if (threadIdx.x == 0) record_error(p.err, T0B_DEVERR_SHAPE);
    return;
  }
  const uint32_t rank = cluster_rank();
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::OFF_BAR);  // [NS] bytes of both CTAs (CTA 0's)
  uint64_t *empty = full + NS;       // [NS] the stage's MMAs are done (each CTA's)
  uint64_t *raw_full = empty + NS;   // [NS] up rows' scales as they are held (each CTA's; ROT)
  uint64_t *rot_full = raw_full + NS;  // [NS] and moved to the tile's rows, both CTAs (CTA 0's; ROT)
  uint64_t *acc_full = rot_full + NS;  // each CTA's
  uint64_t *acc_empty = acc_full + 1;  // epilogue warps of both CTAs (CTA 0's)
  uint64_t *mma_done = acc_empty + 1;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(mma_done + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(mma_done + 2);
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int S = (p.K + 255) / 256;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
      mbar_init(&raw_full[i], 1);
      mbar_init(&rot_full[i], 2);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 2 * PAIR_EPI_WARPS);
    mbar_init(mma_done, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_xs);
    prefetch_tmap(&tm_ws);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();
  auto lead = [](const uint64_t *b) { return mapa_shared(smem_u32(b), 0); };
  // first weight row of this CTA's half, and of each half's scales
  auto w_row = [&](int nt, uint32_t half) { return GLU ? nt * 128 + (half ? p.up_row : 0) : nt * 256 + 128 * (int)half; };

  if (warp < 4) {
    setmaxnreg_dec<PAIR_REGS_LOW>();
    if (warp == 0 && elect_one()) {
      // ------------------------------------------------------------ loads (both CTAs)
      uint32_t g = 0;
      for (int tile = pair; tile < p.n_tiles && !*abort_flag; tile += npairs) {
        const int nt = tile % p.n_tiles_n, m0 = tile / p.n_tiles_n * 256 + 128 * (int)rank;
        for (int s = 0; s < S && !*abort_flag; ++s, ++g) {
          const uint32_t sl = g % NS;
          if (g >= NS && !mbar_wait(&empty[sl], (g / NS - 1) & 1, p.err, T0B_DEVERR_WAIT_EMPTY, abort_flag)) break;
          uint8_t *st = smem + sl * C::STAGE;
          if (rank == 0) mbar_arrive_expect_tx(&full[sl], 4 * C::CODES + (ROT ? 4 : 6) * C::SC);
          const uint32_t fb = lead(&full[sl]);
          if (!T0B_CHECK_TMA(s * 128, 1, m0, p.err) || !T0B_CHECK(w_row(nt, 1) >= 0 && s * AT < p.kt, p.err)) continue;
          // (byte, row) of the codes, (tile, row group) of the scales; what lies
          // behind the matrix arrives as zeros
          tma_load_2d_pair(st + C::OFF_A, &tm_x, fb, s * 128, m0);
          tma_load_2d_pair(st + C::OFF_B, &tm_w, fb, s * 128, w_row(nt, rank));
          tma_load_3d_pair(st + C::OFF_SA, &tm_xs, fb, 0, s * AT, m0 >> 7);
          tma_load_3d_pair(st + C::OFF_SB, &tm_ws, fb, 0, s * AT, w_row(nt, 0) >> 7);
          if constexpr (!ROT) {
            tma_load_3d_pair(st + C::OFF_SB + C::SC, &tm_ws, fb, 0, s * AT, w_row(nt, 1) >> 7);
          } else {
            mbar_arrive_expect_tx(&raw_full[sl], 2 * C::SC);
            tma_load_3d(st + C::OFF_RAW, &tm_ws, &raw_full[sl], 0, s * AT, w_row(nt, 1) >> 7);
            tma_load_3d(st + C::OFF_RAW + C::SC, &tm_ws, &raw_full[sl], 0, s * AT, (w_row(nt, 1) >> 7) + 1);
          }
        }
      }
      // Copies in flight have landed before the shared memory is given up, also
      // after a wait that ran out (CTA 0's barriers count both CTAs' copies, and
      // both CTAs leave together).
      for (uint32_t i = g > NS ? g - NS : 0; i < g; ++i) {
        if (rank == 0) mbar_wait(&full[i % NS], (i / NS) & 1, p.err, T0B_DEVERR_WAIT_X, nullptr);
        if (ROT) mbar_wait(&raw_full[i % NS], (i / NS) & 1, p.err, T0B_DEVERR_WAIT_W, nullptr);
      }
    } else if (warp == 1 && rank == 0) {
      // ------------------------------------------------------------ MMA (CTA 0)
      constexpr uint32_t idesc = idesc_fp4<NV>(256, 256);
      const int steps = (p.K + 63) / 64;
      const uint64_t da = sw128_desc(base + C::OFF_A), db = sw128_desc(base + C::OFF_B);
      const uint64_t dsa = scale_desc(base + C::OFF_SA), dsb = scale_desc(base + C::OFF_SB);
      uint32_t sl = 0, phase = 0, it = 0;
      bool ok = true;
      for (int tile = pair; tile < p.n_tiles && ok; tile += npairs, ++it) {
        if (it >= 1) ok = mbar_wait(acc_empty, (it - 1) & 1, p.err, T0B_DEVERR_WAIT_ACC, abort_flag);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        tc_fence_after();
        for (int s = 0; s < S; ++s) {
          ok = mbar_wait(&full[sl], phase, p.err, T0B_DEVERR_WAIT_X, abort_flag) &&
               (!ROT || mbar_wait(&rot_full[sl], phase, p.err, T0B_DEVERR_WAIT_DEQ, abort_flag));
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) break;
          tc_fence_after();
          const uint64_t at = sl * (C::STAGE >> 4);
          const uint32_t sf = tmem + 256 + sl * C::SFC;
          const int n = steps - 4 * s;
          if (elect_one()) {
#pragma unroll
            for (int a = 0; a < AT; ++a) {
              scale_cp_pair(sf + 4 * a, dsa + at + 32 * a);
              scale_cp_pair(sf + 4 * AT + 8 * a, dsb + at + 32 * a);
              scale_cp_pair(sf + 4 * AT + 8 * a + 4, dsb + at + (C::SC >> 4) + 32 * a);
            }
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              if (kk < n) {
                const int a = NV ? kk : kk / 2;
                umma_fp4_pair<NV>(tmem, da + at + 2 * kk, db + at + 2 * kk, idesc | (NV ? 0u : idesc_scale_id(kk % 2 * 2)),
                                  sf + 4 * a, sf + 4 * AT + 8 * a, s > 0 || kk > 0);
              }
            umma_commit_pair_both(&empty[sl]);
            if (s == S - 1) umma_commit_pair_both(acc_full);
          }
          __syncwarp();
          if (++sl == NS) sl = 0, phase ^= 1;
        }
      }
      if (elect_one()) umma_commit_pair(smem_u32(mma_done));
      __syncwarp();
      mbar_wait(mma_done, 0, p.err, T0B_DEVERR_WAIT_ACC, nullptr);
    } else if (ROT && warp == 2) {
      // ------------------------------------------------------------ up rows' scales (both CTAs)
      uint32_t g = 0;
      const int off = p.up_row & 127;
      bool ok = true;
      for (int tile = pair; tile < p.n_tiles && ok && !*abort_flag; tile += npairs) {
        for (int s = 0; s < S; ++s, ++g) {
          const uint32_t sl = g % NS;
          ok = __all_sync(0xFFFFFFFFu, mbar_wait(&raw_full[sl], (g / NS) & 1, p.err, T0B_DEVERR_WAIT_W, abort_flag));
          if (!ok) break;
          uint8_t *st = smem + sl * C::STAGE;
          move_scales<AT>(st + C::OFF_SB + C::SC, st + C::OFF_RAW, off);
          if (lane == 0) mbar_arrive_cluster(lead(&rot_full[sl]));
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    setmaxnreg_inc<PAIR_REGS_EPI>();
    // Lane quarter q; of the tile's columns this warp has W from W h on, and
    // every 4 W further (W: 64 bytes of the result), gated the up ones too.
    constexpr int OT = TY < 0 ? TY_F32 : TY, W = TY == TY_F32 ? 16 : 32, N = (GLU ? 32 : 64) / W;
    const int q = warp & 3, h = (warp - 4) >> 2;
    uint8_t *stg = smem + C::OFF_STG + (4 * q + h) * 2048;
    float *sb = reinterpret_cast<float *>(smem + C::OFF_BIAS) + (warp - 4) * 64;
    uint32_t it = 0;
    for (int tile = pair; tile < p.n_tiles; tile += npairs, ++it) {
      const int nt = tile % p.n_tiles_n, m0 = tile / p.n_tiles_n * 256 + 128 * (int)rank;
      const int n0 = nt * (GLU ? 128 : 256);
      // this warp's 64 biases (gated: 32 gate, 32 up)
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = GLU ? lane : 32 * i + lane, c = n0 + W * h + j / W * 4 * W + j % W;
        sb[32 * i + lane] = p.bias && c < p.n ? p.bias[GLU && i ? p.n + c : c] : 0.0f;
      }
      __syncwarp();
      const int row0 = m0 + 32 * q;
      const uint32_t trow = tmem + ((uint32_t)(32 * q) << 16) + W * h;
      bool have = mbar_wait(acc_full, it & 1, p.err, T0B_DEVERR_WAIT_ACC, abort_flag) && !*abort_flag;
      have = __all_sync(0xFFFFFFFFu, have);
      tc_fence_after();
      uint32_t r[2][32];
      if (have) {
        if constexpr (W == 32) {
          tmem_ld32(trow, r[0]);
          tmem_ld32(trow + 128, r[1]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) tmem_ld16(trow + 64 * i, r[i / 2] + 16 * (i % 2));
        }
        tmem_ld_wait(r[0]);
        tmem_ld_wait(r[1]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(lead(acc_empty));
      if (TY >= 0 && !p.vec) {  // the quarter's warps go on together or not at all
        int all;
        asm volatile("{\n .reg .pred a, b;\n setp.ne.b32 a, %1, 0;\n barrier.cta.red.and.pred b, %2, 128, a;\n selp.b32 %0, 1, 0, b;\n}"
                     : "=r"(all)
                     : "r"((int)have), "r"(2 + q)
                     : "memory");
        have = all;
      }
      if (!have) continue;
      auto store = [&](int i, const float *v) {
        if (p.vec)
          store_rows<OT>(p, &tm_y, stg, row0, n0 + W * h + 4 * W * i, v);
        else
          store_rows_unaligned<OT>(p, smem + C::OFF_STG + q * 8192, q, h, row0, n0 + W * h + 4 * W * i, v);
      };
      if constexpr (!GLU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          float v[W];
#pragma unroll
          for (int j = 0; j < W; j += 4) {
            const float4 b = *reinterpret_cast<const float4 *>(sb + W * i + j);
            const uint32_t *a = r[i * W / 32] + i * W % 32 + j;
            v[j] = fmaf(__uint_as_float(a[0]), p.alpha, b.x);
            v[j + 1] = fmaf(__uint_as_float(a[1]), p.alpha, b.y);
            v[j + 2] = fmaf(__uint_as_float(a[2]), p.alpha, b.z);
            v[j + 3] = fmaf(__uint_as_float(a[3]), p.alpha, b.w);
          }
          store(i, v);
        }
      } else {
        const F2 alpha(p.alpha, p.alpha);
        float *g = reinterpret_cast<float *>(r[0]), *u = reinterpret_cast<float *>(r[1]), *v = g;
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 b = *reinterpret_cast<const float4 *>(sb + j), d = *reinterpret_cast<const float4 *>(sb + 32 + j);
          fma2(F2(g[j], g[j + 1]), alpha, F2(b.x, b.y)).get(g[j], g[j + 1]);
          fma2(F2(g[j + 2], g[j + 3]), alpha, F2(b.z, b.w)).get(g[j + 2], g[j + 3]);
          fma2(F2(u[j], u[j + 1]), alpha, F2(d.x, d.y)).get(u[j], u[j + 1]);
          fma2(F2(u[j + 2], u[j + 3]), alpha, F2(d.z, d.w)).get(u[j + 2], u[j + 3]);
        }
        const float top = absmax_of<32>(g);
        bool body = top <= SILU_TAIL;
        if (!body) {
          float low = 0.0f;
#pragma unroll
          for (int j = 0; j < 32; j += 2) asm("min.f32 %0, %0, %1, %2;" : "+f"(low) : "f"(g[j]), "f"(g[j + 1]));
          body = low >= -SILU_TAIL && top < 1048576.0f;
        }
        if (body) {
#pragma unroll
          for (int j = 0; j < 32; j += 2) silu_mul2(F2(g[j], g[j + 1]), F2(u[j], u[j + 1])).get(v[j], v[j + 1]);
        } else {  // rare: one value at a time, from local memory (unrolled, it cost the others 4 %)
          float lg[32], lu[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) lg[j] = g[j], lu[j] = u[j];
#pragma unroll 1
          for (int j = 0; j < 32; ++j) lg[j] = silu_mul(lg[j], lu[j]);
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = lg[j];
        }
        if constexpr (TY >= 0) {
#pragma unroll
          for (int i = 0; i < N; ++i) store(i, v + W * i);
        } else {
          store_quant32<NV>(p.q, row0 + lane, n0 + 32 * h, v);
        }
      }
    }
    if (lane == 0) bulk_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ------------------------------------------------- product, few tokens
// The product for launches with few pair tiles: a CTA multiplies 128 weight
// rows (MMA rows; gated: 128 gate rows and the 128 matching up rows, two
// accumulators) with up to 128 tokens (MMA columns) over one slice of K, and
// the slices of a tile form a thread-block cluster.  Every SM gets a share of
// the weights, which is what such a product has to read; the partial tiles
// meet in distributed shared memory, each CTA adding the slices of its share
// of the tokens in slice order.  With rows as lanes the results of a token are
// 32 consecutive columns of a warp: stores are coalesced whatever the row
// stride, and a 4-bit result's blocks are joined by shuffles.  FUSED: x is
// plain and each CTA quantises its slice of the tokens into shared memory
// itself (one launch, no 4-bit activations in memory).
// Bound by its chain of latencies (launch, loads, MMA, exchange, stores): 1
// token 512 x 512 3.0 us, 4096 x 4096 4.8 us (the pair kernel: 8.9); 19 tokens
// gated 4096 x 1024 5.2 us (10.1); 333 x 1001 x 1000 5.4 us (9.9).
constexpr int SPLIT_THREADS = 256;
constexpr int SPLIT_MAX_NS = 6;

struct SplitArgs {
  Fp4Args a;
  int NT, CS, SL, NS;       // tokens of a tile (a multiple of 8), K slices, stages of a slice, ring depth
  int rt;                   // weight row tiles
  uint32_t stage;           // bytes of a ring stage
  uint32_t off_x, off_xs;   // FUSED: the slice's activation codes and scales
  uint32_t off_slot, off_bar;
  uint32_t tmem_cols;
  int out_type;             // ggml type of y, or -1: the 4-bit result
  int rot;                  // gated: up rows' scales must be moved (F % 128 != 0)
  int early;                // the previous kernel on the stream does not write the weights
  const void *x;            // FUSED
  int x_type;
  int64_t ldx;
  Fp4Mat xq;                // its scales' constants
  int xalign;               // bytes its rows start on
};

// One value per lane and row, 32 consecutive columns c0 .. c0 + 31 (zeros behind
// the matrix) of `rows` <= 4 rows from r on, to 4 bits: largest magnitudes and
// words of codes by shuffles, the rows side by side so that their latencies
// overlap.  Every lane of the warp calls it; c0 is a multiple of 32.
template <bool NV>
T0B_DEV void quantize_lanes4(const Fp4Mat &q, int r, int rows, int c0, const float *v) {
  constexpr int BLK = NV ? 16 : 32;
  const int lane = threadIdx.x & 31, kt = (q.k + 4 * BLK - 1) / (4 * BLK);
  float top[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) top[j] = fabsf(v[j]);
#pragma unroll
  for (int o = BLK / 2; o; o >>= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) top[j] = absmax(top[j], __shfl_xor_sync(0xFFFFFFFFu, top[j], o), 0.0f);
  uint32_t byte[4], w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const BlockScale<NV> s(__float_as_uint(top[j]), q);
    byte[j] = s.byte;
    w[j] = quantize1<NV>(s, v[j]) << (4 * (lane & 7));
  }
#pragma unroll
  for (int o = 1; o < 8; o *= 2)
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] |= __shfl_xor_sync(0xFFFFFFFFu, w[j], o);
  const int b = (c0 + lane) / BLK;
  const bool has_scale = lane % BLK == 0 && b < 4 * kt, has_codes = lane % 8 == 0 && (c0 + lane) / 2 < (int)code_pitch(q.k);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j >= rows) break;
    if (has_scale) q.scales[scale_at(r + j, b, kt)] = b * BLK < q.k ? (uint8_t)byte[j] : 0;
    if (has_codes) *reinterpret_cast<uint32_t *>(q.codes + (r + j) * code_pitch(q.k) + (c0 + lane) / 2) = w[j];
  }
}

T0B_DEV void scale_cp(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <bool NV>
T0B_DEV void umma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t acc) {
  if constexpr (NV)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
        : "memory");
}
T0B_DEV void umma_commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
T0B_DEV void st_cluster_f32x4(uint32_t addr, const float *v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3])
               : "memory");
}
T0B_DEV void add4(float4 &a, const float4 &b) { a.x += b.x, a.y += b.y, a.z += b.z, a.w += b.w; }

// Bytes of a stage: weight codes, weight scales (gated: two halves, and room
// for the up rows' scales as they are held), then, unless FUSED, the tokens'.
template <bool NV, bool GLU, bool FUSED>
__host__ __device__ constexpr uint32_t split_stage(int NT) {
  const uint32_t sc = (NV ? 4 : 2) * 512;
  const uint32_t n = (GLU ? 2 : 1) * 16384u + (GLU ? 4 : 1) * sc + (FUSED ? 0u : (uint32_t)NT * 128u + sc);
  return (n + 1023u) & ~1023u;
}

template <int TY, bool NV>
T0B_DEV void quantize_slice(const SplitArgs &p, uint8_t *codes, uint8_t *scales, int m0, int toks, int k_begin, int stages) {
  // a warp takes 256 values (a stage) of a token, four such pieces at a time,
  // the next four on their way meanwhile
  constexpr int AT = NV ? 4 : 2, BLK = NV ? 16 : 32, LB = BLK / 8, U = 4, W = SPLIT_THREADS / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const auto *x = reinterpret_cast<const typename Plain<TY>::T *>(p.x);
  const int n = toks * stages;
  const uint32_t inv = (65536u + (uint32_t)stages - 1) / (uint32_t)stages;  // i / stages for i < 4096, stages <= SPLIT_FUSED_MAX_SL
  auto token = [&](int i) { return (int)((uint32_t)i * inv >> 16); };
  Raw8<TY> next[U];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * W, t = token(i);
      if (i < n) next[u].load(x + (int64_t)(m0 + t) * p.ldx, k_begin + (i - t * stages) * 256 + lane * 8, p.a.K, p.xalign);
    }
  };
  fetch(warp);
  for (int i0 = warp; i0 < n; i0 += U * W) {
    Raw8<TY> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = next[u];
    fetch(i0 + U * W);
    auto piece = [&](int u) {
      const int i = i0 + u * W, t = token(i), s = i - t * stages;
      float v[8];
      raw[u].get(v);
      float top = absmax_of<8>(v);
#pragma unroll
      for (int o = 1; o < LB; o *= 2) top = absmax(top, __shfl_xor_sync(0xFFFFFFFFu, top, o), 0.0f);
      const BlockScale<NV> sc(__float_as_uint(top), p.xq);
      // 128-byte rows, 16-byte pieces swizzled by the row
      *reinterpret_cast<uint32_t *>(codes + (s * p.NT + t) * 128 + (((lane >> 2) ^ (t & 7)) << 4) + (lane & 3) * 4) =
          quantize8<NV>(sc, v);
      if (lane % LB == 0)
        scales[(s * AT + lane / (4 * LB)) * 512 + (t & 31) * 16 + (t >> 5) * 4 + lane / LB % 4] =
            k_begin + s * 256 + lane * 8 < p.a.K ? (uint8_t)sc.byte : 0;
    };
    // without branches between them the pieces overlap
    const int left = (n - i0 + W - 1) / W;
    if (left >= 4)
      piece(0), piece(1), piece(2), piece(3);
    else if (left == 3)
      piece(0), piece(1), piece(2);
    else if (left == 2)
      piece(0), piece(1);
    else
      piece(0);
  }
}

// Four values with a gate below -SILU_TAIL among them: rare, and out of the way of the others.
__device__ __noinline__ float4 silu_mul4(float4 g, float4 u) {
  return make_float4(silu_mul(g.x, u.x), silu_mul(g.y, u.y), silu_mul(g.z, u.z), silu_mul(g.w, u.w));
}

// The results of a tile.  Warps 0 .. 3 and 4 .. 7 take alternate groups of 16
// tokens; a thread has one weight row.  The slices' partial sums go to the CTA
// that adds them as [source][four tokens][gate, up][row][token], 16 bytes a
// thread.  OT: result type, -1 the 4-bit result.
template <bool NV, bool GLU, int OT>
T0B_DEV void split_results(const SplitArgs &p, uint8_t *slots, uint32_t tmem, int rank, int n0, int m0, int toks, bool have) {
  constexpr int H = GLU ? 2 : 1, TY = OT < 0 ? TY_F32 : OT;
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int NT = p.NT, CS = p.CS;
  const int half = warp >> 2, row = 32 * (warp & 3) + lane, n = n0 + row;
  const int sh4 = ((NT + CS - 1) / CS + 3) / 4;  // groups of four tokens whose slices a CTA adds
  const uint32_t trow = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
  const float alpha = p.a.alpha;
  float b0 = 0.0f, b1 = 0.0f;
  if (p.a.bias && n < p.a.n) {
    b0 = p.a.bias[n];
    if (GLU) b1 = p.a.bias[p.a.n + n];
  }
  typename Plain<TY>::T *y = reinterpret_cast<typename Plain<TY>::T *>(p.a.y) + m0 * p.a.ld + n;
  const bool in = n < p.a.n;
  auto finish4 = [&](int t0, const float *g, const float *u) {  // tokens t0 .. t0 + 3 of the tile
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = fmaf(g[j], alpha, b0);
    if constexpr (GLU) {
      float h[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = fmaf(u[j], alpha, b1);
      if (fminf(fminf(v[0], v[1]), fminf(v[2], v[3])) >= -SILU_TAIL) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = silu_mul_body(v[j], h[j]);
      } else {
        const float4 r = silu_mul4(make_float4(v[0], v[1], v[2], v[3]), make_float4(h[0], h[1], h[2], h[3]));
        v[0] = r.x, v[1] = r.y, v[2] = r.z, v[3] = r.w;
      }
    }
    if constexpr (OT >= 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (in && t0 + j < toks) y[(t0 + j) * p.a.ld] = Plain<TY>::put(v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = in ? v[j] : 0.0f;
      quantize_lanes4<NV>(p.a.q, m0 + t0, min(4, toks - t0), n0 + 32 * (warp & 3), v);
    }
  };
  for (int t0 = 16 * half; t0 < toks && have; t0 += 32) {
    uint32_t g[16], u[16];
    tmem_ld16(trow + t0, g);
    if (GLU) tmem_ld16(trow + NT + t0, u);
    tmem_ld_wait16(g);
    if (GLU) tmem_ld_wait16(u);
    const float *gf = reinterpret_cast<const float *>(g), *uf = reinterpret_cast<const float *>(u);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int c4 = t0 / 4 + c;
      if (4 * c4 >= toks) break;
      if (CS == 1) {
        finish4(4 * c4, gf + 4 * c, uf + 4 * c);
      } else {
        const int owner = c4 / sh4;
        const uint32_t at = mapa_shared(smem_u32(slots) + (((rank * sh4 + c4 - owner * sh4) * H) * 128 + row) * 16, owner);
        st_cluster_f32x4(at, gf + 4 * c);
        if (GLU) st_cluster_f32x4(at + 2048, uf + 4 * c);
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  if (CS > 1) {
    cluster_sync_all();
    const float4 *slot = reinterpret_cast<const float4 *>(slots) + row;
    for (int c4 = half; c4 < sh4 && have; c4 += 2) {
      const int t0 = 4 * (rank * sh4 + c4);
      if (t0 >= toks) break;
      float4 g[2] = {};
#pragma unroll
      for (int c = 0; c < SPLIT_MAX_CLUSTER; ++c) {
        if (c >= CS) break;
        const float4 *v = slot + (c * sh4 + c4) * H * 128;
        add4(g[0], v[0]);
        if (GLU) add4(g[1], v[128]);
      }
      finish4(t0, &g[0].x, &g[1].x);
    }
  } else {
    __syncthreads();
  }
  if (OT < 0 && m0 + NT >= p.a.M && rank == 0) {
    // zero scales of the last row group's rows behind the last token
    const int m = p.a.M + (int)threadIdx.x % 128;
    constexpr int TILES = NV ? 2 : 1;  // scale tiles of 128 columns
    const int t = n0 / 128 * TILES + (int)threadIdx.x / 128, kt = (p.a.q.k + (NV ? 63 : 127)) / (NV ? 64 : 128);
    if (m < (p.a.M + 127) / 128 * 128 && (int)threadIdx.x / 128 < TILES && t < kt)
      *reinterpret_cast<uint32_t *>(p.a.q.scales + scale_at(m, 4 * t, kt)) = 0;
  }
}

// Waits for the copies of the last of `issued` stages of a ring of NS.
T0B_DEV void drain(uint64_t *full, int NS, int issued, int *err, int code) {
  for (int i = max(0, issued - NS); i < issued; ++i) mbar_wait(&full[i % NS], (i / NS) & 1, err, code, nullptr);
}

template <bool NV, bool GLU, bool FUSED>
__global__ void __launch_bounds__(SPLIT_THREADS, 1)
    fp4_gemm_split_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                          const __grid_constant__ CUtensorMap tm_xs, const __grid_constant__ CUtensorMap tm_ws, SplitArgs p) {
  constexpr int AT = NV ? 4 : 2, H = GLU ? 2 : 1;
  constexpr uint32_t SC = AT * 512, OFF_WS = H * 16384, OFF_RAW = OFF_WS + 2 * SC, OFF_X = OFF_WS + (GLU ? 4 : 1) * SC;
  constexpr uint32_t SFC = AT * 4 * (H + 1);  // TMEM columns of a stage's scales
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t *smem = smem_raw + (base - smem_u32(smem_raw));
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int NT = p.NT, CS = p.CS, NS = p.NS;
  if ((int)cluster_size() != CS) {
    if (threadIdx.x == 0) record_error(p.a.err, T0B_DEVERR_SHAPE);
    return;
  }
  const uint32_t OFF_XS = OFF_X + NT * 128;
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + p.off_bar), *empty = full + SPLIT_MAX_NS, *raw_full = empty + SPLIT_MAX_NS;
  uint64_t *rot_full = raw_full + SPLIT_MAX_NS, *acc_full = rot_full + SPLIT_MAX_NS;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_full + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(acc_full + 2);
  const int rank = blockIdx.x % CS, tile = blockIdx.x / CS;
  const int n0 = tile % p.rt * 128, m0 = tile / p.rt * NT;
  const int toks = min(NT, p.a.M - m0);
  const int S = (p.a.K + 255) / 256, s0 = rank * p.SL, ns = min(p.SL, S - s0);  // the host leaves no slice empty

  if (threadIdx.x == 0) {
    for (int i = 0; i < SPLIT_MAX_NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
      mbar_init(&raw_full[i], 1);
      mbar_init(&rot_full[i], 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 2 && lane == 0) {
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_ws);
    if (!FUSED) {
      prefetch_tmap(&tm_x);
      prefetch_tmap(&tm_xs);
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(p.tmem_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (CS > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // running: its shared memory may be written
  const uint32_t tmem = *tmem_slot;

  auto load_w = [&](int i) {  // stage i of the slice
    const int sl = i % NS, s = s0 + i;
    uint8_t *st = smem + sl * p.stage;
    if (!T0B_CHECK_TMA(s * 128, 1, n0, p.a.err) || !T0B_CHECK(s * AT < p.a.kt && sl < SPLIT_MAX_NS, p.a.err)) return;
    const bool rot = GLU && p.rot;
    mbar_arrive_expect_tx(&full[sl], H * 16384u + (GLU && !rot ? 2 : 1) * SC + (FUSED ? 0u : (uint32_t)NT * 128u + SC));
    tma_load_2d(st, &tm_w, &full[sl], s * 128, n0);
    tma_load_3d(st + OFF_WS, &tm_ws, &full[sl], 0, s * AT, n0 >> 7);
    if constexpr (GLU) {
      const int u0 = p.a.up_row + n0;
      tma_load_2d(st + 16384, &tm_w, &full[sl], s * 128, u0);
      if (!rot) {
        tma_load_3d(st + OFF_WS + SC, &tm_ws, &full[sl], 0, s * AT, u0 >> 7);
      } else {
        mbar_arrive_expect_tx(&raw_full[sl], 2 * SC);
        tma_load_3d(st + OFF_RAW, &tm_ws, &raw_full[sl], 0, s * AT, u0 >> 7);
        tma_load_3d(st + OFF_RAW + SC, &tm_ws, &raw_full[sl], 0, s * AT, (u0 >> 7) + 1);
      }
    }
  };
  auto load_x = [&](int i) {
    const int sl = i % NS, s = s0 + i;
    uint8_t *st = smem + sl * p.stage;
    if (!T0B_CHECK_TMA(s * 128, 1, m0, p.a.err)) return;
    tma_load_2d(st + OFF_X, &tm_x, &full[sl], s * 128, m0);
    tma_load_3d(st + OFF_XS, &tm_xs, &full[sl], 0, s * AT, m0 >> 7);
  };
  const int first = min(ns, NS);
  const bool loader = warp == 0 && elect_one();
  if (loader && p.early)
    for (int i = 0; i < first; ++i) load_w(i);
  pdl_wait();
  pdl_launch_dependents();
  if (loader) {
    if (!p.early)
      for (int i = 0; i < first; ++i) load_w(i);
    if constexpr (!FUSED)
      for (int i = 0; i < first; ++i) load_x(i);
  }
  if constexpr (FUSED) {
    __syncwarp();
    uint8_t *xc = smem + p.off_x, *xs = smem + p.off_xs;
    if (p.x_type == TY_F32)
      quantize_slice<TY_F32, NV>(p, xc, xs, m0, toks, s0 * 256, ns);
    else if (p.x_type == TY_F16)
      quantize_slice<TY_F16, NV>(p, xc, xs, m0, toks, s0 * 256, ns);
    else
      quantize_slice<TY_BF16, NV>(p, xc, xs, m0, toks, s0 * 256, ns);
    fence_proxy_async_smem();
    __syncthreads();
  }
  int issued = first;
  if (loader) {
    for (; issued < ns; ++issued) {
      if (!mbar_wait(&empty[issued % NS], (issued / NS - 1) & 1, p.a.err, T0B_DEVERR_WAIT_EMPTY, abort_flag)) break;
      load_w(issued);
      if constexpr (!FUSED) load_x(issued);
    }
  } else if (warp == 1 && elect_one()) {
    // ------------------------------------------------------------ MMA
    const uint32_t idesc = idesc_fp4<NV>(128, 0) | (uint32_t)(NT >> 3) << 17;
    const int steps = (p.a.K + 63) / 64;
    const uint32_t sf_col = (uint32_t)(m0 & 127) >> 5;  // the tile's first token in its row group's scale columns
    for (int i = 0; i < ns; ++i) {
      const int sl = i % NS;
      if (!mbar_wait(&full[sl], (i / NS) & 1, p.a.err, T0B_DEVERR_WAIT_X, abort_flag)) break;
      if (GLU && p.rot && !mbar_wait(&rot_full[sl], (i / NS) & 1, p.a.err, T0B_DEVERR_WAIT_DEQ, abort_flag)) break;
      tc_fence_after();
      const uint32_t st = base + sl * p.stage, sf = tmem + H * NT + sl * SFC;
      const uint32_t xc = FUSED ? base + p.off_x + i * NT * 128 : st + OFF_X;
      const uint32_t xs = FUSED ? base + p.off_xs + i * SC : st + OFF_XS;
#pragma unroll
      for (int a = 0; a < AT; ++a) {
        scale_cp(sf + 4 * a, scale_desc(xs + 512 * a));
#pragma unroll
        for (int h = 0; h < H; ++h) scale_cp(sf + 4 * AT * (1 + h) + 4 * a, scale_desc(st + OFF_WS + h * SC + 512 * a));
      }
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        if (4 * (s0 + i) + kk >= steps) break;
        const int a = NV ? kk : kk / 2;
#pragma unroll
        for (int h = 0; h < H; ++h)
          umma_fp4<NV>(tmem + h * NT, sw128_desc(st + h * 16384 + 32 * kk), sw128_desc(xc + 32 * kk),
                       idesc | (NV ? 0u : idesc_scale_id(kk % 2 * 2)), sf + 4 * AT * (1 + h) + 4 * a,
                       sf + 4 * a + sf_col, i > 0 || kk > 0);
      }
      umma_commit(&empty[sl]);
    }
    umma_commit(acc_full);  // also after a wait that ran out: what was issued completes before TMEM is given back
  } else if (GLU && warp == 2 && p.rot) {
    const int off = p.a.up_row & 127;
    for (int i = 0; i < ns; ++i) {
      const int sl = i % NS;
      if (!__all_sync(0xFFFFFFFFu, mbar_wait(&raw_full[sl], (i / NS) & 1, p.a.err, T0B_DEVERR_WAIT_W, abort_flag))) break;
      uint8_t *st = smem + sl * p.stage;
      move_scales<AT>(st + OFF_WS + SC, st + OFF_RAW, off);
      if (lane == 0) mbar_arrive(&rot_full[sl]);
    }
  }
  __syncwarp();
  if (CS > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");

  bool have = mbar_wait(acc_full, 0, p.a.err, T0B_DEVERR_WAIT_ACC, abort_flag) && !*abort_flag;
  have = __all_sync(0xFFFFFFFFu, have);
  tc_fence_after();
  uint8_t *slots = smem + p.off_slot;
  if (GLU && p.out_type < 0)
    split_results<NV, GLU, -1>(p, slots, tmem, rank, n0, m0, toks, have);
  else if (p.out_type == TY_F32)
    split_results<NV, GLU, TY_F32>(p, slots, tmem, rank, n0, m0, toks, have);
  else if (p.out_type == TY_F16)
    split_results<NV, GLU, TY_F16>(p, slots, tmem, rank, n0, m0, toks, have);
  else
    split_results<NV, GLU, TY_BF16>(p, slots, tmem, rank, n0, m0, toks, have);
  // after a wait that ran out: copies in flight land before the shared memory is given up
  if (!have && loader) {
    drain(full, NS, issued, p.a.err, T0B_DEVERR_WAIT_X);
    if (GLU && p.rot) drain(raw_full, NS, issued, p.a.err, T0B_DEVERR_WAIT_W);
  }
  __syncwarp();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
  }
}

// ------------------------------------------------------------- host side
// Every kernel here starts while the previous one of the stream ends and
// waits for it (griddepcontrol.wait) before its first access to memory that a
// kernel may have written.
cudaLaunchAttribute dependent_launch() {
  cudaLaunchAttribute a{};
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
  return a;
}

template <typename... P, typename... A>
cudaError_t launch(void (*k)(P...), dim3 grid, dim3 block, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0] = dependent_launch();
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, args...);
}

// Tensor maps of a matrix: codes in boxes of `rows` rows x 128 bytes, scales in
// boxes of one row group's `at` tiles.
bool code_map(CUtensorMap *tm, const Fp4Mat &q, int rows) {
  const uint64_t pitch = (uint64_t)((q.k + 31) / 32) * 16;
  return t0b_make_tmap_u8_2d(tm, q.codes, pitch, (uint64_t)q.rows, pitch, 128, rows);
}
bool scale_map(CUtensorMap *tm, const Fp4Mat &q, int kt, int at) {
  return t0b_make_tmap_f16_3d(tm, q.scales, 256, (uint64_t)kt, (uint64_t)((q.rows + 127) / 128), 512, (uint64_t)kt * 512, 256,
                              (uint32_t)at, 1, false);
}

// Pairs of the kernel that fit on the current device at once, asked once per
// kernel and device.
int max_pairs(const void *kfn, const cudaLaunchConfig_t &cfg) {
  static std::mutex mu;
  static std::map<std::pair<const void *, int>, int> cache;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lk(mu);
  int &n = cache[{kfn, dev}];
  if (n) return n;
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  cudaLaunchConfig_t c = cfg;
  c.gridDim = dim3(sms / 2 * 2);
  if (cudaOccupancyMaxActiveClusters(&n, kfn, &c) != cudaSuccess) {
    cudaGetLastError();
    n = 0;
  }
  return n;
}

// The largest power of two up to 32 that the rows' addresses are multiples of.
int rows_start(const void *p, int64_t ld, int type) {
  const uint64_t a = (uintptr_t)p | (uint64_t)ld * (type == TY_F32 ? 4 : 2) | 32;
  return (int)(a & (~a + 1));
}
bool rows_aligned(const void *p, int64_t ld, int type) { return rows_start(p, ld, type) >= 16; }

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return n;
}

// x_type < 0: x is the 4-bit matrix xm; else plain, to be quantised as xm says.
template <bool NV, bool GLU, bool FUSED>
cudaError_t launch_split(const Fp4Mat &w, const Fp4Mat &xm, const void *x, int x_type, int64_t ldx, const Fp4Args &a, int out_type,
                         const SplitPlan &q, bool early, cudaStream_t st) {
  constexpr int AT = NV ? 4 : 2, H = GLU ? 2 : 1;
  constexpr uint32_t SC = AT * 512, LIMIT = 232448;
  if (!split_plan_ok(q, GLU, FUSED, a.M, a.n, a.K)) return cudaErrorInvalidConfiguration;
  SplitArgs p{};
  p.a = a;
  p.NT = q.NT, p.CS = q.CS, p.SL = q.SL, p.rt = q.rt;
  p.out_type = out_type;
  p.rot = GLU && a.up_row % 128;
  p.early = early;
  p.x = x, p.x_type = x_type, p.ldx = ldx, p.xq = xm;
  p.xalign = FUSED ? rows_start(x, ldx, x_type) : 0;
  p.stage = split_stage<NV, GLU, FUSED>(q.NT);
  const uint32_t fixed = (FUSED ? (uint32_t)q.SL * (q.NT * 128 + SC) : 0) +
                         (q.CS > 1 ? (uint32_t)(((q.NT + q.CS - 1) / q.CS + 3) / 4 * q.CS) * H * 2048 : 0) + 512 + 1024;
  // Tensor memory is given out CTA by CTA: clusters that hold some on one SM
  // and wait for more on another could wait for each other.  So no two CTAs
  // whose columns exceed the 512 fit on an SM: up to 256 columns with over a
  // third of its shared memory, more with over two thirds.
  auto columns = [&] { return H * q.NT + p.NS * AT * 4 * (H + 1); };
  p.NS = q.SL < SPLIT_MAX_NS ? q.SL : SPLIT_MAX_NS;
  while (p.NS > 4 && columns() > 256) --p.NS;
  while (p.NS > 1 && p.NS * p.stage + fixed > LIMIT) --p.NS;
  const uint32_t used = p.NS * p.stage + fixed, least = columns() <= 256 ? 76 * 1024 : 152 * 1024;
  const uint32_t smem = used > least ? used : least;
  if (smem > LIMIT) return cudaErrorInvalidConfiguration;
  p.off_x = p.NS * p.stage;
  p.off_xs = p.off_x + (FUSED ? q.SL * q.NT * 128 : 0);
  p.off_slot = p.off_xs + (FUSED ? q.SL * SC : 0);
  p.off_bar = used - 512 - 1024;
  for (p.tmem_cols = 32; (int)p.tmem_cols < columns();) p.tmem_cols *= 2;
  if (p.tmem_cols > 512 || q.ctas > INT32_MAX) return cudaErrorInvalidConfiguration;
  CUtensorMap tx, tw, txs, tws;
  if (!code_map(&tw, w, 128) || !scale_map(&tws, w, a.kt, AT)) return cudaErrorInvalidValue;
  if (FUSED)
    tx = tw, txs = tws;  // not used
  else if (!code_map(&tx, xm, q.NT) || !scale_map(&txs, xm, a.kt, AT))
    return cudaErrorInvalidValue;
  auto kfn = fp4_gemm_split_kernel<NV, GLU, FUSED>;
  cudaError_t e = t0b_smem_limit((const void *)kfn, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = q.CS;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1] = dependent_launch();
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)q.ctas);
  cfg.blockDim = dim3(SPLIT_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kfn, tx, tw, txs, tws, p);
}

template <bool NV, bool GLU, bool ROT, int TY>
cudaError_t launch_pair(const Fp4Mat &w, const Fp4Mat &x, Fp4Args p, cudaStream_t st) {
  using C = PairCfg<NV, ROT>;
  auto kfn = fp4_gemm_pair_kernel<NV, GLU, ROT, TY>;
  static const int regs = [&] {
    cudaFuncAttributes fa{};
    return cudaFuncGetAttributes(&fa, (const void *)kfn) == cudaSuccess ? fa.numRegs : -1;
  }();
  if (regs != PAIR_REGS) return cudaErrorInvalidConfiguration;
  cudaError_t e = t0b_smem_limit((const void *)kfn, C::SMEM);
  if (e != cudaSuccess) return e;
  CUtensorMap tx, tw, txs, tws;
  if (!code_map(&tx, x, 128) || !code_map(&tw, w, 128) || !scale_map(&txs, x, p.kt, C::AT) || !scale_map(&tws, w, p.kt, C::AT))
    return cudaErrorInvalidValue;
  CUtensorMap ty = tx;  // not used without aligned rows
  if (p.vec && !t0b_make_tmap_rows64(&ty, p.y, TY == TY_F32 ? 4 : 2, (uint64_t)p.n, (uint64_t)p.M, (uint64_t)p.ld))
    return cudaErrorInvalidValue;
  p.n_tiles_n = GLU ? (p.n + 127) / 128 : (p.n + 255) / 256;
  const int64_t tiles = (int64_t)p.n_tiles_n * ((p.M + 255) / 256);
  if (tiles > INT32_MAX / 2) return cudaErrorInvalidValue;
  p.n_tiles = (int)tiles;
  cudaLaunchAttribute at[2];
  at[1] = dependent_launch();
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(PAIR_THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  const int pairs = max_pairs((const void *)kfn, cfg);
  if (pairs < 1) return cudaErrorInvalidConfiguration;
  cfg.gridDim = dim3(2 * (p.n_tiles < pairs ? p.n_tiles : pairs));
  return cudaLaunchKernelEx(&cfg, kfn, tx, tw, txs, tws, ty, p);
}

template <bool NV, int TY>
cudaError_t gemm_ty(const Fp4Mat &w, const Fp4Mat &x, const Fp4Out &out, const Fp4Args &p, cudaStream_t st) {
  if (!out.glu) return launch_pair<NV, false, false, TY < 0 ? TY_F32 : TY>(w, x, p, st);
  // gate and up rows meet in one tile; up rows that do not start at a row group's first row need their scales moved
  return p.up_row % 128 ? launch_pair<NV, true, true, TY>(w, x, p, st) : launch_pair<NV, true, false, TY>(w, x, p, st);
}

template <bool NV>
cudaError_t gemm_fmt(const Fp4Mat &w, const Fp4Mat &x, const Fp4Out &out, const Fp4Args &p, cudaStream_t st) {
  if (out.quant) return gemm_ty<NV, -1>(w, x, out, p, st);
  if (out.type == TY_F32) return gemm_ty<NV, TY_F32>(w, x, out, p, st);
  if (out.type == TY_F16) return gemm_ty<NV, TY_F16>(w, x, out, p, st);
  return gemm_ty<NV, TY_BF16>(w, x, out, p, st);
}

// Lanes along a row: those of one scale tile (8 NV, 16 MX) for rows no wider,
// 16 up to 128 values, else the warp.  65,536 x 16 f16 quantised in 4.2 us (NV)
// and 6.0 us (MX), with the whole warp along a row 11.2 and 10.5 us.
template <int TY, bool NV, bool QUANT>
cudaError_t convert(const void *x, int64_t ld, const Fp4Mat &q, cudaStream_t st) {
  using T = typename Plain<TY>::T;
  constexpr int TILE = NV ? 8 : 16;
  const int align = rows_start(x, ld, TY);
  const int lpr = q.k <= 8 * TILE ? TILE : q.k <= 128 ? 16 : 32;
  const int row_warps = (q.rows + 127) / 128 * lpr;  // of 32 / lpr rows, 32 rows a group
  const int width = QUANT ? (q.k + 8 * TILE - 1) / (8 * TILE) * (8 * TILE) : q.k;  // whole scale tiles
  dim3 grid((row_warps + QT_WARPS - 1) / QT_WARPS, (width + 8 * lpr - 1) / (8 * lpr));
  if constexpr (QUANT) {
    // pieces of a row one after the other in a warp, as long as two waves of CTAs remain
    int chunks = 1;
    while (chunks < QT_CHUNKS && grid.y > 1 && (int64_t)grid.x * grid.y > 2 * 4 * sm_count()) chunks *= 2, grid.y = (grid.y + 1) / 2;
    auto k = lpr == TILE ? fp4_quantize_kernel<TY, NV, TILE, false>
             : lpr == 16 ? fp4_quantize_kernel<TY, NV, 16, false>
             : TY != TY_F32 || align >= 8 ? fp4_quantize_kernel<TY, NV, 32, false>
                                          : fp4_quantize_kernel<TY, NV, 32, TY == TY_F32>;
    return launch(k, grid, 32 * QT_WARPS, st, (const T *)x, ld, q, align, chunks);
  } else {
    auto k = lpr == TILE ? fp4_dequantize_kernel<TY, NV, TILE>
             : lpr == 16 ? fp4_dequantize_kernel<TY, NV, 16>
                         : fp4_dequantize_kernel<TY, NV, 32>;
    // 8 values at once: 32 bytes of f32, 16 of the others
    return launch(k, grid, 32 * QT_WARPS, st, q, (T *)x, ld, align >= (TY == TY_F32 ? 32 : 16));
  }
}
template <bool NV, bool QUANT>
cudaError_t convert_ty(int type, const void *x, int64_t ld, const Fp4Mat &q, cudaStream_t st) {
  if (type == TY_F32) return convert<TY_F32, NV, QUANT>(x, ld, q, st);
  if (type == TY_F16) return convert<TY_F16, NV, QUANT>(x, ld, q, st);
  return convert<TY_BF16, NV, QUANT>(x, ld, q, st);
}

}  // namespace

cudaError_t t0b_launch_fp4_quantize(int x_type, const void *x, int64_t ldx, const Fp4Mat &q, cudaStream_t st) {
  return q.blk == 16 ? convert_ty<true, true>(x_type, x, ldx, q, st) : convert_ty<false, true>(x_type, x, ldx, q, st);
}

cudaError_t t0b_launch_fp4_dequantize(const Fp4Mat &q, int y_type, void *y, int64_t ldy, cudaStream_t st) {
  return q.blk == 16 ? convert_ty<true, false>(y_type, y, ldy, q, st) : convert_ty<false, false>(y_type, y, ldy, q, st);
}

namespace {

Fp4Args product_args(const Fp4Mat &w, const Fp4Mat &x, const Fp4Out &out, int *err) {
  Fp4Args p{};
  p.M = x.rows;
  p.n = out.glu ? w.rows / 2 : w.rows;
  p.K = w.k;
  p.kt = (w.k + 4 * w.blk - 1) / (4 * w.blk);
  p.alpha = w.ts * x.ts;
  p.bias = out.bias;
  p.y = out.y;
  p.ld = out.ld;
  p.q = out.q;
  p.up_row = out.glu ? p.n : 0;
  p.err = err;
  p.vec = !out.quant && rows_aligned(out.y, out.ld, out.type);
  return p;
}

// Values of the activations up to which a CTA of the split kernel quantises
// its slice itself (a piece of 256 takes a warp 0.26 us).  4096 x 4096, 16
// tokens (at the limit): 7.3 us in a graph and 7.9 us a call, with a quantise
// launch 6.6 and 8.7; 32 tokens: 9.7 and 9.9, with a launch 7.0 and 8.8; 1
// token: 5.4 and 6.5, with a launch 6.1 and 9.2.
constexpr int FUSED_MAX_VALUES = 16384;

template <bool FUSED>
cudaError_t split_dispatch(const Fp4Mat &w, const Fp4Mat &xm, const void *x, int x_type, int64_t ldx, const Fp4Out &out,
                           const Fp4Args &a, const SplitPlan &q, bool early, cudaStream_t st) {
  const int ot = out.quant ? -1 : out.type;
  if (w.blk == 16)
    return out.glu ? launch_split<true, true, FUSED>(w, xm, x, x_type, ldx, a, ot, q, early, st)
                   : launch_split<true, false, FUSED>(w, xm, x, x_type, ldx, a, ot, q, early, st);
  return out.glu ? launch_split<false, true, FUSED>(w, xm, x, x_type, ldx, a, ot, q, early, st)
                 : launch_split<false, false, FUSED>(w, xm, x, x_type, ldx, a, ot, q, early, st);
}

}  // namespace

cudaError_t t0b_launch_fp4_gemm(const Fp4Mat &w, const Fp4Mat &x, const Fp4Out &out, bool after_own, int *err, cudaStream_t st) {
  const Fp4Args a = product_args(w, x, out, err);
  const SplitPlan q = choose(out.glu, a.M, a.n, a.K, sm_count());
  if (q.CS) return split_dispatch<false>(w, x, nullptr, -1, 0, out, a, q, after_own, st);
  return w.blk == 16 ? gemm_fmt<true>(w, x, out, a, st) : gemm_fmt<false>(w, x, out, a, st);
}

cudaError_t t0b_launch_fp4_linear(const Fp4Mat &w, int x_type, const void *x, int64_t ldx, const Fp4Mat &xq, const Fp4Out &out,
                                  int *err, cudaStream_t st) {
  if (xq.rows <= 64) {
    const Fp4Args a = product_args(w, xq, out, err);
    const SplitPlan q = choose(out.glu, a.M, a.n, a.K, sm_count());
    // its share of the activations stays in shared memory
    if (q.CS && q.SL <= SPLIT_FUSED_MAX_SL && q.SL * 256 * a.M <= FUSED_MAX_VALUES)
      return split_dispatch<true>(w, xq, x, x_type, ldx, out, a, q, false, st);
  }
  const cudaError_t e = t0b_launch_fp4_quantize(x_type, x, ldx, xq, st);
  return e != cudaSuccess ? e : t0b_launch_fp4_gemm(w, xq, out, true, err, st);
}
