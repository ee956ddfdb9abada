// t0b_fp4.cu -- C entry points of the 4-bit microscaled operators (t0b.h):
// argument checks, the engine's device, then the launchers of k_fp4.cu.
#include <cmath>
#include <cstdio>
#include <cstring>

#include "../../include/t0b.h"
#include "t0b_internal.h"

namespace {

constexpr int kMaxK = 1 << 20, kMaxRows = 1 << 30;

t0b_status fail(t0b_status s, const char *fn, const char *what) {
  char msg[256];
  snprintf(msg, sizeof(msg), "%s: %s", fn, what);
  return t0b_set_error(s, msg);
}

// Makes the engine's device current for the scope and restores the caller's.
struct DeviceScope {
  int prev = -1;
  cudaError_t status;
  explicit DeviceScope(int device) {
    status = cudaGetDevice(&prev);
    if (status == cudaSuccess && prev != device)
      status = cudaSetDevice(device);
    else
      prev = -1;
  }
  ~DeviceScope() {
    if (prev >= 0) cudaSetDevice(prev);
  }
  DeviceScope(const DeviceScope &) = delete;
  DeviceScope &operator=(const DeviceScope &) = delete;
};

bool valid_shape(int rows, int k) { return rows >= 1 && rows < kMaxRows && k >= 1 && k <= kMaxK; }
int block_of(int format) { return format == T0B_FP4_MX ? 32 : format == T0B_FP4_NV ? 16 : 0; }
size_t type_bytes(int type) { return type == T0B_F32 ? 4 : type == T0B_F16 || type == T0B_BF16 ? 2 : 0; }

// A matrix argument; `write`: the call quantises into it.
t0b_status check_mat(const char *fn, const char *name, const t0b_fp4 *m, bool write, Fp4Mat *out) {
  char what[160];
  auto bad = [&](t0b_status s, const char *why) {
    snprintf(what, sizeof(what), "%s %s", name, why);
    return fail(s, fn, what);
  };
  if (!m) return bad(T0B_ERR_INVALID, "is NULL");
  if (!block_of(m->format)) return bad(T0B_ERR_UNSUPPORTED, "has no known format (T0B_FP4_MX or T0B_FP4_NV)");
  if (!valid_shape(m->rows, m->k)) return bad(T0B_ERR_INVALID, "has an empty or too large shape");
  if (!m->codes || !m->scales) return bad(T0B_ERR_INVALID, "has no memory (NULL codes or scales)");
  if (((uintptr_t)m->codes | (uintptr_t)m->scales) % 16)
    return bad(T0B_ERR_INVALID, "codes and scales must be 16-byte aligned");
  const float ts = m->tensor_scale;
  if (m->format == T0B_FP4_MX) {
    if (ts != 1.0f) return bad(T0B_ERR_INVALID, "of format T0B_FP4_MX has tensor_scale 1");
  } else {
    int ex;
    if (!std::isnormal(ts) || ts < 0) return bad(T0B_ERR_INVALID, "needs a positive normal tensor_scale");
    if (write && (std::frexp(ts, &ex) != 0.5f || ex - 1 < -64 || ex - 1 > 64))
      return bad(T0B_ERR_INVALID, "needs a power of two in [2^-64, 2^64] as tensor_scale to be quantised into");
  }
  const double r6 = 1.0 / (6.0 * (double)ts);
  float hi = (float)r6;
  if ((double)hi > r6) hi = std::nextafter(hi, 0.0f);
  *out = Fp4Mat{m->codes, m->scales, m->rows, m->k, block_of(m->format), ts, hi, (float)(r6 - (double)hi)};
  return T0B_OK;
}

// A plain tensor argument [rows, cols] with rows ld elements apart.
t0b_status check_plain(const char *fn, const char *name, int type, const void *p, int64_t ld, int64_t rows, int64_t cols) {
  char what[160];
  const size_t b = type_bytes(type);
  const char *why = nullptr;
  t0b_status s = T0B_ERR_INVALID;
  if (!b)
    why = "must be T0B_F32, T0B_F16 or T0B_BF16", s = T0B_ERR_UNSUPPORTED;
  else if (!p)
    why = "is NULL";
  else if ((uintptr_t)p % b)
    why = "is not aligned to its elements";
  else if (ld < cols || ld > (int64_t(1) << 40) / rows)
    why = "has a row stride below its width or out of range";
  if (!why) return T0B_OK;
  snprintf(what, sizeof(what), "%s %s", name, why);
  return fail(s, fn, what);
}

t0b_status check_bias(const char *fn, const float *b) {
  if ((uintptr_t)b % 4) return fail(T0B_ERR_INVALID, fn, "bias is not aligned to its elements");
  return T0B_OK;
}

t0b_status check_product(const char *fn, const Fp4Mat &w, const Fp4Mat &x) {
  if (w.blk != x.blk) return fail(T0B_ERR_INVALID, fn, "weights and activations must have one format");
  if (w.k != x.k) return fail(T0B_ERR_INVALID, fn, "weights and activations must have one k");
  if (!std::isnormal(w.ts * x.ts)) return fail(T0B_ERR_INVALID, fn, "the tensor scales' product is out of range");
  return T0B_OK;
}

t0b_status cuda_status(const char *fn, cudaError_t e) {
  if (e == cudaSuccess) return T0B_OK;
  cudaGetLastError();  // reported here: not left for the caller's next check
  return fail(T0B_ERR_CUDA, fn, cudaGetErrorString(e));
}

// A C entry's body: no C++ exception leaves it (the host-side caches and the
// error message allocate).
template <class F>
t0b_status guarded(F body) {
  try {
    return body();
  } catch (...) {
    return T0B_ERR_OOM;
  }
}

// Clears the error word unless another error has been recorded since `seen`
// was read: an error is cleared only by a call that reports it.
__global__ void clear_error_kernel(int *err, int seen) { atomicCAS(err, seen, 0); }

#define TRY(expr)                        \
  do {                                   \
    const t0b_status s_ = (expr);        \
    if (s_ != T0B_OK) return s_;         \
  } while (0)

}  // namespace

extern "C" size_t t0b_fp4_code_bytes(int rows, int k) {
  if (!valid_shape(rows, k)) return 0;
  return (size_t)rows * ((k + 31) / 32) * 16;
}

extern "C" size_t t0b_fp4_scale_bytes(int format, int rows, int k) {
  const int blk = block_of(format);
  if (!blk || !valid_shape(rows, k)) return 0;
  return (size_t)((rows + 127) / 128) * ((k + 4 * blk - 1) / (4 * blk)) * 512;
}

extern "C" t0b_status t0b_fp4_quantize(t0b_engine *e, int x_type, const void *x_dev, int64_t ldx, const t0b_fp4 *out,
                                       void *stream) {
  return guarded([&]() -> t0b_status {
    const char *fn = "t0b_fp4_quantize";
    if (!e) return fail(T0B_ERR_INVALID, fn, "engine is NULL");
    Fp4Mat q;
    TRY(check_mat(fn, "out", out, true, &q));
    TRY(check_plain(fn, "x", x_type, x_dev, ldx, q.rows, q.k));
    DeviceScope dev(t0b_engine_device(e));
    TRY(cuda_status(fn, dev.status));
    return cuda_status(fn, t0b_launch_fp4_quantize(x_type, x_dev, ldx, q, (cudaStream_t)stream));
  });
}

extern "C" t0b_status t0b_fp4_dequantize(t0b_engine *e, const t0b_fp4 *in, int y_type, void *y_dev, int64_t ldy,
                                         void *stream) {
  return guarded([&]() -> t0b_status {
    const char *fn = "t0b_fp4_dequantize";
    if (!e) return fail(T0B_ERR_INVALID, fn, "engine is NULL");
    Fp4Mat q;
    TRY(check_mat(fn, "in", in, false, &q));
    TRY(check_plain(fn, "y", y_type, y_dev, ldy, q.rows, q.k));
    DeviceScope dev(t0b_engine_device(e));
    TRY(cuda_status(fn, dev.status));
    return cuda_status(fn, t0b_launch_fp4_dequantize(q, y_type, y_dev, ldy, (cudaStream_t)stream));
  });
}

extern "C" t0b_status t0b_fp4_gemm(t0b_engine *e, const t0b_fp4 *w, const t0b_fp4 *x, const float *bias_dev, int y_type,
                                   void *y_dev, int64_t ldy, void *stream) {
  return guarded([&]() -> t0b_status {
    const char *fn = "t0b_fp4_gemm";
    if (!e) return fail(T0B_ERR_INVALID, fn, "engine is NULL");
    Fp4Mat wm, xm;
    TRY(check_mat(fn, "w", w, false, &wm));
    TRY(check_mat(fn, "x", x, false, &xm));
    TRY(check_product(fn, wm, xm));
    TRY(check_bias(fn, bias_dev));
    TRY(check_plain(fn, "y", y_type, y_dev, ldy, xm.rows, wm.rows));
    DeviceScope dev(t0b_engine_device(e));
    TRY(cuda_status(fn, dev.status));
    const Fp4Out out{y_type, y_dev, ldy, bias_dev, false, false, {}};
    return cuda_status(fn, t0b_launch_fp4_gemm(wm, xm, out, false, t0b_engine_fp4_err(e), (cudaStream_t)stream));
  });
}

extern "C" t0b_status t0b_fp4_glu(t0b_engine *e, const t0b_fp4 *w, const t0b_fp4 *x, const float *bias_dev, int z_type,
                                  void *z_dev, int64_t ldz, const t0b_fp4 *zq, void *stream) {
  return guarded([&]() -> t0b_status {
    const char *fn = "t0b_fp4_glu";
    if (!e) return fail(T0B_ERR_INVALID, fn, "engine is NULL");
    if ((z_dev != nullptr) == (zq != nullptr)) return fail(T0B_ERR_INVALID, fn, "needs either z_dev or zq");
    Fp4Mat wm, xm;
    TRY(check_mat(fn, "w", w, false, &wm));
    TRY(check_mat(fn, "x", x, false, &xm));
    TRY(check_product(fn, wm, xm));
    TRY(check_bias(fn, bias_dev));
    if (wm.rows % 2) return fail(T0B_ERR_INVALID, fn, "w needs gate and up rows in equal number");
    const int F = wm.rows / 2;
    Fp4Out out{z_type, z_dev, ldz, bias_dev, true, zq != nullptr, {}};
    if (zq) {
      TRY(check_mat(fn, "zq", zq, true, &out.q));
      if (out.q.blk != wm.blk || out.q.rows != xm.rows || out.q.k != F)
        return fail(T0B_ERR_INVALID, fn, "zq must have w's format and shape [x->rows, w->rows / 2]");
    } else {
      TRY(check_plain(fn, "z", z_type, z_dev, ldz, xm.rows, F));
    }
    DeviceScope dev(t0b_engine_device(e));
    TRY(cuda_status(fn, dev.status));
    return cuda_status(fn, t0b_launch_fp4_gemm(wm, xm, out, false, t0b_engine_fp4_err(e), (cudaStream_t)stream));
  });
}

extern "C" t0b_status t0b_fp4_linear(t0b_engine *e, const t0b_fp4 *w, int x_type, const void *x_dev, int64_t ldx,
                                     const t0b_fp4 *xq, const float *bias_dev, int y_type, void *y_dev, int64_t ldy,
                                     void *stream) {
  return guarded([&]() -> t0b_status {
    const char *fn = "t0b_fp4_linear";
    if (!e) return fail(T0B_ERR_INVALID, fn, "engine is NULL");
    Fp4Mat wm, xm;
    TRY(check_mat(fn, "w", w, false, &wm));
    TRY(check_mat(fn, "xq", xq, true, &xm));
    TRY(check_product(fn, wm, xm));
    TRY(check_bias(fn, bias_dev));
    TRY(check_plain(fn, "x", x_type, x_dev, ldx, xm.rows, xm.k));
    TRY(check_plain(fn, "y", y_type, y_dev, ldy, xm.rows, wm.rows));
    DeviceScope dev(t0b_engine_device(e));
    TRY(cuda_status(fn, dev.status));
    const Fp4Out out{y_type, y_dev, ldy, bias_dev, false, false, {}};
    return cuda_status(fn, t0b_launch_fp4_linear(wm, x_type, x_dev, ldx, xm, out, t0b_engine_fp4_err(e), (cudaStream_t)stream));
  });
}

extern "C" t0b_status t0b_fp4_mlp(t0b_engine *e, const t0b_fp4 *w0, const t0b_fp4 *w2, int x_type, const void *x_dev,
                                  int64_t ldx, const t0b_fp4 *xq, const t0b_fp4 *zq, const float *b0_dev,
                                  const float *b2_dev, int y_type, void *y_dev, int64_t ldy, void *stream) {
  return guarded([&]() -> t0b_status {
    const char *fn = "t0b_fp4_mlp";
    if (!e) return fail(T0B_ERR_INVALID, fn, "engine is NULL");
    Fp4Mat w0m, w2m, xm, zm;
    TRY(check_mat(fn, "w0", w0, false, &w0m));
    TRY(check_mat(fn, "w2", w2, false, &w2m));
    TRY(check_mat(fn, "xq", xq, true, &xm));
    TRY(check_mat(fn, "zq", zq, true, &zm));
    TRY(check_product(fn, w0m, xm));
    TRY(check_product(fn, w2m, zm));
    TRY(check_bias(fn, b0_dev));
    TRY(check_bias(fn, b2_dev));
    if (w0m.rows % 2) return fail(T0B_ERR_INVALID, fn, "w0 needs gate and up rows in equal number");
    if (zm.rows != xm.rows || zm.k != w0m.rows / 2 || zm.blk != w0m.blk)
      return fail(T0B_ERR_INVALID, fn, "zq must have w0's format and shape [xq->rows, w0->rows / 2]");
    TRY(check_plain(fn, "x", x_type, x_dev, ldx, xm.rows, xm.k));
    TRY(check_plain(fn, "y", y_type, y_dev, ldy, xm.rows, w2m.rows));
    DeviceScope dev(t0b_engine_device(e));
    TRY(cuda_status(fn, dev.status));
    const cudaStream_t st = (cudaStream_t)stream;
    int *err = t0b_engine_fp4_err(e);
    const Fp4Out hid{0, nullptr, 0, b0_dev, true, true, zm};
    TRY(cuda_status(fn, t0b_launch_fp4_linear(w0m, x_type, x_dev, ldx, xm, hid, err, st)));
    const Fp4Out out{y_type, y_dev, ldy, b2_dev, false, false, {}};
    return cuda_status(fn, t0b_launch_fp4_gemm(w2m, zm, out, true, err, st));
  });
}

extern "C" t0b_status t0b_fp4_sync(t0b_engine *e, void *stream) {
  return guarded([&]() -> t0b_status {
    const char *fn = "t0b_fp4_sync";
    if (!e) return fail(T0B_ERR_INVALID, fn, "engine is NULL");
    DeviceScope dev(t0b_engine_device(e));
    TRY(cuda_status(fn, dev.status));
    const cudaStream_t st = (cudaStream_t)stream;
    // refused before anything is queued: a copy or wait would end the capture
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    TRY(cuda_status(fn, cudaStreamIsCapturing(st, &capture)));
    if (capture != cudaStreamCaptureStatusNone) return fail(T0B_ERR_INVALID, fn, "the stream is being captured");
    int *err = t0b_engine_fp4_err(e), herr = 0;
    TRY(cuda_status(fn, cudaMemcpyAsync(&herr, err, sizeof(int), cudaMemcpyDeviceToHost, st)));
    TRY(cuda_status(fn, cudaStreamSynchronize(st)));
    if (!herr) return T0B_OK;
    clear_error_kernel<<<1, 1, 0, st>>>(err, herr);
    TRY(cuda_status(fn, cudaGetLastError()));
    TRY(cuda_status(fn, cudaStreamSynchronize(st)));
    char what[80];
    snprintf(what, sizeof(what), "a kernel reported device error code %d", herr);
    return fail(T0B_ERR_DEVICE, fn, what);
  });
}
