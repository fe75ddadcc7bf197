// Layer normalisation, forward and backward, over the last axis of [R][C] rows and over the channels of an [N][C][S] map.
//
//   mean = sum_c x / C,  var = sum_c (x - mean)^2 / C,  rstd = 1 / sqrt(var + eps),  u = (x - mean) rstd,  y = u w + b
//   g = dy w,  dx = rstd (g - sum_c g / C - u sum_c (g u) / C),  dw = sum_rows dy u,  db = sum_rows dy
//
// Statistics, sums and the parameter gradients are held in 32 bits whatever the type of x; the variance is taken around the
// mean in a second sweep (sum x^2 - C mean^2 cancels where the mean is large against the deviation).  No atomics: every sum has
// one order, so two calls on the same inputs agree bit for bit.  y and dx are rounded once.
#include "common.h"

namespace {

struct LnParam {          // weight / bias (or their gradients): 32 bits or the type of x
  const void* p;
  int f32;
  template <typename T> __device__ __forceinline__ float get(int c, float none) const {
    if (p == nullptr) return none;
    return f32 ? reinterpret_cast<const float*>(p)[c] : to_f(reinterpret_cast<const T*>(p)[c]);
  }
};

// sum of one value per thread over the whole block, the same order on every thread
template <int THREADS> __device__ __forceinline__ float block_sum(float v, float* sh) {
  v = wave_sum(v);
  constexpr int NW = THREADS / 64;
  if (NW == 1) return v;
  __syncthreads();                      // the last reader of sh is done
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = sh[0];
#pragma unroll
  for (int k = 1; k < NW; ++k) s += sh[k];
  return s;
}

// ---- rows of any length: one workgroup a row, three sweeps (the second and third come out of the caches) -------------------
template <typename T>
__global__ __launch_bounds__(256) void ln_rows_fwd_loop(long R, int C, long xs, const T* __restrict__ x, LnParam w, LnParam b,
                                                        float eps, T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float sh[4];
  for (long r = blockIdx.x; r < R; r += gridDim.x) {
    const T* xr = x + r * xs;
    float s = 0.f;
    for (int c = threadIdx.x; c < C; c += 256) s += to_f(xr[c]);
    const float m = block_sum<256>(s, sh) / C;
    float q = 0.f;
    for (int c = threadIdx.x; c < C; c += 256) { const float d = to_f(xr[c]) - m; q += d * d; }
    const float rs = 1.f / sqrtf(block_sum<256>(q, sh) / C + eps);
    T* yr = y + r * C;
    for (int c = threadIdx.x; c < C; c += 256)
      yr[c] = from_f<T>((to_f(xr[c]) - m) * rs * w.get<T>(c, 1.f) + b.get<T>(c, 0.f));
    if (mean != nullptr && threadIdx.x == 0) { mean[r] = m; rstd[r] = rs; }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_rows_dx_loop(long R, int C, long xs, const T* __restrict__ x, const T* __restrict__ dy, LnParam w,
                                                       const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx) {
  __shared__ float sh[4];
  for (long r = blockIdx.x; r < R; r += gridDim.x) {
    const T* xr = x + r * xs;
    const T* gr = dy + r * C;
    const float m = mean[r], rs = rstd[r];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < C; c += 256) {
      const float g = to_f(gr[c]) * w.get<T>(c, 1.f), u = (to_f(xr[c]) - m) * rs;
      s1 += g; s2 += g * u;
    }
    const float a1 = block_sum<256>(s1, sh) / C, a2 = block_sum<256>(s2, sh) / C;
    T* dr = dx + r * C;
    for (int c = threadIdx.x; c < C; c += 256) {
      const float g = to_f(gr[c]) * w.get<T>(c, 1.f), u = (to_f(xr[c]) - m) * rs;
      dr[c] = from_f<T>(rs * (g - a1 - u * a2));
    }
  }
}

// dw / db partial sums: workgroup (column block, row group) -> part[group][2][C]
template <typename T>
__global__ __launch_bounds__(256) void ln_rows_dwb_loop(long R, int C, long xs, const T* __restrict__ x, const T* __restrict__ dy,
                                                        const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ part) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float sw = 0.f, sb = 0.f;
  for (long r = blockIdx.y; r < R; r += gridDim.y) {
    const float g = to_f(dy[r * C + c]);
    sw += g * ((to_f(x[r * xs + c]) - mean[r]) * rstd[r]);
    sb += g;
  }
  float* p = part + (long)blockIdx.y * 2 * C;
  p[c] = sw;
  p[C + c] = sb;
}

// ---- channels of a map, any number: one thread a position ------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void ln_chan_fwd_loop(long P, int C, long S, const T* __restrict__ x, LnParam w, LnParam b, float eps,
                                                        T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  for (long p = blockIdx.x * 256L + threadIdx.x; p < P; p += gridDim.x * 256L) {
    const long n = p / S, o = n * C * S + (p - n * S);
    float s = 0.f;
    for (int c = 0; c < C; ++c) s += to_f(x[o + c * S]);
    const float m = s / C;
    float q = 0.f;
    for (int c = 0; c < C; ++c) { const float d = to_f(x[o + c * S]) - m; q += d * d; }
    const float rs = 1.f / sqrtf(q / C + eps);
    for (int c = 0; c < C; ++c) y[o + c * S] = from_f<T>((to_f(x[o + c * S]) - m) * rs * w.get<T>(c, 1.f) + b.get<T>(c, 0.f));
    if (mean != nullptr) { mean[p] = m; rstd[p] = rs; }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_chan_dx_loop(long P, int C, long S, const T* __restrict__ x, const T* __restrict__ dy, LnParam w,
                                                       const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx) {
  for (long p = blockIdx.x * 256L + threadIdx.x; p < P; p += gridDim.x * 256L) {
    const long n = p / S, o = n * C * S + (p - n * S);
    const float m = mean[p], rs = rstd[p];
    float s1 = 0.f, s2 = 0.f;
    for (int c = 0; c < C; ++c) {
      const float g = to_f(dy[o + c * S]) * w.get<T>(c, 1.f);
      s1 += g; s2 += g * ((to_f(x[o + c * S]) - m) * rs);
    }
    const float a1 = s1 / C, a2 = s2 / C;
    for (int c = 0; c < C; ++c) {
      const float g = to_f(dy[o + c * S]) * w.get<T>(c, 1.f), u = (to_f(x[o + c * S]) - m) * rs;
      dx[o + c * S] = from_f<T>(rs * (g - a1 - u * a2));
    }
  }
}

// workgroup (channel, position group) -> part[group][2][C]
template <typename T>
__global__ __launch_bounds__(256) void ln_chan_dwb_loop(long P, int C, long S, const T* __restrict__ x, const T* __restrict__ dy,
                                                        const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ part) {
  __shared__ float sh[4];
  const int c = blockIdx.x;
  float sw = 0.f, sb = 0.f;
  for (long p = blockIdx.y * 256L + threadIdx.x; p < P; p += gridDim.y * 256L) {
    const long n = p / S, o = (n * C + c) * S + (p - n * S);
    const float g = to_f(dy[o]);
    sw += g * ((to_f(x[o]) - mean[p]) * rstd[p]);
    sb += g;
  }
  sw = block_sum<256>(sw, sh);
  sb = block_sum<256>(sb, sh);
  if (threadIdx.x == 0) {
    part[(long)blockIdx.y * 2 * C + c] = sw;
    part[(long)blockIdx.y * 2 * C + C + c] = sb;
  }
}

// part[G][2][C] -> dw[C], db[C] (either may be absent), groups in ascending order
template <typename T>
__global__ __launch_bounds__(256) void ln_dwb_fold(int G, int C, const float* __restrict__ part, void* dw, void* db, int f32) {
  const int k = blockIdx.x * 256 + threadIdx.x;
  if (k >= 2 * C) return;
  void* out = k < C ? dw : db;
  if (out == nullptr) return;
  float s = 0.f;
  for (int g = 0; g < G; ++g) s += part[(long)g * 2 * C + k];
  const int c = k < C ? k : k - C;
  if (f32) reinterpret_cast<float*>(out)[c] = s;
  else reinterpret_cast<T*>(out)[c] = from_f<T>(s);
}

inline unsigned blocks_for(long n, long most) { return (unsigned)(n < 1 ? 1 : (n < most ? n : most)); }

// groups of the dw / db partial sums
inline int ln_groups(long rows, int C) {
  (void)C;
  const long g = (rows + 63) / 64;
  return (int)(g < 1 ? 1 : (g > 256 ? 256 : g));
}

template <typename T>
int ln_fwd(long R, int C, long S, long xs, const void* x, LnParam w, LnParam b, float eps, void* y, float* mean, float* rstd, hipStream_t st) {
  if (S < 0)
    hipLaunchKernelGGL(ln_rows_fwd_loop<T>, dim3(blocks_for(R, 1 << 20)), dim3(256), 0, st, R, C, xs, (const T*)x, w, b, eps, (T*)y, mean, rstd);
  else
    hipLaunchKernelGGL(ln_chan_fwd_loop<T>, dim3(blocks_for((R + 255) / 256, 1 << 20)), dim3(256), 0, st, R, C, S, (const T*)x, w, b, eps,
                       (T*)y, mean, rstd);
  PXL_LAUNCH_CHECK();
  return PXL_OK;
}

template <typename T>
int ln_bwd(long R, int C, long S, long xs, const void* x, const void* dy, LnParam w, const float* mean, const float* rstd, void* dx,
           void* dw, void* db, int pf32, float* part, hipStream_t st) {
  const int G = ln_groups(R, C);
  if (R > 0 && dx != nullptr) {
    if (S < 0)
      hipLaunchKernelGGL(ln_rows_dx_loop<T>, dim3(blocks_for(R, 1 << 20)), dim3(256), 0, st, R, C, xs, (const T*)x, (const T*)dy, w, mean, rstd, (T*)dx);
    else
      hipLaunchKernelGGL(ln_chan_dx_loop<T>, dim3(blocks_for((R + 255) / 256, 1 << 20)), dim3(256), 0, st, R, C, S, (const T*)x, (const T*)dy, w,
                         mean, rstd, (T*)dx);
    PXL_LAUNCH_CHECK();
  }
  if (dw != nullptr || db != nullptr) {
    if (S < 0)
      hipLaunchKernelGGL(ln_rows_dwb_loop<T>, dim3((C + 255) / 256, G), dim3(256), 0, st, R, C, xs, (const T*)x, (const T*)dy, mean, rstd, part);
    else
      hipLaunchKernelGGL(ln_chan_dwb_loop<T>, dim3(C, G), dim3(256), 0, st, R, C, S, (const T*)x, (const T*)dy, mean, rstd, part);
    PXL_LAUNCH_CHECK();
    hipLaunchKernelGGL(ln_dwb_fold<T>, dim3((2 * C + 255) / 256), dim3(256), 0, st, G, C, part, dw, db, pf32);
    PXL_LAUNCH_CHECK();
  }
  return PXL_OK;
}

int ln_check(const char* what, int dtype, int pdtype, long R, int C) {
  PXL_REQUIRE(dtype == PXL_F32 || dtype == PXL_BF16, "%s: dtype %d is neither PXL_F32 nor PXL_BF16", what, dtype);
  PXL_REQUIRE(pdtype == PXL_F32 || pdtype == dtype, "%s: weight and bias are 32-bit or of the type of x", what);
  PXL_REQUIRE(R >= 0 && C >= 1 && C <= (1 << 30), "%s: bad sizes (rows %ld, features %d)", what, R, C);
  return PXL_OK;
}

}  // namespace

extern "C" size_t pxl_layer_norm_bwd_workspace(long R, int C) {
  return R < 0 || C < 1 ? 0 : (size_t)ln_groups(R, C) * 2 * C * sizeof(float);
}

extern "C" int pxl_layer_norm_fwd(int dtype, int pdtype, long R, int C, long x_stride, const void* x, const void* w, const void* b, float eps,
                                  void* y, float* mean, float* rstd, void* stream) {
  const int rc = ln_check("layer_norm_fwd", dtype, pdtype, R, C);
  if (rc != PXL_OK) return rc;
  if (R == 0) return PXL_OK;
  PXL_REQUIRE(x && y && x_stride >= C && (mean == nullptr) == (rstd == nullptr) && eps >= 0.f, "layer_norm_fwd: bad argument");
  const LnParam pw{w, pdtype == PXL_F32}, pb{b, pdtype == PXL_F32};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return dtype == PXL_F32 ? ln_fwd<float>(R, C, -1, x_stride, x, pw, pb, eps, y, mean, rstd, st)
                          : ln_fwd<bf16_t>(R, C, -1, x_stride, x, pw, pb, eps, y, mean, rstd, st);
}

extern "C" int pxl_layer_norm_bwd(int dtype, int pdtype, long R, int C, long x_stride, const void* x, const void* dy, const void* w,
                                  const float* mean, const float* rstd, void* dx, void* dw, void* db, void* ws, size_t ws_bytes, void* stream) {
  const int rc = ln_check("layer_norm_bwd", dtype, pdtype, R, C);
  if (rc != PXL_OK) return rc;
  PXL_REQUIRE(R == 0 || (x && dy && mean && rstd && x_stride >= C), "layer_norm_bwd: bad argument");
  if ((dw || db) && (ws == nullptr || ws_bytes < pxl_layer_norm_bwd_workspace(R, C)))
    return pxl_set_error(PXL_ERR_WORKSPACE, "layer_norm_bwd: workspace of %zu bytes, %zu needed", ws_bytes, pxl_layer_norm_bwd_workspace(R, C));
  const LnParam pw{w, pdtype == PXL_F32};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  float* part = reinterpret_cast<float*>(ws);
  return dtype == PXL_F32 ? ln_bwd<float>(R, C, -1, x_stride, x, dy, pw, mean, rstd, dx, dw, db, pdtype == PXL_F32, part, st)
                          : ln_bwd<bf16_t>(R, C, -1, x_stride, x, dy, pw, mean, rstd, dx, dw, db, pdtype == PXL_F32, part, st);
}

extern "C" int pxl_layer_norm_nchw_fwd(int dtype, int pdtype, long N, int C, long S, const void* x, const void* w, const void* b, float eps,
                                       void* y, float* mean, float* rstd, void* stream) {
  PXL_REQUIRE(N >= 0 && S >= 0, "layer_norm_nchw_fwd: bad sizes (maps %ld, positions %ld)", N, S);
  const int rc = ln_check("layer_norm_nchw_fwd", dtype, pdtype, N * S, C);
  if (rc != PXL_OK) return rc;
  if (N * S == 0) return PXL_OK;
  PXL_REQUIRE(x && y && (mean == nullptr) == (rstd == nullptr) && eps >= 0.f, "layer_norm_nchw_fwd: bad argument");
  const LnParam pw{w, pdtype == PXL_F32}, pb{b, pdtype == PXL_F32};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return dtype == PXL_F32 ? ln_fwd<float>(N * S, C, S, 0, x, pw, pb, eps, y, mean, rstd, st)
                          : ln_fwd<bf16_t>(N * S, C, S, 0, x, pw, pb, eps, y, mean, rstd, st);
}

extern "C" size_t pxl_layer_norm_nchw_bwd_workspace(long N, int C, long S) {
  return N < 0 || S < 0 || C < 1 ? 0 : (size_t)ln_groups(N * S, C) * 2 * C * sizeof(float);
}

extern "C" int pxl_layer_norm_nchw_bwd(int dtype, int pdtype, long N, int C, long S, const void* x, const void* dy, const void* w,
                                       const float* mean, const float* rstd, void* dx, void* dw, void* db, void* ws, size_t ws_bytes,
                                       void* stream) {
  PXL_REQUIRE(N >= 0 && S >= 0, "layer_norm_nchw_bwd: bad sizes (maps %ld, positions %ld)", N, S);
  const int rc = ln_check("layer_norm_nchw_bwd", dtype, pdtype, N * S, C);
  if (rc != PXL_OK) return rc;
  PXL_REQUIRE(N * S == 0 || (x && dy && mean && rstd), "layer_norm_nchw_bwd: bad argument");
  if ((dw || db) && (ws == nullptr || ws_bytes < pxl_layer_norm_nchw_bwd_workspace(N, C, S)))
    return pxl_set_error(PXL_ERR_WORKSPACE, "layer_norm_nchw_bwd: workspace of %zu bytes, %zu needed", ws_bytes,
                         pxl_layer_norm_nchw_bwd_workspace(N, C, S));
  const LnParam pw{w, pdtype == PXL_F32};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  float* part = reinterpret_cast<float*>(ws);
  return dtype == PXL_F32 ? ln_bwd<float>(N * S, C, S, 0, x, dy, pw, mean, rstd, dx, dw, db, pdtype == PXL_F32, part, st)
                          : ln_bwd<bf16_t>(N * S, C, S, 0, x, dy, pw, mean, rstd, dx, dw, db, pdtype == PXL_F32, part, st);
}
