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

// ---- 16-byte pieces at any element alignment --------------------------------------------------------------------------------
template <typename T> struct Piece {
  static constexpr int N = 16 / (int)sizeof(T);
  // `valid` elements from p on (all N: one unaligned 16-byte access), the others 0
  static __device__ __forceinline__ uint4 load(const T* p, int valid) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (valid >= N) {
      __builtin_memcpy(&v, p, 16);
    } else if (valid > 0) {
      T t[N];
#pragma unroll
      for (int e = 0; e < N; ++e) t[e] = e < valid ? p[e] : T(0);
      __builtin_memcpy(&v, t, 16);
    }
    return v;
  }
  static __device__ __forceinline__ void store(T* p, const float* f, int valid) {
    const uint4 v = Chunk<T>::pack(f);
    if (valid >= N) {
      __builtin_memcpy(p, &v, 16);
    } else if (valid > 0) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (e < valid) p[e] = from_f<T>(f[e]);
    }
  }
};

template <int LPR> __device__ __forceinline__ float row_sum(float v, float* sh) {
  if constexpr (LPR == 256) return block_sum<256>(v, sh);
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// ---- rows that fit into registers: LPR lanes hold a row in NV pieces each, one sweep over memory; weight and bias stay in registers
// over the rows of a workgroup --------------------------------------------------------------------------------------------------
template <typename T, int LPR, int NV>
__global__ __launch_bounds__(256) void ln_rows_fwd(long R, int C, long xs, const T* __restrict__ x, LnParam w, LnParam b, float eps,
                                                   T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int V = Piece<T>::N, RPB = 256 / LPR;
  __shared__ float sh[4];
  const int lane = threadIdx.x % LPR;
  float wv[NV][V], bv[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = (j * LPR + lane) * V + e;
      wv[j][e] = c < C ? w.get<T>(c, 1.f) : 0.f;
      bv[j][e] = c < C ? b.get<T>(c, 0.f) : 0.f;
    }
  const float inv = 1.f / C;
  for (long r0 = (long)blockIdx.x * RPB; r0 < R; r0 += (long)gridDim.x * RPB) {
    const long r = r0 + threadIdx.x / LPR;
    const bool live = RPB == 1 || r < R;
    float f[NV][V];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * LPR + lane) * V;
      Chunk<T>::unpack(Piece<T>::load(x + r * xs + c, live ? C - c : 0), f[j]);
#pragma unroll
      for (int e = 0; e < V; ++e) s += f[j][e];
    }
    const float m = row_sum<LPR>(s, sh) / C;           // (divided: a row of equal values has its mean exactly)
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int left = C - (j * LPR + lane) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[j][e] -= m;
        if (e < left) q += f[j][e] * f[j][e];
      }
    }
    const float rs = 1.f / sqrtf(row_sum<LPR>(q, sh) * inv + eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * LPR + lane) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) f[j][e] = f[j][e] * rs * wv[j][e] + bv[j][e];
      Piece<T>::store(y + r * C + c, f[j], live ? C - c : 0);
    }
    if (mean != nullptr && lane == 0 && live) { mean[r] = m; rstd[r] = rs; }
  }
}

// dx and, kept in registers over the rows of a workgroup, its share of dw / db -> part[workgroup][2][C]
template <typename T, int LPR, int NV>
__global__ __launch_bounds__(256) void ln_rows_bwd(long R, int C, long xs, const T* __restrict__ x, const T* __restrict__ dy, LnParam w,
                                                   const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx,
                                                   float* __restrict__ part) {
  constexpr int V = Piece<T>::N, RPB = 256 / LPR;
  __shared__ float sh[4];
  const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  float wv[NV][V], aw[NV][V], ab[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = (j * LPR + lane) * V + e;
      wv[j][e] = c < C ? w.get<T>(c, 1.f) : 0.f;
      aw[j][e] = ab[j][e] = 0.f;
    }
  const float inv = 1.f / C;
  for (long r0 = (long)blockIdx.x * RPB; r0 < R; r0 += (long)gridDim.x * RPB) {
    const long r = r0 + sub;
    const bool live = RPB == 1 || r < R;
    const float m = live ? mean[r] : 0.f, rs = live ? rstd[r] : 0.f;
    float u[NV][V], g[NV][V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * LPR + lane) * V;
      Chunk<T>::unpack(Piece<T>::load(x + r * xs + c, live ? C - c : 0), u[j]);
      Chunk<T>::unpack(Piece<T>::load(dy + r * C + c, live ? C - c : 0), g[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        u[j][e] = (u[j][e] - m) * rs;
        const float d = g[j][e];            // 0 behind the row's end
        if (part != nullptr) {
          aw[j][e] += d * u[j][e];
          ab[j][e] += d;
        }
        g[j][e] = d * wv[j][e];
        s1 += g[j][e];
        s2 += g[j][e] * u[j][e];
      }
    if (dx == nullptr) continue;
    const float a1 = row_sum<LPR>(s1, sh) * inv, a2 = row_sum<LPR>(s2, sh) * inv;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * LPR + lane) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) g[j][e] = rs * (g[j][e] - a1 - u[j][e] * a2);
      Piece<T>::store(dx + r * C + c, g[j], live ? C - c : 0);
    }
  }
  if (part == nullptr) return;
  float* p = part + (long)blockIdx.x * 2 * C;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * LPR + lane) * V;
      Piece<float>::store(p + c, aw[j], C - c);
      Piece<float>::store(p + C + c, ab[j], C - c);
      if constexpr (V == 8) {
        Piece<float>::store(p + c + 4, aw[j] + 4, C - c - 4);
        Piece<float>::store(p + C + c + 4, ab[j] + 4, C - c - 4);
      }
    }
  } else {
    // the row lanes of the workgroup one after the other into one copy
    __shared__ float acc[2][LPR * NV * V];
    for (int k = 0; k < RPB; ++k) {
      if (sub == k) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const int at = (j * V + e) * LPR + lane;
            acc[0][at] = k == 0 ? aw[j][e] : acc[0][at] + aw[j][e];
            acc[1][at] = k == 0 ? ab[j][e] : acc[1][at] + ab[j][e];
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < C; c += 256) {
      const int piece = c / V, e = c - piece * V, j = piece / LPR, l = piece - j * LPR;
      p[c] = acc[0][(j * V + e) * LPR + l];
      p[C + c] = acc[1][(j * V + e) * LPR + l];
    }
  }
}

// ---- channels that fit into registers: a workgroup takes all C channels of TSV pieces of consecutive positions; a thread holds NV
// channels (CY apart) of one piece ------------------------------------------------------------------------------------------------
// sums over the channels, per position of the piece: over the lanes of the wave, then over the waves through LDS
template <int THREADS, int TSV, int V, int NS>
__device__ __forceinline__ void chan_sum(float (&s)[NS][V], float* sh) {
  constexpr int NW = THREADS / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sv = threadIdx.x % TSV;
#pragma unroll
  for (int o = TSV; o < 64; o <<= 1)
#pragma unroll
    for (int k = 0; k < NS; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) s[k][e] += __shfl_xor(s[k][e], o, 64);
  constexpr int W = NS * TSV * V;                     // values per wave
  if (lane < TSV) {
#pragma unroll
    for (int k = 0; k < NS; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) sh[wave * W + (k * TSV + sv) * V + e] = s[k][e];
  }
  __syncthreads();
  if (threadIdx.x < W) {
    float t = sh[threadIdx.x];
#pragma unroll
    for (int q = 1; q < NW; ++q) t += sh[q * W + threadIdx.x];
    sh[NW * W + threadIdx.x] = t;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < NS; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) s[k][e] = sh[NW * W + (k * TSV + sv) * V + e];
}

template <typename T, int THREADS, int TSV, int NV>
__global__ __launch_bounds__(THREADS) void ln_chan_fwd(int tiles, int per, int C, long S, const T* __restrict__ x, LnParam w, LnParam b, float eps,
                                                       T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int V = Piece<T>::N, CY = THREADS / TSV, TS = TSV * V;
  __shared__ float sh[(THREADS / 64 + 1) * TS];
  const int sv = threadIdx.x % TSV, cy = threadIdx.x / TSV;
  const float inv = 1.f / C;
  const int t = xcd_remap(blockIdx.x, tiles);
  const long n = t / per;
  const long s0 = (long)(t - n * per) * TS + sv * V;
  const int left = S - s0 >= V ? V : (S - s0 > 0 ? (int)(S - s0) : 0);
  const long base = n * C * S + s0;
  uint4 raw[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = j * CY + cy;
    raw[j] = Piece<T>::load(x + base + c * S, c < C ? left : 0);
  }
  float s[1][V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[0][e] = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float f[V];
    Chunk<T>::unpack(raw[j], f);
#pragma unroll
    for (int e = 0; e < V; ++e) s[0][e] += f[e];
  }
  chan_sum<THREADS, TSV, V, 1>(s, sh);
  float m[V];
#pragma unroll
  for (int e = 0; e < V; ++e) { m[e] = s[0][e] / C; s[0][e] = 0.f; }           // (divided: equal values have their mean exactly)
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float f[V];
    Chunk<T>::unpack(raw[j], f);
    if (j * CY + cy < C) {
#pragma unroll
      for (int e = 0; e < V; ++e) s[0][e] += (f[e] - m[e]) * (f[e] - m[e]);
    }
  }
  __syncthreads();                    // the last readers of sh are done
  chan_sum<THREADS, TSV, V, 1>(s, sh);
  float rs[V];
#pragma unroll
  for (int e = 0; e < V; ++e) rs[e] = 1.f / sqrtf(s[0][e] * inv + eps);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = j * CY + cy;
    if (c >= C) continue;
    const float wc = w.get<T>(c, 1.f), bc = b.get<T>(c, 0.f);
    float f[V];
    Chunk<T>::unpack(raw[j], f);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = (f[e] - m[e]) * rs[e] * wc + bc;
    Piece<T>::store(y + base + c * S, f, left);
  }
  if (mean != nullptr && cy == 0) {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < left) { mean[n * S + s0 + e] = m[e]; rstd[n * S + s0 + e] = rs[e]; }
  }
}

template <typename T, int THREADS, int TSV, int NV>
__global__ __launch_bounds__(THREADS) void ln_chan_bwd(int tiles, int per, int C, long S, const T* __restrict__ x, const T* __restrict__ dy, LnParam w,
                                                       const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx,
                                                       float* __restrict__ part) {
  constexpr int V = Piece<T>::N, CY = THREADS / TSV, TS = TSV * V;
  __shared__ float sh[(THREADS / 64 + 1) * 2 * TS];
  const int sv = threadIdx.x % TSV, cy = threadIdx.x / TSV;
  const float inv = 1.f / C;
  float aw[NV], ab[NV], wv[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = j * CY + cy;
    aw[j] = ab[j] = 0.f;
    wv[j] = c < C ? w.get<T>(c, 1.f) : 0.f;
  }
  // consecutive tiles (they share cache lines where rows start anywhere) to one workgroup
  const int G = gridDim.x, g = xcd_remap(blockIdx.x, G);
  const int t0 = (int)((long)tiles * g / G), t1 = (int)((long)tiles * (g + 1) / G);
  for (int t = t0; t < t1; ++t) {
    const long n = t / per;
    const long s0 = (long)(t - n * per) * TS + sv * V;
    const int left = S - s0 >= V ? V : (S - s0 > 0 ? (int)(S - s0) : 0);
    const long base = n * C * S + s0;
    uint4 rx[NV], rg[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = j * CY + cy;
      rx[j] = Piece<T>::load(x + base + c * S, c < C ? left : 0);
      rg[j] = Piece<T>::load(dy + base + c * S, c < C ? left : 0);
    }
    float m[V], rs[V], s[2][V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      m[e] = e < left ? mean[n * S + s0 + e] : 0.f;
      rs[e] = e < left ? rstd[n * S + s0 + e] : 0.f;
      s[0][e] = s[1][e] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float u[V], d[V];
      Chunk<T>::unpack(rx[j], u);
      Chunk<T>::unpack(rg[j], d);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        u[e] = (u[e] - m[e]) * rs[e];
        aw[j] += d[e] * u[e];
        ab[j] += d[e];
        s[0][e] += d[e] * wv[j];
        s[1][e] += d[e] * wv[j] * u[e];
      }
    }
    if (dx == nullptr) continue;
    chan_sum<THREADS, TSV, V, 2>(s, sh);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = j * CY + cy;
      if (c >= C) continue;
      float u[V], d[V];
      Chunk<T>::unpack(rx[j], u);
      Chunk<T>::unpack(rg[j], d);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        u[e] = (u[e] - m[e]) * rs[e];
        d[e] = rs[e] * (d[e] * wv[j] - s[0][e] * inv - u[e] * (s[1][e] * inv));
      }
      Piece<T>::store(dx + base + c * S, d, left);
    }
    __syncthreads();                  // the last readers of sh are done
  }
  if (part == nullptr) return;
  float* p = part + (long)g * 2 * C;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = j * CY + cy;
#pragma unroll
    for (int o = 1; o < TSV; o <<= 1) {
      aw[j] += __shfl_xor(aw[j], o, 64);
      ab[j] += __shfl_xor(ab[j], o, 64);
    }
    if (sv == 0 && c < C) { p[c] = aw[j]; p[C + c] = ab[j]; }
  }
}

// part[G][2][C] -> dw[C], db[C] (either may be absent): 16 columns a workgroup, 16 lanes over the groups, in ascending order each
template <typename T>
__global__ __launch_bounds__(256) void ln_dwb_fold(int G, int C, const float* __restrict__ part, void* dw, void* db, int f32) {
  __shared__ float sh[16][17];
  const int col = threadIdx.x & 15, gl = threadIdx.x >> 4;
  const int k = blockIdx.x * 16 + col;
  float s = 0.f;
  if (k < 2 * C)
    for (int g = gl; g < G; g += 16) s += part[(long)g * 2 * C + k];
  sh[gl][col] = s;
  __syncthreads();
  if (gl != 0 || k >= 2 * C) return;
#pragma unroll
  for (int q = 1; q < 16; ++q) s += sh[q][col];
  void* out = k < C ? dw : db;
  if (out == nullptr) return;
  const int c = k < C ? k : k - C;
  if (f32) reinterpret_cast<float*>(out)[c] = s;
  else reinterpret_cast<T*>(out)[c] = from_f<T>(s);
}

inline unsigned blocks_for(long n, long most) { return (unsigned)(n < 1 ? 1 : (n < most ? n : most)); }

// How a call is run.  Rows: 8 .. 64 lanes (a wave or a part of it) hold a row in at most 4 pieces each, else a workgroup holds it in at
// most 4 (fp32: 8); channels: at most 16 pieces a thread; beyond: the three-sweep kernels, which take any length.
struct LnShape { int lanes, nv, threads, tsv; int groups; long tiles; };
LnShape ln_rows_shape(int dtype, long R, int C) {
  LnShape s = {0, 0, 256, 0, 1, 0};
  const int v = dtype == PXL_F32 ? 4 : 8, pieces = (C + v - 1) / v;
  if (pieces <= 256) {
    s.lanes = 8;
    while (s.lanes < 64 && s.lanes < pieces) s.lanes *= 2;
    s.nv = pieces <= s.lanes ? 1 : (pieces <= 2 * s.lanes ? 2 : 4);
  } else if (pieces <= 1024 || (dtype == PXL_F32 && pieces <= 2048)) {
    s.lanes = 256;
    s.nv = pieces <= 512 ? 2 : (pieces <= 1024 ? 4 : 8);
  }
  if (s.lanes) {
    const long passes = (R + 256 / s.lanes - 1) / (256 / s.lanes);
    s.groups = (int)(passes < 1 ? 1 : (passes > 512 ? 512 : passes));
  } else {
    const long g = (R + 63) / 64;
    s.groups = (int)(g < 1 ? 1 : (g > 256 ? 256 : g));
  }
  return s;
}
LnShape ln_chan_shape(int dtype, long N, int C, long S) {
  LnShape s = {0, 0, 256, 8, 1, 0};
  if (C <= 256) {
    s.nv = C <= 32 ? 1 : (C <= 64 ? 2 : (C <= 128 ? 4 : 8));
  } else if (C <= 2048) {
    s.threads = 512;
    s.tsv = C <= 512 ? 8 : 4;
    s.nv = C <= 1024 ? 8 : 16;
  }
  if (s.nv) {
    const int ts = s.tsv * (dtype == PXL_F32 ? 4 : 8);
    s.lanes = s.tsv;
    s.tiles = N * ((S + ts - 1) / ts);
    const long most = s.threads == 256 ? 1024 : 512;
    if (s.tiles >= (1l << 30)) s.lanes = s.nv = 0;
    s.groups = (int)(s.tiles < 1 ? 1 : (s.tiles > most ? most : s.tiles));
  }
  if (!s.nv) {
    const long g = (N * S + 63) / 64;
    s.groups = (int)(g < 1 ? 1 : (g > 256 ? 256 : g));
  }
  return s;
}
inline LnShape ln_shape(int dtype, long R, int C, long S) { return S < 0 ? ln_rows_shape(dtype, R, C) : ln_chan_shape(dtype, S > 0 ? R / S : 0, C, S); }

#define LN_ROWS(KERNEL, BLOCKS, ...)                                                                                   \
  do {                                                                                                                 \
    const dim3 grid(BLOCKS);                                                                                           \
    const int key = s.lanes * 16 + s.nv;                                                                               \
    if (key == 8 * 16 + 1) hipLaunchKernelGGL((KERNEL<T, 8, 1>), grid, dim3(256), 0, st, __VA_ARGS__);                 \
    else if (key == 16 * 16 + 1) hipLaunchKernelGGL((KERNEL<T, 16, 1>), grid, dim3(256), 0, st, __VA_ARGS__);          \
    else if (key == 32 * 16 + 1) hipLaunchKernelGGL((KERNEL<T, 32, 1>), grid, dim3(256), 0, st, __VA_ARGS__);          \
    else if (key == 64 * 16 + 1) hipLaunchKernelGGL((KERNEL<T, 64, 1>), grid, dim3(256), 0, st, __VA_ARGS__);          \
    else if (key == 64 * 16 + 2) hipLaunchKernelGGL((KERNEL<T, 64, 2>), grid, dim3(256), 0, st, __VA_ARGS__);          \
    else if (key == 64 * 16 + 4) hipLaunchKernelGGL((KERNEL<T, 64, 4>), grid, dim3(256), 0, st, __VA_ARGS__);          \
    else if (key == 256 * 16 + 2) hipLaunchKernelGGL((KERNEL<T, 256, 2>), grid, dim3(256), 0, st, __VA_ARGS__);        \
    else if (key == 256 * 16 + 4) hipLaunchKernelGGL((KERNEL<T, 256, 4>), grid, dim3(256), 0, st, __VA_ARGS__);        \
    else if constexpr (sizeof(T) == 4) hipLaunchKernelGGL((KERNEL<T, 256, 8>), grid, dim3(256), 0, st, __VA_ARGS__);   \
  } while (0)
#define LN_CHAN(KERNEL, BLOCKS, ...)                                                                                                 \
  do {                                                                                                                               \
    const dim3 grid(BLOCKS);                                                                                                         \
    if (s.threads == 256) {                                                                                                          \
      if (s.nv == 1) hipLaunchKernelGGL((KERNEL<T, 256, 8, 1>), grid, dim3(256), 0, st, __VA_ARGS__);                                \
      else if (s.nv == 2) hipLaunchKernelGGL((KERNEL<T, 256, 8, 2>), grid, dim3(256), 0, st, __VA_ARGS__);                           \
      else if (s.nv == 4) hipLaunchKernelGGL((KERNEL<T, 256, 8, 4>), grid, dim3(256), 0, st, __VA_ARGS__);                           \
      else hipLaunchKernelGGL((KERNEL<T, 256, 8, 8>), grid, dim3(256), 0, st, __VA_ARGS__);                                          \
    } else if (s.tsv == 8) hipLaunchKernelGGL((KERNEL<T, 512, 8, 8>), grid, dim3(512), 0, st, __VA_ARGS__);                          \
    else if (s.nv == 8) hipLaunchKernelGGL((KERNEL<T, 512, 4, 8>), grid, dim3(512), 0, st, __VA_ARGS__);                             \
    else hipLaunchKernelGGL((KERNEL<T, 512, 4, 16>), grid, dim3(512), 0, st, __VA_ARGS__);                                           \
  } while (0)

template <typename T>
int ln_fwd(long R, int C, long S, long xs, const void* x, LnParam w, LnParam b, float eps, void* y, float* mean, float* rstd, hipStream_t st) {
  const LnShape s = ln_shape(Elem<T>::DTYPE, R, C, S);
  if (S < 0) {
    if (s.lanes) {
      const long passes = (R + 256 / s.lanes - 1) / (256 / s.lanes);
      LN_ROWS(ln_rows_fwd, blocks_for(passes, 2048), R, C, xs, (const T*)x, w, b, eps, (T*)y, mean, rstd);
    } else {
      hipLaunchKernelGGL(ln_rows_fwd_loop<T>, dim3(blocks_for(R, 1 << 20)), dim3(256), 0, st, R, C, xs, (const T*)x, w, b, eps, (T*)y, mean, rstd);
    }
  } else if (s.lanes) {
    const int per = (int)(s.tiles / (R / S));
    LN_CHAN(ln_chan_fwd, (unsigned)s.tiles, (int)s.tiles, per, C, S, (const T*)x, w, b, eps, (T*)y, mean, rstd);
  } else {
    hipLaunchKernelGGL(ln_chan_fwd_loop<T>, dim3(blocks_for((R + 255) / 256, 1 << 20)), dim3(256), 0, st, R, C, S, (const T*)x, w, b, eps,
                       (T*)y, mean, rstd);
  }
  PXL_LAUNCH_CHECK();
  return PXL_OK;
}

template <typename T>
int ln_bwd(long R, int C, long S, long xs, const void* x, const void* dy, LnParam w, const float* mean, const float* rstd, void* dx,
           void* dw, void* db, int pf32, float* part, hipStream_t st) {
  const LnShape s = ln_shape(Elem<T>::DTYPE, R, C, S);
  const int G = s.groups;
  const bool params = dw != nullptr || db != nullptr;
  if (R > 0 && s.lanes && (dx != nullptr || params)) {
    float* p = params ? part : nullptr;
    if (S < 0) {
      LN_ROWS(ln_rows_bwd, (unsigned)G, R, C, xs, (const T*)x, (const T*)dy, w, mean, rstd, (T*)dx, p);
    } else {
      const int per = (int)(s.tiles / (R / S));
      LN_CHAN(ln_chan_bwd, (unsigned)G, (int)s.tiles, per, C, S, (const T*)x, (const T*)dy, w, mean, rstd, (T*)dx, p);
    }
    PXL_LAUNCH_CHECK();
  } else if (R > 0) {
    if (dx != nullptr) {
      if (S < 0)
        hipLaunchKernelGGL(ln_rows_dx_loop<T>, dim3(blocks_for(R, 1 << 20)), dim3(256), 0, st, R, C, xs, (const T*)x, (const T*)dy, w, mean, rstd, (T*)dx);
      else
        hipLaunchKernelGGL(ln_chan_dx_loop<T>, dim3(blocks_for((R + 255) / 256, 1 << 20)), dim3(256), 0, st, R, C, S, (const T*)x, (const T*)dy, w,
                           mean, rstd, (T*)dx);
      PXL_LAUNCH_CHECK();
    }
    if (params) {
      if (S < 0)
        hipLaunchKernelGGL(ln_rows_dwb_loop<T>, dim3((C + 255) / 256, G), dim3(256), 0, st, R, C, xs, (const T*)x, (const T*)dy, mean, rstd, part);
      else
        hipLaunchKernelGGL(ln_chan_dwb_loop<T>, dim3(C, G), dim3(256), 0, st, R, C, S, (const T*)x, (const T*)dy, mean, rstd, part);
      PXL_LAUNCH_CHECK();
    }
  }
  if (params) {
    hipLaunchKernelGGL(ln_dwb_fold<T>, dim3((2 * C + 15) / 16), dim3(256), 0, st, R > 0 ? G : 0, C, part, dw, db, pf32);
    PXL_LAUNCH_CHECK();
  }
  return PXL_OK;
}

// (the workspace queries do not know the type)
inline int ln_rows_most(long R, int C) { const int a = ln_rows_shape(PXL_F32, R, C).groups, b = ln_rows_shape(PXL_BF16, R, C).groups; return a > b ? a : b; }
inline int ln_chan_most(long N, int C, long S) { const int a = ln_chan_shape(PXL_F32, N, C, S).groups, b = ln_chan_shape(PXL_BF16, N, C, S).groups; return a > b ? a : b; }

int ln_check(const char* what, int dtype, int pdtype, long R, int C) {
  PXL_REQUIRE(dtype == PXL_F32 || dtype == PXL_BF16, "%s: dtype %d is neither PXL_F32 nor PXL_BF16", what, dtype);
  PXL_REQUIRE(pdtype == PXL_F32 || pdtype == dtype, "%s: weight and bias are 32-bit or of the type of x", what);
  PXL_REQUIRE(R >= 0 && C >= 1 && C <= (1 << 30), "%s: bad sizes (rows %ld, features %d)", what, R, C);
  return PXL_OK;
}

}  // namespace

extern "C" size_t pxl_layer_norm_bwd_workspace(long R, int C) {
  return R < 0 || C < 1 ? 0 : (size_t)ln_rows_most(R, C) * 2 * C * sizeof(float);
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
  return N < 0 || S < 0 || C < 1 ? 0 : (size_t)ln_chan_most(N, C, S) * 2 * C * sizeof(float);
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
