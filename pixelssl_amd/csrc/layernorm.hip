// Layer normalisation, forward and backward, over the last axis of [R][C] rows and over the channels of an [N][C][S] map.
//
//   mean = sum_c x / C,  var = sum_c (x - mean)^2 / C,  rstd = 1 / sqrt(var + eps),  u = (x - mean) rstd,  y = u w + b
//   g = dy w,  dx = rstd (g - sum_c g / C - u sum_c (g u) / C),  dw = sum_rows dy u,  db = sum_rows dy
//
// Statistics, sums and the parameter gradients are held in 32 bits or more whatever the type of x; the variance is taken around the
// mean in a second sweep (sum x^2 - C mean^2 cancels where the mean is large against the deviation).  No atomics: every sum has
// one order, so two calls on the same inputs agree bit for bit.  y and dx are rounded once.
//
// Bound by memory: forward moves x and y once, backward x, dy and dx once (rows and channels live in registers between the sweeps), at
// 5.1 TB/s of a large copy.  Measured, us (rate): 33800 x 2048 bf16 forward 51 (5.4 TB/s), backward 87 (4.8); 8 x 256 x 129 x 129 fp32 64 (4.3)
// and 100 (4.1); 8 x 2048 x 65 x 65 bf16 87 (3.2) and 180 (2.3) -- rows of 8450 bytes, so pieces lie across cache lines, and one workgroup a CU
// that loads, sums and stores in turn.  Partial dw / db: under 5 us to write and to add.  Small calls are bound by the launches (5 us a
// kernel) and, forward + backward, by the host: 65 us, of which an engine pass with a trivial node takes 44 - 47.
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

// Sums of any number of terms (up to 2^24 features, 2^31 rows and more a call) are taken in 64 bits: one after the other in 32 bits, 10^6 terms of
// one sign are off by up to 1 %.  out: over the threads of one place (threadIdx.x % TP) of a workgroup of 256, on each of them
template <int TP> __device__ __forceinline__ double long_sum(double v, double (*sh)[TP < 64 ? TP : 64]) {
#pragma unroll
  for (int o = TP < 64 ? TP : 64; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
  constexpr int W = TP < 64 ? TP : 64;
  const int at = threadIdx.x & (W - 1);
  __syncthreads();                      // the last reader of sh is done
  if ((threadIdx.x & 63) < W) sh[threadIdx.x >> 6][at] = v;
  __syncthreads();
  return (sh[0][at] + sh[1][at]) + (sh[2][at] + sh[3][at]);
}

// ---- rows of any length: one workgroup a row, three sweeps (the second and third come out of the caches) -------------------
template <typename T>
__global__ __launch_bounds__(256) void ln_rows_fwd_loop(long R, int C, long xs, const T* __restrict__ x, LnParam w, LnParam b,
                                                        float eps, T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ double sh[4][1];
  for (long r = blockIdx.x; r < R; r += gridDim.x) {
    const T* xr = x + r * xs;
    double s = 0.0;
    for (int c = threadIdx.x; c < C; c += 256) s += to_f(xr[c]);
    const float m = (float)(long_sum<1>(s, sh) / C);
    double q = 0.0;
    for (int c = threadIdx.x; c < C; c += 256) { const float d = to_f(xr[c]) - m; q += d * d; }
    const float rs = 1.f / sqrtf((float)(long_sum<1>(q, sh) / C) + eps);
    T* yr = y + r * C;
    for (int c = threadIdx.x; c < C; c += 256)
      yr[c] = from_f<T>((to_f(xr[c]) - m) * rs * w.get<T>(c, 1.f) + b.get<T>(c, 0.f));
    if (mean != nullptr && threadIdx.x == 0) { mean[r] = m; rstd[r] = rs; }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_rows_dx_loop(long R, int C, long xs, const T* __restrict__ x, const T* __restrict__ dy, LnParam w,
                                                       const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx) {
  __shared__ double sh[4][1];
  for (long r = blockIdx.x; r < R; r += gridDim.x) {
    const T* xr = x + r * xs;
    const T* gr = dy + r * C;
    const float m = mean[r], rs = rstd[r];
    double s1 = 0.0, s2 = 0.0;
    for (int c = threadIdx.x; c < C; c += 256) {
      const float g = to_f(gr[c]) * w.get<T>(c, 1.f), u = (to_f(xr[c]) - m) * rs;
      s1 += g; s2 += g * u;
    }
    const float a1 = (float)(long_sum<1>(s1, sh) / C), a2 = (float)(long_sum<1>(s2, sh) / C);
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
  double sw = 0.0, sb = 0.0;
  for (long r = blockIdx.y; r < R; r += gridDim.y) {
    const float g = to_f(dy[r * C + c]);
    sw += g * ((to_f(x[r * xs + c]) - mean[r]) * rstd[r]);
    sb += g;
  }
  float* p = part + (long)blockIdx.y * 2 * C;
  p[c] = (float)sw;
  p[C + c] = (float)sb;
}

// ---- channels of a map, any number: TP positions a workgroup, 256 / TP threads over the channels of each; xn: elements from one map of x to
// the next (rows shorter than a piece come here too, as maps of one position) -----------------------------------------------------------
template <typename T, int TP>
__global__ __launch_bounds__(256) void ln_chan_fwd_loop(long P, int C, long S, long xn, const T* __restrict__ x, LnParam w, LnParam b, float eps,
                                                        T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ double sh[4][TP < 64 ? TP : 64];
  constexpr int CL = 256 / TP;
  const int cl = threadIdx.x / TP;
  auto sum = [&](double v) { return CL == 1 ? v : long_sum<TP>(v, sh); };
  for (long p0 = (long)blockIdx.x * TP; p0 < P; p0 += (long)gridDim.x * TP) {
    const long at = p0 + threadIdx.x % TP, p = at < P ? at : P - 1;         // past the end: the last position again, stored by none
    const long n = p / S, i = p - n * S, o = n * C * S + i, ox = n * xn + i;
    double s = 0.0;
    for (int c = cl; c < C; c += CL) s += to_f(x[ox + c * S]);
    const float m = (float)(sum(s) / C);
    double q = 0.0;
    for (int c = cl; c < C; c += CL) { const float d = to_f(x[ox + c * S]) - m; q += d * d; }
    const float rs = 1.f / sqrtf((float)(sum(q) / C) + eps);
    if (at >= P) continue;
    for (int c = cl; c < C; c += CL) y[o + c * S] = from_f<T>((to_f(x[ox + c * S]) - m) * rs * w.get<T>(c, 1.f) + b.get<T>(c, 0.f));
    if (mean != nullptr && cl == 0) { mean[p] = m; rstd[p] = rs; }
  }
}

template <typename T, int TP>
__global__ __launch_bounds__(256) void ln_chan_dx_loop(long P, int C, long S, long xn, const T* __restrict__ x, const T* __restrict__ dy, LnParam w,
                                                       const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx) {
  __shared__ double sh[4][TP < 64 ? TP : 64];
  constexpr int CL = 256 / TP;
  const int cl = threadIdx.x / TP;
  auto sum = [&](double v) { return CL == 1 ? v : long_sum<TP>(v, sh); };
  for (long p0 = (long)blockIdx.x * TP; p0 < P; p0 += (long)gridDim.x * TP) {
    const long at = p0 + threadIdx.x % TP, p = at < P ? at : P - 1;
    const long n = p / S, i = p - n * S, o = n * C * S + i, ox = n * xn + i;
    const float m = mean[p], rs = rstd[p];
    double s1 = 0.0, s2 = 0.0;
    for (int c = cl; c < C; c += CL) {
      const float g = to_f(dy[o + c * S]) * w.get<T>(c, 1.f);
      s1 += g; s2 += g * ((to_f(x[ox + c * S]) - m) * rs);
    }
    const float a1 = (float)(sum(s1) / C), a2 = (float)(sum(s2) / C);
    if (at >= P) continue;
    for (int c = cl; c < C; c += CL) {
      const float g = to_f(dy[o + c * S]) * w.get<T>(c, 1.f), u = (to_f(x[ox + c * S]) - m) * rs;
      dx[o + c * S] = from_f<T>(rs * (g - a1 - u * a2));
    }
  }
}

// workgroup (channel from c0 on, position group) -> part[group][2][C]
template <typename T>
__global__ __launch_bounds__(256) void ln_chan_dwb_loop(int c0, long P, int C, long S, long xn, const T* __restrict__ x, const T* __restrict__ dy,
                                                        const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ part) {
  __shared__ double sh[4][1];
  const int c = c0 + blockIdx.x;
  double sw = 0.0, sb = 0.0;
  for (long p = blockIdx.y * 256L + threadIdx.x; p < P; p += gridDim.y * 256L) {
    const long n = p / S, i = p - n * S, o = (n * C + c) * S + i, ox = n * xn + c * S + i;
    const float g = to_f(dy[o]);
    sw += g * ((to_f(x[ox]) - mean[p]) * rstd[p]);
    sb += g;
  }
  sw = long_sum<1>(sw, sh);
  sb = long_sum<1>(sb, sh);
  if (threadIdx.x == 0) {
    part[(long)blockIdx.y * 2 * C + c] = (float)sw;
    part[(long)blockIdx.y * 2 * C + C + c] = (float)sb;
  }
}

// ---- 16-byte pieces at any element alignment.  A piece that would pass the end of its run is moved back to end there: it holds `dup`
// elements that the piece before it holds too, which count once in sums and are written twice with the same bits ----------------
template <typename T> struct Piece {
  static constexpr int N = 16 / (int)sizeof(T);
  static __device__ __forceinline__ uint4 load(const T* p) {
    uint4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
  }
  static __device__ __forceinline__ void store(T* p, const float* f) {
    const uint4 v = Chunk<T>::pack(f);
    __builtin_memcpy(p, &v, 16);
  }
};

// a piece's worth of parameters from c on, in 16-byte loads (one by one, 64 loads a lane of 2048 features: a row 8.0 us, so 3.8)
template <typename T> __device__ __forceinline__ void param_piece(const LnParam& w, int c, float none, float* f) {
  constexpr int N = Piece<T>::N;
  if (w.p == nullptr) {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = none;
  } else if (sizeof(T) == 4 || w.f32) {
    __builtin_memcpy(f, reinterpret_cast<const float*>(w.p) + c, 4 * N);
  } else {
    Chunk<T>::unpack(Piece<T>::load(reinterpret_cast<const T*>(w.p) + c), f);
  }
}

// makes the compiler take a piece as new: what is unpacked from it after this is unpacked again, not kept in registers from before
__device__ __forceinline__ void renew(uint4& v) { asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w)); }

template <int LPR> __device__ __forceinline__ float row_sum(float v, float* sh) {
  if constexpr (LPR == 256) return block_sum<256>(v, sh);
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// ---- rows that fit into registers: LPR lanes hold a row in NV pieces each, one sweep over memory; weight and bias stay in registers
// over the rows of a workgroup.  TAIL: C is no multiple of a piece --------------------------------------------------------------
// (Three sweeps over memory by a workgroup a row: 503 us forward + backward of 33800 x 2048 bf16, this 142.)
// start of piece j of a lane, moved back where it would pass C; dup: elements it shares with the piece before (N or more: all)
template <int N, int LPR, bool TAIL> __device__ __forceinline__ int piece_at(int j, int lane, int C, int& dup) {
  const int c = (j * LPR + lane) * N;
  if (!TAIL) { dup = c < C ? 0 : N; return c < C ? c : 0; }
  const int at = c + N <= C ? c : C - N;
  dup = c - at;
  return at;
}

template <typename T, int LPR, int NV, bool TAIL>
__global__ __launch_bounds__(256) void ln_rows_fwd(long R, int C, long xs, const T* __restrict__ x, LnParam w, LnParam b, float eps,
                                                   T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int V = Piece<T>::N, RPB = 256 / LPR;
  __shared__ float sh[4];
  const int lane = threadIdx.x % LPR;
  float wv[NV][V], bv[NV][V];
  int at[NV], dup[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) at[j] = piece_at<V, LPR, TAIL>(j, lane, C, dup[j]);
  const float inv = 1.f / C;
  const long step = (long)gridDim.x * RPB;
  uint4 raw[NV];
  auto fetch = [&](long r) {
    const T* xr = x + (r < R ? r : R - 1) * xs;            // past the end: the last row again
#pragma unroll
    for (int j = 0; j < NV; ++j) raw[j] = Piece<T>::load(xr + at[j]);
  };
  fetch((long)blockIdx.x * RPB + threadIdx.x / LPR);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    param_piece<T>(w, at[j], 1.f, wv[j]);
    param_piece<T>(b, at[j], 0.f, bv[j]);
  }
  for (long r0 = (long)blockIdx.x * RPB; r0 < R; r0 += step) {
    const long r = r0 + threadIdx.x / LPR;
    float f[NV][V];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Chunk<T>::unpack(raw[j], f[j]);
#pragma unroll
      for (int e = 0; e < V; ++e) s += e >= dup[j] ? f[j][e] : 0.f;
    }
    fetch(r + step);                                       // the next row, while this one is reduced
    const float m = row_sum<LPR>(s, sh) / C;               // (divided: a row of equal values has its mean exactly)
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[j][e] -= m;
        q += e >= dup[j] ? f[j][e] * f[j][e] : 0.f;
      }
    const float rs = 1.f / sqrtf(row_sum<LPR>(q, sh) * inv + eps);
    if (RPB > 1 && r >= R) continue;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < V; ++e) f[j][e] = f[j][e] * rs * wv[j][e] + bv[j][e];
      if (dup[j] < V) Piece<T>::store(y + r * C + at[j], f[j]);
    }
    if (mean != nullptr && lane == 0) { mean[r] = m; rstd[r] = rs; }
  }
}

// dx and, kept in registers over the rows of a workgroup, its share of dw / db -> part[workgroup][2][C]
template <typename T, int LPR, int NV, bool TAIL>
__global__ __launch_bounds__(256) void ln_rows_bwd(long R, int C, long xs, const T* __restrict__ x, const T* __restrict__ dy, LnParam w,
                                                   const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx,
                                                   float* __restrict__ part) {
  constexpr int V = Piece<T>::N, RPB = 256 / LPR;
  __shared__ float sh[4];
  const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  float wv[NV][V], aw[NV][V], ab[NV][V];
  int at[NV], dup[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    at[j] = piece_at<V, LPR, TAIL>(j, lane, C, dup[j]);
#pragma unroll
    for (int e = 0; e < V; ++e) aw[j][e] = ab[j][e] = 0.f;
    param_piece<T>(w, at[j], 1.f, wv[j]);
  }
  const float inv = 1.f / C;
  for (long r0 = (long)blockIdx.x * RPB; r0 < R; r0 += (long)gridDim.x * RPB) {
    const bool live = RPB == 1 || r0 + sub < R;
    const long r = live ? r0 + sub : R - 1;                // past the end: the last row again, counted nowhere
    const float m = mean[r], rs = rstd[r];
    float u[NV][V], g[NV][V];
    float s1 = 0.f, s2 = 0.f;
    uint4 ru[NV], rg[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      ru[j] = Piece<T>::load(x + r * xs + at[j]);
      rg[j] = Piece<T>::load(dy + r * C + at[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Chunk<T>::unpack(ru[j], u[j]);
      Chunk<T>::unpack(rg[j], g[j]);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        u[j][e] = (u[j][e] - m) * rs;
        const float d = g[j][e];
        if (live) {
          aw[j][e] += d * u[j][e];
          ab[j][e] += d;
        }
        g[j][e] = d * wv[j][e];
        s1 += e >= dup[j] ? g[j][e] : 0.f;
        s2 += e >= dup[j] ? g[j][e] * u[j][e] : 0.f;
        asm volatile("" : "+v"(aw[j][e]), "+v"(ab[j][e]));
      }
    }
    if (dx == nullptr) continue;
    const float a1 = row_sum<LPR>(s1, sh) * inv, a2 = row_sum<LPR>(s2, sh) * inv;
    if (!live) continue;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < V; ++e) g[j][e] = rs * (g[j][e] - a1 - u[j][e] * a2);
      if (dup[j] < V) Piece<T>::store(dx + r * C + at[j], g[j]);
    }
  }
  if (part == nullptr) return;
  // a shared column has the same sums in both of its pieces: either is written
  float* p = part + (long)blockIdx.x * 2 * C;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (dup[j] < V) {
#pragma unroll
        for (int e = 0; e < V; e += 4) {
          Piece<float>::store(p + at[j] + e, &aw[j][e]);
          Piece<float>::store(p + C + at[j] + e, &ab[j][e]);
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
            const int i = (j * V + e) * LPR + lane;
            acc[0][i] = k == 0 ? aw[j][e] : acc[0][i] + aw[j][e];
            acc[1][i] = k == 0 ? ab[j][e] : acc[1][i] + ab[j][e];
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < C; c += 256) {
      const int piece = c / V, j = piece / LPR, l = piece - j * LPR;
      int shared;
      const int e = c - piece_at<V, LPR, TAIL>(j, l, C, shared);
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

// addresses: a base per j that the whole workgroup shares, and one 32-bit byte offset per lane (CY S <= 2^8 2^22 elements of 4 bytes)
template <typename T> __device__ __forceinline__ const T* lane_at(const T* base, unsigned off) {
  return reinterpret_cast<const T*>(reinterpret_cast<const unsigned char*>(base) + off);
}
template <typename T> __device__ __forceinline__ T* lane_at(T* base, unsigned off) {
  return reinterpret_cast<T*>(reinterpret_cast<unsigned char*>(base) + off);
}

template <typename T, int THREADS, int TSV, int NV>
__global__ __launch_bounds__(THREADS) void ln_chan_fwd(int first, int per, int C, int S, const T* __restrict__ x, LnParam w, LnParam b, float eps,
                                                       T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int V = Piece<T>::N, CY = THREADS / TSV, TS = TSV * V;
  __shared__ float sh[(THREADS / 64 + 1) * TS];
  const int sv = threadIdx.x % TSV, cy = threadIdx.x / TSV;
  const float inv = 1.f / C;
  const int t = first + xcd_remap(blockIdx.x, gridDim.x);
  const int n = t / per, s0 = (t - n * per) * TS + sv * V;
  const int at = s0 + V <= S ? s0 : S - V, dup = s0 - at;
  const long base = (long)n * C * S, step = (long)CY * S;
  uint4 raw[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int b0 = j * CY < C ? j * CY : C - 1, c = b0 + cy < C ? cy : C - 1 - b0;      // past the channels: the last one again
    raw[j] = Piece<T>::load(lane_at(x + base + (long)b0 * S, (unsigned)(c * S + at) * (unsigned)sizeof(T)));
  }
  // parameters on their way while the channels are summed (16 channels a thread: read where they are used, no registers for them)
  constexpr bool KEEP = NV <= 8;
  float wk[KEEP ? NV : 1], bk[KEEP ? NV : 1];
  if (KEEP) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = j * CY + cy < C ? j * CY + cy : C - 1;
      wk[KEEP ? j : 0] = w.get<T>(c, 1.f);
      bk[KEEP ? j : 0] = b.get<T>(c, 0.f);
    }
  }
  float s[1][V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[0][e] = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float f[V];
    Chunk<T>::unpack(raw[j], f);
    if (j * CY + cy < C) {
#pragma unroll
      for (int e = 0; e < V; ++e) s[0][e] += f[e];
    }
  }
  chan_sum<THREADS, TSV, V, 1>(s, sh);
  float m[V];
#pragma unroll
  for (int e = 0; e < V; ++e) { m[e] = s[0][e] / C; s[0][e] = 0.f; }           // (divided: equal values have their mean exactly)
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float f[V];
    renew(raw[j]);
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
  if (dup >= V) return;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = j * CY + cy;
    if (c >= C) continue;
    const float wc = KEEP ? wk[KEEP ? j : 0] : w.get<T>(c, 1.f), bc = KEEP ? bk[KEEP ? j : 0] : b.get<T>(c, 0.f);
    float f[V];
    renew(raw[j]);
    Chunk<T>::unpack(raw[j], f);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = (f[e] - m[e]) * rs[e] * wc + bc;
    Piece<T>::store(lane_at(y + base + j * step, (unsigned)(cy * S + at) * (unsigned)sizeof(T)), f);
  }
  if (mean != nullptr && cy == 0) {
#pragma unroll
    for (int e = 0; e < V; ++e) { mean[(long)n * S + at + e] = m[e]; rstd[(long)n * S + at + e] = rs[e]; }
  }
}

// FULL: every thread has NV channels.  Else what channels past the end would add to the sums is replaced by 0 (times a weight of 0, an infinite
// dy of the last channel made every channel's sums NaN): forward + backward of 8 x 2000 x 65 x 65 bf16 272 us, 268 without; replaced where dy is
// loaded or unpacked, in all threads, it cost registers (8 x 2048 x 65 x 65 289 - 300 us, so 270).
template <typename T, int THREADS, int TSV, int NV, bool FULL>
__global__ __launch_bounds__(THREADS) void ln_chan_bwd(int tiles, int per, int C, int S, const T* __restrict__ x, const T* __restrict__ dy, LnParam w,
                                                       const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx,
                                                       float* __restrict__ part) {
  constexpr int V = Piece<T>::N, CY = THREADS / TSV, TS = TSV * V;
  __shared__ float sh[(THREADS / 64 + 1) * 2 * TS];
  const int sv = threadIdx.x % TSV, cy = threadIdx.x / TSV;
  const float inv = 1.f / C;
  const long step = (long)CY * S;
  constexpr bool KEEP = NV <= 8;                           // weights in registers, or read again where they are used
  float aw[NV], ab[NV], wk[KEEP ? NV : 1];
  auto weight = [&](int j) { return j * CY + cy < C ? w.get<T>(j * CY + cy, 1.f) : 0.f; };     // (0: a channel past the end adds nothing)
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    aw[j] = ab[j] = 0.f;
    if (KEEP) wk[j] = weight(j);
  }
  // Rows start anywhere, so neighbouring tiles share a cache line per row and channel: an XCD (one L2) takes a run of tiles, and its workgroups
  // neighbouring ones at a time (each a run of its own: 3 times the bytes from beyond the L2, 306 us in place of 149 for 8 x 2048 x 65 x 65 bf16)
  const int G = gridDim.x, g = xcd_remap(blockIdx.x, G);
  const int xcd = blockIdx.x & 7, mine = (G - xcd + 7) >> 3, lead = g - (blockIdx.x >> 3);      // workgroups of this XCD, the first of them
  const int t0 = (int)((long)tiles * lead / G) + (blockIdx.x >> 3), t1 = (int)((long)tiles * (lead + mine) / G);
  for (int t = t0; t < t1; t += mine) {
    const int n = t / per, s0 = (t - n * per) * TS + sv * V;
    const int at = s0 + V <= S ? s0 : S - V, dup = s0 - at;
    const long base = (long)n * C * S;
    uint4 rx[NV], rg[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int b0 = j * CY < C ? j * CY : C - 1, c = b0 + cy < C ? cy : C - 1 - b0;    // past the channels: the last one again
      const unsigned off = (unsigned)(c * S + at) * (unsigned)sizeof(T);
      rx[j] = Piece<T>::load(lane_at(x + base + (long)b0 * S, off));
      rg[j] = Piece<T>::load(lane_at(dy + base + (long)b0 * S, off));
    }
    float m[V], rs[V], s[2][V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      m[e] = mean[(long)n * S + at + e];
      rs[e] = rstd[(long)n * S + at + e];
      s[0][e] = s[1][e] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float u[V], d[V];
      const float wj = KEEP ? wk[KEEP ? j : 0] : weight(j);
      Chunk<T>::unpack(rx[j], u);
      Chunk<T>::unpack(rg[j], d);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        u[e] = (u[e] - m[e]) * rs[e];
        const float own = e >= dup ? d[e] : 0.f;          // a position that the piece before holds too counts there
        aw[j] += e >= dup ? d[e] * u[e] : 0.f;
        ab[j] += own;
        const float gj = FULL || j * CY + cy < C ? d[e] * wj : 0.f;
        s[0][e] += gj;
        s[1][e] += gj * u[e];
      }
      // every sum is taken here: left to the compiler, some sink to the loop's end and keep all pieces unpacked until then (196 registers, 144 so)
      asm volatile("" : "+v"(aw[j]), "+v"(ab[j]));
#pragma unroll
      for (int e = 0; e < V; ++e) asm volatile("" : "+v"(s[0][e]), "+v"(s[1][e]));
    }
    if (dx == nullptr) continue;
    chan_sum<THREADS, TSV, V, 2>(s, sh);
    if (dup < V) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = j * CY + cy;
        if (c >= C) continue;
        float u[V], d[V];
        const float wj = KEEP ? wk[KEEP ? j : 0] : weight(j);
        renew(rx[j]);
        renew(rg[j]);
        Chunk<T>::unpack(rx[j], u);
        Chunk<T>::unpack(rg[j], d);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          u[e] = (u[e] - m[e]) * rs[e];
          d[e] = rs[e] * (d[e] * wj - s[0][e] * inv - u[e] * (s[1][e] * inv));
        }
        Piece<T>::store(lane_at(dx + base + j * step, (unsigned)(cy * S + at) * (unsigned)sizeof(T)), d);
      }
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

// part[G][2][C] -> dw[C], db[C] (either may be absent): 16 columns a workgroup, 64 lanes over the groups, in ascending order each
template <typename T>
__global__ __launch_bounds__(1024) void ln_dwb_fold(int G, int C, const float* __restrict__ part, void* dw, void* db, int f32) {
  __shared__ double sh[64][17];
  const int col = threadIdx.x & 15, gl = threadIdx.x >> 4;
  const int k = blockIdx.x * 16 + col;
  double s = 0.0;                             // (up to 8192 shares)
  if (k < 2 * C) {
    int g = gl;
    for (; g + 192 < G; g += 256) {           // four loads in flight
      float t[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) t[q] = part[(long)(g + 64 * q) * 2 * C + k];
#pragma unroll
      for (int q = 0; q < 4; ++q) s += t[q];
    }
    for (; g < G; g += 64) s += part[(long)g * 2 * C + k];
  }
  sh[gl][col] = s;
  __syncthreads();
  if (gl != 0 || k >= 2 * C) return;
  s = 0.0;
#pragma unroll 16
  for (int q = 0; q < 64; ++q) s += sh[q][col];
  void* out = k < C ? dw : db;
  if (out == nullptr) return;
  const int c = k < C ? k : k - C;
  if (f32) reinterpret_cast<float*>(out)[c] = (float)s;
  else reinterpret_cast<T*>(out)[c] = from_f<T>((float)s);
}

constexpr long LN_MOST = 1l << 22;        // workgroups a launch at most: of up to 1024 threads, and a grid has fewer than 2^32
inline unsigned blocks_for(long n, long most) { return (unsigned)(n < 1 ? 1 : (n < most ? n : most)); }

// How a call is run.  Rows: 8 .. 64 lanes (a wave or a part of it) hold a row in at most 4 pieces each, else a workgroup holds it in at
// most 4 (fp32: 8); channels: at most 16 pieces a thread; beyond: the three-sweep kernels, which take any length.
struct LnShape { int lanes, nv, threads, tsv; int groups; long tiles; };
// Workgroups of a backward pass over `n` turns: as many as run at once, the turns evenly over them; several times as many where a thread would add
// up the parameters' gradients over more than `longest` turns, one after the other in 32 bits (2^20 x 2048 fp32 of a constant gradient: 2048 turns, db
// 1.6e-5 off, with 256 2e-6; the plain sum 2e-6) -- up to 8192, whose shares take 128 KB a 2 features.
inline int ln_groups(long n, long resident, long longest) {
  long most = resident * ((n + resident * longest - 1) / (resident * longest));
  if (most < resident) most = resident;
  if (most > 8192) most = 8192 / resident * resident;
  const long each = (n + most - 1) / most;
  return (int)(n < 1 ? 1 : (n + each - 1) / each);
}
LnShape ln_rows_shape(int dtype, long R, int C) {
  LnShape s = {0, 0, 256, 0, 1, 0};
  const int v = dtype == PXL_F32 ? 4 : 8, pieces = (C + v - 1) / v;
  if (C < v) {
    s.lanes = 0;                          // shorter than a piece
  } else if (pieces <= 256) {
    s.lanes = 8;
    while (s.lanes < 64 && s.lanes < pieces) s.lanes *= 2;
    s.nv = pieces <= s.lanes ? 1 : (pieces <= 2 * s.lanes ? 2 : 4);
  } else if (pieces <= 1024 || (dtype == PXL_F32 && pieces <= 2048)) {
    s.lanes = 256;
    s.nv = pieces <= 512 ? 2 : (pieces <= 1024 ? 4 : 8);
  }
  if (s.lanes) {
    const long passes = (R + 256 / s.lanes - 1) / (256 / s.lanes);
    s.groups = ln_groups(passes, 512, 256);
  } else {
    const long g = (R + 63) / 64;
    s.groups = (int)(g < 1 ? 1 : (g > 256 ? 256 : g));
  }
  return s;
}
LnShape ln_chan_shape(int dtype, long N, int C, long S) {
  LnShape s = {0, 0, 256, 8, 1, 0};
  const int v = dtype == PXL_F32 ? 4 : 8;
  if (S < v || S >= (1l << 22)) {
    s.nv = 0;                             // shorter than a piece; a lane's offsets past 32 bits
  } else if (C <= 256) {
    s.nv = C <= 32 ? 1 : (C <= 64 ? 2 : (C <= 128 ? 4 : 8));
  } else if (C <= 2048) {
    s.tsv = 4;
    s.threads = C <= 512 ? 256 : 512;
    s.nv = C <= 1024 ? 8 : 16;
  }
  if (s.nv) {
    const int ts = s.tsv * v;
    s.lanes = s.tsv;
    s.tiles = N * ((S + ts - 1) / ts);
    if (s.tiles >= (1l << 30)) s.lanes = s.nv = 0;
    // backward: as many workgroups as are resident at once (of 1024 threads 1 a CU, of 512 2, of 256 5), the tiles evenly over them: fewer partial
    // sums too (8 x 64 x 257 x 257 fp32 108 us + 5 to add 1175 of them, a workgroup for every 4 tiles 106 + 20)
    const int threads = s.nv >= 8 ? 2 * s.threads : s.threads;
    const long most = threads == 1024 ? 256 : (threads == 512 ? 512 : 1280);
    s.groups = ln_groups(s.tiles, most, 128 / v);
  }
  if (!s.nv) {
    const long g = (N * S + 63) / 64;
    s.groups = (int)(g < 1 ? 1 : (g > 256 ? 256 : g));
  }
  return s;
}
inline LnShape ln_shape(int dtype, long R, int C, long S) { return S < 0 ? ln_rows_shape(dtype, R, C) : ln_chan_shape(dtype, S > 0 ? R / S : 0, C, S); }

#define LN_ROWS_TAIL(KERNEL, L, N, ...)                                                                                \
  do {                                                                                                                 \
    if (C % (16 / (int)sizeof(T))) hipLaunchKernelGGL((KERNEL<T, L, N, true>), grid, dim3(256), 0, st, __VA_ARGS__);   \
    else hipLaunchKernelGGL((KERNEL<T, L, N, false>), grid, dim3(256), 0, st, __VA_ARGS__);                            \
  } while (0)
#define LN_ROWS(KERNEL, BLOCKS, ...)                                                                                   \
  do {                                                                                                                 \
    const dim3 grid(BLOCKS);                                                                                           \
    const int key = s.lanes * 16 + s.nv;                                                                               \
    if (key == 8 * 16 + 1) LN_ROWS_TAIL(KERNEL, 8, 1, __VA_ARGS__);                                                    \
    else if (key == 16 * 16 + 1) LN_ROWS_TAIL(KERNEL, 16, 1, __VA_ARGS__);                                             \
    else if (key == 32 * 16 + 1) LN_ROWS_TAIL(KERNEL, 32, 1, __VA_ARGS__);                                             \
    else if (key == 64 * 16 + 1) LN_ROWS_TAIL(KERNEL, 64, 1, __VA_ARGS__);                                             \
    else if (key == 64 * 16 + 2) LN_ROWS_TAIL(KERNEL, 64, 2, __VA_ARGS__);                                             \
    else if (key == 64 * 16 + 4) LN_ROWS_TAIL(KERNEL, 64, 4, __VA_ARGS__);                                             \
    else if (key == 256 * 16 + 2) LN_ROWS_TAIL(KERNEL, 256, 2, __VA_ARGS__);                                           \
    else if (key == 256 * 16 + 4) LN_ROWS_TAIL(KERNEL, 256, 4, __VA_ARGS__);                                           \
    else if constexpr (sizeof(T) == 4) LN_ROWS_TAIL(KERNEL, 256, 8, __VA_ARGS__);                                      \
  } while (0)
// Backward (H = 2), which holds x and dy: 8 channels a thread and more go to twice the threads with half of them each (8 x 256 x 129 x 129 fp32
// 100 us, with 8 a thread 109; 8 x 2048 x 65 x 65 bf16 180 us, with 16 a thread 194; forward the other way round, 87 with 16 and 104 with 8)
#define LN_CHAN_FWD(TH, TSV, NV, ...) hipLaunchKernelGGL((ln_chan_fwd<T, TH, TSV, NV>), grid, dim3(TH), 0, st, __VA_ARGS__)
#define LN_CHAN_BWD(TH, TSV, NV, ...)                                                                                                \
  do {                                                                                                                               \
    if (C == TH / TSV * NV) hipLaunchKernelGGL((ln_chan_bwd<T, TH, TSV, NV, true>), grid, dim3(TH), 0, st, __VA_ARGS__);             \
    else hipLaunchKernelGGL((ln_chan_bwd<T, TH, TSV, NV, false>), grid, dim3(TH), 0, st, __VA_ARGS__);                               \
  } while (0)
#define LN_CHAN(LAUNCH, H, BLOCKS, ...)                                                                                              \
  do {                                                                                                                               \
    const dim3 grid(BLOCKS);                                                                                                         \
    if (s.tsv == 8) {                                                                                                                \
      if (s.nv == 1) LAUNCH(256, 8, 1, __VA_ARGS__);                                                                                 \
      else if (s.nv == 2) LAUNCH(256, 8, 2, __VA_ARGS__);                                                                            \
      else if (s.nv == 4) LAUNCH(256, 8, 4, __VA_ARGS__);                                                                            \
      else LAUNCH((256 * H), 8, (8 / H), __VA_ARGS__);                                                                               \
    } else if (s.threads == 256) LAUNCH((256 * H), 4, (8 / H), __VA_ARGS__);                                                         \
    else if (s.nv == 8) LAUNCH((512 * H), 4, (8 / H), __VA_ARGS__);                                                                  \
    else LAUNCH((512 * H), 4, (16 / H), __VA_ARGS__);                                                                                \
  } while (0)

// Channels beyond the register kernels: up to 16 of them one thread a position, more 8 positions a workgroup (forward + backward of 2^18 maps of
// 2 positions, us, one thread a position / so: bf16 17 channels 179 / 219, 24 329 / 232, 64 1432 / 432; fp32 368 / 259, 551 / 298, 1720 / 625)
#define LN_CHAN_LOOP(KERNEL, ...)                                                                                                   \
  do {                                                                                                                              \
    if (C <= 16) hipLaunchKernelGGL((KERNEL<T, 256>), dim3(blocks_for((R + 255) / 256, 1 << 20)), dim3(256), 0, st, __VA_ARGS__);   \
    else hipLaunchKernelGGL((KERNEL<T, 8>), dim3(blocks_for((R + 7) / 8, 1 << 20)), dim3(256), 0, st, __VA_ARGS__);                 \
  } while (0)

template <typename T>
int ln_fwd(long R, int C, long S, long xs, const void* x, LnParam w, LnParam b, float eps, void* y, float* mean, float* rstd, hipStream_t st) {
  const LnShape s = ln_shape(Elem<T>::DTYPE, R, C, S);
  if (S < 0) {
    if (s.lanes) {
      // as many workgroups as are resident at once (registers: 3 a CU with 4 pieces a lane, else 6 and more), the rows evenly over them
      const long passes = (R + 256 / s.lanes - 1) / (256 / s.lanes), most = s.nv >= 4 ? 768 : 1536, each = (passes + most - 1) / most;
      LN_ROWS(ln_rows_fwd, blocks_for((passes + each - 1) / each, most), R, C, xs, (const T*)x, w, b, eps, (T*)y, mean, rstd);
    } else if (C < Piece<T>::N) {
      LN_CHAN_LOOP(ln_chan_fwd_loop, R, C, 1, xs, (const T*)x, w, b, eps, (T*)y, mean, rstd);
    } else {
      hipLaunchKernelGGL(ln_rows_fwd_loop<T>, dim3(blocks_for(R, 1 << 20)), dim3(256), 0, st, R, C, xs, (const T*)x, w, b, eps, (T*)y, mean, rstd);
    }
  } else if (s.lanes) {
    const int per = (int)(s.tiles / (R / S));
    for (long t = 0; t < s.tiles; t += LN_MOST)
      LN_CHAN(LN_CHAN_FWD, 1, (unsigned)(s.tiles - t < LN_MOST ? s.tiles - t : LN_MOST), (int)t, per, C, (int)S, (const T*)x, w, b, eps, (T*)y, mean, rstd);
  } else {
    LN_CHAN_LOOP(ln_chan_fwd_loop, R, C, S, C * S, (const T*)x, w, b, eps, (T*)y, mean, rstd);
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
      LN_CHAN(LN_CHAN_BWD, 2, (unsigned)G, (int)s.tiles, per, C, (int)S, (const T*)x, (const T*)dy, w, mean, rstd, (T*)dx, p);
    }
    PXL_LAUNCH_CHECK();
  } else if (R > 0) {
    if (dx != nullptr) {
      if (S < 0 && C < Piece<T>::N)
        LN_CHAN_LOOP(ln_chan_dx_loop, R, C, 1, xs, (const T*)x, (const T*)dy, w, mean, rstd, (T*)dx);
      else if (S < 0)
        hipLaunchKernelGGL(ln_rows_dx_loop<T>, dim3(blocks_for(R, 1 << 20)), dim3(256), 0, st, R, C, xs, (const T*)x, (const T*)dy, w, mean, rstd, (T*)dx);
      else
        LN_CHAN_LOOP(ln_chan_dx_loop, R, C, S, C * S, (const T*)x, (const T*)dy, w, mean, rstd, (T*)dx);
      PXL_LAUNCH_CHECK();
    }
    if (params) {
      if (S < 0 && C >= Piece<T>::N)
        hipLaunchKernelGGL(ln_rows_dwb_loop<T>, dim3((C + 255) / 256, G), dim3(256), 0, st, R, C, xs, (const T*)x, (const T*)dy, mean, rstd, part);
      else
        for (long c = 0; c < C; c += LN_MOST)
          hipLaunchKernelGGL(ln_chan_dwb_loop<T>, dim3((unsigned)(C - c < LN_MOST ? C - c : LN_MOST), G), dim3(256), 0, st, (int)c, R, C, S < 0 ? 1 : S,
                             S < 0 ? xs : C * S, (const T*)x, (const T*)dy, mean, rstd, part);
      PXL_LAUNCH_CHECK();
    }
  }
  if (params) {
    hipLaunchKernelGGL(ln_dwb_fold<T>, dim3((2 * C + 15) / 16), dim3(1024), 0, st, R > 0 ? G : 0, C, part, dw, db, pf32);
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
  PXL_REQUIRE(R >= 0 && C >= 1 && C <= (1 << 24), "%s: bad sizes (rows %ld, features %d: 1 .. 2^24)", what, R, C);
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
  if (S == 1) return pxl_layer_norm_fwd(dtype, pdtype, N, C, C, x, w, b, eps, y, mean, rstd, stream);          // rows of C without gaps
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
  if (S == 1) return pxl_layer_norm_bwd_workspace(N, C);
  return N < 0 || S < 0 || C < 1 ? 0 : (size_t)ln_chan_most(N, C, S) * 2 * C * sizeof(float);
}

extern "C" int pxl_layer_norm_nchw_bwd(int dtype, int pdtype, long N, int C, long S, const void* x, const void* dy, const void* w,
                                       const float* mean, const float* rstd, void* dx, void* dw, void* db, void* ws, size_t ws_bytes,
                                       void* stream) {
  PXL_REQUIRE(N >= 0 && S >= 0, "layer_norm_nchw_bwd: bad sizes (maps %ld, positions %ld)", N, S);
  if (S == 1) return pxl_layer_norm_bwd(dtype, pdtype, N, C, C, x, dy, w, mean, rstd, dx, dw, db, ws, ws_bytes, stream);
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
