// Orthogonalised updates (the Muon optimizer): Newton-Schulz iteration on every weight matrix of a call at once.
//
//   X0 = G / max(|G|_F, eps),   X <- X (a + b L + c L^2)  with  L = X' X (or X X': the smaller),  one (a, b, c) per step
//
// drives every singular value of G to about 1.  With m = min(rows, cols), n = max, one step as written costs m^2 n (the symmetric
// product at half price) + m^3 + 2 m^2 n operations.  All factors of several steps are polynomials of the SAME symmetric A = X X' and
// commute, so a run of steps ("segment") needs X only at its ends:
//   A = X X';  per step  Q = a + b A + c A^2,  P <- Q P,  A <- Q (Q A);   at the end  X <- P X
// Rounding of A by e turns into eigenvalues of size e next to zero, which every recursion multiplies by q(0)^2 = a^2 = 11.9 for the
// usual coefficients: a segment ends (X is multiplied out and A formed afresh, exactly positive) before that passes 16 for 32-bit
// results (2 + 2 + 1 of 5 steps) and 2^15 for bf16 results (all 5 steps: 11.9^4 2^-24 = 1.2e-3, under bf16's half step of 3.9e-3).
//
// Products run on the fp16 matrix instructions.  A 32-bit matrix is held as two fp16 planes, hi = fp16(x s), lo = fp16(x s - hi), s a
// power of two that puts the largest possible entry (|x_ij| <= the spectral norm, which the coefficients bound from step to step)
// under 2^15: 22 bits and more; a product is hi hi + hi lo + lo hi summed in fp32 -- 3 of the 16-bit instructions, five times the rate
// of the fp32 ones.  A bf16 matrix scaled by a power of two IS one fp16 plane (8 of 11 bits), its norm's remainder is applied to A and
// to the result.
//
// No atomics, no state between calls, every sum in one order.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <vector>

#include "common.h"

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int NS_MAX_CLASSES = 12;      // shapes per set of launches (kernel arguments); more shapes: further sets, one after the other
constexpr int NS_MAX_STEPS = 16;
constexpr int NS_TABLE = 64;            // items per table-writing launch
constexpr int NS_CHUNK = 8192;          // elements a workgroup of the norm pass takes at least
constexpr int NS_PARTS = 1024;          // partial sums of squares per matrix at most

// one matrix, in device memory
struct NsItem { void* p; const void* g; float* mom; float scale; int pad; };
struct NsTable { NsItem it[NS_TABLE]; };

// matrices of one shape, in kernel arguments.  Offsets in bytes from the workspace; the matrices of a class lie `stride` apart.
struct NsClass {
  int first, count;                     // in the device table
  int rows, cols, m, n, mp, np;         // mp / np: m / n rounded up (zero padding)
  int start, per;                       // first workgroup and workgroups per matrix of THIS launch
  int chunk, parts;                     // norm pass: elements per workgroup, workgroups per matrix
  int tn, pad;                          // tiles across (this launch)
  size_t base, stride;
};
struct NsClasses { NsClass c[NS_MAX_CLASSES]; int n; };

__device__ __forceinline__ int find_class(const NsClasses& cs, int b) {
  int k = 0;
#pragma unroll 1
  while (k + 1 < cs.n && b >= cs.c[k + 1].start) ++k;
  return k;
}

__global__ void ns_table_kernel(NsTable t, int n, NsItem* __restrict__ dst) {
  const int k = threadIdx.x;
  if (k < n) dst[k] = t.it[k];
}

struct MuonArgs { float lr, mu, nu, keep; int nesterov; };       // nu = 1 - mu, keep = 1 - lr * decay: from 64 bits (1.f - 0.95f is off by 2^-22)

// momentum (in place) and the update it gives
__device__ __forceinline__ float muon_momentum(float m, float g, const MuonArgs& a) { return __fmaf_rn(a.mu, m, a.nu * g); }
__device__ __forceinline__ float muon_update(float m, float g, const MuonArgs& a) { return a.nesterov ? __fmaf_rn(a.mu, m, a.nu * g) : m; }

// ---- pass 1: momentum, partial sums of squares (in 64 bits: squares of any fp32 value fit) -----------------------------------
template <typename T>
__global__ __launch_bounds__(256) void ns_norm_kernel(NsClasses cs, const NsItem* __restrict__ table, double* __restrict__ part, MuonArgs a) {
  __shared__ double sh[4];
  const int k = find_class(cs, blockIdx.x);
  const NsClass& c = cs.c[k];
  const int local = blockIdx.x - c.start, i = local / c.per, j = local - i * c.per;
  const NsItem it = table[c.first + i];
  const long size = (long)c.rows * c.cols, lo = (long)j * c.chunk, hi = lo + c.chunk < size ? lo + c.chunk : size;
  const T* g = reinterpret_cast<const T*>(it.g);
  double s = 0.0;
  for (long e = lo + threadIdx.x; e < hi; e += 256) {
    float u = to_f(g[e]);
    if (it.mom != nullptr) {
      const float m = muon_momentum(it.mom[e], u, a);
      it.mom[e] = m;
      u = muon_update(m, u, a);
    }
    s += (double)u * u;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[(long)(c.first + i) * NS_PARTS + j] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// ---- pass 2: scaled fp16 planes of X in both layouts: Xk [mp][np], Xt [np][mp] ------------------------------------------------
// residue[i]: what X's entries are still to be multiplied by (1 with two planes)
template <typename T, int NP>
__global__ __launch_bounds__(256) void ns_split_kernel(NsClasses cs, const NsItem* __restrict__ table, const double* __restrict__ part,
                                                       float* __restrict__ residue, unsigned char* __restrict__ ws, size_t off_k, size_t off_t,
                                                       float eps, float sx, MuonArgs a) {
  __shared__ double shn[4];
  __shared__ float tile[64][65];
  const int k = find_class(cs, blockIdx.x);
  const NsClass& c = cs.c[k];
  const int local = blockIdx.x - c.start, i = local / c.per, t = local - i * c.per;
  const int tr = t / c.tn, tc = t - tr * c.tn;             // 64 x 64 tile of [mp][np]
  const NsItem it = table[c.first + i];
  double s = 0.0;
  for (int e = threadIdx.x; e < c.parts; e += 256) s += part[(long)(c.first + i) * NS_PARTS + e];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) shn[threadIdx.x >> 6] = s;
  __syncthreads();
  const double square = (shn[0] + shn[1]) + (shn[2] + shn[3]);
  const double norm = fmax(sqrt(square), (double)eps);
  double mul;
  float left = 1.f;
  if (NP == 2) {
    mul = (double)sx / norm;
  } else {
    int e;
    frexp(norm, &e);                                       // norm in [2^(e-1), 2^e): entries below 1 after 2^-e
    mul = ldexp((double)sx, -e);
    left = (float)(ldexp(1.0, e) / norm);
  }
  if (!(square < HUGE_VAL)) mul = nan("");                 // a NaN or an infinity in the matrix: all of its result is NaN
  if (t == 0 && threadIdx.x == 0) residue[c.first + i] = left;
  const T* g = reinterpret_cast<const T*>(it.g);
  const bool tall = c.rows > c.cols;
  // tile[r][q]: r along m, q along n; read along the memory's rows
  for (int e = threadIdx.x; e < 4096; e += 256) {
    const int hi = e >> 6, lo = e & 63;
    const int r = tall ? lo : hi, q = tall ? hi : lo;
    const int im = tr * 64 + r, in = tc * 64 + q;
    float v = 0.f;
    if (im < c.m && in < c.n) {
      const long at = tall ? (long)in * c.cols + im : (long)im * c.cols + in;
      v = to_f(g[at]);
      if (it.mom != nullptr) v = muon_update(it.mom[at], v, a);
      v = (float)((double)v * mul);
    }
    tile[r][q] = v;
  }
  __syncthreads();
  unsigned char* base = ws + c.base + (size_t)i * c.stride;
  const size_t plane = (size_t)c.mp * c.np * 2;
  for (int e = threadIdx.x; e < 4096; e += 256) {
    const int hi = e >> 6, lo = e & 63;
    if (tr * 64 + hi < c.mp && tc * 64 + lo < c.np) {
      const float v = tile[hi][lo];
      const _Float16 h = (_Float16)v;
      _Float16* d = reinterpret_cast<_Float16*>(base + off_k * plane) + (size_t)(tr * 64 + hi) * c.np + tc * 64 + lo;
      d[0] = h;
      if (NP == 2) d[plane / 2] = (_Float16)(v - (float)h);
    }
    if (tc * 64 + hi < c.np && tr * 64 + lo < c.mp) {
      const float v = tile[lo][hi];
      const _Float16 h = (_Float16)v;
      _Float16* d = reinterpret_cast<_Float16*>(base + off_t * plane) + (size_t)(tc * 64 + hi) * c.mp + tr * 64 + lo;
      d[0] = h;
      if (NP == 2) d[plane / 2] = (_Float16)(v - (float)h);
    }
  }
}

// ---- products: C[i][j] = sum_k a[i][k] b[j][k] over fp16 planes, both operands with k contiguous ------------------------------
enum { EPI_GRAM = 0, EPI_Q = 1, EPI_MUL = 2, EPI_X = 3, EPI_OUT = 4 };

// operand / result slots of a matrix's workspace region: X planes first (units of mp * np * 2 bytes), then m x m pairs of planes
struct NsSlot { int x, mm; };           // x planes, then mm pairs
__device__ __forceinline__ size_t slot_off(const NsClass& c, int xplanes, int slot) {
  const size_t px = (size_t)c.mp * c.np * 2, pm = (size_t)c.mp * c.mp * 2;
  return slot < xplanes ? (size_t)slot * px : (size_t)xplanes * px + (size_t)(slot - xplanes) * 2 * pm;
}

struct NsJob { int a, b, out, out2; };  // slots
struct NsGemm {
  NsJob job[2];
  int xplanes;                          // X slots of a region
  float unscale, scale;                 // accumulator -> value, value -> planes
  float qa, qb, qc, sa_inv;             // EPI_Q: coefficients, 1 / scale of A's planes
  int res_pow;                          // EPI_GRAM: value *= residue^2;  EPI_OUT / EPI_X: value *= residue
  float lr, decay;                      // EPI_OUT of a Muon step
  int muon;
};

__device__ __forceinline__ void put_split(_Float16* d, size_t plane, float v) {
  const _Float16 h = (_Float16)v;
  d[0] = h;
  d[plane] = (_Float16)(v - (float)h);
}

// lower-triangular tile number t -> (row, column), row >= column
__device__ __forceinline__ void tri_tile(int t, int& r, int& q) {
  r = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
  while ((r + 1) * (r + 2) / 2 <= t) ++r;
  while (r * (r + 1) / 2 > t) --r;
  q = t - r * (r + 1) / 2;
}

// T x T tile per workgroup of 4 waves (2 x 2), K steps of 32, two LDS buffers; LDS rows of 64 bytes, 16-byte chunk c of row r at
// c ^ ((r >> 2) & 3): the 16 lanes that read one chunk column in a phase then hit 16 different bank groups
template <int EPI, int NA, int NB, int T, typename OutT>
__global__ __launch_bounds__(256) void ns_gemm_kernel(NsClasses cs, NsGemm p, const NsItem* __restrict__ table, const float* __restrict__ residue,
                                                      unsigned char* __restrict__ ws) {
  constexpr bool SYM = EPI <= EPI_MUL;
  constexpr int W = T / 64;                     // 32 x 32 accumulators per wave and direction
  constexpr int PL = T * 64;                    // bytes of one plane's tile
  constexpr int CH = T / 64;                    // 16-byte chunks a thread moves per plane
  __shared__ __attribute__((aligned(16))) unsigned char lds[2][(NA + NB) * PL];
  const int k = find_class(cs, blockIdx.x);
  const NsClass& c = cs.c[k];
  const int local = blockIdx.x - c.start, i = local / c.per, t = local - i * c.per;
  int tr, tc;
  if (SYM) tri_tile(t, tr, tc);
  else { tr = t / c.tn; tc = t - tr * c.tn; }
  const NsJob job = p.job[blockIdx.z];
  unsigned char* base = ws + c.base + (size_t)i * c.stride;
  const bool xa = EPI == EPI_GRAM;              // operands: the X planes, or m x m pairs
  const int K = xa ? c.np : c.mp;
  const int rowsA = c.mp, rowsB = EPI >= EPI_X ? c.np : c.mp;
  const size_t plane_a = (size_t)rowsA * K, plane_b = (size_t)rowsB * K;
  const _Float16* A = reinterpret_cast<const _Float16*>(base + slot_off(c, p.xplanes, job.a));
  const _Float16* B = reinterpret_cast<const _Float16*>(base + slot_off(c, p.xplanes, job.b));

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wr = wave >> 1, wc = wave & 1;
  u32x4 ra[NA][CH], rb[NB][CH];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int e = tid + q * 256, r = e >> 2, ch = e & 3;
      int ia = tr * T + r, ib = tc * T + r;     // rows past the matrix: the last one again (never stored)
      if (ia >= rowsA) ia = rowsA - 1;
      if (ib >= rowsB) ib = rowsB - 1;
      const _Float16* pa = A + (size_t)ia * K + k0 + ch * 8;
      const _Float16* pb = B + (size_t)ib * K + k0 + ch * 8;
#pragma unroll
      for (int z = 0; z < NA; ++z) ra[z][q] = *reinterpret_cast<const u32x4*>(pa + z * plane_a);
#pragma unroll
      for (int z = 0; z < NB; ++z) rb[z][q] = *reinterpret_cast<const u32x4*>(pb + z * plane_b);
    }
  };
  auto stash = [&](int buf) {
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int e = tid + q * 256, r = e >> 2, ch = e & 3;
      const int at = r * 64 + ((ch ^ ((r >> 2) & 3)) << 4);
#pragma unroll
      for (int z = 0; z < NA; ++z) *reinterpret_cast<u32x4*>(&lds[buf][z * PL + at]) = ra[z][q];
#pragma unroll
      for (int z = 0; z < NB; ++z) *reinterpret_cast<u32x4*>(&lds[buf][(NA + z) * PL + at]) = rb[z][q];
    }
  };
  f32x16 acc[W][W];
#pragma unroll
  for (int u = 0; u < W; ++u)
#pragma unroll
    for (int v = 0; v < W; ++v)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[u][v][e] = 0.f;

  fetch(0);
  stash(0);
  __syncthreads();
  const int steps = K >> 5;
  for (int s = 0; s < steps; ++s) {
    if (s + 1 < steps) fetch((s + 1) << 5);
    const unsigned char* buf = lds[s & 1];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      f16x8 fa[NA][W], fb[NB][W];
#pragma unroll
      for (int u = 0; u < W; ++u) {
        const int r = wr * (T / 2) + u * 32 + (lane & 31), ch = kk * 2 + (lane >> 5);
        const int q = wc * (T / 2) + u * 32 + (lane & 31);
#pragma unroll
        for (int z = 0; z < NA; ++z) fa[z][u] = *reinterpret_cast<const f16x8*>(buf + z * PL + r * 64 + ((ch ^ ((r >> 2) & 3)) << 4));
#pragma unroll
        for (int z = 0; z < NB; ++z) fb[z][u] = *reinterpret_cast<const f16x8*>(buf + (NA + z) * PL + q * 64 + ((ch ^ ((q >> 2) & 3)) << 4));
      }
#pragma unroll
      for (int u = 0; u < W; ++u)
#pragma unroll
        for (int v = 0; v < W; ++v) {
          if (NB == 2) acc[u][v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[0][u], fb[NB - 1][v], acc[u][v], 0, 0, 0);
          if (NA == 2) acc[u][v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[NA - 1][u], fb[0][v], acc[u][v], 0, 0, 0);
          acc[u][v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[0][u], fb[0][v], acc[u][v], 0, 0, 0);
        }
    }
    if (s + 1 < steps) stash((s + 1) & 1);
    __syncthreads();
  }

  // accumulator element e of lane: row 8 (e / 4) + 4 (lane / 32) + e % 4, column lane % 32
  const float res = EPI == EPI_Q || EPI == EPI_MUL ? 1.f : (p.res_pow == 0 ? 1.f : (p.res_pow == 2 ? residue[c.first + i] * residue[c.first + i] : residue[c.first + i]));
  const float un = p.unscale * res;
  const size_t pm = (size_t)c.mp * c.mp, px = (size_t)c.mp * c.np;
  _Float16* out = reinterpret_cast<_Float16*>(base + slot_off(c, p.xplanes, job.out));
  _Float16* out2 = reinterpret_cast<_Float16*>(base + slot_off(c, p.xplanes, job.out2));
  const NsItem it = table[c.first + i];
  const bool tall = c.rows > c.cols;
#pragma unroll
  for (int u = 0; u < W; ++u)
#pragma unroll
    for (int v = 0; v < W; ++v)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int r0 = tr * T + wr * (T / 2) + u * 32 + 8 * e4 + 4 * (lane >> 5);
        const int q = tc * T + wc * (T / 2) + v * 32 + (lane & 31);
        float val[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) val[e] = acc[u][v][e4 * 4 + e] * un;
        if (EPI == EPI_OUT) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = r0 + e;
            if (r >= c.m || q >= c.n) continue;
            const size_t at = tall ? (size_t)q * c.cols + r : (size_t)r * c.cols + q;
            OutT* o = reinterpret_cast<OutT*>(it.p) + at;
            if (p.muon) *o = from_f<OutT>(to_f(*o) * p.decay - p.lr * it.scale * val[e]);
            else *o = from_f<OutT>(val[e]);
          }
          continue;
        }
        if (r0 >= c.mp || q >= (EPI == EPI_X ? c.np : c.mp)) continue;      // (mp, np are multiples of 32)
        if (EPI == EPI_Q) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const _Float16* am = A + (size_t)(r0 + e) * c.mp + q;
            val[e] = p.qc * val[e] + p.qb * (((float)am[0] + (float)am[pm]) * p.sa_inv) + (r0 + e == q ? p.qa : 0.f);
          }
        }
        const int ld = EPI == EPI_X ? c.np : c.mp;
        const size_t pl = EPI == EPI_X ? px : pm;
        f16x4 h, l;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = val[e] * p.scale;
          h[e] = (_Float16)x;
          l[e] = (_Float16)(x - (float)h[e]);
          _Float16* d = out + (size_t)(r0 + e) * ld + q;
          d[0] = h[e];
          if (EPI != EPI_X || NB == 2) d[pl] = l[e];
        }
        if (EPI == EPI_X || tr != tc) {           // the other layout of X; the mirrored tile of a symmetric product
          const int ld2 = EPI == EPI_X ? c.mp : c.mp;
          _Float16* d = (EPI == EPI_X ? out2 : out) + (size_t)q * ld2 + r0;
          *reinterpret_cast<f16x4*>(d) = h;
          if (EPI != EPI_X || NB == 2) *reinterpret_cast<f16x4*>(d + pl) = l;
        }
      }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------
struct NsPlan {
  struct Set { std::vector<NsClass> cls; std::vector<int> order; size_t bytes; int items; };
  std::vector<Set> sets;
  int np;                               // planes of X
  int xplanes;
  size_t head;                          // table + norms + residues, for the largest set
  size_t bytes;
};

inline int round_up(int v, int to) { return (v + to - 1) / to * to; }
inline size_t round_up_z(size_t v, size_t to) { return (v + to - 1) / to * to; }

// slots of a region: Xk, Xt, Xu (the next Xt), NP planes each, then A, T and three for Q / P
int ns_plan(const char* what, int dtype, const pxl_ns_item* items, int n, NsPlan& plan) {
  PXL_REQUIRE(dtype == PXL_F32 || dtype == PXL_BF16, "%s: dtype %d is neither PXL_F32 nor PXL_BF16", what, dtype);
  PXL_REQUIRE(n >= 0 && (n == 0 || items != nullptr), "%s: bad item list", what);
  plan.np = dtype == PXL_F32 ? 2 : 1;
  plan.xplanes = 3 * plan.np;
  std::vector<NsPlan::Set>& sets = plan.sets;
  for (int i = 0; i < n; ++i) {
    PXL_REQUIRE(items[i].rows >= 1 && items[i].cols >= 1 && items[i].rows <= (1 << 24) && items[i].cols <= (1 << 24) &&
                    (items[i].rows < items[i].cols ? items[i].rows : items[i].cols) <= (1 << 15),
                "%s: item %d is %d x %d (1 .. 2^24, the smaller side at most 32768)", what, i, items[i].rows, items[i].cols);
    int sk = -1, ck = -1;
    for (size_t s = 0; s < sets.size() && sk < 0; ++s)
      for (size_t k = 0; k < sets[s].cls.size(); ++k)
        if (sets[s].cls[k].rows == items[i].rows && sets[s].cls[k].cols == items[i].cols) { sk = (int)s; ck = (int)k; break; }
    if (sk < 0) {
      if (sets.empty() || sets.back().cls.size() == (size_t)NS_MAX_CLASSES) sets.emplace_back();
      NsClass c;
      memset(&c, 0, sizeof(c));
      c.rows = items[i].rows;
      c.cols = items[i].cols;
      c.m = c.rows < c.cols ? c.rows : c.cols;
      c.n = c.rows < c.cols ? c.cols : c.rows;
      c.mp = round_up(c.m, 32);
      c.np = round_up(c.n, 32);
      const long size = (long)c.rows * c.cols;
      long chunk = NS_CHUNK;
      while ((size + chunk - 1) / chunk > NS_PARTS) chunk *= 2;
      PXL_REQUIRE(chunk < (1l << 30), "%s: item %d of %ld elements is too large", what, i, size);
      c.chunk = (int)chunk;
      c.parts = (int)((size + chunk - 1) / chunk);
      c.stride = round_up_z((size_t)plan.xplanes * c.mp * c.np * 2 + (size_t)5 * 2 * c.mp * c.mp * 2, 256);
      sets.back().cls.push_back(c);
      sk = (int)sets.size() - 1;
      ck = (int)sets.back().cls.size() - 1;
    }
    sets[sk].cls[ck].count++;
  }
  plan.head = plan.bytes = 0;
  for (auto& s : sets) {
    int first = 0;
    for (auto& c : s.cls) { c.first = first; first += c.count; }
    s.items = first;
    const size_t head = round_up_z(first * sizeof(NsItem), 256) + round_up_z(first * sizeof(double) * NS_PARTS, 256) + round_up_z(first * sizeof(float), 256);
    if (head > plan.head) plan.head = head;
  }
  for (auto& s : sets) {
    size_t at = plan.head;
    for (auto& c : s.cls) { c.base = at; at += c.stride * c.count; }
    s.bytes = at;
    if (at > plan.bytes) plan.bytes = at;
  }
  return PXL_OK;
}

// bounds of the iteration on singular values in [0, 1], and where its segments end
struct NsStep { double a, b, c, sigma, lam, q, t, gain; int last; };     // bounds BEFORE the step: sigma, lam; OF it: |q|, |lam q|
int ns_schedule(const char* what, int steps, const float* coef, int np, std::vector<NsStep>& st) {
  PXL_REQUIRE(steps >= 1 && steps <= NS_MAX_STEPS && coef != nullptr, "%s: 1 .. %d steps with three coefficients each", what, NS_MAX_STEPS);
  const double limit = np == 2 ? 16.0 : 32768.0;
  double sigma = 1.0, grown = 1.0;
  for (int s = 0; s < steps; ++s) {
    NsStep d;
    d.a = coef[3 * s]; d.b = coef[3 * s + 1]; d.c = coef[3 * s + 2];
    PXL_REQUIRE(std::isfinite(d.a) && std::isfinite(d.b) && std::isfinite(d.c), "%s: coefficients of step %d are not finite", what, s);
    d.sigma = sigma;
    d.lam = sigma * sigma;
    double next = 0.0;
    d.q = d.t = 0.0;
    for (int e = 0; e <= 4096; ++e) {
      const double x = sigma * e / 4096, l = x * x, q = fabs(d.a + l * (d.b + d.c * l));
      next = fmax(next, x * q);
      d.q = fmax(d.q, q);
      d.t = fmax(d.t, l * q);
    }
    PXL_REQUIRE(next <= 16.0 && d.q <= 1e4, "%s: step %d lets singular values grow to %g", what, s, next);
    sigma = next * 1.01 + 1e-3;
    d.gain = d.q * d.q > 1.0 ? d.q * d.q : 1.0;
    d.last = s == steps - 1;
    if (!d.last) {
      if (grown * d.gain > limit) { d.last = 1; grown = 1.0; }
      else grown *= d.gain;
    }
    st.push_back(d);
  }
  return PXL_OK;
}

// the largest power of two that keeps `bound` below 2^15
inline float plane_scale(double bound) {
  int e;
  frexp(bound < 1e-6 ? 1e-6 : bound, &e);
  return (float)ldexp(1.0, 15 - e);
}

struct NsRun {
  hipStream_t st;
  NsClasses cs;
  NsItem* table;
  double* part;
  float* residue;
  unsigned char* ws;
};

template <int EPI, int NA, int NB, typename OutT>
int ns_gemm(NsRun& r, const NsGemm& g, int jobs) {
  constexpr int T = 64;
  int at = 0;
  for (int k = 0; k < r.cs.n; ++k) {
    NsClass& c = r.cs.c[k];
    const int tm = (c.mp + T - 1) / T, tn = (c.np + T - 1) / T;
    c.tn = EPI <= EPI_MUL ? tm : tn;
    c.per = EPI <= EPI_MUL ? tm * (tm + 1) / 2 : tm * tn;
    c.start = at;
    at += c.per * c.count;
  }
  hipLaunchKernelGGL((ns_gemm_kernel<EPI, NA, NB, T, OutT>), dim3(at, 1, jobs), dim3(256), 0, r.st, r.cs, g, r.table, r.residue, r.ws);
  PXL_LAUNCH_CHECK();
  return PXL_OK;
}

#define NS_TRY(expr)            \
  do {                          \
    const int _rc = (expr);     \
    if (_rc != PXL_OK) return _rc; \
  } while (0)

template <typename T, int NP>
int ns_run_set(NsRun& r, const std::vector<NsStep>& steps, float eps, const MuonArgs& ma, int muon) {
  const int XK = 0, XT = NP, XU = 2 * NP, xplanes = 3 * NP, MA = xplanes, MT = xplanes + 1;
  int blocks = 0;
  for (int k = 0; k < r.cs.n; ++k) {
    NsClass& c = r.cs.c[k];
    c.per = c.parts;
    c.start = blocks;
    blocks += c.per * c.count;
  }
  hipLaunchKernelGGL(ns_norm_kernel<T>, dim3(blocks), dim3(256), 0, r.st, r.cs, r.table, r.part, ma);
  PXL_LAUNCH_CHECK();
  blocks = 0;
  for (int k = 0; k < r.cs.n; ++k) {
    NsClass& c = r.cs.c[k];
    c.tn = (c.np + 63) / 64;
    c.per = c.tn * ((c.mp + 63) / 64);
    c.start = blocks;
    blocks += c.per * c.count;
  }
  float sx = plane_scale(1.0);
  hipLaunchKernelGGL((ns_split_kernel<T, NP>), dim3(blocks), dim3(256), 0, r.st, r.cs, r.table, r.part, r.residue, r.ws, (size_t)XK, (size_t)XT, eps, sx, ma);
  PXL_LAUNCH_CHECK();

  NsGemm g;
  memset(&g, 0, sizeof(g));
  g.xplanes = xplanes;
  int first = 1, xt = XT, xu = XU;
  size_t s = 0;
  while (s < steps.size()) {
    double lam = steps[s].lam, pbound = 1.0;
    float sA = plane_scale(lam), sP = 1.f;
    g.job[0] = {XK, XK, MA, MA};
    g.unscale = 1.f / (sx * sx);
    g.scale = sA;
    g.res_pow = NP == 1 && first ? 2 : 0;
    NS_TRY((ns_gemm<EPI_GRAM, NP, NP, T>(r, g, 1)));
    int P = -1;
    for (;; ++s) {
      const NsStep& d = steps[s];
      int q = xplanes + 2;
      while (q == P) ++q;
      const float sQ = plane_scale(d.q);
      g.job[0] = {MA, MA, q, q};
      g.unscale = 1.f / (sA * sA);
      g.scale = sQ;
      g.qa = (float)d.a; g.qb = (float)d.b; g.qc = (float)d.c;
      g.sa_inv = 1.f / sA;
      NS_TRY((ns_gemm<EPI_Q, 2, 2, T>(r, g, 1)));
      pbound *= d.q;
      const float sP2 = plane_scale(pbound), sT = plane_scale(d.t);
      if (P < 0) {
        P = q;
        sP = sQ;
      } else {
        int p2 = xplanes + 2;
        while (p2 == P || p2 == q) ++p2;
        g.job[0] = {q, P, p2, p2};
        g.unscale = 1.f / (sQ * sP);
        g.scale = sP2;
        NS_TRY((ns_gemm<EPI_MUL, 2, 2, T>(r, g, 1)));
        P = p2;
        sP = sP2;
      }
      if (d.last) break;
      g.job[0] = {q, MA, MT, MT};
      g.unscale = 1.f / (sQ * sA);
      g.scale = sT;
      NS_TRY((ns_gemm<EPI_MUL, 2, 2, T>(r, g, 1)));
      const float sA2 = plane_scale(steps[s + 1].lam);
      g.job[0] = {q, MT, MA, MA};
      g.unscale = 1.f / (sQ * sT);
      g.scale = sA2;
      NS_TRY((ns_gemm<EPI_MUL, 2, 2, T>(r, g, 1)));
      sA = sA2;
    }
    ++s;
    g.unscale = 1.f / (sP * sx);
    g.res_pow = NP == 1 && first ? 1 : 0;
    if (s == steps.size()) {
      g.job[0] = {P, xt, 0, 0};
      g.muon = muon;
      g.lr = ma.lr;
      g.decay = ma.keep;
      NS_TRY((ns_gemm<EPI_OUT, 2, NP, T>(r, g, 1)));
    } else {
      const float sx2 = plane_scale(steps[s].sigma);
      g.job[0] = {P, xt, XK, xu};
      g.scale = sx2;
      NS_TRY((ns_gemm<EPI_X, 2, NP, T>(r, g, 1)));
      sx = sx2;
      const int o = xt;
      xt = xu;
      xu = o;
      first = 0;
    }
  }
  return PXL_OK;
}

// what is written (results, momenta) overlaps nothing else of the call (a result over its own matrix apart)
int ns_overlap(const char* what, int dtype, const pxl_ns_item* items, int n, int muon) {
  struct Span { uintptr_t lo, hi; bool written; };
  std::vector<Span> v;
  v.reserve(3 * (size_t)n);
  for (int i = 0; i < n; ++i) {
    const size_t size = (size_t)items[i].rows * items[i].cols, bytes = size * (dtype == PXL_F32 ? 4 : 2);
    const uintptr_t p = (uintptr_t)items[i].p, g = (uintptr_t)items[i].g, m = (uintptr_t)items[i].mom;
    v.push_back({p, p + bytes, true});
    if (muon || g != p) v.push_back({g, g + bytes, false});
    if (muon) v.push_back({m, m + size * 4, true});
  }
  std::sort(v.begin(), v.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
  uintptr_t written = 0, any = 0;
  for (const Span& s : v) {
    PXL_REQUIRE(s.lo >= (s.written ? any : written), "%s: the same memory appears twice (at %p)", what, (void*)s.lo);
    if (s.written) written = std::max(written, s.hi);
    any = std::max(any, s.hi);
  }
  return PXL_OK;
}

int ns_run(const char* what, int dtype, const pxl_ns_item* items, int n, int steps, const float* coef, float eps, const MuonArgs& ma, int muon,
           void* ws, size_t ws_bytes, void* stream) {
  NsPlan plan;
  NS_TRY(ns_plan(what, dtype, items, n, plan));
  std::vector<NsStep> st;
  NS_TRY(ns_schedule(what, steps, coef, plan.np, st));
  PXL_REQUIRE(eps > 0.f, "%s: eps %g", what, eps);
  for (int i = 0; i < n; ++i)
    PXL_REQUIRE(items[i].p != nullptr && items[i].g != nullptr && (!muon || items[i].mom != nullptr), "%s: item %d has a null pointer", what, i);
  if (n == 0) return PXL_OK;
  NS_TRY(ns_overlap(what, dtype, items, n, muon));
  if (ws == nullptr || ws_bytes < plan.bytes)
    return pxl_set_error(PXL_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, ws_bytes, plan.bytes);
  NsRun r;
  r.st = reinterpret_cast<hipStream_t>(stream);
  r.ws = reinterpret_cast<unsigned char*>(ws);
  for (auto& set : plan.sets) {
    r.table = reinterpret_cast<NsItem*>(ws);
    r.part = reinterpret_cast<double*>(r.ws + round_up_z(set.items * sizeof(NsItem), 256));
    r.residue = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(r.part) + round_up_z(set.items * sizeof(double) * NS_PARTS, 256));
    r.cs.n = (int)set.cls.size();
    for (int k = 0; k < r.cs.n; ++k) r.cs.c[k] = set.cls[k];
    std::vector<NsItem> list;
    for (auto& c : set.cls)
      for (int i = 0; i < n; ++i)
        if (items[i].rows == c.rows && items[i].cols == c.cols)
          list.push_back(NsItem{items[i].p, items[i].g, muon ? items[i].mom : nullptr, items[i].scale, 0});
    for (size_t at = 0; at < list.size(); at += NS_TABLE) {
      NsTable t;
      const int cnt = (int)(list.size() - at < (size_t)NS_TABLE ? list.size() - at : NS_TABLE);
      memcpy(t.it, &list[at], cnt * sizeof(NsItem));
      hipLaunchKernelGGL(ns_table_kernel, dim3(1), dim3(64), 0, r.st, t, cnt, r.table + at);
      PXL_LAUNCH_CHECK();
    }
    if (dtype == PXL_F32) NS_TRY((ns_run_set<float, 2>(r, st, eps, ma, muon)));
    else NS_TRY((ns_run_set<bf16_t, 1>(r, st, eps, ma, muon)));
  }
  return PXL_OK;
}

}  // namespace

extern "C" size_t pxl_ns_workspace(int dtype, const pxl_ns_item* items, int n) {
  try {
    NsPlan plan;
    return ns_plan("ns_workspace", dtype, items, n, plan) == PXL_OK ? plan.bytes : 0;
  } catch (...) {
    return 0;
  }
}

extern "C" int pxl_orthogonalize(int dtype, const pxl_ns_item* items, int n, int steps, const float* coef, float eps, void* ws, size_t ws_bytes,
                                 void* stream) {
  try {
    return ns_run("orthogonalize", dtype, items, n, steps, coef, eps, MuonArgs{0.f, 0.f, 0.f, 0.f, 0}, 0, ws, ws_bytes, stream);
  } catch (...) {
    return pxl_set_error(PXL_ERR_ARG, "orthogonalize: out of host memory");
  }
}

extern "C" int pxl_muon_step(int dtype, const pxl_ns_item* items, int n, int steps, const float* coef, float eps, double lr, double momentum,
                             int nesterov, double weight_decay, void* ws, size_t ws_bytes, void* stream) {
  if (!(momentum >= 0.0 && momentum < 1.0) || !std::isfinite(lr) || !std::isfinite(weight_decay))
    return pxl_set_error(PXL_ERR_ARG, "muon_step: lr %g, momentum %g (0 <= momentum < 1), weight decay %g", lr, momentum, weight_decay);
  try {
    return ns_run("muon_step", dtype, items, n, steps, coef, eps, MuonArgs{(float)lr, (float)momentum, (float)(1.0 - momentum), (float)(1.0 - lr * weight_decay), nesterov}, 1, ws, ws_bytes, stream);
  } catch (...) {
    return pxl_set_error(PXL_ERR_ARG, "muon_step: out of host memory");
  }
}
