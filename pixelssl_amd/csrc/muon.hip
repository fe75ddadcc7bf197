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
// results (2 + 2 + 1 of 5 steps) and 2^15 for bf16 results (all 5 steps).  What that leaves of a bf16 result before its rounding: errors of A of
// 2^-22 of its entries, spread over all directions, are within 1e-5 of |O| on noise with strong directions in it, and 8e-4 at most on spectra of
// one strong direction, 1 / i^2 and six decades (measured, 60 x 130 to 256 x 1024), where the rounding to bf16 is 1.7e-3 of |O|.
//
// Products run on the fp16 matrix instructions.  A 32-bit matrix is held as two fp16 planes, hi = fp16(x s), lo = fp16(x s - hi), s a
// power of two that puts the largest possible entry (|x_ij| <= the spectral norm, which the coefficients bound from step to step)
// under 2^15: 22 bits of every entry down to 2^-17 of that, fewer below (fp16 ends at 2^-24): rows 2^-24 below the matrix' norm, or its eps where
// that is larger, keep about 14 bits and rows 2^-38 below it vanish; a product is hi hi + hi lo + lo hi summed in fp32 -- 3 of the 16-bit
// instructions, five times the rate of the fp32 ones.  A bf16 matrix scaled by a power of two IS one fp16 plane (8 of 11 bits), its norm's remainder is applied to A and
// to the result.  (A Muon step's update is a 32-bit matrix, of bf16 parameters too: two planes.)
//
// Measured (5 steps, us): 64 x 147 fp32 34, 23 x 256 x 2304 fp32 341 - 349, 23 x 1024 x 256 bf16 191 - 196, 2 x 2048 x 4608 fp32 2090 - 2150 (0.77 PF
// of fp16 products against 1.09 of a large library product: power brings the clock from 2.4 to 1.7 - 1.8 GHz), Muon steps of 3 x 512 x 4608 350 - 354
// (bf16 parameters too) and of 4 x 21 x 18432 74.  Below some hundred rows the chain of dependent products bounds it: 4.5 us a launch until its first product, 2 us its stores.
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
constexpr int NS_CHUNK = 2048;          // elements a workgroup of the norm pass takes at least
constexpr int NS_PARTS = 1024;          // partial sums of squares per matrix at most

// one matrix, in device memory
struct NsItem { void* p; const void* g; float* mom; float scale; int pad; };
struct NsTable { NsItem it[NS_TABLE]; };
// up to 32 of them travel in the kernel arguments of the three kernels that need them: no table launch
constexpr int NS_INLINE = 32;
struct NsInline { NsItem it[NS_INLINE]; };
__device__ __forceinline__ NsItem ns_item(const NsInline& few, const NsItem* table, int i) { return table != nullptr ? table[i] : few.it[i]; }

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// four elements at any element alignment
__device__ __forceinline__ void load4(const float* p, float* v) { __builtin_memcpy(v, p, 16); }
__device__ __forceinline__ void load4(const bf16_t* p, float* v) {
  uint2 w;
  __builtin_memcpy(&w, p, 8);
  v[0] = bf_lo(w.x); v[1] = bf_hi(w.x); v[2] = bf_lo(w.y); v[3] = bf_hi(w.y);
}
__device__ __forceinline__ void store4(float* p, const float* v) { __builtin_memcpy(p, v, 16); }
__device__ __forceinline__ void store4(bf16_t* p, const float* v) {
  const uint2 w = make_uint2(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]));
  __builtin_memcpy(p, &w, 8);
}

// matrices of one shape, in kernel arguments.  Offsets in bytes from the workspace; the matrices of a class lie `stride` apart.
struct NsClass {
  int first, count;                     // in the device table
  int rows, cols, m, n, mp, np;         // mp / np: m / n rounded up (zero padding)
  int start, per;                       // first workgroup and workgroups per matrix of THIS launch
  int chunk, parts;                     // norm pass: elements per workgroup, workgroups per matrix
  int tn, ks;                           // tiles across (this launch); split products: k a share
  size_t base, stride;
};
struct NsClasses { NsClass c[NS_MAX_CLASSES]; int n; };

// the class of workgroup b, by value: the first one's fields are fetched together with the other arguments (one shape: no further round trip)
__device__ __forceinline__ NsClass find_class(const NsClasses& cs, int b) {
  NsClass c = cs.c[0];
  if (cs.n > 1 && b >= cs.c[1].start) {
    int k = 1;
#pragma unroll 1
    while (k + 1 < cs.n && b >= cs.c[k + 1].start) ++k;
    c = cs.c[k];
  }
  return c;
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
__global__ __launch_bounds__(256) void ns_norm_kernel(NsClasses cs, NsInline few, const NsItem* __restrict__ table, double* __restrict__ part, MuonArgs a) {
  __shared__ double sh[4];
  const NsClass c = find_class(cs, blockIdx.x);
  const int local = blockIdx.x - c.start, i = local / c.per, j = local - i * c.per;
  const NsItem it = ns_item(few, table, c.first + i);
  const long size = (long)c.rows * c.cols, lo = (long)j * c.chunk, hi = lo + c.chunk < size ? lo + c.chunk : size;
  const T* g = reinterpret_cast<const T*>(it.g);
  double s = 0.0;
  long e = lo + threadIdx.x * 4;
  for (; e + 4 <= hi; e += 1024) {
    float u[4];
    load4(g + e, u);
    if (it.mom != nullptr) {
      float m[4];
      load4(it.mom + e, m);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        m[q] = muon_momentum(m[q], u[q], a);
        u[q] = muon_update(m[q], u[q], a);
      }
      store4(it.mom + e, m);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) s += (double)u[q] * u[q];
  }
  for (; e < hi; ++e) {                  // the one thread whose four pass the end
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

// ---- pass 2: scaled fp16 planes of X [mp][np] (the smaller side first whatever the matrix is) ---------------------------------
// residue[i]: what X's entries are still to be multiplied by (1 with two planes)
template <typename T, int NP>
__global__ __launch_bounds__(256) void ns_split_kernel(NsClasses cs, NsInline few, const NsItem* __restrict__ table, const double* __restrict__ part,
                                                       float* __restrict__ residue, unsigned char* __restrict__ ws, float eps, float sx, MuonArgs a) {
  __shared__ double shn[4];
  __shared__ float tile[64][65];
  const NsClass c = find_class(cs, blockIdx.x);
  const int local = blockIdx.x - c.start, i = local / c.per, t = local - i * c.per;
  const int tr = t / c.tn, tc = t - tr * c.tn;             // 64 x 64 tile of [mp][np]
  const NsItem it = ns_item(few, table, c.first + i);
  const T* g = reinterpret_cast<const T*>(it.g);
  const bool tall = c.rows > c.cols;
  // tile[r][q]: r along m, q along n; read along the memory's rows, four elements a thread -- before the norm is there
  const int lines = tall ? c.n : c.m, line0 = tall ? tc * 64 : tr * 64, col0 = tall ? tr * 64 : tc * 64;
  const int col = col0 + (threadIdx.x & 15) * 4, l0 = threadIdx.x >> 4;
  float u[4][4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int line = line0 + l0 + q * 16;
#pragma unroll
    for (int e = 0; e < 4; ++e) u[q][e] = 0.f;
    if (line < lines) {
      const long at = (long)line * c.cols + col;
      if (col + 4 <= c.cols) {
        load4(g + at, u[q]);
        if (it.mom != nullptr) {
          float m[4];
          load4(it.mom + at, m);
#pragma unroll
          for (int e = 0; e < 4; ++e) u[q][e] = muon_update(m[e], u[q][e], a);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < c.cols) {
            u[q][e] = to_f(g[at + e]);
            if (it.mom != nullptr) u[q][e] = muon_update(it.mom[at + e], u[q][e], a);
          }
      }
    }
  }
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
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = (float)((double)u[q][e] * mul);
      if (tall) tile[(threadIdx.x & 15) * 4 + e][l0 + q * 16] = x;
      else tile[l0 + q * 16][(threadIdx.x & 15) * 4 + e] = x;
    }
  __syncthreads();
  unsigned char* base = ws + c.base + (size_t)i * c.stride;
  const size_t plane = (size_t)c.mp * c.np;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = l0 + q * 16, im = tr * 64 + r, in = tc * 64 + (threadIdx.x & 15) * 4;
    if (im >= c.mp || in >= c.np) continue;
    f16x4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = tile[r][(threadIdx.x & 15) * 4 + e];
      h[e] = (_Float16)v;
      l[e] = (_Float16)(v - (float)h[e]);
    }
    _Float16* d = reinterpret_cast<_Float16*>(base) + (size_t)im * c.np + in;
    *reinterpret_cast<f16x4*>(d) = h;
    if (NP == 2) *reinterpret_cast<f16x4*>(d + plane) = l;
  }
}

// ---- products over fp16 planes ------------------------------------------------------------------------------------------------
// GRAM, PART, Q, MUL: C[i][j] = sum_k a[i][k] b[j][k], symmetric: tiles on and below the diagonal, mirrored when stored
// X, OUT:             C[i][j] = sum_k a[i][k] b[k][j]   (a = P, b = X)
enum { EPI_GRAM = 0, EPI_PART = 1, EPI_Q = 2, EPI_MUL = 3, EPI_X = 4, EPI_OUT = 5 };

// slots of a matrix's workspace region: X planes first (units of mp * np * 2 bytes), then m x m pairs of planes
__device__ __forceinline__ size_t slot_off(const NsClass& c, int xplanes, int slot) {
  const size_t px = (size_t)c.mp * c.np * 2, pm = (size_t)c.mp * c.mp * 2;
  return slot < xplanes ? (size_t)slot * px : (size_t)xplanes * px + (size_t)(slot - xplanes) * 2 * pm;
}

struct NsJob { int a, b, out; };        // slots
struct NsGemm {
  NsJob job[2];                         // MUL may do two products of one kind in a launch (blockIdx.z)
  int xplanes;                          // X slots of a region
  float unscale[2], scale[2];           // accumulator -> value, value -> planes
  float qa, qb, qc, sa_inv;             // EPI_Q: coefficients, 1 / scale of A's planes
  int res_pow;                          // GRAM: value *= residue^2;  OUT / X: value *= residue
  float lr, decay;                      // OUT of a Muon step
  int muon;
  float* part;                          // PART: [share][tile][T * T] accumulators;  cut tiles: [job][tile][share][T * T]
  int full, cut;                        // symmetric products in 128 x 128 tiles: tiles from `full` on run in `cut` shares of K each (1: none do)
};

// lower-triangular tile number t -> (row, column), row >= column
__device__ __forceinline__ void tri_tile(int t, int& r, int& q) {
  r = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
  while ((r + 1) * (r + 2) / 2 <= t) ++r;
  while (r * (r + 1) / 2 > t) --r;
  q = t - r * (r + 1) / 2;
}

// Where a lane's accumulators of one 32 x 32 block lie: element e at row 8 (e / 4) + 4 (lane / 32) + e % 4, column lane % 32.
// One block of a symmetric product at (r, q) -> both planes of the result: what lies on or below the diagonal, and its mirror image.  EXACTLY
// symmetric matrices are what keeps the recursion one of commuting factors: with the two halves rounded apart, an error across strong and
// weak directions grows by a^2 a step where a symmetric one does not grow at all (one strong direction over 1e-3: 15 % off after 5 steps).
// (A's elements of the block, EPI_Q, come from there too: four at a time)
struct NsOld { f16x4 h[4], l[4]; };
__device__ __forceinline__ NsOld ns_load_sym(const NsClass& c, const _Float16* A, int r, int q) {
  const int lane = threadIdx.x & 63;
  const size_t pm = (size_t)c.mp * c.mp;
  NsOld o;
  if (r >= c.mp || q >= c.mp || r < q) {
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) o.h[e4] = o.l[e4] = f16x4{0, 0, 0, 0};
    return o;
  }
  const _Float16* a = A + (size_t)(q + (lane & 31)) * c.mp + r + 4 * (lane >> 5);
#pragma unroll
  for (int e4 = 0; e4 < 4; ++e4) {
    o.h[e4] = *reinterpret_cast<const f16x4*>(a + 8 * e4);
    o.l[e4] = *reinterpret_cast<const f16x4*>(a + pm + 8 * e4);
  }
  return o;
}
template <int EPI>
__device__ __forceinline__ void ns_store_sym(const NsClass& c, const NsGemm& p, const NsOld& old, _Float16* out, int r, int q, float un, float scale, const f32x16& acc) {
  const int lane = threadIdx.x & 63;
  if (r >= c.mp || q >= c.mp || r < q) return;                // (blocks are 32 wide, mp is a multiple of 32; a block above the diagonal)
  const size_t pm = (size_t)c.mp * c.mp;
  q += lane & 31;
  r += 4 * (lane >> 5);
#pragma unroll
  for (int e4 = 0; e4 < 4; ++e4) {
    const int r0 = r + 8 * e4;
    f16x4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float val = acc[e4 * 4 + e] * un;
      _Float16* d = out + (size_t)(r0 + e) * c.mp + q;
      if (EPI == EPI_Q) val = p.qc * val + p.qb * (((float)old.h[e4][e] + (float)old.l[e4][e]) * p.sa_inv) + (r0 + e == q ? p.qa : 0.f);
      const float x = val * scale;
      h[e] = (_Float16)x;
      l[e] = (_Float16)(x - (float)h[e]);
      if (r0 + e >= q) {
        d[0] = h[e];
        d[pm] = l[e];
      }
    }
    _Float16* d = out + (size_t)q * c.mp + r0;
    if (r0 > q) {
      *reinterpret_cast<f16x4*>(d) = h;
      *reinterpret_cast<f16x4*>(d + pm) = l;
    } else {
#pragma unroll
      for (int e = 1; e < 4; ++e)
        if (r0 + e > q) {
          d[e] = h[e];
          d[pm + e] = l[e];
        }
    }
  }
}

// One T x T tile per workgroup of 4 waves.  T = 128: K steps of 32, the waves 2 x 2 on the tile.  T = 64 (few tiles): K steps of 64, each wave
// takes 16 of them for the WHOLE tile and the four sums are added at the end in order: an LDS read feeds as many matrix instructions as with
// T = 128 (32 x 32 a wave would be bound by LDS reads), and a barrier stands between 12 of them instead of 6.
// Global memory -> registers, D steps ahead (2; 4 in launches of at most a workgroup per CU, which then have all registers) -> LDS, two buffers, one barrier a step.  LDS images: rows of one K step for a, and for b in [j][k],
// 16-byte chunks permuted within the row; rows of T columns per k for b in [k][j], 32-byte segments permuted, read with the transposing LDS load
// (within 16 lanes, lane j receives 16-bit slot j % 4 of lanes j / 4 + 4 e): 4 k of one column.  The permutations keep every group of lanes that
// is served at once on different banks.
template <int T> __device__ __forceinline__ int chunk_at(int r, int ch) {          // byte of chunk ch of row r
  return T == 128 ? r * 64 + ((ch ^ ((r >> 2) & 3)) << 4) : r * 128 + ((ch ^ ((r >> 1) & 7)) << 4);
}
template <int T> __device__ __forceinline__ int segment_at(int k, int seg) {       // byte of 32-byte segment seg of row k
  return T == 128 ? k * 256 + ((seg ^ ((k & 3) << 1)) << 5) : k * 128 + ((seg ^ (k & 2)) << 5);
}
// k of a share of a cut tile
__host__ __device__ inline int ns_cut(int K, int cut) { return (K / 32 + cut - 1) / cut * 32; }
template <int EPI, int NA, int NB, int T, int D, typename OutT>
__global__ __launch_bounds__(256, D == 2 ? 2 : 1) void ns_gemm_kernel(NsClasses cs, NsGemm p, NsInline few, const NsItem* __restrict__ table,
                                                         const float* __restrict__ residue, unsigned char* __restrict__ ws) {
  constexpr bool SYM = EPI <= EPI_MUL, NN = EPI >= EPI_X;
  constexpr int KS = T == 128 ? 32 : 64;        // k a step
  constexpr int PL = T * KS * 2;                // bytes of one plane's tile
  constexpr int BUF = (NA + NB) * PL;
  __shared__ __attribute__((aligned(16))) unsigned char lds[T == 64 && 2 * BUF < 65536 ? 65536 : 2 * BUF];
  constexpr bool CUTS = T == 128 && SYM && EPI != EPI_PART;
  const bool cut = CUTS && (int)blockIdx.x >= p.full;
  const int bid = !CUTS ? xcd_remap(blockIdx.x, gridDim.x) : (cut ? p.full + (int)(blockIdx.x - p.full) / p.cut : xcd_remap(blockIdx.x, p.full));
  const NsClass c = find_class(cs, bid);
  const int local = bid - c.start, i = local / c.per, t = local - i * c.per;
  int tr, tc;
  if (SYM) tri_tile(t, tr, tc);
  else { tr = t / c.tn; tc = t - tr * c.tn; }
  unsigned char* base = ws + c.base + (size_t)i * c.stride;
  const int K = EPI <= EPI_PART ? c.np : c.mp;          // (a multiple of 32)
  const size_t plane_a = (size_t)c.mp * K, plane_b = NN ? (size_t)c.mp * c.np : (size_t)c.mp * K;
  const int z = EPI == EPI_MUL ? blockIdx.z : 0;
  const NsJob job = p.job[z];
  const _Float16* A = reinterpret_cast<const _Float16*>(base + slot_off(c, p.xplanes, job.a));
  const _Float16* B = reinterpret_cast<const _Float16*>(base + slot_off(c, p.xplanes, job.b));

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wr = wave >> 1, wc = wave & 1;
  int k0 = 0, k1 = K;
  if (EPI == EPI_PART) {
    k0 = blockIdx.y * c.ks;
    k1 = k0 + c.ks < K ? k0 + c.ks : K;
    if (k0 >= k1) return;                       // (shapes with fewer shares than the grid has: never read)
  }
  const int share = cut ? (int)(blockIdx.x - p.full) % p.cut : 0;
  if (cut) {
    const int ks = ns_cut(K, p.cut);
    k0 = share * ks;
    k1 = k0 + ks < K ? k0 + ks : K;
    if (k0 >= k1) return;                       // (never read)
  }
  const int steps = (k1 - k0 + KS - 1) / KS;
  // byte offsets of a thread's chunks from the tile's first element, and where they go in LDS
  constexpr int RC = KS / 8;                    // chunks a row
  unsigned oa[2], ob[2];
  int la[2], lb[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int e = tid + q * 256, r = e / RC, ch = e % RC;
    const int ia = tr * T + r < c.mp ? r : c.mp - 1 - tr * T;      // rows past the matrix: the last one again (never stored; tr * T < mp)
    oa[q] = (unsigned)(ia * K + ch * 8) * 2u;
    la[q] = chunk_at<T>(r, ch);
    if (NN) {
      const int kr = e / (T / 8), cc = e % (T / 8);
      const int col = tc * T + cc * 8 < c.np ? cc * 8 : 0;         // chunks past the matrix: the tile's first again (never stored)
      ob[q] = (unsigned)(kr * c.np + col) * 2u;
      lb[q] = segment_at<T>(kr, cc >> 1) + ((cc & 1) << 4);
    } else {
      const int ib = tc * T + r < c.mp ? r : c.mp - 1 - tc * T;
      ob[q] = (unsigned)(ib * K + ch * 8) * 2u;
      lb[q] = la[q];
    }
  }
  // Buffer loads: the moving base stays in scalar registers, and what lies past the end of a plane reads as zero (the last step of 64 where K is
  // an odd multiple of 32: what else it reads there is not used).  Offsets within a window stay below 2^31.
  size_t pa = ((size_t)tr * T * K + k0) * 2, pb = (NN ? (size_t)k0 * c.np + tc * T : (size_t)tc * T * K + k0) * 2;
  const size_t step_b = NN ? (size_t)KS * 2 * c.np : KS * 2;
  auto window = [](const _Float16* plane, size_t at, size_t bytes) {
    const size_t left = bytes - at;
    return __builtin_amdgcn_make_buffer_rsrc((void*)(reinterpret_cast<const unsigned char*>(plane) + at), 0, (int)(left < 0x7fffffff ? left : 0x7fffffff), 0x00020000);
  };
  u32x4 ra[D][NA][2], rb[D][NB][2];
  int fetched = 0;
  auto fetch = [&](int slot) {
#pragma unroll
    for (int z = 0; z < NA; ++z) {
      const auto w = window(A + z * plane_a, pa, plane_a * 2);
#pragma unroll
      for (int q = 0; q < 2; ++q) ra[slot][z][q] = __builtin_amdgcn_raw_buffer_load_b128(w, (int)oa[q], 0, 0);
    }
#pragma unroll
    for (int z = 0; z < NB; ++z) {
      const auto w = window(B + z * plane_b, pb, plane_b * 2);
#pragma unroll
      for (int q = 0; q < 2; ++q) rb[slot][z][q] = __builtin_amdgcn_raw_buffer_load_b128(w, (int)ob[q], 0, 0);
    }
    // (past the last step: that one again, in bounds and unused -- a fetch under a condition would make every wait one for all loads)
    const bool more = ++fetched < steps;
    pa += more ? KS * 2 : 0;
    pb += more ? step_b : 0;
  };
  f32x16 acc[2][2];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[u][v][e] = 0.f;

#pragma unroll
  for (int d = 0; d < D; ++d) {
    fetch(d);
    __builtin_amdgcn_sched_barrier(0);          // (in this order: the waits count)
  }
  NsOld old[EPI == EPI_Q && T == 128 ? 4 : 1];
  if (EPI == EPI_Q && T == 64) old[0] = ns_load_sym(c, A, tr * 64 + wr * 32, tc * 64 + wc * 32);
  // fragments of k 16 kk .. 16 kk + 15 of a step
  struct Frags { f16x8 a[NA][2], b[NB][2]; };
  auto read = [&](Frags& f, const unsigned char* buf, int kk) {
    const int ro = T == 128 ? wr * 64 : 0, qo = T == 128 ? wc * 64 : 0, ch = kk * 2 + (lane >> 5);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = ro + u * 32 + (lane & 31), q = qo + u * 32 + (lane & 31);
#pragma unroll
      for (int z = 0; z < NA; ++z) f.a[z][u] = *reinterpret_cast<const f16x8*>(buf + z * PL + chunk_at<T>(r, ch));
#pragma unroll
      for (int z = 0; z < NB; ++z) {
        if (NN) {
          // lanes 0-15 / 16-31: columns 0-15 / 16-31 of these 32, k 0-7; lanes 32-63: the same columns, k 8-15
          f16x4 half[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int kr = kk * 16 + 8 * (lane >> 5) + 4 * h + ((lane & 15) >> 2);
            half[h] = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(
                buf + (NA + z) * PL + segment_at<T>(kr, (qo + u * 32) / 16 + ((lane >> 4) & 1)) + ((lane & 3) << 3))));
          }
          f.b[z][u] = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
          f.b[z][u] = *reinterpret_cast<const f16x8*>(buf + (NA + z) * PL + chunk_at<T>(q, ch));
        }
      }
    }
  };
  auto multiply = [&](const Frags& f) {
    // X: the operands the other way round, so that a lane holds four consecutive columns of one row of the result
#define NS_MFMA(A_, B_, C_) (EPI == EPI_X ? __builtin_amdgcn_mfma_f32_32x32x16_f16(B_, A_, C_, 0, 0, 0) : __builtin_amdgcn_mfma_f32_32x32x16_f16(A_, B_, C_, 0, 0, 0))
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        if (NB == 2) acc[u][v] = NS_MFMA(f.a[0][u], f.b[NB - 1][v], acc[u][v]);
        if (NA == 2) acc[u][v] = NS_MFMA(f.a[NA - 1][u], f.b[0][v], acc[u][v]);
        acc[u][v] = NS_MFMA(f.a[0][u], f.b[0][v], acc[u][v]);
      }
#undef NS_MFMA
  };
  auto put = [&](int s, int slot) {
    unsigned char* buf = lds + (s & 1) * BUF;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int z = 0; z < NA; ++z) *reinterpret_cast<u32x4*>(buf + z * PL + la[q]) = ra[slot][z][q];
#pragma unroll
      for (int z = 0; z < NB; ++z) *reinterpret_cast<u32x4*>(buf + (NA + z) * PL + lb[q]) = rb[slot][z][q];
    }
    fetch(slot);
  };
  if constexpr (T == 128) {
    // LDS is read ahead of the matrix instructions by half a step: while those of one half run, the other half's operands arrive and the next
    // step's tiles are written.  (The last step writes and reads on, in bounds and unused.)
    static_assert(D == 2, "slots by the parity of the step");
    Frags f0, f1;
    auto step = [&](int s, int next) {
      const unsigned char *buf = lds + (s & 1) * BUF, *then = lds + ((s + 1) & 1) * BUF;
      read(f1, buf, 1);
      multiply(f0);
      put(s + 1, next);
      __syncthreads();
      read(f0, then, 0);
      multiply(f1);
    };
    put(0, 0);
    __syncthreads();
    read(f0, lds, 0);
    int s = 0;
    for (; s + 2 <= steps; s += 2) {
      step(s, 1);
      step(s + 1, 0);
    }
    if (s < steps) step(s, 1);
  } else {
    auto step = [&](int s, int slot) {
      put(s, slot);
      __syncthreads();
      if (k0 + s * KS + wave * 16 < k1) {
        Frags f;
        read(f, lds + (s & 1) * BUF, wave);
        multiply(f);
      }
    };
    int s = 0;
    for (; s + D <= steps; s += D) {
#pragma unroll
      for (int d = 0; d < D; ++d) step(s + d, d);
    }
#pragma unroll
    for (int d = 0; d < D - 1; ++d)
      if (s + d < steps) step(s + d, d);
  }

  // T = 64: the waves' sums through LDS; wave w goes on with block (w / 2, w % 2)
  f32x16 sum;
  if constexpr (T == 64) {
    __syncthreads();
    float4* x = reinterpret_cast<float4*>(lds);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4)
          x[((wave * 4 + u * 2 + v) * 4 + e4) * 64 + lane] = make_float4(acc[u][v][e4 * 4], acc[u][v][e4 * 4 + 1], acc[u][v][e4 * 4 + 2], acc[u][v][e4 * 4 + 3]);
    __syncthreads();
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      float4 a = x[(wave * 4 + e4) * 64 + lane];
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        const float4 b = x[((w * 4 + wave) * 4 + e4) * 64 + lane];
        a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
      }
      sum[e4 * 4] = a.x; sum[e4 * 4 + 1] = a.y; sum[e4 * 4 + 2] = a.z; sum[e4 * 4 + 3] = a.w;
    }
    __syncthreads();
  }
  // blocks of this wave: (number, row, column, accumulators)
  auto blocks = [&](auto&& f) {
    if constexpr (T == 64) {
      f(wave, tr * 64 + wr * 32, tc * 64 + wc * 32, sum);
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int v = 0; v < 2; ++v) f(wave * 4 + u * 2 + v, tr * 128 + wr * 64 + u * 32, tc * 128 + wc * 64 + v * 32, acc[u][v]);
    }
  };

  if constexpr (EPI == EPI_PART) {
    // [share][tile][block][e / 4][lane] float4: the pass that adds the shares has the same lanes
    blocks([&](int n, int, int, const f32x16& a) {
      float4* o = reinterpret_cast<float4*>(p.part) + (((size_t)blockIdx.y * gridDim.x + bid) * (T * T / 1024) + n) * 256 + lane;
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) o[e4 * 64] = make_float4(a[e4 * 4], a[e4 * 4 + 1], a[e4 * 4 + 2], a[e4 * 4 + 3]);
    });
    return;
  }
  if constexpr (CUTS) {
    if (cut) {
      const size_t tile = ((size_t)z * ((gridDim.x - p.full) / p.cut) + (bid - p.full)) * p.cut + share;
      blocks([&](int n, int, int, const f32x16& a) {
        float4* o = reinterpret_cast<float4*>(p.part) + (tile * 16 + n) * 256 + lane;
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) o[e4 * 64] = make_float4(a[e4 * 4], a[e4 * 4 + 1], a[e4 * 4 + 2], a[e4 * 4 + 3]);
      });
      return;
    }
  }
  const float scale = p.scale[z];
  float un = p.unscale[z];
  if (EPI != EPI_Q && EPI != EPI_MUL && p.res_pow) {
    const float rs = residue[c.first + i];
    un *= p.res_pow == 2 ? rs * rs : rs;
  }
  _Float16* out = reinterpret_cast<_Float16*>(base + slot_off(c, p.xplanes, job.out));
  if constexpr (SYM) {
    if (EPI == EPI_Q && T == 128) blocks([&](int n, int r, int q, const f32x16&) { old[EPI == EPI_Q && T == 128 ? n & 3 : 0] = ns_load_sym(c, A, r, q); });
    blocks([&](int n, int r, int q, const f32x16& a) { ns_store_sym<EPI>(c, p, old[EPI == EPI_Q && T == 128 ? n & 3 : 0], out, r, q, un, scale, a); });
  } else if constexpr (EPI == EPI_X) {
    // through LDS, one plane after the other: rows of T columns, 16-byte stores.  Lane: row lane % 32, columns 8 e4 + 4 (lane / 32) + 0 .. 3
    constexpr int PITCH = T + 8;
    _Float16* stage = reinterpret_cast<_Float16*>(lds);
    static_assert(sizeof(lds) >= (size_t)T * PITCH * 2, "a plane's tile fits");
    const size_t px = (size_t)c.mp * c.np;
#pragma unroll
    for (int z = 0; z < NB; ++z) {
      __syncthreads();
      blocks([&](int, int r, int q, const f32x16& a) {
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          f16x4 h;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = a[e4 * 4 + e] * un * scale;
            h[e] = (_Float16)x;
            if (z == 1) h[e] = (_Float16)(x - (float)h[e]);
          }
          *reinterpret_cast<f16x4*>(stage + (r - tr * T + (lane & 31)) * PITCH + q - tc * T + 8 * e4 + 4 * (lane >> 5)) = h;
        }
      });
      __syncthreads();
#pragma unroll
      for (int q = 0; q < T * T / 8 / 256; ++q) {
        const int e = tid + q * 256, r = e / (T / 8), cc = e % (T / 8) * 8;
        if (tr * T + r < c.mp && tc * T + cc < c.np)
          *reinterpret_cast<u32x4*>(out + z * px + (size_t)(tr * T + r) * c.np + tc * T + cc) = *reinterpret_cast<const u32x4*>(stage + r * PITCH + cc);
      }
    }
  } else {
    const NsItem it = ns_item(few, table, c.first + i);
    const bool tall = c.rows > c.cols;
    const float f = p.muon ? -p.lr * it.scale : 1.f;
    OutT* o = reinterpret_cast<OutT*>(it.p);
    // element (r, q) of [m][n]; four consecutive r of a lane are consecutive in memory where the matrix is tall
    auto place = [&](int r, int q) { return tall ? (size_t)q * c.cols + r : (size_t)r * c.cols + q; };
    // a Muon step's parameters are read before any is written: one wait for all of them (interleaved: 53 us in place of 37 for 3 x 512 x 4608)
    f32x16 was[T == 64 ? 1 : 4];
    if (p.muon) {
      blocks([&](int n, int r, int qb, const f32x16&) {
        f32x16& w = was[T == 64 ? 0 : n & 3];
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const int r0 = r + 8 * e4 + 4 * (lane >> 5), q = qb + (lane & 31);
          if (tall && r0 + 4 <= c.m && q < c.n) {
            float v[4];
            load4(o + place(r0, q), v);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e4 * 4 + e] = v[e];
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e4 * 4 + e] = r0 + e < c.m && q < c.n ? to_f(o[place(r0 + e, q)]) : 0.f;
          }
        }
      });
    }
    blocks([&](int n, int r, int qb, const f32x16& a) {
      const f32x16& w = was[T == 64 ? 0 : n & 3];
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int r0 = r + 8 * e4 + 4 * (lane >> 5), q = qb + (lane & 31);
        if (r0 >= c.m || q >= c.n) continue;
        float val[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) val[e] = a[e4 * 4 + e] * un * f + (p.muon ? w[e4 * 4 + e] * p.decay : 0.f);
        if (tall && r0 + 4 <= c.m) {
          store4(o + place(r0, q), val);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (r0 + e < c.m) o[place(r0 + e, q)] = from_f<OutT>(val[e]);
        }
      }
    });
  }
}

// number of shares of a class's Gram product
__device__ __forceinline__ int ns_shares(const NsClass& c) { return (c.np + c.ks - 1) / c.ks; }

// one block's share sums, in the order of the shares
template <int UNROLL> __device__ __forceinline__ f32x16 ns_share_sum(const float* part, int shares, size_t per_share, size_t at) {
  f32x16 a;
#pragma unroll
  for (int e = 0; e < 16; ++e) a[e] = 0.f;
  const float4* x = reinterpret_cast<const float4*>(part) + at * 256 + (threadIdx.x & 63);
#pragma unroll UNROLL
  for (int s = 0; s < shares; ++s) {
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const float4 v = x[(size_t)s * per_share * 256 + e4 * 64];
      a[e4 * 4] += v.x; a[e4 * 4 + 1] += v.y; a[e4 * 4 + 2] += v.z; a[e4 * 4 + 3] += v.w;
    }
  }
  return a;
}

// a split Gram product's shares -> A; one wave a block of 32 x 32
template <int T>
__global__ __launch_bounds__(64) void ns_fold_kernel(NsClasses cs, NsGemm p, int tiles, const float* __restrict__ residue, unsigned char* __restrict__ ws) {
  constexpr int NBL = T * T / 1024, SIDE = T / 32;
  const int bid = blockIdx.x / NBL, n = blockIdx.x % NBL;
  const NsClass c = find_class(cs, bid);
  const int local = bid - c.start, i = local / c.per, t = local - i * c.per;
  int tr, tc;
  tri_tile(t, tr, tc);
  // block n of a tile, as the product numbers them
  const int br = T == 64 ? n >> 1 : (n >> 3) * 2 + ((n >> 1) & 1), bc = T == 64 ? n & 1 : ((n >> 2) & 1) * 2 + (n & 1);
  static_assert(SIDE * SIDE == NBL, "blocks of a tile");
  const f32x16 a = ns_share_sum<4>(p.part, ns_shares(c), (size_t)tiles * NBL, (size_t)bid * NBL + n);
  const float rs = residue[c.first + i];
  _Float16* out = reinterpret_cast<_Float16*>(ws + c.base + (size_t)i * c.stride + slot_off(c, p.xplanes, p.job[0].out));
  ns_store_sym<EPI_GRAM>(c, p, NsOld(), out, tr * T + br * 32, tc * T + bc * 32, p.unscale[0] * (p.res_pow == 2 ? rs * rs : 1.f), p.scale[0], a);
}

// the shares of a product's cut tiles -> its result; one wave a block of 32 x 32
template <int EPI>
__global__ __launch_bounds__(64) void ns_cut_fold_kernel(NsClasses cs, NsGemm p, const float* __restrict__ residue, unsigned char* __restrict__ ws) {
  const int j = blockIdx.x >> 4, n = blockIdx.x & 15, bid = p.full + j, z = blockIdx.z;
  const NsClass c = find_class(cs, bid);
  const int local = bid - c.start, i = local / c.per, t = local - i * c.per;
  int tr, tc;
  tri_tile(t, tr, tc);
  const int r = tr * 128 + ((n >> 3) * 2 + ((n >> 1) & 1)) * 32, q = tc * 128 + (((n >> 2) & 1) * 2 + (n & 1)) * 32;
  const int K = EPI == EPI_GRAM ? c.np : c.mp, ks = ns_cut(K, p.cut);
  unsigned char* base = ws + c.base + (size_t)i * c.stride;
  NsOld old;
  if (EPI == EPI_Q) old = ns_load_sym(c, reinterpret_cast<const _Float16*>(base + slot_off(c, p.xplanes, p.job[z].a)), r, q);
  const f32x16 a = ns_share_sum<4>(p.part, (K + ks - 1) / ks, 16, ((size_t)z * (gridDim.x >> 4) + j) * p.cut * 16 + n);
  float un = p.unscale[z];
  if (EPI == EPI_GRAM && p.res_pow) un *= residue[c.first + i] * residue[c.first + i];
  ns_store_sym<EPI>(c, p, old, reinterpret_cast<_Float16*>(base + slot_off(c, p.xplanes, p.job[z].out)), r, q, un, p.scale[z], a);
}

// ---- the recursion of a whole segment on one CU, for matrices of at most 32 MT rows ---------------------------------------------------
// Wave (I, J) = (wave / MT, wave % MT) holds its 32 x 32 block of A, P and what it multiplies next in registers; LDS holds the planes of
// the two operands of the product at hand (all symmetric: C[i][j] = sum_k x[i][k] y[j][k]).  In place of 3 to 5 launches a step.
// The matrices are kept EXACTLY symmetric (ns_store_sym says why).  Blocks (I, J) and (J, I) are the same sums in the same order with the
// operands of the matrix instructions exchanged, a block on the diagonal is the mean of its product and the exchanged one: so every wave
// writes its block alone, four elements (r0 .. r0 + 3, q) as one access at row q, columns r0 .. r0 + 3.
struct NsRecStep {                      // one step: factors from a product's sums to what is stored, plane scales (powers of two) in them
  float g, ia, a;                       // Q = g (A A)' + ia A' + a
  float fP, fT, fA;                     // P = fP (Q P)',  T = fT (Q A)',  next A = fA (Q T)'
  float sP, pad;                        // planes of P where it is the segment's last step
};
struct NsRec {
  int steps, xplanes, out;              // of this segment; slot of P
  float unscale;                        // share sums -> A
  int res_pow;
  const float* part;
  float sA[NS_MAX_STEPS];               // planes of A where a segment begins
  NsRecStep step[NS_MAX_STEPS];
};
template <int MT> struct NsOnCu {
  static constexpr int ROW = 64 * MT, PL = 32 * MT * ROW, SLOT = 2 * PL;      // bytes of a row, a plane, both planes
  unsigned char* lds;                   // two slots
  int mp, lane, I, J;
  bool inside;                          // this wave has a block (mp is a multiple of 32); the others only wait
  int mine[4];
  // 16-byte chunk ch of row r
  static __device__ __forceinline__ int at(int r, int ch) { return r * ROW + ((MT == 2 ? ch ^ ((r >> 1) & 7) : ch ^ (r & 15)) << 4); }
  static __device__ __forceinline__ int elem(int r, int q) { return at(r, q >> 3) + (q & 7) * 2; }
  __device__ __forceinline__ NsOnCu(unsigned char* lds_, int mp_, int wave, int lane_) : lds(lds_), mp(mp_), lane(lane_), I(wave / MT), J(wave % MT) {
    inside = I < MT && I * 32 < mp && J * 32 < mp;
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) mine[e4] = elem(J * 32 + (lane & 31), (I < MT ? I : 0) * 32 + 8 * e4 + 4 * (lane >> 5));
  }
  __device__ __forceinline__ void put(int slot, const f32x16& v) {
    unsigned char* at0 = lds + slot * SLOT;
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      f16x4 h, l;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        h[e] = (_Float16)v[e4 * 4 + e];
        l[e] = (_Float16)(v[e4 * 4 + e] - (float)h[e]);
      }
      *reinterpret_cast<f16x4*>(at0 + mine[e4]) = h;
      *reinterpret_cast<f16x4*>(at0 + PL + mine[e4]) = l;
    }
  }
  // Products, KT times 16 along k: WHERE 0 a block on the diagonal, 1 below, 2 above it.  hi lo, lo hi, hi hi; above the
  // diagonal with the operands exchanged -- the same sum in the same order as its mirror image's.  On the diagonal: the sum of the product
  // and of the exchanged one (2 C: f below makes up for it).
  template <int WHERE, int KT, typename X, typename Y> static __device__ __forceinline__ f32x16 sums(const X& x, const Y& y) {
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    f32x16 turned = acc;
#pragma unroll(MT == 2 ? KT : 2)
    for (int k = 0; k < KT; ++k) {
      const f16x8 xh = x.hi(k), xl = x.lo(k), yh = y.hi(k), yl = y.lo(k);
      if (WHERE == 2) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(yl, xh, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(yh, xl, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(yh, xh, acc, 0, 0, 0);
        continue;
      }
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(xh, yl, acc, 0, 0, 0);
      if (WHERE == 0) turned = __builtin_amdgcn_mfma_f32_32x32x16_f16(yl, xh, turned, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(xl, yh, acc, 0, 0, 0);
      if (WHERE == 0) turned = __builtin_amdgcn_mfma_f32_32x32x16_f16(yh, xl, turned, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(xh, yh, acc, 0, 0, 0);
      if (WHERE == 0) turned = __builtin_amdgcn_mfma_f32_32x32x16_f16(yh, xh, turned, 0, 0, 0);
    }
    if (WHERE == 0) {
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[e] += turned[e];
    }
    return acc;
  }
  // fragments of 32 rows of an operand: in LDS, or in registers (what several products share is read once)
  struct Lds {
    const unsigned char* x;
    int row, half;
    __device__ __forceinline__ f16x8 hi(int k) const { return *reinterpret_cast<const f16x8*>(x + at(row, 2 * k + half)); }
    __device__ __forceinline__ f16x8 lo(int k) const { return *reinterpret_cast<const f16x8*>(x + PL + at(row, 2 * k + half)); }
  };
  template <int KT> struct Regs {
    f16x8 h[KT], l[KT];
    __device__ __forceinline__ f16x8 hi(int k) const { return h[k]; }
    __device__ __forceinline__ f16x8 lo(int k) const { return l[k]; }
  };
  __device__ __forceinline__ Lds rows_of(int slot, int u) const { return Lds{lds + slot * SLOT, u * 32 + (lane & 31), lane >> 5}; }
  // this wave's block of x y, times f: from the rows max(I, J) of x and min(I, J) of y
  template <int KT, typename X> __device__ __forceinline__ f32x16 product(const X& x, int y, float f) const {
    const Lds l = rows_of(y, I < J ? I : J);
    f32x16 r;
    if (I == J) r = sums<0, KT>(x, l);
    else if (I > J) r = sums<1, KT>(x, l);
    else r = sums<2, KT>(x, l);
    if (I == J) f *= 0.5f;
#pragma unroll
    for (int e = 0; e < 16; ++e) r[e] *= f;
    return r;
  }
  // block (bi, bj) of a Gram product, on or below the diagonal, with its mirror image -> slot 0; on the diagonal what lies above it from below
  __device__ __forceinline__ void put_gram(const f32x16& v, float s, int bi, int bj) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int r = bi * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3), q = bj * 32 + (lane & 31);
      const float x = v[e] * s;
      const _Float16 h = (_Float16)x, l = (_Float16)(x - (float)h);
      if (r >= q) {
        *reinterpret_cast<_Float16*>(lds + elem(r, q)) = h;
        *reinterpret_cast<_Float16*>(lds + PL + elem(r, q)) = l;
        *reinterpret_cast<_Float16*>(lds + elem(q, r)) = h;
        *reinterpret_cast<_Float16*>(lds + PL + elem(q, r)) = l;
      }
    }
  }
  // steps first .. last from A in slot 0 (a barrier has been passed since it was written) -> this wave's block of P, times its planes'
  // scale.  Every thread of the workgroup calls it.  Slot 1 is read until its end.
  __device__ __forceinline__ f32x16 run(const NsRec& p, int first, int last) {
    if constexpr (MT == 2) return run_k<4>(p, first, last);          // (mp = 32: ns_rec_one)
    else return mp == 32 * MT ? run_k<2 * MT>(p, first, last) : run_k<2 * MT - 2>(p, first, last);
  }
  template <int KT> __device__ __forceinline__ f32x16 run_k(const NsRec& p, int first, int last) {
    const int u = I < J ? J : I;
    f32x16 P, V, tq;
    for (int s = first; s <= last; ++s) {
      const NsRecStep d = p.step[s];                     // (fetched at once, ahead of the products)
      if (inside) {
        V = product<KT>(rows_of(0, u), 0, d.g);
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const f16x4 h = *reinterpret_cast<const f16x4*>(lds + mine[e4]), l = *reinterpret_cast<const f16x4*>(lds + PL + mine[e4]);
#pragma unroll
          for (int e = 0; e < 4; ++e) V[e4 * 4 + e] = __fmaf_rn(d.ia, (float)h[e], __fmaf_rn(d.ia, (float)l[e], V[e4 * 4 + e]));
        }
        if (I == J) {
#pragma unroll
          for (int e = 0; e < 16; ++e) V[e] += 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3) == (lane & 31) ? d.a : 0.f;
        }
        put(1, V);                      // (slot 1 is free: its last readers have passed a barrier since)
      }
      __syncthreads();
      const Lds ql = rows_of(1, u);
      Regs<KT> qr;                      // (16 waves have no registers for it)
      if (MT == 2 && inside) {
#pragma unroll
        for (int k = 0; k < KT; ++k) { qr.h[k] = ql.hi(k); qr.l[k] = ql.lo(k); }
      }
      auto with_q = [&](float f) { return MT == 2 ? product<KT>(qr, 0, f) : product<KT>(ql, 0, f); };
      if (s < last && inside) tq = with_q(d.fT);         // Q A
      if (s == first) {
        P = V;
      } else {
        __syncthreads();
        if (inside) put(0, P);
        __syncthreads();
        if (inside) P = with_q(d.fP);
      }
      if (s == last) break;
      __syncthreads();
      if (inside) put(0, tq);
      __syncthreads();
      if (inside) V = with_q(d.fA);                      // Q (Q A)
      __syncthreads();
      if (inside) put(0, V);
      __syncthreads();
    }
    return P;
  }
};

// ---- the same for at most 32 rows: one wave, everything in its registers and in fp32 ---------------------------------------------------------
// Planes of 22 bits, whose rounding acts on whole rows of Q and P, left results of so few rows further off than a plain fp32 iteration is (16 x 300
// 2.3e-6 of the norm, so 1.3e-6, for 1.0e-6).  The fp32 matrix instructions take 1024 cycles a product, and no operand has to be moved: of a symmetric
// matrix, element e of a lane (row 8 (e / 4) + 4 (lane / 32) + e % 4, column lane % 32) is both what the lane has to bring as left operand (that
// column's row, that row's column) and as right operand, with k running over the rows in the order of e.
__device__ __forceinline__ f32x16 ns_product_one(const f32x16& x, const f32x16& y) {
  f32x16 r;
#pragma unroll
  for (int e = 0; e < 16; ++e) r[e] = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) r = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], r, 0, 0, 0);
  return r;
}
// f times the mean of v and its transpose, exactly symmetric; through 32 x 33 floats of LDS that no other wave uses
__device__ __forceinline__ f32x16 ns_symmetric_one(const f32x16& v, float f, float* t) {
  const int lane = threadIdx.x & 63, q = lane & 31, h = 4 * (lane >> 5);
#pragma unroll
  for (int e = 0; e < 16; ++e) t[(8 * (e >> 2) + h + (e & 3)) * 33 + q] = v[e];
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  f32x16 r;
  f *= 0.5f;
#pragma unroll
  for (int e = 0; e < 16; ++e) r[e] = (v[e] + t[q * 33 + 8 * (e >> 2) + h + (e & 3)]) * f;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  return r;
}
// steps first .. last from the sums A (times `un`) of a segment's first product -> P, times its planes' scale
__device__ __forceinline__ f32x16 ns_rec_one(const NsRec& p, int first, int last, const f32x16& sums, float un, float* t) {
  const int lane = threadIdx.x & 63;
  f32x16 A = ns_symmetric_one(sums, un * p.sA[first], t), P;
  for (int s = first; s <= last; ++s) {
    const NsRecStep d = p.step[s];
    f32x16 Q = ns_product_one(A, A);                     // (x y summed in the order of y x: symmetric as it is)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      Q[e] = __fmaf_rn(d.g, Q[e], d.ia * A[e]);
      Q[e] += 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3) == (lane & 31) ? d.a : 0.f;
    }
    P = s == first ? Q : ns_symmetric_one(ns_product_one(Q, P), d.fP, t);
    if (s < last) {
      const f32x16 T = ns_symmetric_one(ns_product_one(Q, A), d.fT, t);
      A = ns_symmetric_one(ns_product_one(Q, T), d.fA, t);
    }
  }
  return P;
}

template <int MT>
__global__ __launch_bounds__(MT == 2 ? 512 : 1024) void ns_rec_kernel(NsClasses cs, NsRec p, int tiles, const float* __restrict__ residue, unsigned char* __restrict__ ws) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[2 * NsOnCu<MT>::SLOT];
  const NsClass c = find_class(cs, blockIdx.x);
  const int i = blockIdx.x - c.start;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  NsOnCu<MT> m(lds, c.mp, wave, lane);
  const int I = m.I, J = m.J;
  const bool lower = m.inside && J <= I;
  const float rs = residue[c.first + i];
  const float un = p.unscale * (p.res_pow == 2 ? rs * rs : 1.f);
  f32x16 V;
  if (MT == 2) {
    // one tile, often many shares: two groups of waves add a part of their block's each; of 32 rows, which have one block, all eight
    const int nb = c.mp > 32 ? 4 : 1, groups = 8 / nb, blk = wave % nb, group = wave / nb;
    const int n = ns_shares(c), each = (n + groups - 1) / groups, from = group * each;
    const size_t per_share = (size_t)tiles * 4, first = ((size_t)c.tn + (size_t)i * c.per) * 4 + blk;
    V = ns_share_sum<8>(p.part + (size_t)from * per_share * 1024, n - from < each ? n - from : each, per_share, first);
    float4* x = reinterpret_cast<float4*>(lds) + blk * 256 + lane;
    if (group > 0) {
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) x[(group - 1) * nb * 256 + e4 * 64] = make_float4(V[e4 * 4], V[e4 * 4 + 1], V[e4 * 4 + 2], V[e4 * 4 + 3]);
    }
    __syncthreads();
    if (lower) {
      for (int q = 0; q < groups - 1; ++q)
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const float4 v = x[q * nb * 256 + e4 * 64];
          V[e4 * 4] += v.x; V[e4 * 4 + 1] += v.y; V[e4 * 4 + 2] += v.z; V[e4 * 4 + 3] += v.w;
        }
    }
    __syncthreads();
  } else if (lower) {                  // A from the shares of the 64 x 64 tiles on and below the diagonal
    const int t = (I >> 1) * ((I >> 1) + 1) / 2 + (J >> 1);
    V = ns_share_sum<2>(p.part, ns_shares(c), (size_t)tiles * 4, ((size_t)c.tn + (size_t)i * c.per + t) * 4 + (I & 1) * 2 + (J & 1));
  }
  f32x16 P;
  if (MT == 2 && c.mp == 32) {
    if (!m.inside) return;              // (one wave has a block)
    P = ns_rec_one(p, 0, p.steps - 1, V, un, reinterpret_cast<float*>(lds));
  } else {
    if (lower) {
#pragma unroll
      for (int e = 0; e < 16; ++e) V[e] *= un;
      m.put_gram(V, p.sA[0], I, J);
    }
    __syncthreads();
    P = m.run(p, 0, p.steps - 1);
    if (!m.inside) return;
  }
  _Float16* out = reinterpret_cast<_Float16*>(ws + c.base + (size_t)i * c.stride + slot_off(c, p.xplanes, p.out));
  const size_t pm = (size_t)c.mp * c.mp;
#pragma unroll
  for (int e4 = 0; e4 < 4; ++e4) {
    f16x4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = P[e4 * 4 + e];
      h[e] = (_Float16)x;
      l[e] = (_Float16)(x - (float)h[e]);
    }
    _Float16* d = out + (size_t)(J * 32 + (lane & 31)) * c.mp + I * 32 + 8 * e4 + 4 * (lane >> 5);
    *reinterpret_cast<f16x4*>(d) = h;
    *reinterpret_cast<f16x4*>(d + pm) = l;
  }
}

// ---- P X for matrices of at most 64 rows: X's planes, and the shares of the NEXT segment's Gram product; or the result ----------------------
// A wave takes all rows of 64 columns at a time, in LDS of its own (no barrier): [row][64] per plane, chunks permuted as in the products (chunk_at).
// P's fragments stay in registers, X's come through the transposing LDS load, the result goes back in place, from there to memory in rows of 128
// bytes and, K being columns now, into the Gram product's sums: a launch less a segment, and no tiles of 64 rows for matrices of 32.  5 steps of
// 4 x 21 x 18432 fp32 121 -> 78 us (74 with the recursion in fp32), of 32 x 2304 x 64 110 -> 102, of 1 x 64 x 576 64 either way.
struct NsSlim {
  int xplanes, p, x, out;               // slots
  float unscale, scale;                 // sums -> value;  value -> planes
  int use_res;                          // value *= residue
  float lr, decay;
  int muon;
  float* part;                          // [share][matrix][4 blocks][1024]
  int matrices;
};
template <int NP> constexpr int NS_SLIM_X = 4 * NP * 64 * 128;      // bytes of LDS: columns of four waves
constexpr int NS_SLIM_P = 2 * 64 * 128;                              // P
template <int NP, int MT, bool LAST, typename T>
__device__ __forceinline__ void ns_slim_rows(const NsClass& c, const NsSlim& p, const NsItem& it, const float* __restrict__ residue, unsigned char* __restrict__ ws,
                                             unsigned char* lds, int i, int share) {
  static_assert(LAST || NP == 2, "a single plane has one segment");
  constexpr int PL = 64 * 128;          // a plane of a wave's columns
  constexpr int mp = 32 * MT;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5;
  unsigned char *base = ws + c.base + (size_t)i * c.stride, *x = lds + wave * NP * PL, *lp = lds + NS_SLIM_X<NP>;
  const size_t px = (size_t)mp * c.np, pm = (size_t)mp * mp;
  const _Float16* X = reinterpret_cast<const _Float16*>(base + slot_off(c, p.xplanes, p.x));
  const _Float16* P = reinterpret_cast<const _Float16*>(base + slot_off(c, p.xplanes, p.p));
  _Float16* out = reinterpret_cast<_Float16*>(base + slot_off(c, p.xplanes, p.out));
  const float un = p.unscale * (p.use_res ? residue[c.first + i] : 1.f);
  const bool tall = c.rows > c.cols;

  // P -> LDS, both planes: 16-byte chunks
#pragma unroll
  for (int e = 0; e < MT * MT; ++e) {
    const int n = threadIdx.x + e * 256, z = n / (mp * mp / 8), r = n % (mp * mp / 8) / (mp / 8), ch = n % (mp / 8);
    *reinterpret_cast<u32x4*>(lp + z * PL + chunk_at<64>(r, ch)) = *reinterpret_cast<const u32x4*>(P + z * pm + (size_t)r * mp + ch * 8);
  }
  __syncthreads();
  f32x16 gram[MT == 2 ? 3 : 1];
#pragma unroll
  for (int b = 0; b < (MT == 2 ? 3 : 1); ++b)
#pragma unroll
    for (int e = 0; e < 16; ++e) gram[b][e] = 0.f;

  const int end = (share + 1) * c.ks < c.np ? (share + 1) * c.ks : c.np;
  for (int col = share * c.ks + wave * 64; col < end; col += 256) {
    // columns -> LDS; eight rows of 128 bytes at a time, zero behind the last column (np is a multiple of 32)
    const int lr = lane >> 3, ch = lane & 7;
    const bool in = col + ch * 8 < c.np;
    u32x4 g[NP][4 * MT];
#pragma unroll
    for (int z = 0; z < NP; ++z)
#pragma unroll
      for (int k = 0; k < 4 * MT; ++k) {
        g[z][k] = u32x4{0u, 0u, 0u, 0u};
        if (in) g[z][k] = *reinterpret_cast<const u32x4*>(X + z * px + (size_t)(k * 8 + lr) * c.np + col + ch * 8);
      }
#pragma unroll
    for (int z = 0; z < NP; ++z)
#pragma unroll
      for (int k = 0; k < 4 * MT; ++k)
        *reinterpret_cast<u32x4*>(x + z * PL + chunk_at<64>(k * 8 + lr, ch)) = g[z][k];
#pragma unroll
    for (int cb = 0; cb < 2; ++cb) {
      f32x16 y[MT];
#pragma unroll
      for (int v = 0; v < MT; ++v)
#pragma unroll
        for (int e = 0; e < 16; ++e) y[v][e] = 0.f;
#pragma unroll
      for (int k = 0; k < 2 * MT; ++k) {
        f16x8 xf[NP];
#pragma unroll
        for (int z = 0; z < NP; ++z) {
          f16x4 half[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int kr = k * 16 + 8 * hi + 4 * h + ((lane & 15) >> 2), q = cb * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
            half[h] = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(x + z * PL + chunk_at<64>(kr, q >> 3) + (q & 7) * 2)));
          }
          xf[z] = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
#pragma unroll
        for (int v = 0; v < MT; ++v) {
          const int o = chunk_at<64>(v * 32 + (lane & 31), 2 * k + hi);
          const f16x8 ph = *reinterpret_cast<const f16x8*>(lp + o), pl = *reinterpret_cast<const f16x8*>(lp + PL + o);
          if (NP == 2) y[v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xf[NP - 1], ph, y[v], 0, 0, 0);
          y[v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xf[0], pl, y[v], 0, 0, 0);
          y[v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xf[0], ph, y[v], 0, 0, 0);
        }
      }
      // a lane: row 32 v + lane % 32, columns 32 cb + 8 e4 + 4 (lane / 32) + 0 .. 3
      if constexpr (!LAST) {
#pragma unroll
        for (int v = 0; v < MT; ++v) {
#pragma unroll
          for (int e4 = 0; e4 < 4; ++e4) {
            f16x4 h, l;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float w = y[v][e4 * 4 + e] * un * p.scale;
              h[e] = (_Float16)w;
              l[e] = (_Float16)(w - (float)h[e]);
            }
            const int q = cb * 32 + 8 * e4 + 4 * hi, o = chunk_at<64>(v * 32 + (lane & 31), q >> 3) + (q & 7) * 2;
            *reinterpret_cast<f16x4*>(x + o) = h;
            *reinterpret_cast<f16x4*>(x + PL + o) = l;
          }
        }
      } else {
        T* o = reinterpret_cast<T*>(it.p);
        const float f = p.muon ? -p.lr * it.scale : 1.f;
        auto place = [&](int r, int q) { return tall ? (size_t)q * c.cols + r : (size_t)r * c.cols + q; };
        float was[MT][16];               // a Muon step's parameters: all read before any is written
#pragma unroll
        for (int v = 0; v < MT; ++v)
#pragma unroll
          for (int e4 = 0; e4 < 4; ++e4) {
            const int r = v * 32 + (lane & 31), q = col + cb * 32 + 8 * e4 + 4 * hi;
#pragma unroll
            for (int e = 0; e < 4; ++e) was[v][e4 * 4 + e] = 0.f;
            if (!p.muon || r >= c.m || q >= c.n) continue;
            if (!tall && q + 4 <= c.n) {
              load4(o + place(r, q), &was[v][e4 * 4]);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (q + e < c.n) was[v][e4 * 4 + e] = to_f(o[place(r, q + e)]);
            }
          }
#pragma unroll
        for (int v = 0; v < MT; ++v)
#pragma unroll
          for (int e4 = 0; e4 < 4; ++e4) {
            const int r = v * 32 + (lane & 31), q = col + cb * 32 + 8 * e4 + 4 * hi;
            if (r >= c.m || q >= c.n) continue;
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = y[v][e4 * 4 + e] * un * f + (p.muon ? was[v][e4 * 4 + e] * p.decay : 0.f);
            if (!tall && q + 4 <= c.n) {
              store4(o + place(r, q), w);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (q + e < c.n) o[place(r, q + e)] = from_f<T>(w[e]);
            }
          }
      }
    }
    if constexpr (!LAST) {
#pragma unroll
      for (int z = 0; z < NP; ++z)
#pragma unroll
        for (int k = 0; k < 4 * MT; ++k)
          if (in)
            *reinterpret_cast<u32x4*>(out + z * px + (size_t)(k * 8 + lr) * c.np + col + ch * 8) = *reinterpret_cast<const u32x4*>(x + z * PL + chunk_at<64>(k * 8 + lr, ch));
#pragma unroll
      for (int k = 0; k < 4; ++k) {      // 64 columns
        f16x8 r[MT][NP];
#pragma unroll
        for (int v = 0; v < MT; ++v)
#pragma unroll
          for (int z = 0; z < NP; ++z)
            r[v][z] = *reinterpret_cast<const f16x8*>(x + z * PL + chunk_at<64>(v * 32 + (lane & 31), 2 * k + hi));
#pragma unroll
        for (int b = 0; b < (MT == 2 ? 3 : 1); ++b) {
          const int bi = b > 0, bj = b == 2;
          gram[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(r[bi][0], r[bj][NP - 1], gram[b], 0, 0, 0);
          gram[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(r[bi][NP - 1], r[bj][0], gram[b], 0, 0, 0);
          gram[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(r[bi][0], r[bj][0], gram[b], 0, 0, 0);
        }
      }
    }
  }
  if constexpr (!LAST) {
    // the waves' sums, in order; wave w the blocks (0, 0), (1, 0), (1, 1)
    __syncthreads();
    float4* sum = reinterpret_cast<float4*>(lds);
#pragma unroll
    for (int b = 0; b < (MT == 2 ? 3 : 1); ++b)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) sum[((wave * 3 + b) * 4 + e4) * 64 + lane] = make_float4(gram[b][e4 * 4], gram[b][e4 * 4 + 1], gram[b][e4 * 4 + 2], gram[b][e4 * 4 + 3]);
    __syncthreads();
    if (wave < (MT == 2 ? 3 : 1)) {
      float4* o = reinterpret_cast<float4*>(p.part) + (((size_t)share * p.matrices + c.first + i) * 4 + (wave == 0 ? 0 : wave + 1)) * 256 + lane;
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        float4 a = sum[(wave * 4 + e4) * 64 + lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
          const float4 b = sum[((w * 3 + wave) * 4 + e4) * 64 + lane];
          a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
        }
        o[e4 * 64] = a;
      }
    }
  }
}
template <int NP, bool LAST, typename T>
__global__ __launch_bounds__(256, 2) void ns_slim_kernel(NsClasses cs, NsSlim p, NsInline few, const NsItem* __restrict__ table,
                                                         const float* __restrict__ residue, unsigned char* __restrict__ ws) {
  constexpr int BYTES = NS_SLIM_X<NP> + NS_SLIM_P;
  __shared__ __attribute__((aligned(16))) unsigned char lds[BYTES < 49152 ? 49152 : BYTES];
  const NsClass c = find_class(cs, blockIdx.x);
  const int local = blockIdx.x - c.start, i = local / c.per, share = local - i * c.per;
  const NsItem it = ns_item(few, table, c.first + i);
  if (c.mp == 32) ns_slim_rows<NP, 1, LAST, T>(c, p, it, residue, ws, lds, i, share);
  else ns_slim_rows<NP, 2, LAST, T>(c, p, it, residue, ws, lds, i, share);
}

// ---- matrices that fit one CU's LDS whole: norm, all steps and the update in ONE launch, a workgroup of 8 waves a matrix ----------------------
// At most 64 on the smaller side, 448 (bf16: 384) on the other.  X lives in LDS as planes [mp][pitch]: 16-byte chunk ch of row r at
// ch ^ ((r >> 2) & 3), a pitch of an odd number of 64 bytes -- 16 rows of one chunk, and the four rows of a transposing read, lie on different
// banks.  The products are the ones of the larger matrices; only what is moved differs.
// Measured, this against the launches of the larger ones (5 steps, us): fp32 64 x 147 34 / 61, 64 x 448 56 / 63 (what LDS holds);
// bf16 64 x 256 34 / 39, 64 x 384 40 / 40, 64 x 448 43 / 40: the limits.  What bounds it is one CU's chain of small products
// (1 us each: 24 matrix instructions of 32 cycles on the diagonal, 512 cycles of LDS reads, the split into planes, two barriers).
template <int NP> constexpr int NS_TINY_N = NP == 2 ? 448 : 384;
__host__ __device__ inline int ns_tiny_pitch(int np) { return np * 2 + (np & 32 ? 0 : 64); }
struct NsTiny {
  NsRec rec;                            // scales and coefficients of all steps
  unsigned ends;                        // bit s: step s ends a segment
  float sx[NS_MAX_STEPS + 1];           // scale of X's planes where a segment begins with step s
  float eps, lr, decay;
  int muon;
};
// ONE: at most 32 rows (a kernel of its own: in the other's registers its recursion cost that one 2 %)
template <typename T, int NP, bool ONE>
__global__ __launch_bounds__(512) void ns_tiny_kernel(NsClasses cs, NsTiny p, NsInline few, const NsItem* __restrict__ table, MuonArgs ma) {
  constexpr int XB = 64 * (NS_TINY_N<NP> * 2 + 64);             // bytes of one plane of X at most
  constexpr int GROUPS = 64 * NS_TINY_N<NP> / 4 / 512;          // fours of elements a thread holds at most
  __shared__ __attribute__((aligned(16))) unsigned char x[NP * XB];
  __shared__ __attribute__((aligned(16))) unsigned char lds[2 * NsOnCu<2>::SLOT];
  __shared__ double sh[8];
  const NsClass c = find_class(cs, blockIdx.x);
  const int i = blockIdx.x - c.start;
  const NsItem it = ns_item(few, table, c.first + i);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int pitch = ns_tiny_pitch(c.np), plane = c.mp * pitch;
  auto xat = [&](int r, int q) { return r * pitch + (((q >> 3) ^ ((r >> 2) & 3)) << 4) + (q & 7) * 2; };
  const T* g = reinterpret_cast<const T*>(it.g);
  const bool tall = c.rows > c.cols;

  // momentum, update and its norm; the update stays in registers
  // fours of a line, 512 further each time (no division a step)
  const int per_line = (c.cols + 3) >> 2, lines = 512 / per_line, fours = 512 - lines * per_line;
  const int line0 = tid / per_line, four0 = tid - line0 * per_line;
  float u[GROUPS][4];
  double s = 0.0;
  int line = line0, four = four0;
  auto next = [&]() {
    line += lines;
    four += fours;
    if (four >= per_line) { four -= per_line; ++line; }
  };
#pragma unroll
  for (int k = 0; k < GROUPS; ++k, next()) {
#pragma unroll
    for (int e = 0; e < 4; ++e) u[k][e] = 0.f;
    if (line < c.rows) {
      const int col = four * 4;
      const long at = (long)line * c.cols + col;
      if (col + 4 <= c.cols) {
        load4(g + at, u[k]);
        if (it.mom != nullptr) {
          float m[4];
          load4(it.mom + at, m);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            m[e] = muon_momentum(m[e], u[k][e], ma);
            u[k][e] = muon_update(m[e], u[k][e], ma);
          }
          store4(it.mom + at, m);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < c.cols) {
            float v = to_f(g[at + e]);
            if (it.mom != nullptr) {
              const float m = muon_momentum(it.mom[at + e], v, ma);
              it.mom[at + e] = m;
              v = muon_update(m, v, ma);
            }
            u[k][e] = v;
          }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s += (double)u[k][e] * u[k][e];
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane == 0) sh[wave] = s;
  for (int e = tid * 16; e < NP * plane; e += 512 * 16) *reinterpret_cast<uint4*>(x + e) = make_uint4(0u, 0u, 0u, 0u);     // the padding
  __syncthreads();
  double square = 0.0;
#pragma unroll
  for (int w = 0; w < 8; ++w) square += sh[w];
  const double norm = fmax(sqrt(square), (double)p.eps);
  double mul;
  float left = 1.f;
  if (NP == 2) {
    mul = (double)p.sx[0] / norm;
  } else {
    int e;
    frexp(norm, &e);
    mul = ldexp((double)p.sx[0], -e);
    left = (float)(ldexp(1.0, e) / norm);
  }
  if (!(square < HUGE_VAL)) mul = nan("");                  // a NaN or an infinity in the matrix: all of its result is NaN
  // (in 32 bits where they hold the factor: 2^-24 of a common factor; 64-bit operations run at half their rate)
  const float mf = (float)mul;
  const bool narrow = mf >= 1.2e-38f && mf <= 3e38f;
  line = line0;
  four = four0;
#pragma unroll
  for (int k = 0; k < GROUPS; ++k, next()) {
    if (line < c.rows) {
      const int col = four * 4;
      f16x4 h, l;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = narrow ? u[k][e] * mf : (float)((double)u[k][e] * mul);     // (0 behind a line's end: padding)
        h[e] = (_Float16)v;
        l[e] = (_Float16)(v - (float)h[e]);
      }
      if (!tall) {
        *reinterpret_cast<f16x4*>(x + xat(line, col)) = h;
        if (NP == 2) *reinterpret_cast<f16x4*>(x + plane + xat(line, col)) = l;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          *reinterpret_cast<_Float16*>(x + xat(col + e, line)) = h[e];
          if (NP == 2) *reinterpret_cast<_Float16*>(x + plane + xat(col + e, line)) = l[e];
        }
      }
    }
  }
  __syncthreads();

  NsOnCu<2> m(lds, c.mp, wave, lane);
  const int steps = p.rec.steps, hi = lane >> 5;
  int s0 = 0;
  while (true) {
    int s1 = s0;
    while (!(p.ends >> s1 & 1)) ++s1;
    const float sx = p.sx[s0], res = s0 == 0 ? left : 1.f;
    // A = X X': wave w has block w % nb of the nb on and below the diagonal, and every (8 / nb)-th 16 of K from w / nb on
    constexpr int nb = ONE ? 1 : 3, parts = 8 / nb;
    const int blk = wave % nb, part = wave / nb;
    const int bi = blk > 0, bj = blk == 2;
    f32x16 a;
#pragma unroll
    for (int e = 0; e < 16; ++e) a[e] = 0.f;
    if (part < parts) {
      for (int k = part * 16; k < c.np; k += parts * 16) {
        const int oa = xat(bi * 32 + (lane & 31), k + 8 * hi), ob = xat(bj * 32 + (lane & 31), k + 8 * hi);
        const f16x8 ah = *reinterpret_cast<const f16x8*>(x + oa), bh = *reinterpret_cast<const f16x8*>(x + ob);
        if (NP == 2) {
          const f16x8 al = *reinterpret_cast<const f16x8*>(x + plane + oa), bl = *reinterpret_cast<const f16x8*>(x + plane + ob);
          a = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, a, 0, 0, 0);
          a = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, a, 0, 0, 0);
        }
        a = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, a, 0, 0, 0);
      }
      if (part > 0) {
        float4* o = reinterpret_cast<float4*>(lds) + ((part - 1) * nb + blk) * 256 + lane;          // at most 7 blocks of 4 KB
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) o[e4 * 64] = make_float4(a[e4 * 4], a[e4 * 4 + 1], a[e4 * 4 + 2], a[e4 * 4 + 3]);
      }
    }
    __syncthreads();
    if (part == 0) {
      for (int q = 1; q < parts; ++q) {
        const float4* o = reinterpret_cast<const float4*>(lds) + ((q - 1) * nb + blk) * 256 + lane;
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const float4 v = o[e4 * 64];
          a[e4 * 4] += v.x; a[e4 * 4 + 1] += v.y; a[e4 * 4 + 2] += v.z; a[e4 * 4 + 3] += v.w;
        }
      }
    }
    __syncthreads();
    const float una = res * res / (sx * sx);
    if constexpr (ONE) {
      if (wave == 0) m.put(0, ns_rec_one(p.rec, s0, s1, a, una, reinterpret_cast<float*>(lds + NsOnCu<2>::SLOT)));
    } else {
      if (part == 0) {
#pragma unroll
        for (int e = 0; e < 16; ++e) a[e] *= una;
        m.put_gram(a, p.rec.sA[s0], bi, bj);
      }
      __syncthreads();
      const f32x16 P = m.run(p.rec, s0, s1);
      __syncthreads();
      if (m.inside) m.put(0, P);
    }
    __syncthreads();
    // X <- P X in place: a wave takes blocks of 32 columns, all rows of them (nobody else reads those columns)
    const bool done = s1 == steps - 1;
    const float un = res / (p.rec.step[s1].sP * sx), to = p.sx[s1 + 1];
    for (int nblk = wave; nblk * 32 < c.np; nblk += 8) {
      f32x16 y[2];
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int e = 0; e < 16; ++e) y[v][e] = 0.f;
      for (int k = 0; k < c.mp; k += 16) {
        // columns of X as rows of the first operand: 4 k of one column a lane and read
        f16x8 xf[NP];
#pragma unroll
        for (int z = 0; z < NP; ++z) {
          f16x4 half[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int kr = k + 8 * hi + 4 * h + ((lane & 15) >> 2), col = nblk * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
            half[h] = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(x + z * plane + xat(kr, col))));
          }
          xf[z] = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          if (v * 32 >= c.mp) continue;
          const int o = NsOnCu<2>::at(v * 32 + (lane & 31), (k >> 3) + hi);
          const f16x8 ph = *reinterpret_cast<const f16x8*>(lds + o), pl = *reinterpret_cast<const f16x8*>(lds + NsOnCu<2>::PL + o);
          if (NP == 2) y[v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xf[NP - 1], ph, y[v], 0, 0, 0);
          y[v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xf[0], pl, y[v], 0, 0, 0);
          y[v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xf[0], ph, y[v], 0, 0, 0);
        }
      }
      // a lane: row 32 v + lane % 32, columns 32 nblk + 8 e4 + 4 (lane / 32) + 0 .. 3
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        if (v * 32 >= c.mp) continue;
        const int r = v * 32 + (lane & 31);
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const int q = nblk * 32 + 8 * e4 + 4 * hi;
          if (NP == 2 && !done) {        // (a single plane has one segment)
            f16x4 h, l;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float w = y[v][e4 * 4 + e] * un * to;
              h[e] = (_Float16)w;
              l[e] = (_Float16)(w - (float)h[e]);
            }
            *reinterpret_cast<f16x4*>(x + xat(r, q)) = h;
            *reinterpret_cast<f16x4*>(x + plane + xat(r, q)) = l;
          } else if (r < c.m) {
            T* o = reinterpret_cast<T*>(it.p);
            const float f = p.muon ? -p.lr * it.scale : 1.f;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (q + e < c.n) {
                const size_t at = tall ? (size_t)(q + e) * c.cols + r : (size_t)r * c.cols + q + e;
                const float w = y[v][e4 * 4 + e] * un * f;
                o[at] = from_f<T>(p.muon ? to_f(o[at]) * p.decay + w : w);
              }
          }
        }
      }
    }
    if (done) break;
    __syncthreads();
    s0 = s1 + 1;
  }
}

// ---- matrices of up to 64 x 64 and 32 x 128 on one CU: in fp32, step by step as written --------------------------------------------------------
// Near-square matrices of so few rows have weak directions, which the iteration amplifies 485 times, beside strong ones, which the P of several steps
// has to keep in spite of its size (11.9 after two); with planes and with fp32 alike that showed against a plain fp32 iteration: 32 x 32 1.4e-6 of the norm,
// 64 x 64 1.4e-6 (all in fp32 1.8e-6), 94 x 22 1.7e-6 for 0.9e-6, 1.0e-6, 1.0e-6.  Here X X', its square and (b A + c A^2) X are the only
// products of a step, three of nearly the same size, so that commuting factors would save none: X <- a X + (b A + c A^2) X.
// The fp32 instructions take 64 cycles for 32 x 32 x 2: 2048 a product of 64 x 64 on each wave.  Rows of X and of the symmetric matrices lie in LDS an
// odd number of 16 bytes apart; wave w < 3 has block (w > 0, w == 2) of those on and below the diagonal and writes its mirror image too.
// Measured (5 steps, us, with planes before): 16 x 27 15 / 24, 32 x 128 18 / 26, 64 x 64 29 / 30; bf16, where planes are exact enough, 15 / 20, 18 / 21,
// 29 / 27.  32 x 300 so would take 40, with planes and the recursion in fp32 26 at 1.3e-6 of the norm for the plain iteration's 1.0e-6.
struct NsF32 {
  static constexpr int PM = 64 + 4;
  int q, h, I, J;
  // sum over k of a[32 I + row][k] b[32 J + column][k]
  static __device__ __forceinline__ f32x16 rows(const float* a, const float* b, int from, int to, int step, f32x16 r) {
#pragma unroll 4
    for (int k = from; k < to; k += step) {
      const float4 x = *reinterpret_cast<const float4*>(a + k), y = *reinterpret_cast<const float4*>(b + k);
      r = __builtin_amdgcn_mfma_f32_32x32x2f32(x.x, y.x, r, 0, 0, 0);
      r = __builtin_amdgcn_mfma_f32_32x32x2f32(x.y, y.y, r, 0, 0, 0);
      r = __builtin_amdgcn_mfma_f32_32x32x2f32(x.z, y.z, r, 0, 0, 0);
      r = __builtin_amdgcn_mfma_f32_32x32x2f32(x.w, y.w, r, 0, 0, 0);
    }
    return r;
  }
  static __device__ __forceinline__ f32x16 zero() {
    f32x16 r;
#pragma unroll
    for (int e = 0; e < 16; ++e) r[e] = 0.f;
    return r;
  }
  // this wave's block of the product of two symmetric 64 x 64 matrices
  __device__ __forceinline__ f32x16 product(const float* a, const float* b) const {
    return rows(a + (32 * I + q) * PM + h, b + (32 * J + q) * PM + h, 0, 64, 8, zero());
  }
  // exactly symmetric: of a block on the diagonal the elements on and below it
  __device__ __forceinline__ void put(float* m, const f32x16& v) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r0 = 32 * I + 8 * i + h, c = 32 * J + q;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (I > J || r0 + e >= c) {
          m[(r0 + e) * PM + c] = v[i * 4 + e];
          m[c * PM + r0 + e] = v[i * 4 + e];
        }
    }
  }
  __device__ __forceinline__ f32x16 get(const float* m) const {
    f32x16 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 t = *reinterpret_cast<const float4*>(m + (32 * J + q) * PM + 32 * I + 8 * i + h);
      v[i * 4] = t.x; v[i * 4 + 1] = t.y; v[i * 4 + 2] = t.z; v[i * 4 + 3] = t.w;
    }
    return v;
  }
};
struct NsF32Args {
  int steps;
  float a[NS_MAX_STEPS], b[NS_MAX_STEPS], c[NS_MAX_STEPS];
  float eps, lr, decay;
  int muon;
};
template <typename T>
__global__ __launch_bounds__(256) void ns_f32_kernel(NsClasses cs, NsF32Args p, NsInline few, const NsItem* __restrict__ table, MuonArgs ma) {
  constexpr int PM = NsF32::PM, GROUPS = 64 * 64 / 4 / 256;
  __shared__ __attribute__((aligned(16))) float x[64 * PM];          // (32 * 132 is less)
  __shared__ __attribute__((aligned(16))) float mat[2][64 * PM];
  __shared__ double sh[4];
  const NsClass c = find_class(cs, blockIdx.x);
  const int i = blockIdx.x - c.start;
  const NsItem it = ns_item(few, table, c.first + i);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const T* g = reinterpret_cast<const T*>(it.g);
  const bool tall = c.rows > c.cols;

  // momentum, update and its norm; the update stays in registers (fours of a line, 256 further each time)
  const int per_line = (c.cols + 3) >> 2, lines = 256 / per_line, fours = 256 - lines * per_line;
  const int line0 = tid / per_line, four0 = tid - line0 * per_line;
  float u[GROUPS][4];
  double s = 0.0;
  int line = line0, four = four0;
  auto next = [&]() {
    line += lines;
    four += fours;
    if (four >= per_line) { four -= per_line; ++line; }
  };
#pragma unroll
  for (int k = 0; k < GROUPS; ++k, next()) {
#pragma unroll
    for (int e = 0; e < 4; ++e) u[k][e] = 0.f;
    if (line < c.rows) {
      const int col = four * 4;
      const long at = (long)line * c.cols + col;
      if (col + 4 <= c.cols) {
        load4(g + at, u[k]);
        if (it.mom != nullptr) {
          float m[4];
          load4(it.mom + at, m);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            m[e] = muon_momentum(m[e], u[k][e], ma);
            u[k][e] = muon_update(m[e], u[k][e], ma);
          }
          store4(it.mom + at, m);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < c.cols) {
            float v = to_f(g[at + e]);
            if (it.mom != nullptr) {
              const float m = muon_momentum(it.mom[at + e], v, ma);
              it.mom[at + e] = m;
              v = muon_update(m, v, ma);
            }
            u[k][e] = v;
          }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s += (double)u[k][e] * u[k][e];
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane == 0) sh[wave] = s;
  const int px = c.np + 4;
  for (int e = tid * 4; e < c.mp * px; e += 1024) *reinterpret_cast<float4*>(x + e) = make_float4(0.f, 0.f, 0.f, 0.f);     // the padding
  __syncthreads();
  const double square = (sh[0] + sh[1]) + (sh[2] + sh[3]);
  // (a NaN or an infinity in the matrix: all of its result is NaN)
  const double mul = square < HUGE_VAL ? 1.0 / fmax(sqrt(square), (double)p.eps) : nan("");
  line = line0;
  four = four0;
#pragma unroll
  for (int k = 0; k < GROUPS; ++k, next()) {
    if (line >= c.rows) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (four * 4 + e < c.cols) x[tall ? (four * 4 + e) * px + line : line * px + four * 4 + e] = (float)((double)u[k][e] * mul);
  }
  __syncthreads();

  const NsF32 m{lane & 31, 4 * (lane >> 5), wave > 0, wave == 2};
  const int q = m.q, h = m.h;
  const bool two = c.mp > 32;
  // block of X <- a X + S X that a wave has: four at most
  const int v = two ? wave & 1 : 0, col = (two ? wave >> 1 : wave) * 32;
  const bool mine = col < c.np;
  float *A = mat[0], *S = mat[1];
  for (int st = 0;; ++st) {
    const float ca = p.a[st], cb = p.b[st], cc = p.c[st];
    if (two) {                             // (wave 3 only waits)
      if (wave < 3) m.put(A, NsF32::rows(x + (32 * m.I + q) * px + h, x + (32 * m.J + q) * px + h, 0, c.np, 8, NsF32::zero()));
      __syncthreads();
      if (wave < 3) {
        f32x16 t = m.product(A, A);
        const f32x16 a = m.get(A);
#pragma unroll
        for (int e = 0; e < 16; ++e) t[e] = __fmaf_rn(cc, t[e], cb * a[e]);
        m.put(S, t);
      }
    } else {
      // four waves share the sum over K
      f32x16 t = NsF32::rows(x + q * px + h, x + q * px + h, wave * 8, c.np, 32, NsF32::zero());
      float4* o = reinterpret_cast<float4*>(A);
      if (wave > 0) {
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) o[((wave - 1) * 4 + e4) * 64 + lane] = make_float4(t[e4 * 4], t[e4 * 4 + 1], t[e4 * 4 + 2], t[e4 * 4 + 3]);
      }
      __syncthreads();
      if (wave == 0) {
        for (int w = 0; w < 3; ++w)
#pragma unroll
          for (int e4 = 0; e4 < 4; ++e4) {
            const float4 a = o[(w * 4 + e4) * 64 + lane];
            t[e4 * 4] += a.x; t[e4 * 4 + 1] += a.y; t[e4 * 4 + 2] += a.z; t[e4 * 4 + 3] += a.w;
          }
        const f32x16 w = ns_product_one(t, t);         // (sums of x y in the order of y x: t is symmetric as it is)
#pragma unroll
        for (int e = 0; e < 16; ++e) t[e] = __fmaf_rn(cc, w[e], cb * t[e]);
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) *reinterpret_cast<float4*>(S + q * PM + 8 * e4 + h) = make_float4(t[e4 * 4], t[e4 * 4 + 1], t[e4 * 4 + 2], t[e4 * 4 + 3]);
      }
    }
    __syncthreads();
    // X <- a X + S X.  A lane: rows 32 v + 8 e4 + h + 0 .. 3, column col + q
    f32x16 y = NsF32::zero();
    if (mine) {
#pragma unroll 4
      for (int k = 0; k < c.mp; k += 8) {
        const float4 a = *reinterpret_cast<const float4*>(S + (32 * v + q) * PM + k + h);
        const float* b = x + (k + h) * px + col + q;
        y = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x, b[0], y, 0, 0, 0);
        y = __builtin_amdgcn_mfma_f32_32x32x2f32(a.y, b[px], y, 0, 0, 0);
        y = __builtin_amdgcn_mfma_f32_32x32x2f32(a.z, b[2 * px], y, 0, 0, 0);
        y = __builtin_amdgcn_mfma_f32_32x32x2f32(a.w, b[3 * px], y, 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) y[e] = __fmaf_rn(ca, x[(32 * v + 8 * (e >> 2) + h + (e & 3)) * px + col + q], y[e]);
    }
    if (st == p.steps - 1) {
      if (!mine || col + q >= c.n) return;
      T* o = reinterpret_cast<T*>(it.p);
      const float f = p.muon ? -p.lr * it.scale : 1.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int r = 32 * v + 8 * (e >> 2) + h + (e & 3), n = col + q;
        if (r >= c.m) continue;
        const size_t at = tall ? (size_t)n * c.cols + r : (size_t)r * c.cols + n;
        const float w = y[e] * f;
        o[at] = from_f<T>(p.muon ? to_f(o[at]) * p.decay + w : w);
      }
      return;
    }
    __syncthreads();
    if (mine) {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[(32 * v + 8 * (e >> 2) + h + (e & 3)) * px + col + q] = y[e];
    }
    __syncthreads();
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------
struct NsPlan {
  struct Set { std::vector<NsClass> cls; size_t bytes; int items; };
  std::vector<Set> sets;
  int np;                               // planes of X
  int xplanes;
  size_t head;                          // table + norms + residues, for the largest set; then the shares of split products
  size_t bytes;
};

inline int sym_tiles(int mp, int t) { const int k = (mp + t - 1) / t; return k * (k + 1) / 2; }

// A symmetric product of `jobs` times the classes' matrices.  Tile: 128 x 128, or about four times as many of 64 x 64, by rounds over the 256 CUs
// of 0.82 us a K step of 32 of a large tile; a small one takes 0.4 of its time.  full / cut: large tiles that pass a multiple of 256 run last, in
// `cut` shares of K over the whole card, which a pass of their own adds up: 65 KB written and read a share at 5 TB/s, 4 us for the launch.
// (2 products of 2048 x 2048 x 2048 in 272 tiles: 105 us as two rounds, 106 us in 1056 small tiles, 84 + 8 us with 16 tiles in 8 shares)
struct NsTiling { int tile, full, cut; double time; };
NsTiling ns_sym_tiling(const NsClass* c, int n, bool gram, int jobs) {
  long big = 0, few = 0;
  int K = 0;
  for (int k = 0; k < n; ++k) {
    big += (long)sym_tiles(c[k].mp, 128) * c[k].count;
    few += (long)sym_tiles(c[k].mp, 64) * c[k].count;
    const int kk = gram ? c[k].np : c[k].mp;
    K = kk > K ? kk : K;
  }
  const double round = K / 32 * 0.82, small = (jobs * few + 255) / 256 * 0.4 * round;
  NsTiling r = {128, (int)big, 1, (jobs * big + 255) / 256 * round};
  const long full = big / 256 * 256, rest = big - full;
  if (full > 0 && rest > 0)
    for (int s = 2; s <= 16 && s * rest <= 256; ++s) {
      const double time = jobs * (full / 256 * round + round / s + s * rest * 131072 / 5e6) + 4.0;
      if (time < r.time) { r.time = time; r.full = (int)full; r.cut = s; }
    }
  if (jobs * big < 128 || small < r.time) r = {64, 0, 1, small};
  return r;
}
// other products: 23 x P X of 256 x 2304 39 us in 828 large, 51 us in 3312 small tiles
inline bool ns_big_tiles(long big, long few) { return (big + 255) / 256 * 10 <= (few + 255) / 256 * 4 && big >= 128; }

inline int round_up(int v, int to) { return (v + to - 1) / to * to; }
inline size_t round_up_z(size_t v, size_t to) { return (v + to - 1) / to * to; }

// How the matrices of one set run.  small: all have at most 128 on their smaller side, their recursion runs on one CU each.
// Gram products may be cut along K (n) into shares that are added up in order; tile and share (K a workgroup takes) by a model of their
// time: rounds of workgroups over the 256 CUs, 0.82 us a K step of 32 of a large tile and 0.66 us a K step of 64 of a small one (measured, whether
// one or two workgroups are on a CU), shares written and read at 5 TB/s and 4 us for the launch that adds them
// (small: 1.2 us for every 16 of them in the recursion's workgroup).  23 x 256 x 2304: 230 small
// tiles in one share 24 us (model) against 34 measured for 8 shares of 69 large ones; 3 x 512 x 4608: 8 shares of 30 large tiles.
struct NsSplit { int tile, shares, tiles, small, mt, tiny, full, cut; size_t bytes; int slim[NS_MAX_CLASSES]; };      // bytes: of all shares, cut tiles' too
inline bool ns_is_f32(const NsClass& c, int planes) { return c.mp == 32 ? c.np <= 128 : c.np <= 64 && planes == 2; }          // (and tiny with it)
inline bool ns_is_tiny(const NsClass& c, int planes) { return c.mp <= 64 && c.np <= (planes == 2 ? NS_TINY_N<2> : NS_TINY_N<1>); }
NsSplit ns_split_plan(std::vector<NsClass>& cls, int planes) {
  NsSplit r = {64, 1, 0, 1, 2, 0, 0, 1, 0, {}};
  if (ns_is_tiny(cls[0], planes)) {               // (and with it all of the set)
    r.tiny = ns_is_f32(cls[0], planes) ? 2 : 1;
    return r;
  }
  int longest = 0;
  for (auto& c : cls) {
    if (c.mp > 64) r.mt = 4;
    if (c.mp > 128) r.small = 0;
    longest = c.np > longest ? c.np : longest;
  }
  double best = 1e30;
  int ks = 0;
  for (int t = 64; t <= (r.small ? 64 : 128); t *= 2)
    for (int s = 1; s <= 128 && (s == 1 || longest / s >= 128); ++s) {
      const int k = ((longest + s - 1) / s + 63) / 64 * 64;
      long wg = 0;
      double bytes = 0.0;
      for (auto& c : cls) {
        const long n = (long)sym_tiles(c.mp, t) * c.count * ((c.np + k - 1) / k);
        wg += n;
        bytes += (double)n * t * t * 8.0;
      }
      const int rounds = (int)((wg + 255) / 256);
      const double time = rounds * (t == 128 ? k / 32 * 0.82 : k / 64 * 0.66) + (s > 1 || r.small ? bytes / 5e6 : 0.0) + (s > 1 && !r.small ? 4.0 : 0.0) + (r.small ? (s + 15) / 16 * 1.2 : 0.0);
      if (time < best) { best = time; r.tile = t; ks = k; }
    }
  NsTiling cut = {0, 0, 1, 0.0};
  if (!r.small) {
    cut = ns_sym_tiling(cls.data(), (int)cls.size(), true, 1);
    if (cut.cut > 1 && cut.time < best) { r.tile = 128; ks = (longest + 63) / 64 * 64; }
    else cut.cut = 1;
  }
  for (auto& c : cls) {
    c.ks = ks;
    const int n = (c.np + ks - 1) / ks;
    if (n > r.shares) r.shares = n;
    r.tiles += sym_tiles(c.mp, r.tile) * c.count;
  }
  r.full = cut.cut > 1 ? cut.full : r.tiles;
  r.cut = cut.cut;
  // matrices of up to 64 rows: columns a workgroup of the kernel that joins P X and the next Gram product takes, at most 128 shares
  int most = r.shares;
  for (size_t k = 0; r.small && r.mt == 2 && k < cls.size(); ++k) {
    const int share = ((cls[k].np + 127) / 128 + 255) / 256 * 256, n = (cls[k].np + share - 1) / share;
    r.slim[k] = share;
    most = n > most ? n : most;
  }
  if (r.shares > 1 || r.small) r.bytes = (size_t)most * r.tiles * r.tile * r.tile * sizeof(float);
  // cut tiles of any of the set's products: at most 256 a job
  if (!r.small) {
    const int n = (int)cls.size();
    const bool any = cut.cut > 1 || ns_sym_tiling(cls.data(), n, false, 1).cut > 1 || ns_sym_tiling(cls.data(), n, false, 2).cut > 1;
    if (any) r.bytes = std::max(r.bytes, (size_t)2 * 256 * 128 * 128 * sizeof(float));
  }
  return r;
}

// slots of a region: X and its successor, two planes each (of a single plane, with one segment: X alone), then A, T and three for Q / P
constexpr int ns_xplanes(int planes) { return planes == 2 ? 4 : 1; }
int ns_plan(const char* what, int dtype, const pxl_ns_item* items, int n, int planes, NsPlan& plan) {
  PXL_REQUIRE(dtype == PXL_F32 || dtype == PXL_BF16, "%s: dtype %d is neither PXL_F32 nor PXL_BF16", what, dtype);
  PXL_REQUIRE(n >= 0 && n <= (1 << 22) && (n == 0 || items != nullptr), "%s: bad item list (%d matrices, at most 2^22)", what, n);
  plan.np = planes;
  plan.xplanes = ns_xplanes(planes);
  std::vector<NsPlan::Set>& sets = plan.sets;
  for (int i = 0; i < n; ++i) {
    PXL_REQUIRE(items[i].rows >= 1 && items[i].cols >= 1 && items[i].rows <= (1 << 23) && items[i].cols <= (1 << 23) &&
                    (items[i].rows < items[i].cols ? items[i].rows : items[i].cols) <= (1 << 15),
                "%s: item %d is %d x %d (1 .. 2^23, the smaller side at most 32768)", what, i, items[i].rows, items[i].cols);
    int sk = -1, ck = -1;
    for (size_t s = 0; s < sets.size() && sk < 0; ++s)
      for (size_t k = 0; k < sets[s].cls.size(); ++k)
        if (sets[s].cls[k].rows == items[i].rows && sets[s].cls[k].cols == items[i].cols) { sk = (int)s; ck = (int)k; break; }
    if (sk < 0) {
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
      // matrices that run on one CU whole, those whose recursion does, by its two sizes, and the others: in sets of their own
      auto kind = [&](const NsClass& x) { return ns_is_f32(x, plan.np) ? -1 : ns_is_tiny(x, plan.np) ? (x.mp == 32 ? -2 : 0) : (x.mp <= 64 ? 1 : (x.mp <= 128 ? 2 : 3)); };
      if (ns_is_tiny(c, plan.np)) c.stride = 0;
      for (size_t q = 0; q < sets.size(); ++q)
        if (kind(sets[q].cls[0]) == kind(c) && sets[q].cls.size() < (size_t)NS_MAX_CLASSES) sk = (int)q;
      if (sk < 0) {
        sets.emplace_back();
        sk = (int)sets.size() - 1;
      }
      sets[sk].cls.push_back(c);
      ck = (int)sets[sk].cls.size() - 1;
    }
    sets[sk].cls[ck].count++;
  }
  plan.head = plan.bytes = 0;
  for (auto& s : sets) {
    int first = 0;
    for (auto& c : s.cls) { c.first = first; first += c.count; }
    s.items = first;
    // no launch of a set has more workgroups than the larger of these two passes; one of 256 threads each, and a grid has fewer than 2^32
    long norm = 0, split = 0;
    for (auto& c : s.cls) {
      norm += (long)c.parts * c.count;
      split += (long)((c.np + 63) / 64) * ((c.mp + 63) / 64) * c.count;
    }
    PXL_REQUIRE(ns_is_tiny(s.cls[0], plan.np) || (norm < (1l << 24) && split < (1l << 24)),
                "%s: %d matrices like %d x %d are too many for one call (2^24 tiles of 64 x 64, 2^35 elements)", what, first, s.cls[0].rows, s.cls[0].cols);
    const size_t table = round_up_z(first * sizeof(NsItem), 256);
    const size_t head = ns_is_tiny(s.cls[0], plan.np) ? table : table + round_up_z(first * sizeof(double) * NS_PARTS, 256) + round_up_z(first * sizeof(float), 256);
    if (head > plan.head) plan.head = head;
  }
  for (auto& s : sets) {
    const NsSplit sp = ns_split_plan(s.cls, plan.np);
    size_t at = plan.head + sp.bytes;
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
    for (int e = 0; e <= 256; ++e) {                       // (smooth: the maxima to 2e-4, under the 1 % added below)
      const double x = sigma * e / 256, l = x * x, q = fabs(d.a + l * (d.b + d.c * l));
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
  NsInline few;
  NsItem* table;                        // NULL: the items are in `few`
  double* part;
  float* residue;
  float* shares;
  unsigned char* ws;
  NsSplit split;
};

#define NS_TRY(expr)            \
  do {                          \
    const int _rc = (expr);     \
    if (_rc != PXL_OK) return _rc; \
  } while (0)

template <int EPI, int NA, int NB, int T, typename OutT>
int ns_launch(NsRun& r, NsGemm& g, int jobs = 1, int full = 0, int cut = 1) {
  int at = 0;
  for (int k = 0; k < r.cs.n; ++k) {
    NsClass& c = r.cs.c[k];
    const int tm = (c.mp + T - 1) / T, tn = (c.np + T - 1) / T;
    c.tn = EPI <= EPI_MUL ? tm : tn;
    c.per = EPI <= EPI_MUL ? tm * (tm + 1) / 2 : tm * tn;
    c.start = at;
    at += c.per * c.count;
  }
  g.full = cut > 1 ? full : at;
  g.cut = cut;
  const int rest = at - g.full;
  const dim3 grid(g.full + rest * cut, EPI == EPI_PART ? r.split.shares : 1, jobs);
  if (T == 64 && at * jobs <= 256 && (EPI == EPI_Q || EPI == EPI_MUL))
    hipLaunchKernelGGL((ns_gemm_kernel<EPI, NA, NB, T, T == 64 && (EPI == EPI_Q || EPI == EPI_MUL) ? 4 : 2, OutT>), grid, dim3(256), 0, r.st, r.cs, g, r.few,
                       r.table, r.residue, r.ws);
  else
    hipLaunchKernelGGL((ns_gemm_kernel<EPI, NA, NB, T, 2, OutT>), grid, dim3(256), 0, r.st, r.cs, g, r.few, r.table, r.residue, r.ws);
  PXL_LAUNCH_CHECK();
  if constexpr (T == 128 && (EPI == EPI_GRAM || EPI == EPI_Q || EPI == EPI_MUL)) {
    if (rest > 0) {
      hipLaunchKernelGGL((ns_cut_fold_kernel<EPI>), dim3(rest * 16, 1, jobs), dim3(64), 0, r.st, r.cs, g, r.residue, r.ws);
      PXL_LAUNCH_CHECK();
    }
  }
  if (EPI == EPI_PART && !r.split.small) {
    hipLaunchKernelGGL((ns_fold_kernel<T>), dim3(at * (T * T / 1024)), dim3(64), 0, r.st, r.cs, g, at, r.residue, r.ws);
    PXL_LAUNCH_CHECK();
  }
  return PXL_OK;
}

template <int EPI, int NA, int NB, typename OutT>
int ns_gemm(NsRun& r, NsGemm& g, int jobs = 1) {
  if constexpr (EPI == EPI_GRAM) {
    if (r.split.shares > 1 || r.split.small)
      return r.split.tile == 128 ? ns_launch<EPI_PART, NA, NB, 128, OutT>(r, g) : ns_launch<EPI_PART, NA, NB, 64, OutT>(r, g);
    return r.split.tile == 128 ? ns_launch<EPI, NA, NB, 128, OutT>(r, g, 1, r.split.full, r.split.cut) : ns_launch<EPI, NA, NB, 64, OutT>(r, g);
  } else if constexpr (EPI <= EPI_MUL) {
    const NsTiling t = ns_sym_tiling(r.cs.c, r.cs.n, false, jobs);
    return t.tile == 128 ? ns_launch<EPI, NA, NB, 128, OutT>(r, g, jobs, t.full, t.cut) : ns_launch<EPI, NA, NB, 64, OutT>(r, g, jobs);
  } else {
    long big = 0, few = 0;
    for (int k = 0; k < r.cs.n; ++k) {
      const NsClass& c = r.cs.c[k];
      big += (long)((c.mp + 127) / 128) * ((c.np + 127) / 128) * c.count;
      few += (long)((c.mp + 63) / 64) * ((c.np + 63) / 64) * c.count;
    }
    return ns_big_tiles(big, few) ? ns_launch<EPI, NA, NB, 128, OutT>(r, g) : ns_launch<EPI, NA, NB, 64, OutT>(r, g);
  }
}

// coefficients and plane scales of steps [s, e), one segment, at places [at, ...)
void ns_rec_scales(NsRec& q, const std::vector<NsStep>& steps, size_t s, size_t e, size_t at) {
  double pbound = 1.0;
  float sP = 1.f;
  q.sA[at] = plane_scale(steps[s].lam);
  for (size_t k = s; k < e; ++k) {
    const NsStep& d = steps[k];
    NsRecStep& o = q.step[at + k - s];
    const float sA = plane_scale(d.lam), sQ = plane_scale(d.q), sT = plane_scale(d.t), before = sP;
    pbound *= d.q;
    o.sP = sP = plane_scale(pbound);                     // (the first step's P is Q: the same scale)
    o.g = (float)d.c * sQ / (sA * sA);
    o.ia = (float)d.b * sQ / sA;
    o.a = (float)d.a * sQ;
    o.fP = sP / (sQ * before);
    o.fT = sT / (sQ * sA);
    o.fA = (k + 1 < e ? plane_scale(steps[k + 1].lam) : 1.f) / (sQ * sT);
  }
}

// the recursion of steps [s, e) of a small set: shares -> P in slot `out`; -> the scale of P's planes
int ns_rec(NsRun& r, const std::vector<NsStep>& steps, size_t s, size_t e, float unscale, int res_pow, int xplanes, int out, float* sP) {
  NsRec q;
  memset(&q, 0, sizeof(q));
  q.steps = (int)(e - s);
  q.xplanes = xplanes;
  q.out = out;
  q.unscale = unscale;
  q.res_pow = res_pow;
  q.part = r.shares;
  ns_rec_scales(q, steps, s, e, 0);
  *sP = q.step[q.steps - 1].sP;
  int at = 0, tiles = 0;
  for (int k = 0; k < r.cs.n; ++k) {
    NsClass& c = r.cs.c[k];
    c.per = sym_tiles(c.mp, 64);
    c.tn = tiles;                       // first tile of the class among the product's
    c.start = at;
    at += c.count;
    tiles += c.per * c.count;
  }
  if (r.split.mt == 2) hipLaunchKernelGGL((ns_rec_kernel<2>), dim3(at), dim3(512), 0, r.st, r.cs, q, tiles, r.residue, r.ws);
  else hipLaunchKernelGGL((ns_rec_kernel<4>), dim3(at), dim3(1024), 0, r.st, r.cs, q, tiles, r.residue, r.ws);
  PXL_LAUNCH_CHECK();
  return PXL_OK;
}

// X <- P X with the shares of its Gram product, or the result
template <int NP, bool LAST, typename T>
int ns_slim(NsRun& r, const NsGemm& g) {
  NsSlim q;
  memset(&q, 0, sizeof(q));
  q.xplanes = g.xplanes;
  q.p = g.job[0].a;
  q.x = g.job[0].b;
  q.out = g.job[0].out;
  q.unscale = g.unscale[0];
  q.scale = g.scale[0];
  q.use_res = g.res_pow;
  q.lr = g.lr;
  q.decay = g.decay;
  q.muon = g.muon;
  q.part = r.shares;
  int at = 0;
  for (int k = 0; k < r.cs.n; ++k) {
    NsClass& c = r.cs.c[k];
    c.ks = r.split.slim[k];             // (and what the recursion adds up next)
    c.per = (c.np + c.ks - 1) / c.ks;
    c.start = at;
    at += c.per * c.count;
    q.matrices += c.count;
  }
  hipLaunchKernelGGL((ns_slim_kernel<NP, LAST, T>), dim3(at), dim3(256), 0, r.st, r.cs, q, r.few, r.table, r.residue, r.ws);
  PXL_LAUNCH_CHECK();
  return PXL_OK;
}

template <typename T, int NP>
int ns_run_tiny(NsRun& r, const std::vector<NsStep>& steps, float eps, const MuonArgs& ma, int muon) {
  NsTiny q;
  memset(&q, 0, sizeof(q));
  q.rec.steps = (int)steps.size();
  for (size_t s = 0; s < steps.size();) {
    size_t e = s;
    while (!steps[e].last) ++e;
    ns_rec_scales(q.rec, steps, s, e + 1, s);
    q.ends |= 1u << e;
    q.sx[s] = plane_scale(s == 0 ? 1.0 : steps[s].sigma);
    s = e + 1;
  }
  q.eps = eps;
  q.muon = muon;
  q.lr = ma.lr;
  q.decay = ma.keep;
  int at = 0;
  for (int k = 0; k < r.cs.n; ++k) {
    r.cs.c[k].start = at;
    at += r.cs.c[k].count;
  }
  if (r.cs.c[0].mp == 32) hipLaunchKernelGGL((ns_tiny_kernel<T, NP, true>), dim3(at), dim3(512), 0, r.st, r.cs, q, r.few, r.table, ma);
  else hipLaunchKernelGGL((ns_tiny_kernel<T, NP, false>), dim3(at), dim3(512), 0, r.st, r.cs, q, r.few, r.table, ma);
  PXL_LAUNCH_CHECK();
  return PXL_OK;
}

template <typename T>
int ns_run_f32(NsRun& r, const std::vector<NsStep>& steps, float eps, const MuonArgs& ma, int muon) {
  NsF32Args q;
  memset(&q, 0, sizeof(q));
  q.steps = (int)steps.size();
  for (size_t s = 0; s < steps.size(); ++s) { q.a[s] = (float)steps[s].a; q.b[s] = (float)steps[s].b; q.c[s] = (float)steps[s].c; }
  q.eps = eps;
  q.lr = ma.lr;
  q.decay = ma.keep;
  q.muon = muon;
  int at = 0;
  for (int k = 0; k < r.cs.n; ++k) {
    r.cs.c[k].start = at;
    at += r.cs.c[k].count;
  }
  hipLaunchKernelGGL((ns_f32_kernel<T>), dim3(at), dim3(256), 0, r.st, r.cs, q, r.few, r.table, ma);
  PXL_LAUNCH_CHECK();
  return PXL_OK;
}

template <typename T, int NP>
int ns_run_set(NsRun& r, const std::vector<NsStep>& steps, float eps, const MuonArgs& ma, int muon) {
  if (r.split.tiny == 2) return ns_run_f32<T>(r, steps, eps, ma, muon);
  if (r.split.tiny) return ns_run_tiny<T, NP>(r, steps, eps, ma, muon);
  constexpr int xplanes = ns_xplanes(NP);
  const int MA = xplanes, MT = xplanes + 1;
  int blocks = 0;
  for (int k = 0; k < r.cs.n; ++k) {
    NsClass& c = r.cs.c[k];
    c.per = c.parts;
    c.start = blocks;
    blocks += c.per * c.count;
  }
  hipLaunchKernelGGL(ns_norm_kernel<T>, dim3(blocks), dim3(256), 0, r.st, r.cs, r.few, r.table, r.part, ma);
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
  hipLaunchKernelGGL((ns_split_kernel<T, NP>), dim3(blocks), dim3(256), 0, r.st, r.cs, r.few, r.table, r.part, r.residue, r.ws, eps, sx, ma);
  PXL_LAUNCH_CHECK();

  NsGemm g;
  memset(&g, 0, sizeof(g));
  g.xplanes = xplanes;
  g.part = r.shares;
  int first = 1, x = 0, x2 = NP;
  size_t s = 0;
  while (s < steps.size()) {
    double pbound = 1.0;
    float sA = plane_scale(steps[s].lam), sP = 1.f;
    g.job[0] = {x, x, MA};
    g.unscale[0] = 1.f / (sx * sx);
    g.scale[0] = sA;
    g.res_pow = NP == 1 && first ? 2 : 0;
    const bool slim = r.split.small && r.split.mt == 2;
    if (!slim || first) NS_TRY((ns_gemm<EPI_GRAM, NP, NP, float>(r, g)));       // (slim: later ones come with P X)
    int P = -1;
    if (r.split.small) {
      size_t e = s;
      while (!steps[e].last) ++e;
      P = xplanes + 2;
      NS_TRY(ns_rec(r, steps, s, e + 1, g.unscale[0], g.res_pow, xplanes, P, &sP));
      s = e;
    }
    g.res_pow = 0;
    for (; !r.split.small; ++s) {
      const NsStep& d = steps[s];
      int q = xplanes + 2;
      while (q == P) ++q;
      const float sQ = plane_scale(d.q);
      g.job[0] = {MA, MA, q};
      g.unscale[0] = 1.f / (sA * sA);
      g.scale[0] = sQ;
      g.qa = (float)d.a; g.qb = (float)d.b; g.qc = (float)d.c;
      g.sa_inv = 1.f / sA;
      NS_TRY((ns_gemm<EPI_Q, 2, 2, float>(r, g)));
      pbound *= d.q;
      const float sP2 = plane_scale(pbound), sT = plane_scale(d.t);
      // P <- Q P and T = Q A, in one launch where there are both
      int jobs = 0;
      if (P < 0) {
        P = q;
        sP = sQ;
      } else {
        int p2 = xplanes + 2;
        while (p2 == P || p2 == q) ++p2;
        g.job[0] = {q, P, p2};
        g.unscale[0] = 1.f / (sQ * sP);
        g.scale[0] = sP2;
        jobs = 1;
        P = p2;
        sP = sP2;
      }
      if (!d.last) {
        g.job[jobs] = {q, MA, MT};
        g.unscale[jobs] = 1.f / (sQ * sA);
        g.scale[jobs++] = sT;
      }
      if (jobs) NS_TRY((ns_gemm<EPI_MUL, 2, 2, float>(r, g, jobs)));
      if (d.last) break;
      const float sA2 = plane_scale(steps[s + 1].lam);
      g.job[0] = {q, MT, MA};
      g.unscale[0] = 1.f / (sQ * sT);
      g.scale[0] = sA2;
      NS_TRY((ns_gemm<EPI_MUL, 2, 2, float>(r, g)));
      sA = sA2;
    }
    ++s;
    g.unscale[0] = 1.f / (sP * sx);
    g.res_pow = NP == 1 && first ? 1 : 0;
    if (s == steps.size()) {
      g.job[0] = {P, x, 0};
      g.muon = muon;
      g.lr = ma.lr;
      g.decay = ma.keep;
      if (slim) NS_TRY((ns_slim<NP, true, T>(r, g)));
      else NS_TRY((ns_gemm<EPI_OUT, 2, NP, T>(r, g)));
    } else if constexpr (NP == 2) {
      const float sx2 = plane_scale(steps[s].sigma);
      g.job[0] = {P, x, x2};
      g.scale[0] = sx2;
      if (slim) {
        g.job[0].out = x2;
        NS_TRY((ns_slim<NP, false, T>(r, g)));
      } else {
        NS_TRY((ns_gemm<EPI_X, 2, NP, float>(r, g)));
      }
      sx = sx2;
      const int o = x;
      x = x2;
      x2 = o;
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

// The steps of a call and its matrices' planes.  A bf16 matrix is one plane; the update of a Muon step is formed in 32 bits from a 32-bit momentum
// whatever the gradient's type, so two (rounded to one, 11 bits: the orthogonalised update of 256 x 1024 with six directions 50 times the noise is off
// by 2e-2).  Nor is X a bf16 matrix any more behind a first segment: steps that do not fit into one run as those of 32-bit matrices
int ns_form(const char* what, int dtype, int steps, const float* coef, int muon, int& planes, std::vector<NsStep>& st) {
  planes = dtype == PXL_F32 || muon ? 2 : 1;
  NS_TRY(ns_schedule(what, steps, coef, planes, st));
  if (planes == 1 && std::any_of(st.begin(), st.end() - 1, [](const NsStep& d) { return d.last; })) {
    planes = 2;
    st.clear();
    NS_TRY(ns_schedule(what, steps, coef, planes, st));
  }
  return PXL_OK;
}

// everything about a call but its workspace; nothing is launched
int ns_check(const char* what, int dtype, const pxl_ns_item* items, int n, int steps, const float* coef, float eps, int muon, NsPlan& plan,
             std::vector<NsStep>& st) {
  int planes;
  NS_TRY(ns_form(what, dtype, steps, coef, muon, planes, st));
  NS_TRY(ns_plan(what, dtype, items, n, planes, plan));
  PXL_REQUIRE(eps > 0.f, "%s: eps %g", what, eps);
  for (int i = 0; i < n; ++i)
    PXL_REQUIRE(items[i].p != nullptr && items[i].g != nullptr && (!muon || items[i].mom != nullptr), "%s: item %d has a null pointer", what, i);
  if (n > 0) NS_TRY(ns_overlap(what, dtype, items, n, muon));
  return PXL_OK;
}

int ns_run(const char* what, int dtype, const pxl_ns_item* items, int n, int steps, const float* coef, float eps, const MuonArgs& ma, int muon,
           void* ws, size_t ws_bytes, void* stream) {
  NsPlan plan;
  std::vector<NsStep> st;
  NS_TRY(ns_check(what, dtype, items, n, steps, coef, eps, muon, plan, st));
  if (n == 0) return PXL_OK;
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
    r.split = ns_split_plan(set.cls, plan.np);
    r.shares = reinterpret_cast<float*>(r.ws + plan.head);
    for (int k = 0; k < r.cs.n; ++k) r.cs.c[k] = set.cls[k];
    std::vector<NsItem> list;
    for (auto& c : set.cls)
      for (int i = 0; i < n; ++i)
        if (items[i].rows == c.rows && items[i].cols == c.cols)
          list.push_back(NsItem{items[i].p, items[i].g, muon ? items[i].mom : nullptr, items[i].scale, 0});
    memset(&r.few, 0, sizeof(r.few));
    if (list.size() <= (size_t)NS_INLINE) {
      memcpy(r.few.it, list.data(), list.size() * sizeof(NsItem));
      r.table = nullptr;
    } else {
      for (size_t at = 0; at < list.size(); at += NS_TABLE) {
        NsTable t;
        const int cnt = (int)(list.size() - at < (size_t)NS_TABLE ? list.size() - at : NS_TABLE);
        memcpy(t.it, &list[at], cnt * sizeof(NsItem));
        hipLaunchKernelGGL(ns_table_kernel, dim3(1), dim3(64), 0, r.st, t, cnt, r.table + at);
        PXL_LAUNCH_CHECK();
      }
    }
    if (dtype == PXL_F32) NS_TRY((ns_run_set<float, 2>(r, st, eps, ma, muon)));
    else if (plan.np == 2) NS_TRY((ns_run_set<bf16_t, 2>(r, st, eps, ma, muon)));
    else NS_TRY((ns_run_set<bf16_t, 1>(r, st, eps, ma, muon)));
  }
  return PXL_OK;
}

}  // namespace

extern "C" size_t pxl_ns_workspace(int dtype, const pxl_ns_item* items, int n) {
  try {
    size_t bytes = 0;                   // (of either form: bf16 matrices run with one plane or two)
    for (int planes = dtype == PXL_F32 ? 2 : 1; planes <= 2; ++planes) {
      NsPlan plan;
      if (ns_plan("ns_workspace", dtype, items, n, planes, plan) != PXL_OK) return 0;
      bytes = std::max(bytes, plan.bytes);
    }
    return bytes;
  } catch (...) {
    return 0;
  }
}

extern "C" size_t pxl_orthogonalize_workspace(int dtype, const pxl_ns_item* items, int n, int steps, const float* coef) {
  try {
    int planes;
    std::vector<NsStep> st;
    NsPlan plan;
    return ns_form("orthogonalize_workspace", dtype, steps, coef, 0, planes, st) == PXL_OK && ns_plan("orthogonalize_workspace", dtype, items, n, planes, plan) == PXL_OK
               ? plan.bytes : 0;
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

static int muon_scalars(double lr, double momentum, double weight_decay) {
  if (!(momentum >= 0.0 && momentum < 1.0) || !std::isfinite(lr) || !std::isfinite(weight_decay))
    return pxl_set_error(PXL_ERR_ARG, "muon_step: lr %g, momentum %g (0 <= momentum < 1), weight decay %g", lr, momentum, weight_decay);
  return PXL_OK;
}

extern "C" int pxl_muon_check(int dtype, const pxl_ns_item* items, int n, int steps, const float* coef, float eps, double lr, double momentum,
                              double weight_decay) {
  NS_TRY(muon_scalars(lr, momentum, weight_decay));
  try {
    NsPlan plan;
    std::vector<NsStep> st;
    return ns_check("muon_step", dtype, items, n, steps, coef, eps, 1, plan, st);
  } catch (...) {
    return pxl_set_error(PXL_ERR_ARG, "muon_step: out of host memory");
  }
}

extern "C" int pxl_muon_step(int dtype, const pxl_ns_item* items, int n, int steps, const float* coef, float eps, double lr, double momentum,
                             int nesterov, double weight_decay, void* ws, size_t ws_bytes, void* stream) {
  NS_TRY(muon_scalars(lr, momentum, weight_decay));
  try {
    return ns_run("muon_step", dtype, items, n, steps, coef, eps, MuonArgs{(float)lr, (float)momentum, (float)(1.0 - momentum), (float)(1.0 - lr * weight_decay), nesterov}, 1, ws, ws_bytes, stream);
  } catch (...) {
    return pxl_set_error(PXL_ERR_ARG, "muon_step: out of host memory");
  }
}
