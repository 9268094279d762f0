// Orthogonalisation of a matrix (or a stack) by Newton-Schulz products, gpx_orthogonalize in include/gpx.h:
//   X = G / (|G|_F + eps);  repeat: A = X X^T, B = b A + c A A, X <- a X + B X      (X is n x m, n <= m)
//
// Numbers.  The polynomial keeps every singular value of X below a bound r that the host computes from the
// coefficients (1.21 for the usual ones), so |X_ij| <= r, |A_ij| <= r^2 and |B_ij| <= max |b t + c t^2|: the
// intermediates are stored in fp16, each scaled by the power of two that puts its bound just under fp16's largest
// value, which leaves values down to 2^-28 of the bound as normal numbers.  Values are two fp16 planes, v = hi + lo with 22 bits,
// and a product three (hi hi + hi lo + lo hi): 1.5e-6 off at worst here, as an fp32 product, at a third of the fp16 rate -- five times
// that of the fp32 matrix instructions.  A bf16 result's error is then that of its rounding alone.
// For bf16 results the caller may choose one plane (GPX_BF16 without GPX_TWO_PLANES) for A, B, X^T and what products read of X, a third of
// the products: 4096 x 4096 3744 -> 1543 us, 1024 x 1024 193 -> 142.  fp16's 11 bits run at bf16's matrix rate and lie 8 times
// nearer.  X itself stays in two planes there, because the term a X hands its rounding on from step to step (a = 3.4 at small singular
// values).  The result's error grows to 1.03 (1024 x 1024) .. 1.07 (512 x 512) .. 1.23 (130 x 260) times that of rounding the exact
// result; with one plane of X to 1.6 times at 512 x 512.
//
// Layout.  Every product has both operands k-contiguous: A needs rows of X; A is symmetric, so A A does too; and
// B X needs rows of X^T, so the step's epilogue writes X in both orientations.  Buffers are padded to multiples of 64
// with zeros, which the iteration preserves.
// The symmetric products compute tiles on and below the diagonal and write them twice.
#include <algorithm>
#include <cmath>

#include "gpx_internal.h"

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16acc __attribute__((ext_vector_type(16)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int PAD = 64;
constexpr int PARTS = 1024;   // partial sums of the norm per matrix

__host__ __device__ inline int pad64(int x) { return (x + PAD - 1) / PAD * PAD; }

template <typename T> __device__ __forceinline__ double to_f64(T v) { return (double)(float)v; }
template <> __device__ __forceinline__ double to_f64<double>(double v) { return v; }

// ---- |G|_F^2: fixed partials per matrix --------------------------------------------------------------------------
// 16 bytes of G at p (16-byte aligned: vec) or its elements one by one, `count` of them valid
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  T x[N];
  __device__ __forceinline__ void load(const T* p, long fs, int count, bool vec) {
    if (vec && count >= N) {
      *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(p);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = e < count ? p[e * fs] : T(0);
    }
  }
};

// whether 16-byte accesses fit: dense along the fast index, every line and matrix on a 16-byte boundary
template <typename T>
__device__ __forceinline__ bool vector_ok(const T* g, long bs, long ss, long fs) {
  constexpr int N = 16 / sizeof(T);
  return fs == 1 && ss % N == 0 && bs % N == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == 0;
}

// Threads run along the unit stride of G (fast index), blocks over the other one; four 16-byte loads under way per thread.
template <typename T>
__global__ __launch_bounds__(256) void ns_norm_kernel(const T* G, long bs, long ss, long fs, int slow, int fast, double* part) {
  constexpr int N = Vec<T>::N, U = 4;
  __shared__ double sm[4];
  const T* g = G + (long)blockIdx.y * bs;
  const bool vec = vector_ok(G, bs, ss, fs);
  double v = 0.0;
  const int per = (fast + 256 * N - 1) / (256 * N);   // a thread's pieces of one line
  const int lines = (slow - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  const long total = (long)lines * per;
  int line = blockIdx.x, piece = 0;
  for (long k = 0; k < total; k += U) {
    Vec<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = (piece * 256 + threadIdx.x) * N;
      const int count = line < slow ? fast - j : 0;
      x[u].load(g + line * ss + j * fs, fs, count, vec);
      if (++piece == per) {
        piece = 0;
        line += gridDim.x;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) v = fma(to_f64(x[u].x[e]), to_f64(x[u].x[e]), v);
  }
  for (int o = 32; o > 0; o >>= 1) v += __shfl_down(v, o);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) part[(long)blockIdx.y * PARTS + blockIdx.x] = (sm[0] + sm[1]) + (sm[2] + sm[3]);
}

// 1 / (sqrt(sum of the partials) + eps); every thread gets it
__device__ __forceinline__ double inv_norm(const double* part, int nparts, double eps, double* sm /* 4 */) {
  double v = 0.0;
  for (int i = threadIdx.x; i < nparts; i += 256) v += part[i];
  for (int o = 32; o > 0; o >>= 1) v += __shfl_down(v, o);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
  __syncthreads();
  return 1.0 / (sqrt((sm[0] + sm[1]) + (sm[2] + sm[3])) + eps);
}

// Where column c of a row is, and from there its low plane, in a row of ld columns: two planes that products read both alternate
// every 32 columns, so that a k-tile of 32 is one line of 128 bytes; otherwise the low plane follows the high one.
template <int NPL> __host__ __device__ __forceinline__ int in_row(int c) { return NPL == 2 ? (c >> 5) * 64 + (c & 31) : c; }
template <int NPL> __host__ __device__ __forceinline__ int to_lo(int ld) { return NPL == 2 ? 32 : ld; }

// ---- X and X^T from G --------------------------------------------------------------------------------------------
// One 64 x 64 tile through LDS, read along G's unit stride, written along rows of X and of X^T.
template <typename T, int NPL>
__global__ __launch_bounds__(256) void ns_pack_kernel(const T* G, long bs, long rs, long cs, int n, int m, const double* part,
                                                      int nparts, double eps, double scale, _Float16* X, _Float16* XT,
                                                      long xs, long ts) {
  __shared__ float tile[64][65];
  __shared__ double sm[4];
  const int z = blockIdx.z, i0 = blockIdx.y * 64, j0 = blockIdx.x * 64, t = threadIdx.x;
  const int np = pad64(n), mp = pad64(m);
  const double f = inv_norm(part + (long)z * PARTS, nparts, eps, sm) * scale;
  const T* g = G + z * bs;
  const bool along_rows = rs == 1 && cs != 1;
  {
    constexpr int N = Vec<T>::N, LANES = 64 / N, LINES = 256 / LANES;   // threads of a line, lines at a time
    const long ss = along_rows ? cs : rs, fs = along_rows ? rs : cs;
    const bool vec = vector_ok(G, bs, ss, fs);
    const int slow0 = along_rows ? j0 : i0, fast0 = along_rows ? i0 : j0, slow = along_rows ? m : n, fast = along_rows ? n : m;
    const int b = (t % LANES) * N;
    Vec<T> x[64 / LINES];
#pragma unroll
    for (int q = 0; q < 64 / LINES; ++q) {
      const int a = q * LINES + t / LANES;
      x[q].load(g + (slow0 + a) * ss + (fast0 + b) * fs, fs, slow0 + a < slow ? fast - fast0 - b : 0, vec);
    }
#pragma unroll
    for (int q = 0; q < 64 / LINES; ++q) {
      const int a = q * LINES + t / LANES;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float v = (float)(to_f64(x[q].x[e]) * f);
        if (along_rows) tile[b + e][a] = v; else tile[a][b + e] = v;
      }
    }
  }
  __syncthreads();
  const int r = t >> 2, c0 = (t & 3) * 16;
  X += z * xs;
  XT += z * ts;
  for (int half = 0; half < 2; ++half) {
    h8 xh, xl, th, tl;
    for (int e = 0; e < 8; ++e) {
      const int c = c0 + half * 8 + e;
      const float x = tile[r][c], y = tile[c][r];
      xh[e] = (_Float16)x;
      xl[e] = (_Float16)(x - (float)xh[e]);
      th[e] = (_Float16)y;
      if (NPL == 2) tl[e] = (_Float16)(y - (float)th[e]);
    }
    const long px = (long)(i0 + r) * 2 * mp + in_row<NPL>(j0 + c0 + half * 8), pt = (long)(j0 + r) * NPL * np + in_row<NPL>(i0 + c0 + half * 8);
    *reinterpret_cast<h8*>(X + px) = xh;
    *reinterpret_cast<h8*>(X + px + to_lo<NPL>(mp)) = xl;
    *reinterpret_cast<h8*>(XT + pt) = th;
    if (NPL == 2) *reinterpret_cast<h8*>(XT + pt + to_lo<NPL>(np)) = tl;
  }
}

#define NS_TRY(expr)          \
  do {                        \
    int rc_ = (expr);         \
    if (rc_ != 0) return rc_; \
  } while (0)

// ---- the product -------------------------------------------------------------------------------------------------
// v = ca * E + cc * (A B^T); v goes to D [row][col], to DT [col][row], or as alpha * v + beta * base to the caller's
// matrix.
struct NsGemm {
  const _Float16 *A, *B, *E;   // A: M rows, B: N rows, both K long; E like D
  _Float16 *D, *DT;
  long lda, ldb;               // elements from row to row of A and B, all planes
  int dpl;                     // planes of D and E; DT has the products' planes
  long sa, sb, sd, st;         // strides of the stack: A, B, D and E, DT
  int M, N, K;                 // padded to 64
  int lower;                   // M == N, tiles on and below the diagonal, DT == D
  float ca, cc;
  // last step only
  int out_type;                // -1: none
  void* out;
  const void* base;
  long obs, ors, ocs, bbs, brs, bcs;
  int n, m;
  float alpha, beta;
  // K split over `parts` workgroups per tile: their sums, [part][matrix][M][N], for ns_join_kernel
  float* sums;
  int parts;
};

// the k-tiles of this workgroup, from blockIdx.z
__device__ __forceinline__ void k_range(const NsGemm& g, int nk, int& first, int& count) {
  first = (int)((long)nk * blockIdx.z / g.parts);
  count = (int)((long)nk * (blockIdx.z + 1) / g.parts) - first;
}

// the sums of one part, EM x EN of them at (row0, col0): stage() leaves them in st (pitch EN + 4)
template <int EM, int EN, typename F>
__device__ __forceinline__ void keep_sums(const NsGemm& g, const float* st, long z, int row0, int col0, int lane, F stage) {
  constexpr int RL = EN / 4, RR = 64 / RL;   // lanes per row, rows at a time
  float* dst = g.sums + (((long)blockIdx.z * gridDim.y + z) * g.M + row0) * g.N + col0 + (lane % RL) * 4;
  stage();
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int r = lane / RL; r < EM; r += RR)
    *reinterpret_cast<f4*>(dst + (long)r * g.N) = *reinterpret_cast<const f4*>(st + r * (EN + 4) + (lane % RL) * 4);
  __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, unsigned voff, unsigned soff, char* dst_wave) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst_wave, 16, voff, soff, 0, 0);
}

// alpha * v + beta * base to the caller's matrix, lanes along its unit stride, 16 elements of base under way at once
template <typename T, int EM, int EN, int P>
__device__ __forceinline__ void write_out(const NsGemm& g, const float* st, long z, int row0, int col0, int lane) {
  const bool along_rows = g.ors == 1 && g.ocs != 1;
  const int fast = along_rows ? EM : EN, per = 64 / fast;   // lanes of a line, lines at a time
  const int lines = (along_rows ? EN : EM) / per, f = lane % fast, l0 = lane / fast;
  T* out = reinterpret_cast<T*>(g.out) + z * g.obs;
  const T* base = g.base == nullptr ? nullptr : reinterpret_cast<const T*>(g.base) + z * g.bbs;
  for (int q0 = 0; q0 < lines; q0 += 16) {
    float old[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const int l = (q0 + u) * per + l0, i = row0 + (along_rows ? f : l), j = col0 + (along_rows ? l : f);
      old[u] = base != nullptr && i < g.n && j < g.m ? (float)base[i * g.brs + j * g.bcs] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const int l = (q0 + u) * per + l0, r = along_rows ? f : l, c = along_rows ? l : f, i = row0 + r, j = col0 + c;
      if (i < g.n && j < g.m) {
        float v = g.alpha * st[r * P + c];
        if (base != nullptr) v = fmaf(g.beta, old[u], v);
        out[i * g.ors + j * g.ocs] = (T)v;
      }
    }
  }
}

// The end of a product for EM x EN of its elements at (row0, col0): stage() leaves the sums in st (pitch EN + 4); every load of E is
// under way before.
template <int NPL, int EM, int EN, typename F>
__device__ __forceinline__ void finish(const NsGemm& g, float* st, long z, int row0, int col0, int lane, bool mirror, F stage) {
  constexpr int P = EN + 4;
  constexpr int RL = EN / 8, RR = 64 / RL, RQ = EM / RR;   // row pass: lanes per row, rows at a time, times
  constexpr int CL = EM / 8, CR = 64 / CL, CQ = EN / CR;   // column pass
  const long ldd = (long)g.dpl * g.N, ldt = (long)NPL * g.M;
  const bool two = g.dpl == 2;
  const _Float16* E = g.E == nullptr ? nullptr : g.E + z * g.sd;
  _Float16* D = g.D == nullptr ? nullptr : g.D + z * g.sd;
  _Float16* DT = g.DT == nullptr ? nullptr : g.DT + z * g.st;
  h8 eh[RQ], el[RQ];
#pragma unroll
  for (int q = 0; q < RQ; ++q) {
    eh[q] = el[q] = h8{0, 0, 0, 0, 0, 0, 0, 0};
    if (E != nullptr) {
      const _Float16* src = E + (row0 + q * RR + lane / RL) * ldd + in_row<NPL>(col0 + (lane % RL) * 8);
      eh[q] = *reinterpret_cast<const h8*>(src);
      if (two) el[q] = *reinterpret_cast<const h8*>(src + to_lo<NPL>(g.N));
    }
  }
  stage();
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int q = 0; q < RQ; ++q) {
    const int r = q * RR + lane / RL, c = (lane % RL) * 8;
    float* p = st + r * P + c;
    float v[8];
    h8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = fmaf(g.ca, (float)eh[q][e] + (float)el[q][e], g.cc * p[e]);
      hi[e] = (_Float16)v[e];
      lo[e] = (_Float16)(v[e] - (float)hi[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = v[e];
    if (D != nullptr) {
      _Float16* dst = D + (row0 + r) * ldd + in_row<NPL>(col0 + c);
      *reinterpret_cast<h8*>(dst) = hi;
      if (two) *reinterpret_cast<h8*>(dst + to_lo<NPL>(g.N)) = lo;
    }
  }
  __builtin_amdgcn_wave_barrier();
  if (DT != nullptr && mirror) {
#pragma unroll
    for (int q = 0; q < CQ; ++q) {
      const int c = q * CR + lane / CL, r = (lane % CL) * 8;
      h8 hi, lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = st[(r + e) * P + c];
        hi[e] = (_Float16)v;
        lo[e] = (_Float16)(v - (float)hi[e]);
      }
      _Float16* dst = DT + (col0 + c) * ldt + in_row<NPL>(row0 + r);
      *reinterpret_cast<h8*>(dst) = hi;
      if (NPL == 2) *reinterpret_cast<h8*>(dst + to_lo<NPL>(g.M)) = lo;
    }
  }
  if (g.out_type == GPX_F32) write_out<float, EM, EN, P>(g, st, z, row0, col0, lane);
  else if (g.out_type == GPX_F16) write_out<_Float16, EM, EN, P>(g, st, z, row0, col0, lane);
  else if (g.out_type == GPX_BF16) write_out<__bf16, EM, EN, P>(g, st, z, row0, col0, lane);
  __builtin_amdgcn_wave_barrier();
}

// The tile of this workgroup.  Workgroups with equal id % 8 share an XCD and its L2: each XCD takes a run of consecutive
// tiles, four tile rows high.
__device__ __forceinline__ void tile_of(int lower, int tiles_m, int tiles_n, int& ti, int& tj) {
  const unsigned per = gridDim.x >> 3, rest = gridDim.x & 7, x = blockIdx.x & 7;
  const unsigned id = x * per + min(x, rest) + (blockIdx.x >> 3);
  if (lower) {
    unsigned r = (unsigned)((sqrtf(8.f * (float)id + 1.f) - 1.f) * 0.5f);
    while ((r + 1) * (r + 2) / 2 <= id) ++r;
    while (r * (r + 1) / 2 > id) --r;
    ti = r;
    tj = id - r * (r + 1) / 2;
  } else {
    const unsigned band = id / (4 * tiles_n), in = id % (4 * tiles_n), high = min(4u, (unsigned)tiles_m - band * 4);
    ti = band * 4 + in % high;
    tj = in / high;
  }
}

// Tile BM x BN, WAVES_M x WAVES_N waves of (BM / WAVES_M) x (BN / WAVES_N) each in 32 x 32 x 16 matrix instructions.
// A k-tile is 64 / NPL long: an LDS row is 128 bytes either way, 8 chunks of 16 bytes (NPL = 2: four of hi, four of
// lo), chunk c of row r in slot c ^ (r >> 1 & 7): 16 rows cover the 64 banks once in a 16-byte fragment read.
template <int BM, int BN, int WAVES_M, int WAVES_N, int NPL, int STAGES>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N) void ns_gemm_kernel(const NsGemm g, int tiles_m, int tiles_n) {
  constexpr int NW = WAVES_M * WAVES_N, NT = 64 * NW;
  constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, TM = WM / 32, TN = WN / 32;
  constexpr int BK = 64 / NPL, KS = BK / 16;
  constexpr int ABYTES = BM * 128, STAGE = (BM + BN) * 128;
  extern __shared__ __align__(16) char smem[];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  int ti, tj;
  tile_of(g.lower, tiles_m, tiles_n, ti, tj);
  const int i0 = ti * BM, j0 = tj * BN;
  const long z = blockIdx.y;
  const long lda = g.lda * 2, ldb = g.ldb * 2;   // bytes
  const __amdgpu_buffer_rsrc_t ra =
      __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)(g.A + z * g.sa) + i0 * lda), 0, 0x7fffffff, 0x00020000);
  const __amdgpu_buffer_rsrc_t rb =
      __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)(g.B + z * g.sb) + j0 * ldb), 0, 0x7fffffff, 0x00020000);
  // per-lane sources of the DMA: piece p of NT lanes covers rows p * (NT / 8) ..; rows behind the matrix repeat its last
  constexpr int PA = BM * 8 / NT, PB = BN * 8 / NT;
  unsigned va[PA], vb[PB];
#pragma unroll
  for (int p = 0; p < PA; ++p) {
    const int s = p * NT + t, r = s >> 3, c = (s & 7) ^ ((r >> 1) & 7);
    const int rr = min(r, g.M - 1 - i0);
    va[p] = (unsigned)(rr * lda + c * 16);
  }
#pragma unroll
  for (int p = 0; p < PB; ++p) {
    const int s = p * NT + t, r = s >> 3, c = (s & 7) ^ ((r >> 1) & 7);
    const int rr = min(r, g.N - 1 - j0);
    vb[p] = (unsigned)(rr * ldb + c * 16);
  }
  auto load = [&](int kt, char* stage) {
    char* sA = stage + wave * 1024;
    char* sB = sA + ABYTES;
    const unsigned so = (unsigned)kt * 128;
#pragma unroll
    for (int p = 0; p < PA; ++p) dma16(ra, va[p], so, sA + p * (NT * 16));
#pragma unroll
    for (int p = 0; p < PB; ++p) dma16(rb, vb[p], so, sB + p * (NT * 16));
  };
  f16acc acc[TM][TN];
#pragma unroll
  for (int a = 0; a < TM; ++a)
#pragma unroll
    for (int b = 0; b < TN; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[a][b][e] = 0.f;
  const int wm = wave / WAVES_N, wn = wave % WAVES_N;
  const int r32 = lane & 31, kh = lane >> 5;
  const int nk = g.K / BK;
  const int offA = (wm * WM + r32) * 128, offB = ABYTES + (wn * WN + r32) * 128;
  h8 fa[2][TM][NPL], fb[2][TN][NPL];
  auto fetch = [&](const char* stage, int s, int set) {
    const int o0 = (((s * 2 + kh) ^ ((r32 >> 1) & 7)) * 16);
#pragma unroll
    for (int pl = 0; pl < NPL; ++pl) {
      const int o = o0 ^ (pl * 64);
#pragma unroll
      for (int a = 0; a < TM; ++a) fa[set][a][pl] = *reinterpret_cast<const h8*>(stage + offA + a * 32 * 128 + o);
#pragma unroll
      for (int b = 0; b < TN; ++b) fb[set][b][pl] = *reinterpret_cast<const h8*>(stage + offB + b * 32 * 128 + o);
    }
  };
  auto multiply = [&](int set) {
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
      for (int b = 0; b < TN; ++b) {
        if (NPL == 2) {
          acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[set][a][0], fb[set][b][NPL - 1], acc[a][b], 0, 0, 0);
          acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[set][a][NPL - 1], fb[set][b][0], acc[a][b], 0, 0, 0);
        }
        acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[set][a][0], fb[set][b][0], acc[a][b], 0, 0, 0);
      }
  };
  // STAGES k-tiles are in flight.  The one barrier of a k-tile comes before its last matrix instructions, when every wave holds
  // its last fragments: the stage is refilled and the next tile's first fragments are read under those.
  constexpr int L = PA + PB;
#pragma unroll
  for (int p = 0; p < STAGES; ++p)
    if (p < nk) load(p, smem + p * STAGE);
  if (nk >= STAGES)
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * L) : "memory");
  else
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  fetch(smem, 0, 0);
  int cur = 0;
  for (int kt = 0; kt < nk; ++kt) {
    const int nxt = cur + 1 == STAGES ? 0 : cur + 1;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if (s + 1 < KS) {
        fetch(smem + cur * STAGE, s + 1, (s + 1) & 1);
      } else if (kt + 1 < nk) {
        if (kt + STAGES <= nk)   // tiles kt + 1 .. kt + STAGES - 1 are under way: wait for the first of them
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * L) : "memory");
        else
          asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (kt + STAGES < nk) load(kt + STAGES, smem + cur * STAGE);
        fetch(smem + nxt * STAGE, 0, (s + 1) & 1);
      }
      multiply(s & 1);
    }
    cur = nxt;
  }
  static_assert(KS % 2 == 0, "the fragment sets alternate");
  static_assert((STAGES - 1) * L < 64, "vmcnt has six bits");
  __syncthreads();   // the stages become the waves' own staging of 64 x 64 blocks
  constexpr int EM = WM % 64 ? 32 : 64, EN = WN % 64 ? 32 : 64, P = EN + 4;
  float* st = reinterpret_cast<float*>(smem) + wave * (EM * P);
#pragma unroll
  for (int bi = 0; bi < WM / EM; ++bi)
#pragma unroll
    for (int bj = 0; bj < WN / EN; ++bj) {
      const int row0 = i0 + wm * WM + bi * EM, col0 = j0 + wn * WN + bj * EN;
      if (row0 >= g.M || col0 >= g.N) continue;   // uniform in the wave; sizes are multiples of 64
      finish<NPL, EM, EN>(g, st, z, row0, col0, lane, !(g.lower && ti == tj), [&] {
#pragma unroll
        for (int a = 0; a < EM / 32; ++a)
#pragma unroll
          for (int b = 0; b < EN / 32; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              st[(a * 32 + (e >> 2) * 8 + kh * 4 + (e & 3)) * P + b * 32 + r32] = acc[bi * (EM / 32) + a][bj * (EN / 32) + b][e];
      });
    }
}

// Small problems, where latency counts and not the rate: a 64 x 64 tile per workgroup, whose W waves take every
// W-th k-tile each, with stages of their own and no barrier, and add their sums through LDS in the order of the waves.  n = 1024, one
// plane: 8.4 us for A A, about 4 of which a launch takes that does nothing else; 16 TB/s from L2.
template <int W, int NPL, int STAGES, bool SPLIT>
__global__ __launch_bounds__(64 * W) void ns_small_kernel(const NsGemm g, int tiles_m, int tiles_n) {
  constexpr int BK = 64 / NPL, KS = BK / 16, STAGE = 128 * 128, P = 68, L = 16, ROWS = 64 / W;
  static_assert(STAGES * L < 64, "vmcnt has six bits");
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int ti, tj;
  tile_of(g.lower, tiles_m, tiles_n, ti, tj);
  const int i0 = ti * 64, j0 = tj * 64;
  const long z = blockIdx.y;
  const long lda = g.lda * 2, ldb = g.ldb * 2;   // bytes
  const __amdgpu_buffer_rsrc_t ra =
      __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)(g.A + z * g.sa) + i0 * lda), 0, 0x7fffffff, 0x00020000);
  const __amdgpu_buffer_rsrc_t rb =
      __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)(g.B + z * g.sb) + j0 * ldb), 0, 0x7fffffff, 0x00020000);
  // piece p: rows 8 p .. 8 p + 7 of a tile, whose sizes are multiples of 64
  unsigned va[8], vb[8];
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const int r = p * 8 + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
    va[p] = (unsigned)(r * lda + c * 16);
    vb[p] = (unsigned)(r * ldb + c * 16);
  }
  char* mine = smem + wave * (STAGES * STAGE);
  auto load = [&](int kt, int stage) {
    char* d = mine + stage * STAGE;
    const unsigned so = (unsigned)kt * 128;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      dma16(ra, va[p], so, d + p * 1024);
      dma16(rb, vb[p], so, d + 8192 + p * 1024);
    }
  };
  f16acc acc[2][2];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[a][b][e] = 0.f;
  const int r32 = lane & 31, kh = lane >> 5;
  int k0 = 0, nk = g.K / BK;
  if (SPLIT) k_range(g, g.K / BK, k0, nk);
  const int own = nk > wave ? (nk - wave + W - 1) / W : 0;   // k-tiles wave, wave + W, ..
#pragma unroll
  for (int p = 0; p < STAGES; ++p)
    if (p < own) load(k0 + wave + p * W, p);
  int cur = 0;
  for (int n = 0; n < own; ++n) {
    if (n + STAGES <= own)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * L) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const char* sA = mine + cur * STAGE + r32 * 128;
    h8 fa[KS][2][NPL], fb[KS][2][NPL];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int pl = 0; pl < NPL; ++pl) {
        const int o = (((s * 2 + kh) ^ ((r32 >> 1) & 7)) * 16) ^ (pl * 64);
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          fa[s][a][pl] = *reinterpret_cast<const h8*>(sA + a * 4096 + o);
          fb[s][a][pl] = *reinterpret_cast<const h8*>(sA + 8192 + a * 4096 + o);
        }
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // in registers: the stage may be filled again
    if (n + STAGES < own) load(k0 + wave + (n + STAGES) * W, cur);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if (NPL == 2) {
            acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[s][a][0], fb[s][b][NPL - 1], acc[a][b], 0, 0, 0);
            acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[s][a][NPL - 1], fb[s][b][0], acc[a][b], 0, 0, 0);
          }
          acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[s][a][0], fb[s][b][0], acc[a][b], 0, 0, 0);
        }
    cur = cur + 1 == STAGES ? 0 : cur + 1;
  }
  __syncthreads();   // the stages become the waves' sums, 64 x 64 each
  float* sum = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        sum[(wave * 64 + a * 32 + (e >> 2) * 8 + kh * 4 + (e & 3)) * P + b * 32 + r32] = acc[a][b][e];
  __syncthreads();
  // wave w: the rows ROWS w .. of all sums; they end in the first
  float* st = sum + wave * ROWS * P;
  auto stage = [&] {
    constexpr int Q = ROWS * 64 / 4 / 64;   // four columns a lane
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = q * 64 + lane, r = i >> 4, c = (i & 15) * 4;
      f4 v = *reinterpret_cast<const f4*>(st + r * P + c);
#pragma unroll
      for (int w = 1; w < W; ++w) v += *reinterpret_cast<const f4*>(st + w * 64 * P + r * P + c);
      *reinterpret_cast<f4*>(st + r * P + c) = v;
    }
  };
  if (SPLIT)
    keep_sums<ROWS, 64>(g, st, z, i0 + wave * ROWS, j0, lane, stage);
  else
    finish<NPL, ROWS, 64>(g, st, z, i0 + wave * ROWS, j0, lane, !(g.lower && ti == tj), stage);
}

// The end of a product whose K was split: 64 x 64 a workgroup, the parts added in their order.
__global__ __launch_bounds__(256) void ns_join_kernel(const NsGemm g, int tiles_m, int tiles_n) {
  constexpr int P = 68, ROWS = 16, Q = ROWS * 64 / 4 / 64;
  __shared__ __align__(16) float smem[4 * ROWS * P];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int ti, tj;
  tile_of(g.lower, tiles_m, tiles_n, ti, tj);
  const long z = blockIdx.y;
  const int row0 = ti * 64 + wave * ROWS, col0 = tj * 64;
  float* st = smem + wave * ROWS * P;
  finish<2, ROWS, 64>(g, st, z, row0, col0, lane, !(g.lower && ti == tj), [&] {
    const long part = (long)gridDim.y * g.M * g.N;
    const float* src = g.sums + (z * g.M + row0) * g.N + col0;
    f4 v[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) v[q] = f4{0, 0, 0, 0};
#pragma unroll 4
    for (int p = 0; p < g.parts; ++p, src += part)
#pragma unroll
      for (int q = 0; q < Q; ++q) v[q] += *reinterpret_cast<const f4*>(src + (long)(q * 4 + (lane >> 4)) * g.N + (lane & 15) * 4);
#pragma unroll
    for (int q = 0; q < Q; ++q) *reinterpret_cast<f4*>(st + (q * 4 + (lane >> 4)) * P + (lane & 15) * 4) = v[q];
  });
}

template <int BM, int BN, int WAVES_M, int WAVES_N, int NPL, int STAGES>
int launch_cfg(hipStream_t s, const NsGemm& g, int batch) {
  constexpr int NW = WAVES_M * WAVES_N;
  constexpr size_t lds = std::max<size_t>(STAGES * (BM + BN) * 128, (size_t)NW * (BM / WAVES_M % 64 ? 32 : 64) * ((BN / WAVES_N % 64 ? 32 : 64) + 4) * 4);
  static_assert(BM * 8 % (64 * NW) == 0 && BN * 8 % (64 * NW) == 0 && BM / WAVES_M % 32 == 0 && BN / WAVES_N % 32 == 0, "tile");
  static_assert(lds <= 160 * 1024, "LDS");
  GPX_REQUIRE(!g.lower || BM == BN, "ns_gemm: half products need square tiles");
  const int tm = (g.M + BM - 1) / BM, tn = (g.N + BN - 1) / BN;
  const unsigned tiles = g.lower ? (unsigned)tm * (tm + 1) / 2 : (unsigned)tm * tn;
  static thread_local bool set[GPX_MAX_DEVICES] = {};
  int dev = 0;
  GPX_HIP(hipGetDevice(&dev));
  if (dev < GPX_MAX_DEVICES && !set[dev]) {
    GPX_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&ns_gemm_kernel<BM, BN, WAVES_M, WAVES_N, NPL, STAGES>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    set[dev] = true;
  }
  hipLaunchKernelGGL((ns_gemm_kernel<BM, BN, WAVES_M, WAVES_N, NPL, STAGES>), dim3(tiles, batch), dim3(64 * NW), lds, s, g, tm, tn);
  GPX_HIP(hipGetLastError());
  return 0;
}

template <int W, int NPL, int STAGES, bool SPLIT>
int launch_small(hipStream_t s, const NsGemm& g, int batch) {
  constexpr size_t lds = std::max<size_t>((size_t)W * STAGES * 128 * 128, (size_t)W * 64 * 68 * 4);
  static_assert(lds <= 160 * 1024, "LDS");
  const int tm = g.M / 64, tn = g.N / 64;
  static thread_local bool set[GPX_MAX_DEVICES] = {};
  int dev = 0;
  GPX_HIP(hipGetDevice(&dev));
  if (dev < GPX_MAX_DEVICES && !set[dev]) {
    GPX_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&ns_small_kernel<W, NPL, STAGES, SPLIT>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    set[dev] = true;
  }
  hipLaunchKernelGGL((ns_small_kernel<W, NPL, STAGES, SPLIT>), dim3(g.lower ? (unsigned)tm * (tm + 1) / 2 : (unsigned)tm * tn, batch, SPLIT ? g.parts : 1),
                     dim3(64 * W), lds, s, g, tm, tn);
  GPX_HIP(hipGetLastError());
  return 0;
}

// Tile by estimated time: rounds of the chip times what one round of a tile takes (measured at K = 4096, one plane, us;
// two planes keep the ratios): 64 x 64 with 4 waves (ns_small_kernel), two on a CU, 34; 128 x 128 with 8 waves 42; 192 x 192 with 6 waves
// 84; 256 x 256 with 8 waves 110.  Larger tiles read LDS less per product, smaller ones fill the chip: A A at n = 4096
// takes 162 / 117 / 84 / 97 us with them, B X 233 / 173 / 169 / 140, at n = 1024 8.4 / 14 / 26 / 35 and 9.3 / 14 / 27 / 36.
//
// A product A A^T of two planes with few tiles and a long K leaves most of the chip idle while a tile's time goes with the bytes
// that its CU loads, 5 to 7 ns per k.  K is then split over workgroups, at the price of a launch and of the sums to memory and back,
// as far as all run at once: 10 tiles with K = 4096 24 -> 14 us, 55 with 4032 26 -> 17, 66 with 2560 21 -> 16; not 136 of K = 3008
// (which would be a second round: 23 -> 25), not of one plane (10 tiles with K = 4096 15 -> 14), and not larger tiles, which keep more
// of the chip busy (136 of 128 x 128 with K = 8192 174 -> 148, nothing of it left in the whole call).
struct Choice {
  int tile, parts;   // tile: of TILE
};
constexpr int TILE[4] = {64, 128, 192, 256};
template <int NPL>
Choice choose(int M, int N, int K, int lower, int batch) {
  const int slots[4] = {512, 256, 256, 256};
  const double unit[4] = {34, 42, 84, 110};
  Choice best = {0, 1};
  double least = 0, tiles = 0;
  for (int i = 0; i < 4; ++i) {
    const double tm = (M + TILE[i] - 1) / TILE[i], tn = (N + TILE[i] - 1) / TILE[i], t = (lower ? tm * (tm + 1) / 2 : tm * tn) * batch;
    const double cost = std::ceil(t / slots[i]) * unit[i];
    if (i == 0 || cost < least) {
      best.tile = i;
      least = cost;
      tiles = t;
    }
  }
  if (NPL == 2 && lower && best.tile == 0) {
    double gain = 2;   // us
    for (int p = 2; p <= 8 && tiles * p <= 256; ++p) {
      const double g = K * (0.0048 + tiles * 0.00003) * (1 - 1.0 / p) - 3 - p * (0.8 + tiles * 0.008);
      if (g > gain) {
        gain = g;
        best.parts = p;
      }
    }
  }
  return best;
}

template <int NPL>
int ns_gemm(hipStream_t s, NsGemm g, int batch) {
  const Choice c = choose<NPL>(g.M, g.N, g.K, g.lower, batch);
  g.parts = c.parts;
  if constexpr (NPL == 2) {
    if (c.parts > 1) {
      NS_TRY((launch_small<4, NPL, 1, true>(s, g, batch)));
      const int tm = g.M / 64;
      hipLaunchKernelGGL(ns_join_kernel, dim3((unsigned)tm * (tm + 1) / 2, batch), dim3(256), 0, s, g, tm, tm);
      GPX_HIP(hipGetLastError());
      return 0;
    }
  }
  switch (c.tile) {
    case 0: return launch_small<4, NPL, 1, false>(s, g, batch);
    case 1: return launch_cfg<128, 128, 2, 4, NPL, 4>(s, g, batch);
    case 2: return launch_cfg<192, 192, 2, 3, NPL, 3>(s, g, batch);
    default: return launch_cfg<256, 256, 2, 4, NPL, 2>(s, g, batch);
  }
}

// bytes of the sums that the products of a call keep, two planes
size_t sums_bytes(int np, int mp, int batch) {
  const int parts = std::max(choose<2>(np, np, mp, 1, batch).parts, choose<2>(np, np, np, 1, batch).parts);
  return parts == 1 ? 0 : (size_t)parts * batch * np * np * 4;
}

// ---- fp64: the framework's own products ----------------------------------------------------------------------------
__global__ __launch_bounds__(256) void ns_pack_f64_kernel(const double* G, long bs, long rs, long cs, int n, int m,
                                                          const double* part, int nparts, double eps, double* X, double* Y, int rows, long ldx) {
  __shared__ double tile[64][65];
  __shared__ double sm[4];
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64, t = threadIdx.x;
  const double f = inv_norm(part + (long)blockIdx.z * PARTS, nparts, eps, sm);
  const bool along_rows = rs == 1 && cs != 1;
  G += blockIdx.z * bs;
  X += blockIdx.z * (rows * ldx);
  Y += blockIdx.z * (rows * ldx);
  for (int q = 0; q < 16; ++q) {
    const int a = q * 4 + (t >> 6), b = t & 63;
    const int i = along_rows ? b : a, j = along_rows ? a : b;
    if (i0 + i < n && j0 + j < m) tile[i][j] = G[(i0 + i) * rs + (j0 + j) * cs] * f;
  }
  __syncthreads();
  for (int q = 0; q < 16; ++q) {
    const int i = q * 4 + (t >> 6), j = t & 63;
    if (i0 + i >= rows || j0 + j >= ldx) continue;
    const bool in = i0 + i < n && j0 + j < m;
    X[(i0 + i) * ldx + j0 + j] = in ? tile[i][j] : 0.0;
    if (!in) Y[(i0 + i) * ldx + j0 + j] = 0.0;   // the other buffer's padding too
  }
}

// S = alpha sum of the parts + beta base for symmetric n x n matrices of which the parts hold the lower triangle; S whole, with zeros
// in its padding.  32 x 32 a workgroup, every load under way at once.
template <int PARTS_>
__global__ __launch_bounds__(256) void ns_join_f64_kernel(int n, const double* sums, double alpha, double beta, const double* base,
                                                          double* S, long ld) {
  __shared__ double tile[32][33];
  const int bi = blockIdx.y, bj = blockIdx.x, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  if (bj > bi) return;
  const long part = n * ld;
  sums += blockIdx.z * (PARTS_ * part);
  S += blockIdx.z * part;
  if (base != nullptr) base += blockIdx.z * part;
  double v[4][PARTS_], b[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int i = min(bi * 32 + q * 8 + ty, n - 1), j = min(bj * 32 + tx, i);
    b[q] = base != nullptr ? base[i * ld + j] : 0.0;
#pragma unroll
    for (int p = 0; p < PARTS_; ++p) v[q][p] = sums[p * part + i * ld + j];
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = q * 8 + ty, i = bi * 32 + r, j = bj * 32 + tx;
    double x = v[q][0];
#pragma unroll
    for (int p = 1; p < PARTS_; ++p) x += v[q][p];
    x = base != nullptr ? alpha * x + beta * b[q] : alpha * x;
    tile[r][tx] = x;
    if (i < n && j <= i) S[i * ld + j] = x;
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = q * 8 + ty, i = bj * 32 + r, j = bi * 32 + tx;   // the mirror image
    if (i < n && j > i && j < ld) S[i * ld + j] = j < n ? tile[tx][r] : 0.0;
  }
}

// Y = alpha X + the sum of the parts, n x m; a row of a matrix a workgroup
template <int PARTS_>
__global__ __launch_bounds__(256) void ns_sum_f64_kernel(int n, int m, const double* sums, double alpha, const double* X, double* Y,
                                                         int rows, long ld) {
  const long at = blockIdx.z * (rows * ld) + blockIdx.y * ld, part = n * ld;
  sums += blockIdx.z * (PARTS_ * part) + blockIdx.y * ld;
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= m) return;
  double v[PARTS_], x = alpha * X[at + j];
#pragma unroll
  for (int p = 0; p < PARTS_; ++p) v[p] = sums[p * part + j];
#pragma unroll
  for (int p = 0; p < PARTS_; ++p) x += v[p];
  Y[at + j] = x;
}

__global__ __launch_bounds__(256) void ns_out_f64_kernel(const double* X, long ldx, int n, int m, double* out, long bs, long rs,
                                                         long cs, const double* base, long bbs, long brs, long bcs, double alpha,
                                                         double beta, int rows) {
  __shared__ double tile[64][65];
  X += blockIdx.z * (rows * ldx);
  out += blockIdx.z * bs;
  if (base != nullptr) base += blockIdx.z * bbs;
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64, t = threadIdx.x;
  for (int q = 0; q < 16; ++q) {
    const int i = q * 4 + (t >> 6), j = t & 63;
    if (i0 + i < n && j0 + j < m) tile[i][j] = X[(i0 + i) * ldx + j0 + j];
  }
  __syncthreads();
  const bool along_rows = rs == 1 && cs != 1;
  for (int q = 0; q < 16; ++q) {
    const int a = q * 4 + (t >> 6), b = t & 63;
    const int i = along_rows ? b : a, j = along_rows ? a : b;
    if (i0 + i >= n || j0 + j >= m) continue;
    double v = alpha * tile[i][j];
    if (base != nullptr) v += beta * base[(i0 + i) * brs + (j0 + j) * bcs];
    out[(i0 + i) * rs + (j0 + j) * cs] = v;
  }
}

long pad32(long x) { return (x + 31) / 32 * 32; }

GemmDesc product(const double* A, long lda, const double* B, long ldb, int b_lay, const double* C, double* D, long ldd, int M,
                 int N, int K, double alpha, double beta, int lower) {
  GemmDesc g;
  g.A = A; g.lda = lda; g.a_lay = GPX_LAY_KC; g.a_tri = 0;
  g.B = B; g.ldb = ldb; g.b_lay = b_lay; g.b_tri = 0;
  g.Cin = C; g.ldcin = ldd;
  g.D = D; g.ldd = ldd;
  g.M = M; g.N = N; g.K = K; g.alpha = alpha; g.beta = beta;
  g.c_lower = lower; g.diag_add = 0.0; g.inplace = 0;
  return g;
}

// the largest |s (a + b s^2 + c s^4)| for 0 <= s <= r
double step_bound(const double* k, double r) {
  auto f = [&](double s) { const double t = s * s; return std::fabs(s * (k[0] + t * (k[1] + t * k[2]))); };
  double best = f(r);
  // stationary points: a + 3 b t + 5 c t^2 = 0
  const double A = 5 * k[2], B = 3 * k[1], C = k[0], disc = B * B - 4 * A * C;
  if (A != 0.0 && disc >= 0.0) {
    for (double sg : {-1.0, 1.0}) {
      const double t = (-B + sg * std::sqrt(disc)) / (2 * A);
      if (t > 0 && t < r * r) best = std::fmax(best, f(std::sqrt(t)));
    }
  } else if (A == 0.0 && B != 0.0) {
    const double t = -C / B;
    if (t > 0 && t < r * r) best = std::fmax(best, f(std::sqrt(t)));
  }
  return best;
}
// the largest |b t + c t^2| for 0 <= t <= r^2
double poly_bound(const double* k, double r) {
  auto f = [&](double t) { return std::fabs(t * (k[1] + t * k[2])); };
  double best = f(r * r);
  if (k[2] != 0.0) {
    const double t = -k[1] / (2 * k[2]);
    if (t > 0 && t < r * r) best = std::fmax(best, f(t));
  }
  return best;
}
// exponent that puts values of at most `bound` (and 5 % for rounding) under 2^14, a quarter of fp16's largest; under 1e-30, where a
// polynomial that shrinks X may lead, the factors between the scales would leave fp32's range
int scale_exp(double bound) { return 14 - (int)std::ceil(std::log2(std::fmax(bound, 1e-30) * 1.05)); }

int planes_of(int dtype) { return dtype == GPX_BF16 ? 1 : 2; }

bool dtype_ok(int dtype) { return dtype == GPX_F64 || dtype == GPX_F32 || dtype == GPX_F16 || dtype == GPX_BF16 || dtype == (GPX_BF16 | GPX_TWO_PLANES); }

template <typename T>
int norm_launch(hipStream_t s, const void* G, long bs, long rs, long cs, int n, int m, int batch, double* part, int& nparts) {
  const bool along_rows = rs == 1 && cs != 1;
  const int slow = along_rows ? m : n, fast = along_rows ? n : m;
  // a block for every 8192 elements: more would only make the sums of the partials longer
  const long blocks = std::max(1L, (long)n * m / 8192);
  nparts = (int)std::min<long>(std::min(slow, PARTS), blocks);
  hipLaunchKernelGGL((ns_norm_kernel<T>), dim3(nparts, batch), dim3(256), 0, s, (const T*)G, bs, along_rows ? cs : rs,
                     along_rows ? rs : cs, slow, fast, part);
  GPX_HIP(hipGetLastError());
  return 0;
}

template <typename T, int NPL>
int run_half(hipStream_t s, int dtype, int batch, int n, int m, const void* G, long bs, long rs, long cs, int steps,
             const double* k, double eps, double alpha, double beta, const void* base, const long* bst, void* out, const long* ost,
             char* work) {
  const int np = pad64(n), mp = pad64(m);
  const long xs = (long)np * mp * 2, ts = (long)np * mp * NPL, as = (long)np * np * NPL;
  double* part = reinterpret_cast<double*>(work);
  _Float16* X[2];
  _Float16* XT[2];
  _Float16* p = reinterpret_cast<_Float16*>(work + (size_t)batch * PARTS * 8);
  X[0] = p; p += batch * xs;
  X[1] = p; p += batch * xs;
  XT[0] = p; p += batch * ts;
  XT[1] = p; p += batch * ts;
  _Float16* A = p; p += batch * as;
  _Float16* B = p; p += batch * as;
  float* sums = reinterpret_cast<float*>(p);
  int nparts = 0;
  NS_TRY(norm_launch<T>(s, G, bs, rs, cs, n, m, batch, part, nparts));
  double r = 1.0;
  int sx = scale_exp(r);
  hipLaunchKernelGGL((ns_pack_kernel<T, NPL>), dim3(mp / 64, np / 64, batch), dim3(256), 0, s, (const T*)G, bs, rs, cs, n, m, part,
                     nparts, eps, std::ldexp(1.0, sx), X[0], XT[0], xs, ts);
  GPX_HIP(hipGetLastError());
  for (int it = 0; it < steps; ++it) {
    const int cur = it & 1;
    const int sa = scale_exp(r * r), sb = scale_exp(poly_bound(k, r));
    const double rn = step_bound(k, r);
    const int sn = scale_exp(rn);
    NsGemm g = {};
    g.out_type = -1;
    g.sums = sums;
    // A = X X^T
    g.A = g.B = X[cur]; g.lda = g.ldb = 2L * mp; g.sa = g.sb = xs;
    g.D = g.DT = A; g.dpl = NPL; g.sd = g.st = as;
    g.M = g.N = np; g.K = mp; g.lower = 1;
    g.ca = 0.f; g.cc = (float)std::ldexp(1.0, sa - 2 * sx);
    NS_TRY(ns_gemm<NPL>(s, g, batch));
    // B = b A + c A A
    g.A = g.B = g.E = A; g.lda = g.ldb = (long)NPL * np; g.sa = g.sb = as;
    g.D = g.DT = B; g.K = np;
    g.ca = (float)(k[1] * std::ldexp(1.0, sb - sa));
    g.cc = (float)(k[2] * std::ldexp(1.0, sb - 2 * sa));
    NS_TRY(ns_gemm<NPL>(s, g, batch));
    // X <- a X + B X
    const bool last = it + 1 == steps;
    g.A = B; g.B = XT[cur]; g.sb = ts; g.E = X[cur]; g.dpl = 2; g.sd = xs; g.st = ts;
    g.D = last ? nullptr : X[cur ^ 1];
    g.DT = last ? nullptr : XT[cur ^ 1];
    g.M = np; g.N = mp; g.K = np; g.lower = 0;
    const int so = last ? 0 : sn;
    g.ca = (float)(k[0] * std::ldexp(1.0, so - sx));
    g.cc = (float)std::ldexp(1.0, so - sb - sx);
    if (last) {
      g.out_type = dtype;
      g.out = out; g.obs = ost[0]; g.ors = ost[1]; g.ocs = ost[2];
      g.base = base; g.bbs = bst[0]; g.brs = bst[1]; g.bcs = bst[2];
      g.n = n; g.m = m; g.alpha = (float)alpha; g.beta = (float)beta;
    }
    NS_TRY(ns_gemm<NPL>(s, g, batch));
    r = rn;
    sx = sn;
  }
  return 0;
}

// Parts into which K (padded to 32 with zeros) of a product is split, as a batch of slices of K, until its tiles of 64 x 64 fill most of
// the chip's 512 places.  Whole calls, half products alone: 1024 x 2048 1131 -> 872 us (988 if half of the places will do), 300 x 700
// 669 -> 321 (371 with slices of 128 and more); with X's product 300 x 700 257, 1000 x 1000 845 -> 784.
int parts_f64(long tiles, long k) {
  int parts = 1;
  while (parts < 8 && tiles * parts < 400 && k / (parts * 2) >= 64) parts *= 2;
  return parts;
}
int half_parts_f64(int n, long k, int batch) {
  const long nt = (n + 63) / 64;
  return parts_f64(nt * (nt + 1) / 2 * batch, k);
}
// of the product with X.  Where it is split the half products are, so that B's padding is zeros: they have fewer tiles.
int step_parts_f64(int n, int m, int batch) { return parts_f64((long)((n + 63) / 64) * ((m + 63) / 64) * batch, pad32(n)); }
// elements of the sums that a call keeps, per matrix of the stack
size_t sums_f64(int n, int m, int batch) {
  const long ldx = pad32(m), lda = pad32(n);
  const int half = std::max(half_parts_f64(n, ldx, batch), half_parts_f64(n, lda, batch)), step = step_parts_f64(n, m, batch);
  return std::max(batch == 1 && half == 1 ? 0 : half * (n * lda), step == 1 ? 0 : step * (n * ldx));
}

// S = alpha R R^T + beta base, whole; matrices of a stack follow each other
int symmetric_f64(hipStream_t s, const double* R, long ldr, long rs, int batch, int n, int k, double* S, long ld, double* sums,
                  double alpha, double beta, const double* base) {
  const int parts = half_parts_f64(n, ldr, batch);
  if (batch == 1 && parts == 1) {
    NS_TRY(gpx_gemm_launch(s, product(R, ldr, R, ldr, GPX_LAY_KC, base, S, ld, n, n, k, alpha, beta, 1)));
    return gpx_symmetrize_launch(s, n, S, ld);
  }
  const int slice = parts == 1 ? k : (int)(ldr / parts);   // the padding is zeros
  GemmDesc g = product(R, ldr, R, ldr, GPX_LAY_KC, nullptr, sums, ld, n, n, slice, 1.0, 0.0, 1);
  g.batch = batch * parts;
  g.batch_inner = parts;
  g.stride_a = g.stride_b = slice;
  g.stride_d = n * ld;
  g.stride2_a = g.stride2_b = rs;
  g.stride2_d = parts * g.stride_d;
  NS_TRY(gpx_gemm_launch(s, g));
  const dim3 grid((n + 31) / 32, (n + 31) / 32, batch);
  if (parts == 1) hipLaunchKernelGGL(ns_join_f64_kernel<1>, grid, dim3(256), 0, s, n, sums, alpha, beta, base, S, ld);
  else if (parts == 2) hipLaunchKernelGGL(ns_join_f64_kernel<2>, grid, dim3(256), 0, s, n, sums, alpha, beta, base, S, ld);
  else if (parts == 4) hipLaunchKernelGGL(ns_join_f64_kernel<4>, grid, dim3(256), 0, s, n, sums, alpha, beta, base, S, ld);
  else hipLaunchKernelGGL(ns_join_f64_kernel<8>, grid, dim3(256), 0, s, n, sums, alpha, beta, base, S, ld);
  GPX_HIP(hipGetLastError());
  return 0;
}

int run_f64(hipStream_t s, int batch, int n, int m, const double* G, long bs, long rs, long cs, int steps, const double* k,
            double eps, double alpha, double beta, const double* base, const long* bst, double* out, const long* ost, char* work) {
  const long ldx = pad32(m), lda = pad32(n), xs = lda * ldx, as = n * lda;   // of a matrix: X has zeros for rows up to lda
  double* part = reinterpret_cast<double*>(work);
  double* X[2] = {part + (size_t)batch * PARTS, nullptr};
  X[1] = X[0] + batch * xs;
  double* A = X[1] + batch * xs;
  double* B = A + batch * as;
  double* sums = B + batch * as;
  int nparts = 0;
  NS_TRY(norm_launch<double>(s, G, bs, rs, cs, n, m, batch, part, nparts));
  const dim3 grid((m + 63) / 64, (n + 63) / 64, batch);
  hipLaunchKernelGGL(ns_pack_f64_kernel, grid, dim3(256), 0, s, G, bs, rs, cs, n, m, part, nparts, eps, X[0], X[1],
                     (int)lda, ldx);
  GPX_HIP(hipGetLastError());
  int cur = 0;
  for (int it = 0; it < steps; ++it, cur ^= 1) {
    NS_TRY(symmetric_f64(s, X[cur], ldx, xs, batch, n, m, A, lda, sums, 1.0, 0.0, nullptr));
    NS_TRY(symmetric_f64(s, A, lda, as, batch, n, n, B, lda, sums, k[2], k[1], A));
    const int parts = step_parts_f64(n, m, batch);
    if (parts == 1) {
      GemmDesc g = product(B, lda, X[cur], ldx, GPX_LAY_RC, X[cur], X[cur ^ 1], ldx, n, m, n, 1.0, k[0], 0);
      g.batch = batch;
      g.stride_a = as;
      g.stride_b = g.stride_d = xs;
      NS_TRY(gpx_gemm_launch(s, g));
      continue;
    }
    const int slice = (int)(lda / parts);
    GemmDesc g = product(B, lda, X[cur], ldx, GPX_LAY_RC, nullptr, sums, ldx, n, m, slice, 1.0, 0.0, 0);
    g.batch = batch * parts;
    g.batch_inner = parts;
    g.stride_a = slice;
    g.stride_b = slice * ldx;
    g.stride_d = n * ldx;
    g.stride2_a = as;
    g.stride2_b = xs;
    g.stride2_d = parts * g.stride_d;
    NS_TRY(gpx_gemm_launch(s, g));
    const dim3 rows((m + 255) / 256, n, batch);
    if (parts == 2) hipLaunchKernelGGL(ns_sum_f64_kernel<2>, rows, dim3(256), 0, s, n, m, sums, k[0], X[cur], X[cur ^ 1], (int)lda, ldx);
    else if (parts == 4) hipLaunchKernelGGL(ns_sum_f64_kernel<4>, rows, dim3(256), 0, s, n, m, sums, k[0], X[cur], X[cur ^ 1], (int)lda, ldx);
    else hipLaunchKernelGGL(ns_sum_f64_kernel<8>, rows, dim3(256), 0, s, n, m, sums, k[0], X[cur], X[cur ^ 1], (int)lda, ldx);
    GPX_HIP(hipGetLastError());
  }
  hipLaunchKernelGGL(ns_out_f64_kernel, grid, dim3(256), 0, s, X[cur], ldx, n, m, out, ost[0], ost[1], ost[2], base, bst[0], bst[1],
                     bst[2], alpha, beta, (int)lda);
  GPX_HIP(hipGetLastError());
  return 0;
}

}  // namespace

extern "C" {

size_t gpx_orthogonalize_work_bytes(int dtype, int batch, int n, int m) {
  if (!dtype_ok(dtype) || batch <= 0 || n <= 0 || m <= 0) return 0;
  const int small = n < m ? n : m, large = n < m ? m : n;
  const size_t parts = (size_t)batch * PARTS * 8;
  if (dtype == GPX_F64) {
    const size_t lx = pad32(large), la = pad32(small);
    return parts + 8 * (size_t)batch * (2 * la * lx + 2 * small * la + sums_f64(small, large, batch));
  }
  const size_t np = pad64(small), mp = pad64(large);
  const size_t pl = planes_of(dtype);   // X twice with two planes, X^T twice, A and B
  const size_t sums = pl == 1 ? 0 : sums_bytes((int)np, (int)mp, batch);
  return parts + (size_t)batch * 2 * ((4 + 2 * pl) * np * mp + 2 * pl * np * np) + sums;
}

int gpx_orthogonalize_tile(int dtype, int batch, int n, int m, int product) {
  if (!dtype_ok(dtype) || dtype == GPX_F64 || batch <= 0 || n <= 0 || m <= 0 || product < 0 || product > 2) return 0;
  const int np = pad64(std::min(n, m)), mp = pad64(std::max(n, m)), lower = product < 2;
  const int N = lower ? np : mp, K = product == 0 ? mp : np;
  return TILE[(planes_of(dtype) == 1 ? choose<1>(np, N, K, lower, batch) : choose<2>(np, N, K, lower, batch)).tile];
}

int gpx_orthogonalize(gpx_handle* h, int dtype, int batch, int n, int m, const void* G, const gpx_strided* g_st, int steps,
                      const double* coef_host, double eps, double alpha, double beta, const void* base,
                      const gpx_strided* base_st, void* out, const gpx_strided* out_st, void* work, size_t work_bytes) {
  GPX_REQUIRE(h != nullptr, "null handle");
  GPX_REQUIRE(dtype_ok(dtype), "orthogonalize: unknown element type %d", dtype);
  GPX_REQUIRE(batch >= 0 && n >= 0 && m >= 0, "orthogonalize: negative size");
  GPX_REQUIRE(batch <= 65535 && n <= 65536 && m <= 65536, "orthogonalize: %d matrices of %d x %d are beyond 65535 of 65536 x 65536",
              batch, n, m);
  GPX_REQUIRE(steps >= 1 && steps <= 64, "orthogonalize: %d steps are outside [1, 64]", steps);
  GPX_REQUIRE(coef_host != nullptr, "orthogonalize: null coefficients");
  GPX_REQUIRE(eps >= 0.0 && std::isfinite(alpha) && std::isfinite(beta), "orthogonalize: eps, alpha or beta out of range");
  double r = 1.0;
  for (int i = 0; i < steps; ++i) {
    r = step_bound(coef_host, r);
    GPX_REQUIRE(r <= 1000.0, "orthogonalize: with these coefficients a singular value may grow beyond 1000 by step %d", i + 1);
  }
  if (batch == 0 || n == 0 || m == 0) return 0;
  GPX_REQUIRE(G != nullptr && out != nullptr && g_st != nullptr && out_st != nullptr, "orthogonalize: null matrix");
  GPX_REQUIRE(beta == 0.0 || (base != nullptr && base_st != nullptr), "orthogonalize: beta != 0 needs base");
  GPX_REQUIRE(work != nullptr && gpx_aligned16(work), "orthogonalize: work null or misaligned");
  GPX_REQUIRE(work_bytes >= gpx_orthogonalize_work_bytes(dtype, batch, n, m), "orthogonalize: work holds %zu of %zu bytes", work_bytes,
              gpx_orthogonalize_work_bytes(dtype, batch, n, m));
  for (const gpx_strided* st : {g_st, out_st})
    GPX_REQUIRE(st->bs >= 0 && st->rs >= 0 && st->cs >= 0, "orthogonalize: negative stride");
  DeviceGuard dg(h->device);
  gpx_gemm_set_workspace(nullptr, 0);   // nothing of the handle's scratch: calls on several streams may overlap
  // n <= m: the transpose is only a matter of strides
  const bool tall = n > m;
  auto strides = [&](const gpx_strided* st, long* o) {
    o[0] = st->bs;
    o[1] = tall ? st->cs : st->rs;
    o[2] = tall ? st->rs : st->cs;
  };
  long gst[3], ost[3], bst[3] = {0, 0, 0};
  strides(g_st, gst);
  strides(out_st, ost);
  if (beta == 0.0) base = nullptr;
  if (base != nullptr) strides(base_st, bst);
  const int a = tall ? m : n, b = tall ? n : m;
  char* w = static_cast<char*>(work);
  switch (dtype) {
    case GPX_F64:
      return run_f64(h->stream, batch, a, b, (const double*)G, gst[0], gst[1], gst[2], steps, coef_host, eps, alpha, beta,
                     (const double*)base, bst, (double*)out, ost, w);
    case GPX_F32:
      return run_half<float, 2>(h->stream, dtype, batch, a, b, G, gst[0], gst[1], gst[2], steps, coef_host, eps, alpha, beta, base, bst,
                                out, ost, w);
    case GPX_F16:
      return run_half<_Float16, 2>(h->stream, dtype, batch, a, b, G, gst[0], gst[1], gst[2], steps, coef_host, eps, alpha, beta, base,
                                   bst, out, ost, w);
    case GPX_BF16 | GPX_TWO_PLANES:
      return run_half<__bf16, 2>(h->stream, GPX_BF16, batch, a, b, G, gst[0], gst[1], gst[2], steps, coef_host, eps, alpha, beta, base,
                                 bst, out, ost, w);
    default:
      return run_half<__bf16, 1>(h->stream, dtype, batch, a, b, G, gst[0], gst[1], gst[2], steps, coef_host, eps, alpha, beta, base, bst,
                                 out, ost, w);
  }
}

}  // extern "C"
