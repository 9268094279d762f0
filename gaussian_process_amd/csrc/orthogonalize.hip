// Orthogonalisation of a matrix (or a stack) by Newton-Schulz products, gpx_orthogonalize in include/gpx.h:
//   X = G / (|G|_F + eps);  repeat: A = X X^T, B = b A + c A A, X <- a X + B X      (X is n x m, n <= m)
//
// Numbers.  The polynomial keeps every singular value of X below a bound r that the host computes from the
// coefficients (1.21 for the usual ones), so |X_ij| <= r, |A_ij| <= r^2 and |B_ij| <= max |b t + c t^2|: the
// intermediates are stored in fp16, each scaled by the power of two that puts its bound just under fp16's largest
// value, which leaves values down to 2^-28 of the bound as normal numbers.  fp16's 11 bits run at bf16's matrix
// rate and lie 8 times nearer: five steps on random matrices end 0.0014 (relative, 2-norm) off in fp16 and 0.011 off
// in bf16, against 0.0017 for rounding the exact result to bf16 once.  Results of more than 8 bits (fp32, fp16) use two fp16
// planes per value, v = hi + lo with 22 bits, and three products (hi hi + hi lo + lo hi): 2.6e-7 off, like an fp32
// product, at a third of the fp16 rate -- five times the rate of the fp32 matrix instructions.
//
// Layout.  Every product has both operands k-contiguous: A needs rows of X; A is symmetric, so A A does too; and
// B X needs rows of X^T, so the step's epilogue writes X in both orientations.  Buffers are padded to multiples of 64
// with zeros, which the iteration preserves; an element's planes lie in one row: [row][plane][ld].
// The symmetric products compute tiles on and below the diagonal and write them twice.
#include <cmath>

#include "gpx_internal.h"

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16acc __attribute__((ext_vector_type(16)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int PAD = 64;
constexpr int PARTS = 256;   // partial sums of the norm per matrix

__host__ __device__ inline int pad64(int x) { return (x + PAD - 1) / PAD * PAD; }

template <typename T> __device__ __forceinline__ double to_f64(T v) { return (double)(float)v; }
template <> __device__ __forceinline__ double to_f64<double>(double v) { return v; }

// ---- |G|_F^2: fixed partials per matrix --------------------------------------------------------------------------
// Threads run along the unit stride of G (fast index), blocks over the other one.
template <typename T>
__global__ __launch_bounds__(256) void ns_norm_kernel(const T* G, long bs, long ss, long fs, int slow, int fast, double* part) {
  __shared__ double sm[4];
  const T* g = G + (long)blockIdx.y * bs;
  double v = 0.0;
  for (int i = blockIdx.x; i < slow; i += gridDim.x)
    for (int j = threadIdx.x; j < fast; j += 256) {
      const double x = to_f64(g[i * ss + j * fs]);
      v = fma(x, x, v);
    }
  for (int o = 32; o > 0; o >>= 1) v += __shfl_down(v, o);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) part[(long)blockIdx.y * PARTS + blockIdx.x] = (sm[0] + sm[1]) + (sm[2] + sm[3]);
}

// 1 / (sqrt(sum of the partials) + eps); every thread gets it
__device__ __forceinline__ double inv_norm(const double* part, int nparts, double eps, double* sm /* 4 */) {
  double v = (int)threadIdx.x < nparts ? part[threadIdx.x] : 0.0;
  for (int o = 32; o > 0; o >>= 1) v += __shfl_down(v, o);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
  __syncthreads();
  return 1.0 / (sqrt((sm[0] + sm[1]) + (sm[2] + sm[3])) + eps);
}

// ---- X and X^T from G --------------------------------------------------------------------------------------------
// One 64 x 64 tile through LDS, read along G's unit stride, written along rows of X and of X^T.
template <typename T, int NPL>
__global__ __launch_bounds__(256) void ns_pack_kernel(const T* G, long bs, long rs, long cs, int n, int m, const double* part,
                                                      int nparts, double eps, double scale, _Float16* X, _Float16* XT,
                                                      long plane) {
  __shared__ float tile[64][65];
  __shared__ double sm[4];
  const int z = blockIdx.z, i0 = blockIdx.y * 64, j0 = blockIdx.x * 64, t = threadIdx.x;
  const int np = pad64(n), mp = pad64(m);
  const double f = inv_norm(part + (long)z * PARTS, nparts, eps, sm) * scale;
  const T* g = G + z * bs;
  const bool along_rows = rs == 1 && cs != 1;
  for (int q = 0; q < 16; ++q) {
    const int a = q * 4 + (t >> 6), b = t & 63;
    const int i = along_rows ? b : a, j = along_rows ? a : b;
    float v = 0.f;
    if (i0 + i < n && j0 + j < m) v = (float)(to_f64(g[(i0 + i) * rs + (j0 + j) * cs]) * f);
    tile[i][j] = v;
  }
  __syncthreads();
  const int r = t >> 2, c0 = (t & 3) * 16;
  X += z * plane;
  XT += z * plane;
  for (int half = 0; half < 2; ++half) {
    h8 xh, xl, th, tl;
    for (int e = 0; e < 8; ++e) {
      const int c = c0 + half * 8 + e;
      const float x = tile[r][c], y = tile[c][r];
      xh[e] = (_Float16)x;
      th[e] = (_Float16)y;
      if (NPL == 2) {
        xl[e] = (_Float16)(x - (float)xh[e]);
        tl[e] = (_Float16)(y - (float)th[e]);
      }
    }
    const long px = (long)(i0 + r) * NPL * mp + j0 + c0 + half * 8, pt = (long)(j0 + r) * NPL * np + i0 + c0 + half * 8;
    *reinterpret_cast<h8*>(X + px) = xh;
    *reinterpret_cast<h8*>(XT + pt) = th;
    if (NPL == 2) {
      *reinterpret_cast<h8*>(X + px + mp) = xl;
      *reinterpret_cast<h8*>(XT + pt + np) = tl;
    }
  }
}

// ---- the product -------------------------------------------------------------------------------------------------
// v = ca * E + cc * (A B^T); v goes to D [row][col], to DT [col][row], or as alpha * v + beta * base to the caller's
// matrix.
struct NsGemm {
  const _Float16 *A, *B, *E;   // A: M rows, B: N rows, both K long; E like D
  _Float16 *D, *DT;
  long sa, sb, sd;             // strides of the stack
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
};

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, unsigned voff, unsigned soff, char* dst_wave) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst_wave, 16, voff, soff, 0, 0);
}

template <typename T>
__device__ __forceinline__ void put(void* out, const void* base, long o, long b, float alpha, float beta, float v) {
  float r = alpha * v;
  if (base != nullptr) r += beta * (float)reinterpret_cast<const T*>(base)[b];
  reinterpret_cast<T*>(out)[o] = (T)r;
}

// Tile BM x BN, WAVES_M x WAVES_N waves of (BM / WAVES_M) x (BN / WAVES_N) each in 32 x 32 x 16 matrix instructions.
// A k-tile is 64 / NPL long: an LDS row is 128 bytes either way, 8 chunks of 16 bytes (NPL = 2: four of hi, four of
// lo), chunk c of row r in slot c ^ (r & 7), so that the 16-byte fragment reads meet no bank twice.
template <int BM, int BN, int WAVES_M, int WAVES_N, int NPL>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N) void ns_gemm_kernel(const NsGemm g, int tiles_n) {
  constexpr int NW = WAVES_M * WAVES_N, NT = 64 * NW;
  constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, TM = WM / 32, TN = WN / 32;
  constexpr int BK = 64 / NPL, KS = BK / 16;
  constexpr int ABYTES = BM * 128, STAGE = (BM + BN) * 128;
  extern __shared__ __align__(16) char smem[];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  int ti, tj;
  if (g.lower) {
    const unsigned id = blockIdx.x;
    unsigned r = (unsigned)((sqrtf(8.f * (float)id + 1.f) - 1.f) * 0.5f);
    while ((r + 1) * (r + 2) / 2 <= id) ++r;
    while (r * (r + 1) / 2 > id) --r;
    ti = r;
    tj = id - r * (r + 1) / 2;
  } else {
    ti = blockIdx.x / tiles_n;
    tj = blockIdx.x % tiles_n;
  }
  const int i0 = ti * BM, j0 = tj * BN;
  const long z = blockIdx.y;
  const long lda = (long)NPL * g.K * 2;   // bytes per row of A and of B
  const __amdgpu_buffer_rsrc_t ra =
      __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)(g.A + z * g.sa) + i0 * lda), 0, 0x7fffffff, 0x00020000);
  const __amdgpu_buffer_rsrc_t rb =
      __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)(g.B + z * g.sb) + j0 * lda), 0, 0x7fffffff, 0x00020000);
  // per-lane sources of the DMA: piece p of NT lanes covers rows p * (NT / 8) ..; rows behind the matrix repeat its last
  constexpr int PA = BM * 8 / NT, PB = BN * 8 / NT;
  unsigned va[PA], vb[PB];
#pragma unroll
  for (int p = 0; p < PA; ++p) {
    const int s = p * NT + t, r = s >> 3, c = (s & 7) ^ (r & 7);
    const int rr = min(r, g.M - 1 - i0);
    va[p] = (unsigned)(rr * lda + (NPL == 1 ? c * 16 : (c >> 2) * g.K * 2 + (c & 3) * 16));
  }
#pragma unroll
  for (int p = 0; p < PB; ++p) {
    const int s = p * NT + t, r = s >> 3, c = (s & 7) ^ (r & 7);
    const int rr = min(r, g.N - 1 - j0);
    vb[p] = (unsigned)(rr * lda + (NPL == 1 ? c * 16 : (c >> 2) * g.K * 2 + (c & 3) * 16));
  }
  auto load = [&](int kt, int buf) {
    char* sA = smem + buf * STAGE + wave * 1024;
    char* sB = sA + ABYTES;
    const unsigned so = (unsigned)kt * (BK * 2);
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
  load(0, 0);
  for (int kt = 0; kt < nk; ++kt) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();   // tile kt has landed, and every wave is done with the buffer that tile kt + 1 goes to
    if (kt + 1 < nk) load(kt + 1, (kt + 1) & 1);
    const char* sA = smem + (kt & 1) * STAGE + (wm * WM + r32) * 128;
    const char* sB = smem + (kt & 1) * STAGE + ABYTES + (wn * WN + r32) * 128;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int o0 = (((s * 2 + kh) ^ (r32 & 7)) * 16);
      h8 fa[TM][NPL], fb[TN][NPL];
#pragma unroll
      for (int pl = 0; pl < NPL; ++pl) {
        const int o = o0 ^ (pl * 64);
#pragma unroll
        for (int a = 0; a < TM; ++a) fa[a][pl] = *reinterpret_cast<const h8*>(sA + a * 32 * 128 + o);
#pragma unroll
        for (int b = 0; b < TN; ++b) fb[b][pl] = *reinterpret_cast<const h8*>(sB + b * 32 * 128 + o);
      }
#pragma unroll
      for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int b = 0; b < TN; ++b) {
          if (NPL == 2) {
            acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[a][0], fb[b][NPL - 1], acc[a][b], 0, 0, 0);
            acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[a][NPL - 1], fb[b][0], acc[a][b], 0, 0, 0);
          }
          acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[a][0], fb[b][0], acc[a][b], 0, 0, 0);
        }
    }
  }
  __syncthreads();   // the stages become the waves' own staging of 64 x 64 blocks
  constexpr int P = 68;
  float* st = reinterpret_cast<float*>(smem) + wave * (64 * P);
  const long ldd = (long)NPL * g.N, ldt = (long)NPL * g.M;
  const _Float16* E = g.E == nullptr ? nullptr : g.E + z * g.sd;
  _Float16* D = g.D == nullptr ? nullptr : g.D + z * g.sd;
  _Float16* DT = g.DT == nullptr ? nullptr : g.DT + z * g.sd;
#pragma unroll
  for (int bi = 0; bi < WM / 64; ++bi)
#pragma unroll
    for (int bj = 0; bj < WN / 64; ++bj) {
      const int row0 = i0 + wm * WM + bi * 64, col0 = j0 + wn * WN + bj * 64;
      if (row0 >= g.M || col0 >= g.N) continue;   // uniform in the wave
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            st[(a * 32 + (e >> 2) * 8 + kh * 4 + (e & 3)) * P + b * 32 + r32] = acc[bi * 2 + a][bj * 2 + b][e];
      __builtin_amdgcn_wave_barrier();
      // rows: 8 lanes x 8 columns, 8 rows at a time
      for (int q = 0; q < 8; ++q) {
        const int r = q * 8 + (lane >> 3), c = (lane & 7) * 8;
        float* p = st + r * P + c;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = g.cc * p[e];
        if (E != nullptr) {
          const _Float16* src = E + (row0 + r) * ldd + col0 + c;
          const h8 eh = *reinterpret_cast<const h8*>(src);
          if (NPL == 2) {
            const h8 el = *reinterpret_cast<const h8*>(src + g.N);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += g.ca * ((float)eh[e] + (float)el[e]);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += g.ca * (float)eh[e];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = v[e];
        if (D != nullptr) {
          h8 hi, lo;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            hi[e] = (_Float16)v[e];
            if (NPL == 2) lo[e] = (_Float16)(v[e] - (float)hi[e]);
          }
          _Float16* dst = D + (row0 + r) * ldd + col0 + c;
          *reinterpret_cast<h8*>(dst) = hi;
          if (NPL == 2) *reinterpret_cast<h8*>(dst + g.N) = lo;
        }
      }
      __builtin_amdgcn_wave_barrier();
      if (DT != nullptr && !(g.lower && ti == tj)) {
        for (int q = 0; q < 8; ++q) {   // columns: 8 lanes x 8 rows, 8 columns at a time
          const int c = q * 8 + (lane >> 3), r = (lane & 7) * 8;
          h8 hi, lo;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = st[(r + e) * P + c];
            hi[e] = (_Float16)v;
            if (NPL == 2) lo[e] = (_Float16)(v - (float)hi[e]);
          }
          _Float16* dst = DT + (col0 + c) * ldt + row0 + r;
          *reinterpret_cast<h8*>(dst) = hi;
          if (NPL == 2) *reinterpret_cast<h8*>(dst + g.M) = lo;
        }
      }
      if (g.out_type >= 0) {
        // the caller's matrix, lanes along its unit stride
        const bool along_rows = g.ors == 1 && g.ocs != 1;
        for (int q = 0; q < 64; ++q) {
          const int r = along_rows ? lane : q, c = along_rows ? q : lane;
          const int i = row0 + r, j = col0 + c;
          if (i < g.n && j < g.m) {
            const long o = z * g.obs + i * g.ors + j * g.ocs, b = z * g.bbs + i * g.brs + j * g.bcs;
            const float v = st[r * P + c];
            if (g.out_type == GPX_F32) put<float>(g.out, g.base, o, b, g.alpha, g.beta, v);
            else if (g.out_type == GPX_F16) put<_Float16>(g.out, g.base, o, b, g.alpha, g.beta, v);
            else put<__bf16>(g.out, g.base, o, b, g.alpha, g.beta, v);
          }
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
}

template <int BM, int BN, int WAVES_M, int WAVES_N, int NPL>
int launch_cfg(hipStream_t s, const NsGemm& g, int batch) {
  constexpr int NW = WAVES_M * WAVES_N;
  constexpr size_t lds = std::max<size_t>(2 * (BM + BN) * 128, (size_t)NW * 64 * 68 * 4);
  const int tm = (g.M + BM - 1) / BM, tn = (g.N + BN - 1) / BN;
  const unsigned tiles = g.lower ? (unsigned)tm * (tm + 1) / 2 : (unsigned)tm * tn;
  static thread_local bool set[GPX_MAX_DEVICES] = {};
  int dev = 0;
  GPX_HIP(hipGetDevice(&dev));
  if (dev < GPX_MAX_DEVICES && !set[dev]) {
    GPX_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&ns_gemm_kernel<BM, BN, WAVES_M, WAVES_N, NPL>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    set[dev] = true;
  }
  hipLaunchKernelGGL((ns_gemm_kernel<BM, BN, WAVES_M, WAVES_N, NPL>), dim3(tiles, batch), dim3(64 * NW), lds, s, g, tn);
  GPX_HIP(hipGetLastError());
  return 0;
}

template <int NPL>
int ns_gemm(hipStream_t s, const NsGemm& g, int batch) {
  return launch_cfg<128, 128, 2, 2, NPL>(s, g, batch);
}

// ---- fp64: the framework's own products ----------------------------------------------------------------------------
__global__ __launch_bounds__(256) void ns_pack_f64_kernel(const double* G, long bs, long rs, long cs, int n, int m,
                                                          const double* part, int nparts, double eps, double* X, long ldx) {
  __shared__ double tile[64][65];
  __shared__ double sm[4];
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64, t = threadIdx.x;
  const double f = inv_norm(part, nparts, eps, sm);
  const bool along_rows = rs == 1 && cs != 1;
  for (int q = 0; q < 16; ++q) {
    const int a = q * 4 + (t >> 6), b = t & 63;
    const int i = along_rows ? b : a, j = along_rows ? a : b;
    if (i0 + i < n && j0 + j < m) tile[i][j] = G[(i0 + i) * rs + (j0 + j) * cs] * f;
  }
  __syncthreads();
  for (int q = 0; q < 16; ++q) {
    const int i = q * 4 + (t >> 6), j = t & 63;
    if (i0 + i < n && j0 + j < m) X[(i0 + i) * ldx + j0 + j] = tile[i][j];
  }
}

__global__ __launch_bounds__(256) void ns_out_f64_kernel(const double* X, long ldx, int n, int m, double* out, long rs, long cs,
                                                         const double* base, long brs, long bcs, double alpha, double beta) {
  __shared__ double tile[64][65];
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

#define NS_TRY(expr)          \
  do {                        \
    int rc_ = (expr);         \
    if (rc_ != 0) return rc_; \
  } while (0)

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
// exponent that puts values of at most `bound` (and 5 % for rounding) under 2^14, a quarter of fp16's largest
int scale_exp(double bound) { return 14 - (int)std::ceil(std::log2(std::fmax(bound, 1e-3) * 1.05)); }

int planes_of(int dtype) { return dtype == GPX_BF16 ? 1 : 2; }

bool dtype_ok(int dtype) { return dtype == GPX_F64 || dtype == GPX_F32 || dtype == GPX_F16 || dtype == GPX_BF16; }

template <typename T>
int norm_launch(hipStream_t s, const void* G, long bs, long rs, long cs, int n, int m, int batch, double* part, int& nparts) {
  const bool along_rows = rs == 1 && cs != 1;
  const int slow = along_rows ? m : n, fast = along_rows ? n : m;
  nparts = slow < PARTS ? slow : PARTS;
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
  const long xs = (long)np * mp * NPL, as = (long)np * np * NPL;
  double* part = reinterpret_cast<double*>(work);
  _Float16* X[2];
  _Float16* XT[2];
  _Float16* p = reinterpret_cast<_Float16*>(work + (size_t)batch * PARTS * 8);
  X[0] = p; p += batch * xs;
  X[1] = p; p += batch * xs;
  XT[0] = p; p += batch * xs;
  XT[1] = p; p += batch * xs;
  _Float16* A = p; p += batch * as;
  _Float16* B = p;
  int nparts = 0;
  NS_TRY(norm_launch<T>(s, G, bs, rs, cs, n, m, batch, part, nparts));
  double r = 1.0;
  int sx = scale_exp(r);
  hipLaunchKernelGGL((ns_pack_kernel<T, NPL>), dim3(mp / 64, np / 64, batch), dim3(256), 0, s, (const T*)G, bs, rs, cs, n, m, part,
                     nparts, eps, std::ldexp(1.0, sx), X[0], XT[0], xs);
  GPX_HIP(hipGetLastError());
  for (int it = 0; it < steps; ++it) {
    const int cur = it & 1;
    const int sa = scale_exp(r * r), sb = scale_exp(poly_bound(k, r));
    const double rn = step_bound(k, r);
    const int sn = scale_exp(rn);
    NsGemm g = {};
    g.out_type = -1;
    // A = X X^T
    g.A = g.B = X[cur]; g.sa = g.sb = xs; g.D = g.DT = A; g.sd = as;
    g.M = g.N = np; g.K = mp; g.lower = 1;
    g.ca = 0.f; g.cc = (float)std::ldexp(1.0, sa - 2 * sx);
    NS_TRY(ns_gemm<NPL>(s, g, batch));
    // B = b A + c A A
    g.A = g.B = g.E = A; g.sa = g.sb = as; g.D = g.DT = B; g.K = np;
    g.ca = (float)(k[1] * std::ldexp(1.0, sb - sa));
    g.cc = (float)(k[2] * std::ldexp(1.0, sb - 2 * sa));
    NS_TRY(ns_gemm<NPL>(s, g, batch));
    // X <- a X + B X
    const bool last = it + 1 == steps;
    g.A = B; g.sa = as; g.B = XT[cur]; g.sb = xs; g.E = X[cur]; g.sd = xs;
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

int run_f64(hipStream_t s, int batch, int n, int m, const double* G, long bs, long rs, long cs, int steps, const double* k,
            double eps, double alpha, double beta, const double* base, const long* bst, double* out, const long* ost, char* work) {
  const long ldx = pad32(m), lda = pad32(n);
  double* part = reinterpret_cast<double*>(work);
  double* X[2] = {part + (size_t)batch * PARTS, nullptr};
  X[1] = X[0] + n * ldx;
  double* A = X[1] + n * ldx;
  double* B = A + n * lda;
  int nparts = 0;
  NS_TRY(norm_launch<double>(s, G, bs, rs, cs, n, m, batch, part, nparts));
  const dim3 grid((m + 63) / 64, (n + 63) / 64);
  for (int z = 0; z < batch; ++z) {
    hipLaunchKernelGGL(ns_pack_f64_kernel, grid, dim3(256), 0, s, G + z * bs, bs, rs, cs, n, m, part + (long)z * PARTS, nparts, eps,
                       X[0], ldx);
    GPX_HIP(hipGetLastError());
    int cur = 0;
    for (int it = 0; it < steps; ++it, cur ^= 1) {
      NS_TRY(gpx_gemm_launch(s, product(X[cur], ldx, X[cur], ldx, GPX_LAY_KC, nullptr, A, lda, n, n, m, 1.0, 0.0, 1)));
      NS_TRY(gpx_symmetrize_launch(s, n, A, lda));
      NS_TRY(gpx_gemm_launch(s, product(A, lda, A, lda, GPX_LAY_KC, A, B, lda, n, n, n, k[2], k[1], 1)));
      NS_TRY(gpx_symmetrize_launch(s, n, B, lda));
      NS_TRY(gpx_gemm_launch(s, product(B, lda, X[cur], ldx, GPX_LAY_RC, X[cur], X[cur ^ 1], ldx, n, m, n, 1.0, k[0], 0)));
    }
    hipLaunchKernelGGL(ns_out_f64_kernel, grid, dim3(256), 0, s, X[cur], ldx, n, m, out + z * ost[0], ost[1], ost[2],
                       base == nullptr ? nullptr : base + z * bst[0], bst[1], bst[2], alpha, beta);
    GPX_HIP(hipGetLastError());
  }
  return 0;
}

}  // namespace

extern "C" {

size_t gpx_orthogonalize_work_bytes(int dtype, int batch, int n, int m) {
  if (!dtype_ok(dtype) || batch <= 0 || n <= 0 || m <= 0) return 0;
  const int small = n < m ? n : m, large = n < m ? m : n;
  const size_t parts = (size_t)batch * PARTS * 8;
  if (dtype == GPX_F64)   // the matrices of a stack take their turns in one set of buffers
    return parts + 8 * (2 * (size_t)small * pad32(large) + 2 * (size_t)small * pad32(small));
  const size_t np = pad64(small), mp = pad64(large);
  return parts + (size_t)batch * 2 * planes_of(dtype) * (4 * np * mp + 2 * np * np);
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
    default:
      return run_half<__bf16, 1>(h->stream, dtype, batch, a, b, G, gst[0], gst[1], gst[2], steps, coef_host, eps, alpha, beta, base, bst,
                                 out, ost, w);
  }
}

}  // extern "C"
