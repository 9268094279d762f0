// The gated delta rule, gpx_delta_* in include/gpx.h:
//   Sbar_t = exp(g_t) S_{t-1};  e_t = v_t - Sbar_t^T k_t;  S_t = Sbar_t + beta_t k_t e_t^T;  o_t = scale S_t^T q_t
//
// Chunks of C = 64 tokens.  With G the running sum of g in the chunk, D_ij = exp(G_i - G_j) (i >= j),
// N = strictly lower part of K K^T o D, P = lower part of Q K^T o D, S the state before the chunk:
//   X = V - diag(exp G) K S;   E = T X with T = (I + N diag(beta))^-1;   U = diag(beta) E
//   O = scale (diag(exp G) Q S + P U);   S' = exp(G_C) S + K^T diag(exp(G_C - G)) U
// (in terms of the errors E instead of beta E, so that beta = 0 divides nothing).  Backward, given dO and dS':
//   dU = scale P^T dO + diag(exp(G_C - G)) K dS';   Z = (I + diag(beta) N)^-T dU;   dV = dX = diag(beta) Z
//   dS = exp(G_C) dS' + scale Q^T diag(exp G) dO - K^T diag(exp G) dX
//   dP = scale dO U^T;   dN = -dX U^T;   dQ = scale diag(exp G) dO S^T + (dP o D) K;   dbeta_j = E_j . Z_j
//   dK = dKr + dKc:  dKr = (dN o D) K - diag(exp G) dX S^T        (the key that reads: row of N, of K S)
//                    dKc = (dN o D)^T K + (dP o D)^T Q + diag(exp(G_C - G)) U dS'^T   (the key that writes)
//   dg_t = sum over i >= t > j of (dP o P + dN o N)_ij + sum over i >= t of r_i + sum over j < t of c_j + exp(G_C) <dS', S>
//          r_i = scale exp(G_i) q_i . S dO_i - exp(G_i) k_i . S dX_i,  c_j = exp(G_C - G_j) k_j . dS' U_j
// dg_t is formed from the pairs of tokens on both sides of it, all of which carry the factor exp(g_t): as a sum over the tokens behind
// t of dG_i = q_i . dQ_i + k_i . (dKr - dKc)_i, the pairs on one side cancel only up to their rounding, which hid the whole
// result of fast heads (relative error 7e-4 at g = -8, 0.02 to 0.1 at -12, 0.4 to 1.7 at -16; 3e-7 now, whatever g).
//
// G is summed in 64 bits, since differences of it are taken, and g is read as max(g, -200): exp(-200) is 0 in fp32,
// and a g of -infinity then gives no infinity minus infinity.
//
// Kernels: plan (where packed sequences are), chunk (parallel over chunks: T, P, G, operands in the scans' order), the chain (over the
// chunks of a sequence, parallel over heads and slices of dv, which are independent) and its reverse, and grads (parallel over
// chunks).  Short inputs and single tokens go through the recurrence itself.  8192 tokens x 16 heads, bf16, dk = dv = 128: chunk 60 us,
// chain 237; training on 2 x 4096 tokens: 81, 191 and 182, grads 235.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "gpx_internal.h"

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int C = 64;          // tokens per chunk
constexpr int DVT = 32;        // dv is rounded up to this: columns that the gradients take at a time
constexpr int PC = 68;         // LDS pitch of [..][64] tiles
constexpr float G_MIN = -200.f;

// Where the chunks of a problem are.  Slot numbers need no table: sequence s starts at slot offsets[s] / C + s, which
// leaves room for every sequence's last, partly filled chunk.
struct Plan {
  int sequences, tokens;
  const int* off;        // sanitised offsets (device) or nullptr: sequence s is batch row s
  int chunks_per_row;    // plain batches
  __device__ __forceinline__ int begin(int s) const { return off ? off[s] : 0; }
  __device__ __forceinline__ int end(int s) const { return off ? off[s + 1] : tokens; }
  __device__ __forceinline__ int slot0(int s) const { return off ? off[s] / C + s : s * chunks_per_row; }
  // the sequence and first token of a slot; len = tokens of the chunk (0: no chunk in this slot)
  __device__ __forceinline__ void locate(int slot, int& s, int& t0, int& len) const {
    if (off == nullptr) {
      s = slot / chunks_per_row;
      t0 = (slot % chunks_per_row) * C;
    } else {
      int lo = 0, hi = sequences - 1;   // the last s with slot0(s) <= slot
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (slot0(mid) <= slot) lo = mid; else hi = mid - 1;
      }
      s = lo;
      t0 = begin(s) + (slot - slot0(s)) * C;
    }
    len = min(C, end(s) - t0);
    if (len < 0 || slot < slot0(s)) len = 0;   // behind the sequence's last chunk, or before the first sequence
  }
  __device__ __forceinline__ long row(int s) const { return off ? 0 : s; }   // batch row
  __device__ __forceinline__ int by_length(int i) const { return off ? off[sequences + 1 + i] : i; }   // the i-th sequence to start
};

// One wave.  out: the offsets made non-decreasing and inside [0, tokens] (every later kernel's accesses follow from these), then
// the sequences, the longest first, as the scans start them: their workgroups outnumber the compute units, and one long
// sequence started last is waited for alone.  Lengths within a quarter of a power of two count as equal.
__global__ void delta_plan_kernel(const int* in, int n, int tokens, int* out) {
  __shared__ int start[128];
  const int lane = threadIdx.x, sequences = n - 1;
  start[lane] = start[lane + 64] = 0;
  int carry = 0;
  for (int base = 0; base < n; base += 64) {
    const int i = base + lane;
    int v = i < n ? min(max(in[i], 0), tokens) : 0;
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(v, o);
      if (lane >= o) v = max(v, u);
    }
    v = max(v, carry);
    carry = __shfl(v, 63);
    if (i < n) out[i] = v;
  }
  __syncthreads();
  auto rank = [&](int i) {   // 0: the longest; a length of 2^30 has 16 M chunks
    const unsigned len = (unsigned)(out[i + 1] - out[i]), chunks = len / C + (len % C != 0), w = chunks * 4 + 3;
    const int e = 31 - __clz(w);   // 1 (no chunk) to 26
    return 127 - (e * 4 + (int)(w >> (e - 1) & 1) * 2 + (e > 1 ? (int)(w >> (e - 2) & 1) : 0));
  };
  for (int i = lane; i < sequences; i += 64) atomicAdd(&start[rank(i)], 1);
  __syncthreads();
  const int a = start[2 * lane], b = start[2 * lane + 1];
  int before = a + b;
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(before, o);
    if (lane >= o) before += u;
  }
  before -= a + b;
  __syncthreads();
  start[2 * lane] = before;
  start[2 * lane + 1] = before + a;
  __syncthreads();
  for (int i = lane; i < sequences; i += 64) out[n + atomicAdd(&start[rank(i)], 1)] = i;
}

typedef float f2 __attribute__((ext_vector_type(2)));

struct Args {
  gpx_delta d;
  Plan p;
  int group;                    // value heads per key head
  int parts;                    // prep: workgroups among which a key head's value heads are dealt, 1 or group
  int dvp;                      // dv rounded up to DVT
  float scale;
  // Parts of the workspaces; "per key head", "per head": of a slot and a key or value head.  Fragments are explained below.
  f2* G;                        // per head: C, the sums of g in two parts
  float* fac;                   // per head: exp(G), beta, exp(G_C - G) beta, exp(G_C), exp(G_C - G), exp(G) beta; C each
  __bf16 *Kf, *Qf, *KTf, *QTf;  // per key head: K and Q in state order, K^T and Q^T
  __bf16 *Tf, *Pf, *T2f, *PTf;  // per head: T, P, (I + diag(beta) N)^-T, P^T
  float *Erow, *Srow;           // per head: E, dvp / 16 x C x 16; S, dvp / 16 x DK x 16
  float *Z, *dS;                // per head: Z (dX = beta Z) like E; dS' like S
  float *d_q_part, *d_k_part;   // per head: its part of dQ and dK, C x DK
  const float *state, *d_state_out;
  float *state_out, *d_state, *d_g, *d_beta;
  void *o, *d_q, *d_k, *d_v;
  const void* d_o;
  gpx_strided do_st;
  int save;
};

template <typename T> __device__ __forceinline__ float ld(const void* p, long i) { return (float)reinterpret_cast<const T*>(p)[i]; }
template <typename T> __device__ __forceinline__ void st(void* p, long i, float v) { reinterpret_cast<T*>(p)[i] = (T)v; }

// acc (16 x 16, rows (lane >> 4) * 4 + e, column lane & 15) += A B over k < K (a multiple of 4), A 16 x K, B K x 16
__device__ __forceinline__ f4 mm(const float* A, int pa, const float* B, int pb, int K, f4 acc) {
  const int r = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
  A += r * pa + g;
  B += g * pb + r;
  for (int k = 0; k < K; k += 4) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(A[k], B[k * pb], acc, 0, 0, 0);
  return acc;
}

// Slices of a head read the same keys: blocks with equal id % 8 share an XCD and its L2.
__device__ __forceinline__ bool scan_coords(unsigned id, int slices, int heads, int& slice, int& head) {
  const unsigned per = 8u * slices;
  head = (int)(id / per * 8 + id % 8);
  slice = (int)(id % per / 8);
  return head < heads;
}

// ---- planes -------------------------------------------------------------------------------------------------------------
// Products run on the bf16 matrix cores with values split exactly into bf16 planes, x = x0 + x1 + x2 (8 bits each): a bf16 input
// is one plane, an fp16 one two, anything in fp32 three.  A product of planes i and j is kept for i + j <= 2, which
// leaves 2^-24, fp32's own rounding; the matrix cores sum in fp32.  Three planes against one cost 3/16 of the fp32
// matrix instruction's time, three against three 6/16.
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));

template <typename T> struct Planes { static constexpr int N = 3; };
template <> struct Planes<_Float16> { static constexpr int N = 2; };
template <> struct Planes<__bf16> { static constexpr int N = 1; };

// the high 16 bits of two floats as two bf16 (truncation; the remainders carry the rest)
__device__ __forceinline__ unsigned high_pair(float a, float b) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x07060302u);
}
__device__ __forceinline__ float truncated(float x) {
  return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) & 0xffff0000u);
}
// NV floats -> NPL planes of NV bf16.  Each plane truncates to 8 bits, except the last, which is rounded where it is not exact
// (NPL < 3).  An infinity's remainder is NaN, so infinite values give NaN.
template <int NV, int NPL, typename V>
__device__ __forceinline__ void split(const float* x, V* planes) {
  float r[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) r[i] = x[i];
#pragma unroll
  for (int p = 0; p < NPL; ++p) {
    unsigned w[NV / 2];
    if (p == 2 || p + 1 < NPL) {
#pragma unroll
      for (int i = 0; i < NV; i += 2) w[i / 2] = high_pair(r[i], r[i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < NV; i += 2) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        b2 v;
        v[0] = (__bf16)r[i];
        v[1] = (__bf16)r[i + 1];
        w[i / 2] = __builtin_bit_cast(unsigned, v);
      }
    }
    __builtin_memcpy(&planes[p], w, sizeof(w));
    if (p + 1 < NPL) {
#pragma unroll
      for (int i = 0; i < NV; ++i) r[i] -= truncated(r[i]);
    }
  }
}

// acc += sum of A_i B_j over planes with i + j < LIM
template <int NA, int NB, int LIM>
__device__ __forceinline__ f4 planes_mma(const b8* a, const b8* b, f4 acc) {
#pragma unroll
  for (int n = LIM - 1; n >= 0; --n)   // small terms first
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int j = n - i;
      if (j >= 0 && j < NB) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], acc, 0, 0, 0);
    }
  return acc;
}

// sum over the 16 lanes of a row, in every lane
__device__ __forceinline__ float row_sum(float x) {
  auto add = [&](auto ctrl) {
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  add(std::integral_constant<int, 0xB1>{});    // lane ^ 1
  add(std::integral_constant<int, 0x4E>{});    // lane ^ 2
  add(std::integral_constant<int, 0x141>{});   // mirrored in eight
  add(std::integral_constant<int, 0x140>{});   // mirrored in sixteen
  return x;
}

// Sums of g, in double: kept times log2(e) as a float and what that leaves out.  exp(x - y) has then the error of one rounding
// of x - y and one of the power; powers below 2^-126 become 0.
__device__ __forceinline__ f2 in_parts(double g) {
  g *= 1.4426950408889634;
  const float hi = (float)g;
  return f2{hi, (float)(g - (double)hi)};
}
__device__ __forceinline__ float decay(f2 x, f2 y) { return __builtin_amdgcn_exp2f((x[0] - y[0]) + (x[1] - y[1])); }

// a barrier that waits for this wave's LDS accesses, not for its global ones
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Fragments.  A matrix instruction's operand is 16 rows x 32 terms, lane l holding row l & 15 and 8 terms of group
// g = l >> 4.  Operands that the scan reads are stored fragment by fragment, [plane][row block][term block][lane][8], so that a
// wave loads one with 16 bytes per lane, in a row.  Natural order: terms 32 ks + 8 g + e.  State order: S lives in the
// accumulators of the wave that updates it, lane l holding column l & 15 and rows 4 g + e of each of its DK / 64 tiles, and
// serves from there as the other operand; the terms of wave w are therefore dk = 16 (w DK / 64) + 4 g + e, e < 4, and the
// same of its second tile (none if DK = 64: zeros).

constexpr int KF = 4 * 4 * 64 * 8;   // elements of a plane of K or Q in state order
constexpr int TF = 4 * 2 * 64 * 8;   // of a C x C matrix
constexpr int FACS = 6 * C;          // factors per head

// C rows of one head as planes in LDS, pitch DK + 8: fetch() has all loads under way, put() splits and writes
template <typename T, int DK>
struct Rows {
  static constexpr int IT = C * DK / 8 / 256, W = sizeof(T) / 2;
  uint4 raw[IT][W];
  __device__ __forceinline__ void fetch(const void* src, const gpx_strided& s, long row, int t0, int len, int head, int dk, int t) {
    const T* base = reinterpret_cast<const T*>(src) + row * s.bs + t0 * s.rs + head * s.cs;
    if (((reinterpret_cast<uintptr_t>(base) | (uintptr_t)(s.rs * sizeof(T))) & 15) == 0 && (dk & 7) == 0) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {   // rows and columns behind the end repeat the last
        const int q = i * 256 + t, r = min(q / (DK / 8), len - 1), c = min(q % (DK / 8) * 8, dk - 8);
        const uint4* p = reinterpret_cast<const uint4*>(base + r * s.rs + c);
#pragma unroll
        for (int w = 0; w < W; ++w) raw[i][w] = p[w];
      }
    } else {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int q = i * 256 + t, r = min(q / (DK / 8), len - 1), c = q % (DK / 8) * 8;
        T v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = base[r * s.rs + min(c + e, dk - 1)];
        __builtin_memcpy(raw[i], v, sizeof(v));
      }
    }
  }
  __device__ __forceinline__ void put(__bf16* dst, int len, int dk, int t) const {
    constexpr int P = DK + 8, N = Planes<T>::N;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int q = i * 256 + t, r = q / (DK / 8), c = q % (DK / 8) * 8;
      T v[8];
      __builtin_memcpy(v, raw[i], sizeof(v));
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = r < len && c + e < dk ? (float)v[e] : 0.f;
      b8 p[N];
      split<8, N>(x, p);
#pragma unroll
      for (int k = 0; k < N; ++k) *reinterpret_cast<b8*>(dst + (k * C + r) * P + c) = p[k];
    }
  }
};

// T = (I + A)^-1 for the strictly lower A (LDS, pitch PC), 4 waves.  The 16 x 16 diagonal blocks by substitution, one column
// per lane; then, twice, [T0 0; -T1 A10 T0 T1] of two blocks and what is under them, on the fp32 matrix cores.  tmp: 32 x 36.
__device__ __forceinline__ void unit_lower_inverse(const float* A, float* Ti, float* tmp, int wave, int lane) {
  const int r4 = (lane >> 4) * 4, col = lane & 15;
  for (int j = wave + 1; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) Ti[(wave * 16 + r4 + e) * PC + j * 16 + col] = 0.f;
  if (lane < 16) {
    const float* a = A + wave * 16 * PC + wave * 16;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == lane ? 1.f : 0.f;
      f4 al[4];
#pragma unroll
      for (int l = 0; l < (i + 3) / 4; ++l) al[l] = *reinterpret_cast<const f4*>(a + i * PC + l * 4);
#pragma unroll
      for (int l = 0; l < i; ++l) v = fmaf(-al[l / 4][l % 4], x[l], v);
      x[i] = v;
      Ti[(wave * 16 + i) * PC + wave * 16 + lane] = v;
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 1; n < 3; ++n) {   // blocks of n times 16 rows
    // this wave's 16 x 16 of the products: rows i, columns j of the n x n under the diagonal, in units of 16
    const int lo = n == 1 ? wave * 2 : 0, hi = lo + n, i = n == 1 ? 0 : wave >> 1, j = n == 1 ? 0 : wave & 1;
    const bool works = n == 2 || wave < 2;
    float* mine = tmp + (n == 1 ? wave * 16 : i * 16) * 36 + j * 16;
    if (works) {
      f4 acc = {0, 0, 0, 0};
      for (int l = j; l < n; ++l)
        acc = mm(A + (hi + i) * 16 * PC + (lo + l) * 16, PC, Ti + (lo + l) * 16 * PC + (lo + j) * 16, PC, 16, acc);
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[(r4 + e) * 36 + col] = acc[e];
    }
    __syncthreads();
    if (works) {
      f4 acc = {0, 0, 0, 0};
      for (int l = 0; l <= i; ++l)
        acc = mm(Ti + (hi + i) * 16 * PC + (hi + l) * 16, PC, mine + (l - i) * 16 * 36, 36, 16, acc);
#pragma unroll
      for (int e = 0; e < 4; ++e) Ti[((hi + i) * 16 + r4 + e) * PC + (lo + j) * 16 + col] = -acc[e];
    }
    __syncthreads();
  }
}

// PAST: past the caches
template <bool PAST>
__device__ __forceinline__ void store_frag(__bf16* p, b8 v) {
  if constexpr (PAST) __builtin_nontemporal_store(v, reinterpret_cast<b8*>(p));
  else *reinterpret_cast<b8*>(p) = v;
}

// rows, or with TR columns, of a lower triangular C x C matrix in LDS (pitch PC) as fragments in natural order; those that
// hold only zeros are neither written nor read
template <int NPL, bool TR, bool PAST>
__device__ __forceinline__ void store_square(const float* M, __bf16* dst, int t) {
  for (int i = t; i < TF / 8; i += 256) {
    const int lane = i & 63, ks = i >> 6 & 1, rb = i >> 7;
    const int r = rb * 16 + (lane & 15), c = ks * 32 + (lane >> 4) * 8;
    if (TR ? ks * 2 + 1 < rb : ks * 2 > rb) continue;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = TR ? M[(c + e) * PC + r] : M[r * PC + c + e];
    b8 v[NPL];
    split<8, NPL>(x, v);
#pragma unroll
    for (int k = 0; k < NPL; ++k) store_frag<PAST>(dst + k * TF + i * 8, v[k]);
  }
}

// Planes of what only the output sees (S, P and U there): two (16 bits) under bf16's 8, where the result's error is 1.00003 times that of
// rounding the exact one; under fp16's 11 bits two would make it 1.0024 times
template <typename T> struct OutPlanes { static constexpr int N = std::is_same<T, __bf16>::value ? 2 : 3; };

// ---- prep: one chunk of one key head and its value heads -----------------------------------------------------------------
// Many chunks: bound by memory, mostly its own stores (2048 chunks of 128 x 128 in bf16: 231 MB in 60 us, 337 MB in 84 with what
// training keeps).  Few: by the inverse and its barriers, 24 us for one chunk in fp32, so that value heads that share a key head get a
// workgroup each while these fit the chip twice (fp32, 28 chunks of two heads: 33 -> 25 us; fp16, 348: 28 -> 38, so not there).
// PAST: what it writes goes past the caches, for large training steps, in whose scans it would not last in them (2048 chunks: 83 -> 81 us,
// the scans 193 -> 185; forward alone 59 -> 50, but the scan 239 -> 249; small steps 24 -> 23 and 22 -> 23).
template <typename T, int DK>
constexpr size_t chunk_room() {
  constexpr size_t first = 2 * Planes<T>::N * C * (DK + 8) * 2, second = (2 * C * PC + 32 * 36) * 4;
  return first > second ? first : second;
}

template <typename T, int DK, bool PAST>
__global__ __launch_bounds__(256, Planes<T>::N == 1 ? 4 : 1) void delta_chunk_kernel(const Args a) {
  constexpr int N = Planes<T>::N, P = DK + 8, RT = DK / 64, KSN = DK / 32;
  extern __shared__ __align__(16) char smem[];
  __bf16* K = reinterpret_cast<__bf16*>(smem);
  __bf16* Q = K + N * C * P;
  float* A = reinterpret_cast<float*>(smem);   // over K and Q, once these are in registers and memory
  float* M = A + C * PC;
  float* tmp = M + C * PC;
  f2* G = reinterpret_cast<f2*>(smem + chunk_room<T, DK>());
  float* beta = reinterpret_cast<float*>(G + C);
  const int part = blockIdx.x % a.parts, hk = blockIdx.x / a.parts % a.d.key_heads, slot = blockIdx.x / a.parts / a.d.key_heads;
  const int first = a.group / a.parts * part, last = first + a.group / a.parts;   // value heads of the key head
  int s, t0, len;
  a.p.locate(slot, s, t0, len);
  if (len == 0) return;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), col = lane & 15, g8 = (lane >> 4) * 8;
  const long row = a.p.row(s), atk = (long)slot * a.d.key_heads + hk;
  float gv = 0.f, bv = 0.f;   // wave 0: g and beta of the next value head
  auto load_g = [&](int hv) {
    const int tok = t0 + min(lane, len - 1);
    gv = a.d.g[row * a.d.g_st.bs + tok * a.d.g_st.rs + hv * a.d.g_st.cs];
    bv = a.d.beta[row * a.d.beta_st.bs + tok * a.d.beta_st.rs + hv * a.d.beta_st.cs];
  };
  if (wave == 0) load_g(hk * a.group + first);
  // wave 0: G, beta and the factors of value head hv; the next head's values set off
  auto factors = [&](int hv) {
    const long at = (long)slot * a.d.value_heads + hv;
    const float g = lane < len ? gv : 0.f, b = lane < len ? bv : 0.f;
    load_g(min(hv + 1, a.d.value_heads - 1));
    double x = g < G_MIN ? G_MIN : g;
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(x, o);
      if (lane >= o) x += y;
    }
    const double sum = __shfl(x, 63);
    G[lane] = a.G[at * C + lane] = in_parts(x);
    beta[lane] = b;
    float* f = a.fac + at * FACS + lane;
    const float eg = expf((float)x), tail = expf((float)(sum - x));
    f[0] = eg;
    f[C] = b;
    f[2 * C] = tail * b;
    f[3 * C] = expf((float)sum);
    f[4 * C] = tail;
    f[5 * C] = eg * b;
  };
  {
    Rows<T, DK> k, q;
    k.fetch(a.d.k, a.d.k_st, row, t0, len, hk, a.d.dk, t);
    q.fetch(a.d.q, a.d.q_st, row, t0, len, hk, a.d.dk, t);
    if (wave == 0) factors(hk * a.group + first);
    k.put(K, len, a.d.dk, t);
    q.put(Q, len, a.d.dk, t);
  }
  __syncthreads();
  // K and Q in state order, K^T in natural order
  const int mine = part == 0 ? t : KF;   // one workgroup writes them
  for (int i = mine; i < KF / 8; i += 256) {
    const int l = i & 63, w = i >> 6 & 3, rb = i >> 8;
    const int r = rb * 16 + (l & 15), c = w * RT * 16 + (l >> 4) * 4;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const __bf16* x = K + (k * C + r) * P + c;
      const __bf16* y = Q + (k * C + r) * P + c;
      b4 z = {0, 0, 0, 0};
      const b4 x0 = *reinterpret_cast<const b4*>(x), y0 = *reinterpret_cast<const b4*>(y);
      const b4 x1 = RT == 2 ? *reinterpret_cast<const b4*>(x + 16 * (RT - 1)) : z;
      const b4 y1 = RT == 2 ? *reinterpret_cast<const b4*>(y + 16 * (RT - 1)) : z;
      store_frag<PAST>(a.Kf + (atk * N + k) * KF + i * 8, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
      store_frag<PAST>(a.Qf + (atk * N + k) * KF + i * 8, __builtin_shufflevector(y0, y1, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
  for (int i = mine; i < DK * C / 8; i += 256) {
    const int l = i & 63, ks = i >> 6 & 1, rb = i >> 7;
    const int c = rb * 16 + (l & 15), r = ks * 32 + (l >> 4) * 8;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      b8 v, w;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = K[(k * C + r + e) * P + c];
        w[e] = Q[(k * C + r + e) * P + c];
      }
      store_frag<PAST>(a.KTf + (atk * N + k) * (DK * C) + i * 8, v);
      if (a.save) store_frag<PAST>(a.QTf + (atk * N + k) * (DK * C) + i * 8, w);
    }
  }
  // K K^T and Q K^T: wave w the rows 16 w ..
  f4 nn[4], pp[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    nn[j] = pp[j] = f4{0, 0, 0, 0};
    if (j > wave) continue;
#pragma unroll
    for (int ks = 0; ks < KSN; ++ks) {
      b8 x[N], y[N], z[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        x[k] = *reinterpret_cast<const b8*>(K + (k * C + wave * 16 + col) * P + ks * 32 + g8);
        y[k] = *reinterpret_cast<const b8*>(Q + (k * C + wave * 16 + col) * P + ks * 32 + g8);
        z[k] = *reinterpret_cast<const b8*>(K + (k * C + j * 16 + col) * P + ks * 32 + g8);
      }
      nn[j] = planes_mma<N, N, 3>(x, z, nn[j]);
      pp[j] = planes_mma<N, N, 3>(y, z, pp[j]);
    }
  }
  for (int m = first; m < last; ++m) {
    const int hv = hk * a.group + m;
    int tt = threadIdx.x;
    asm volatile("" : "+v"(tt));   // opaque: addresses of all matrices held over the loop are spilled
    const int t = tt, lane = t & 63, r4 = (lane >> 4) * 4, col = lane & 15;
    const long at = (long)slot * a.d.value_heads + hv;
    if (m > first && wave == 0) factors(hv);
    __syncthreads();
    f4 nd[4];   // N
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = j * 16 + col;
      nd[j] = f4{0, 0, 0, 0};
      if (j <= wave) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = wave * 16 + r4 + e;
          const float D = r >= c ? decay(G[r], G[c]) : 0.f;
          nd[j][e] = r > c ? nn[j][e] * D : 0.f;
          A[r * PC + c] = nd[j][e] * beta[c];
          M[r * PC + c] = r >= c ? pp[j][e] * D : 0.f;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) A[(wave * 16 + r4 + e) * PC + c] = M[(wave * 16 + r4 + e) * PC + c] = 0.f;
      }
    }
    __syncthreads();
    store_square<OutPlanes<T>::N, false, PAST>(M, a.Pf + at * OutPlanes<T>::N * TF, t);
    if (a.save) store_square<3, true, PAST>(M, a.PTf + at * 3 * TF, t);
    __syncthreads();
    unit_lower_inverse(A, M, tmp, wave, lane);
    store_square<3, false, PAST>(M, a.Tf + at * 3 * TF, t);
    if (a.save) {   // (I + diag(beta) N)^-1 = I - diag(beta) T N
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) A[(wave * 16 + r4 + e) * PC + j * 16 + col] = nd[j][e];
      __syncthreads();
      f4 t2[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) t2[j] = f4{0, 0, 0, 0};
#pragma unroll
      for (int l = 0; l < 4; ++l)   // N's block rows, each for up to four sums side by side
        if (l <= wave)
#pragma unroll
          for (int j = 0; j <= l; ++j) t2[j] = mm(M + wave * 16 * PC + l * 16, PC, A + l * 16 * PC + j * 16, PC, 16, t2[j]);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j > wave) continue;   // zeros already
        const int c = j * 16 + col;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = wave * 16 + r4 + e;
          A[r * PC + c] = (r == c ? 1.f : 0.f) - beta[r] * t2[j][e];
        }
      }
      __syncthreads();
      store_square<3, true, PAST>(A, a.T2f + at * 3 * TF, t);
    }
    __syncthreads();
  }
}

// ---- the scans: 16 columns of dv of one value head of one sequence ----------------------------------------------------------------
// Forward, chunk after chunk:    X = V - exp(G) K S;       E = T X;      S <- exp(G_C) S + K^T (exp(G_C - G) beta E)
// Backward (BACK), from the last: X = Y + exp(G_C - G) K dS;  Z = T2^T X;   dS <- exp(G_C) dS - K^T (exp(G) beta Z) + Q^T Of
// (Y = scale P^T dO, Of = scale exp(G) dO).
// Bound by the chain from chunk to chunk: the product with K (each wave with its own rows of S, which are in its accumulators;
// partial sums through LDS), X through LDS, the product with T, U through LDS, the product with K^T: three barriers.  Four waves do that
// and nothing else; four more take S and E from LDS and do what the chain does not wait for -- forward the outputs
// O = scale (exp(G) Q S + P beta E), backward Q^T Of and the next chunk's Y, and all stores.  (A wave waits for its memory accesses
// in order: with the stores in the chain's waves its loads waited for them.)  Fragments come straight from memory, up to a chunk
// ahead (two gained nothing), issued under the latency of LDS reads or matrix instructions; every load is issued whatever comes,
// since loads behind branches make the compiler wait for all that are under way.
// 8192 tokens x 16 heads, bf16, dk = dv = 128, 128 workgroups: 237 us, 1.85 a chunk, of which 78 KB of operands take 0.5 at L1's 64
// bytes a clock; without any access to memory 137; with the outputs in a kernel of their own 256 and 68; with 32 columns to a
// workgroup 349.  Training on 2 x 4096 tokens, 256 workgroups: 191 forward, 130 to 140 without the stores of S and E (200 MB),
// 182 back, where Y from a kernel of its own took 54 more.
__device__ __forceinline__ b8 ld_frag(const __bf16* uniform, unsigned lane_bytes) {
  return *reinterpret_cast<const b8*>(reinterpret_cast<const char*>(uniform) + lane_bytes);
}

template <typename T, int DK, bool BACK, bool TWO>
__global__ __launch_bounds__(512, TWO ? 4 : 2) void delta_chain_kernel(const Args a) {
  constexpr int N = Planes<T>::N, NO = OutPlanes<T>::N, RT = DK / 64, PT = C + 8, PE = C + 4;
  __shared__ f4 part[4][4][64];                  // K S: wave, row block
  constexpr int NS = BACK ? 0 : NO;
  __shared__ b8 Sp[2][4][NS + 1][64];            // planes of S for the outputs: parity of the chunk, wave
  __shared__ f4 Sx[2][4][2][64];                 // S to be stored: parity, wave, tile
  constexpr int NB = BACK ? 1 : 0;
  __shared__ f4 Rx[4][2][64];                    // BACK: Q^T Of, likewise
  __shared__ __align__(16) float Yx[NB + 1][16][PE];       // BACK: Y^T, parity
  __shared__ __align__(16) __bf16 Ox[N][16][PT];           // BACK: dO^T
  __shared__ __align__(16) float Ex[2][16][PE];  // E^T or Z^T, parity of the chunk
  __shared__ __align__(16) __bf16 X[3][16][PT], U[3][16][PT];
  const int heads = a.p.sequences * a.d.value_heads, slices = a.dvp / 16;
  int slice, head;
  if (!scan_coords(blockIdx.x, slices, heads, slice, head)) return;
  const int s = a.p.by_length(head / a.d.value_heads), hv = head % a.d.value_heads, hk = hv / a.group;
  const int c0 = slice * 16;
  const int t = threadIdx.x, lane = t & 63, wave8 = __builtin_amdgcn_readfirstlane(t >> 6), wave = wave8 & 3, r4 = (lane >> 4) * 4,
            col = lane & 15, g8 = (lane >> 4) * 8;
  const int begin = a.p.begin(s), end = a.p.end(s), chunks = (end - begin + C - 1) / C;
  const long slot0 = a.p.slot0(s), row = a.p.row(s);
  const unsigned lb = lane * 16;

  if (wave8 < 4) {   // ---- the chain
    __builtin_amdgcn_s_setprio(3);
    f4 S[RT];
    const float* init = BACK ? a.d_state_out : a.state;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = (wave * RT + i) * 16 + r4 + e, c = c0 + col;
        S[i][e] = init != nullptr && r < a.d.dk && c < a.d.dv ? init[(((long)s * a.d.value_heads + hv) * a.d.dk + r) * a.d.dv + c] : 0.f;
      }
    b8 kf[4][N], tf[2][3], kt[RT][2][N];
    T v[4];
    f4 fx, fu;
    float keep;
    const T* V = reinterpret_cast<const T*>(a.d.v) + row * a.d.v_st.bs + begin * a.d.v_st.rs + hv * a.d.v_st.cs;
    const unsigned vrs = (unsigned)a.d.v_st.rs, vcol = min(c0 + col, a.d.dv - 1);
    auto load_k = [&](long slot) {
      const __bf16* p = a.Kf + (slot * a.d.key_heads + hk) * N * KF + wave * 512;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < N; ++k) kf[i][k] = ld_frag(p + k * KF + i * 4 * 512, lb);
    };
    auto load_x = [&](long at, int m) {
      if (!BACK) {   // rows and columns behind the end repeat the last; they are masked where they are used
        const T* p = V + (long)m * C * a.d.v_st.rs;
        const unsigned last = min(C, end - begin - m * C) - 1;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = p[min((unsigned)(wave * 16 + r4 + e), last) * vrs + vcol];
      }
      fx = *reinterpret_cast<const f4*>(a.fac + at * FACS + (BACK ? 4 * C : 0) + wave * 16 + r4);
    };
    auto load_t = [&](long at) {
      const __bf16* p = (BACK ? a.T2f : a.Tf) + at * 3 * TF + wave * 2 * 512;
      const int k0 = BACK && wave >= 2 ? 512 : 0, k1 = !BACK && wave < 2 ? 0 : 512;   // not the zeros: these are not there
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        tf[0][k] = ld_frag(p + k * TF + k0, lb);
        tf[1][k] = ld_frag(p + k * TF + k1, lb);
      }
      fu = *reinterpret_cast<const f4*>(a.fac + at * FACS + (BACK ? 5 : 2) * C + wave * 16 + r4);
    };
    auto load_kt = [&](long slot, long at) {
      const __bf16* p = a.KTf + (slot * a.d.key_heads + hk) * N * (DK * C) + wave * RT * 2 * 512;
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int k = 0; k < N; ++k) kt[i][ks][k] = ld_frag(p + k * (DK * C) + (i * 2 + ks) * 512, lb);
      keep = a.fac[at * FACS + 3 * C + lane];   // by lane: a scalar load would be waited for with LDS
    };
    auto chunk = [&](int n) {
      const int m = BACK ? chunks - 1 - n : n, nm = BACK ? max(m - 1, 0) : min(m + 1, chunks - 1);
      const long nslot = slot0 + nm, nat = nslot * a.d.value_heads + hv;
      const long slot = slot0 + m, at = slot * a.d.value_heads + hv;
      const int live = BACK ? 0 : end - begin - n * C - wave * 16 - r4;   // rows e < live hold tokens
      {
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = S[0][e];
          x[4 + e] = RT == 2 ? S[RT - 1][e] : 0.f;
        }
        b8 sb[3];
        split<8, 3>(x, sb);
#pragma unroll
        for (int k = 0; k < NS; ++k) Sp[n & 1][wave][k][lane] = sb[k];
        if (BACK || a.save) {
          Sx[n & 1][wave][0][lane] = S[0];
          if (RT == 2) Sx[n & 1][wave][1][lane] = S[RT - 1];
        }
        f4 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = f4{0, 0, 0, 0};
        // plane by plane over the four row blocks: four chains of matrix instructions side by side
#pragma unroll
        for (int q = 2; q >= 0; --q)
#pragma unroll
          for (int k = 0; k < N; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (q >= k) p[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[i][k], sb[q - k], p[i], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (!BACK) load_kt(slot, at);   // this chunk's: used behind its third barrier
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) part[wave][i][lane] = p[i];
      }
      lds_barrier();
      {
        const f4 p0 = part[0][wave][lane], p1 = part[1][wave][lane], p2 = part[2][wave][lane], p3 = part[3][wave][lane];
        const f4 y = BACK ? *reinterpret_cast<const f4*>(&Yx[n & NB][col][wave * 16 + r4]) : f4{0, 0, 0, 0};
        __builtin_amdgcn_sched_barrier(0);
        load_k(nslot);
        __builtin_amdgcn_sched_barrier(0);
        const f4 p = (p0 + p1) + (p2 + p3);
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[e] = BACK ? fmaf(fx[e], p[e], y[e]) : e < live && c0 + col < a.d.dv ? fmaf(-fx[e], p[e], (float)v[e]) : 0.f;
        b4 xp[3];
        split<4, 3>(x, xp);
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<b4*>(&X[k][col][wave * 16 + r4]) = xp[k];
      }
      lds_barrier();
      {
        // T's upper, T2^T's lower half is zeros
        f4 e0 = {0, 0, 0, 0}, e1 = {0, 0, 0, 0};
        b8 xb[2][3];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int k = 0; k < 3; ++k) xb[ks][k] = *reinterpret_cast<const b8*>(&X[k][col][ks * 32 + g8]);
        __builtin_amdgcn_sched_barrier(0);
        load_x(nat, nm);
        __builtin_amdgcn_sched_barrier(0);
        if (!BACK || wave < 2) e0 = planes_mma<3, 3, 3>(tf[0], xb[0], e0);
        if (BACK || wave >= 2) e1 = planes_mma<3, 3, 3>(tf[1], xb[1], e1);
        const f4 fv = fu;
        __builtin_amdgcn_sched_barrier(0);
        load_t(nat);
        __builtin_amdgcn_sched_barrier(0);
        const f4 ev = e0 + e1;
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (BACK ? -fv[e] : fv[e]) * ev[e];
        b4 up[3];
        split<4, 3>(w, up);
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<b4*>(&U[k][col][wave * 16 + r4]) = up[k];
        *reinterpret_cast<f4*>(&Ex[n & 1][col][wave * 16 + r4]) = ev;
      }
      lds_barrier();
      {
        f4 more[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          S[i] *= keep;
          more[i] = BACK ? Rx[wave][i][lane] : f4{0, 0, 0, 0};
        }
        b8 ub[2][3];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int k = 0; k < 3; ++k) ub[ks][k] = *reinterpret_cast<const b8*>(&U[k][col][ks * 32 + g8]);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          S[i] = planes_mma<N, 3, 3>(kt[i][0], ub[0], S[i]);
          more[i] = planes_mma<N, 3, 3>(kt[i][1], ub[1], more[i]);
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) S[i] += more[i];
        __builtin_amdgcn_sched_barrier(0);
        if (BACK) load_kt(nslot, nat);   // a chunk ahead, where registers allow it (forward slower: 245 us for 239)
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (chunks > 0) {
      const int m = BACK ? chunks - 1 : 0;
      const long slot = slot0 + m, at = slot * a.d.value_heads + hv;
      load_k(slot);
      load_x(at, m);
      load_t(at);
      if (BACK) load_kt(slot, at);
      if (BACK) {   // the other waves' start
        lds_barrier();
        lds_barrier();
      }
    }
    for (int n = 0; n < chunks; ++n) chunk(n);
    float* out = BACK ? a.d_state : a.state_out;
    if (out != nullptr) {
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = (wave * RT + i) * 16 + r4 + e, c = c0 + col;
          if (r < a.d.dk && c < a.d.dv) out[(((long)s * a.d.value_heads + hv) * a.d.dk + r) * a.d.dv + c] = S[i][e];
        }
    }
  } else if constexpr (BACK) {
    // ---- beside the chain: Q^T Of of this chunk, Y of the next, all stores
    b8 qt[RT][2][N], of[2][N], pt[2][3];
    f4 eg[4];
    T d[4];
    const int srow = lane >> 2, sc = (lane & 3) * 4;   // S, Z: 4 columns of one row per lane, a kilobyte in a row
    auto slot_of = [&](int n) { return slot0 + chunks - 1 - min(n, chunks - 1); };
    auto load_q = [&](int n) {
      const long slot = slot_of(n), at = slot * a.d.value_heads + hv;
      const __bf16* p = a.QTf + (slot * a.d.key_heads + hk) * N * (DK * C) + wave * RT * 2 * 512;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int k = 0; k < N; ++k) qt[i][ks][k] = ld_frag(p + k * (DK * C) + (i * 2 + ks) * 512, lb);
      const float* f = a.fac + at * FACS + g8;
#pragma unroll
      for (int i = 0; i < 4; ++i) eg[i] = *reinterpret_cast<const f4*>(f + (i >> 1) * 32 + (i & 1) * 4);
    };
    auto load_p = [&](int n) {   // P^T is upper triangular, its zeros are not there
      const __bf16* p = a.PTf + (slot_of(n) * a.d.value_heads + hv) * 3 * TF + wave * 2 * 512;
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        pt[0][k] = ld_frag(p + k * TF + (wave < 2 ? 0 : 512), lb);
        pt[1][k] = ld_frag(p + k * TF + 512, lb);
      }
    };
    const T* dO = reinterpret_cast<const T*>(a.d_o) + row * a.do_st.bs + hv * a.do_st.cs + min(c0 + col, a.d.dv - 1);
    auto load_o = [&](int n) {
      const int tok = begin + (chunks - 1 - min(n, chunks - 1)) * C + wave * 16 + r4;
#pragma unroll
      for (int e = 0; e < 4; ++e) d[e] = dO[min(tok + e, end - 1) * a.do_st.rs];
    };
    auto put_o = [&](int n) {   // what load_o(n) brought
      const int live = end - begin - (chunks - 1 - min(n, chunks - 1)) * C - wave * 16 - r4;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = e < live && c0 + col < a.d.dv ? (float)d[e] : 0.f;
      b4 xp[N];
      split<4, N>(x, xp);
#pragma unroll
      for (int k = 0; k < N; ++k) *reinterpret_cast<b4*>(&Ox[k][col][wave * 16 + r4]) = xp[k];
    };
    auto product_y = [&](int n) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int k = 0; k < N; ++k) of[ks][k] = *reinterpret_cast<const b8*>(&Ox[k][col][ks * 32 + g8]);
      f4 y = {0, 0, 0, 0};
      if (wave < 2) y = planes_mma<3, N, 3>(pt[0], of[0], y);
      y = planes_mma<3, N, 3>(pt[1], of[1], y);
      *reinterpret_cast<f4*>(&Yx[n & NB][col][wave * 16 + r4]) = y * a.scale;
    };
    auto place = [&](float* base, int n, int rows) {
      return base + (slot_of(n) * a.d.value_heads + hv) * (long)(rows * a.dvp) + c0 * rows;
    };
    auto store_z = [&](int n) {
      f4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = Ex[n & 1][sc + e][wave * 16 + srow];
      __builtin_nontemporal_store(v, reinterpret_cast<f4*>(place(a.Z, n, C) + (unsigned)((wave * 16 + srow) * 16 + sc)));
    };
    auto chunk = [&](int n) {
      f4 r[RT];
#pragma unroll
      for (int i = 0; i < RT; ++i) r[i] = f4{0, 0, 0, 0};
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float v = 0.f;
#pragma unroll
          for (int k = 0; k < N; ++k) v += (float)of[ks][k][e];
          x[e] = a.scale * eg[ks * 2 + (e >> 2)][e & 3] * v;
        }
        b8 ob[3];
        split<8, 3>(x, ob);
#pragma unroll
        for (int i = 0; i < RT; ++i) r[i] = planes_mma<N, 3, 3>(qt[i][ks], ob, r[i]);
      }
      put_o(n + 1);
      load_o(n + 2);
      lds_barrier();
#pragma unroll
      for (int i = 0; i < RT; ++i) Rx[wave][i][lane] = r[i];   // the chain has read those of the chunk before
      load_q(n + 1);
      product_y(n + 1);
      load_p(n + 2);
      lds_barrier();
      if (n > 0) store_z(n - 1);
      float* dst = place(a.dS, n, DK) + wave * RT * 256;
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const float* p = reinterpret_cast<const float*>(&Sx[n & 1][wave][i][(srow >> 2) * 16 + sc]) + (srow & 3);
        __builtin_nontemporal_store(f4{p[0], p[4], p[8], p[12]}, reinterpret_cast<f4*>(dst + (unsigned)((i * 16 + srow) * 16 + sc)));
      }
      lds_barrier();
    };
    if (chunks > 0) {
      load_o(0);
      load_q(0);
      load_p(0);
      put_o(0);
      load_o(1);
      lds_barrier();
      product_y(0);
      load_p(1);
      lds_barrier();
      for (int n = 0; n < chunks; ++n) chunk(n);
      store_z(chunks - 1);
    }
  } else {
    // ---- beside the chain, one chunk behind it: the work on chunk n - 1 is spread over the three stretches of chunk n, the longest
    // first, so that no barrier waits for it.
    // Fragments a chunk ahead; where registers allow it, two sets and two chunks (8192 tokens: 237 us for 248).
    constexpr int SETS = TWO ? 1 : 2;
    b8 qf[SETS][4][N], pf[SETS][2][NO];
    f4 eg[SETS], bt[SETS][4], o;
    // S and E go to memory 4 columns of one row per lane, a kilobyte in a row, past the caches that the operands need (2 x 4096 tokens:
    // 207 us in rows of 32 columns, which two workgroups share, 205 in a row, 201 past the caches; backward 200, 194, 185)
    const int srow = lane >> 2, sc = (lane & 3) * 4;
    auto load_q = [&](int u, int n) {
      const long slot = slot0 + min(n, chunks - 1), at = slot * a.d.value_heads + hv;
      const __bf16* q = a.Qf + (slot * a.d.key_heads + hk) * N * KF + wave * 4 * 512;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < N; ++k) qf[u][i][k] = ld_frag(q + k * KF + i * 512, lb);
      eg[u] = *reinterpret_cast<const f4*>(a.fac + at * FACS + wave * 16 + r4);
    };
    auto load_p = [&](int u, int n) {
      const long at = (slot0 + min(n, chunks - 1)) * a.d.value_heads + hv;
      const __bf16* p = a.Pf + at * NO * TF + wave * 2 * 512;
#pragma unroll
      for (int k = 0; k < NO; ++k) {
        pf[u][0][k] = ld_frag(p + k * TF, lb);
        pf[u][1][k] = ld_frag(p + k * TF + (wave < 2 ? 0 : 512), lb);
      }
      const float* f = a.fac + at * FACS + C + g8;
#pragma unroll
      for (int i = 0; i < 4; ++i) bt[u][i] = *reinterpret_cast<const f4*>(f + (i >> 1) * 32 + (i & 1) * 4);
    };
    // Q S, the terms of chain wave w
    auto q_part = [&](int u, int n, int w) {
      b8 sb[NO];
#pragma unroll
      for (int k = 0; k < NS; ++k) sb[k] = Sp[n & 1][w][k][lane];
      o = planes_mma<N, NO, N == 2 ? 3 : NO>(qf[u][w], sb, o);
    };
    // E of chunk n
    auto flush = [&](int n) {
      if (a.save) {
        float* dst = a.Erow + ((slot0 + n) * a.d.value_heads + hv) * (long)(C * a.dvp) + c0 * C + wave * 256;
        f4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = Ex[n & 1][sc + e][wave * 16 + srow];
        __builtin_nontemporal_store(v, reinterpret_cast<f4*>(dst + (unsigned)(srow * 16 + sc)));
      }
    };
    auto first = [&](int u, int n) {
      if (n > 0) flush(n - 1);
      o = f4{0, 0, 0, 0};
      q_part(u, n, 0);
      q_part(u, n, 1);
      q_part(u, n, 2);
      if (a.save) {
        float* dst = a.Srow + ((slot0 + n) * a.d.value_heads + hv) * (long)(DK * a.dvp) + c0 * DK + wave * RT * 256;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          const float* p = reinterpret_cast<const float*>(&Sx[n & 1][wave][i][(srow >> 2) * 16 + sc]) + (srow & 3);
          __builtin_nontemporal_store(f4{p[0], p[4], p[8], p[12]}, reinterpret_cast<f4*>(dst + (unsigned)((i * 16 + srow) * 16 + sc)));
        }
      }
    };
    auto second = [&](int u, int n) {
      q_part(u, n, 3);
      o *= eg[u];
      load_q(u, n + SETS);
    };
    auto third = [&](int u, int n) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        if (ks * 2 > wave) continue;   // P is lower triangular
        const f4 e0 = *reinterpret_cast<const f4*>(&Ex[n & 1][col][ks * 32 + g8]),
                 e1 = *reinterpret_cast<const f4*>(&Ex[n & 1][col][ks * 32 + g8 + 4]);
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = e0[e] * bt[u][ks * 2][e];
          x[4 + e] = e1[e] * bt[u][ks * 2 + 1][e];
        }
        b8 ub[NO];
        split<8, NO>(x, ub);
        o = planes_mma<NO, NO, NO>(pf[u][ks], ub, o);
      }
      load_p(u, n + SETS);
      const int tok = begin + n * C + wave * 16 + r4;
      T* out = reinterpret_cast<T*>(a.o) + ((row * a.d.tokens + tok) * a.d.value_heads + hv) * (long)a.d.dv + c0 + col;
      if (c0 + col < a.d.dv)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (tok + e < end) out[(long)e * a.d.value_heads * a.d.dv] = (T)(a.scale * o[e]);
    };
    // u: the set of chunk n
    auto chunk = [&](int u, int n) {
      if (n > 0) first(SETS - 1 - u, n - 1);
      lds_barrier();
      if (n > 0) second(SETS - 1 - u, n - 1);
      lds_barrier();
      if (n > 0) third(SETS - 1 - u, n - 1);
      lds_barrier();
    };
    if (chunks > 0) {
#pragma unroll
      for (int u = 0; u < SETS; ++u) {
        load_q(u, u);
        load_p(u, u);
      }
      for (int n = 0; n < chunks; n += SETS) {
        chunk(0, n);
        if (SETS == 2 && n + 1 < chunks) chunk(SETS - 1, n + 1);
      }
      auto rest = [&](int u, int n) {
        first(u, n);
        second(u, n);
        third(u, n);
      };
      const int n = chunks - 1;
      if (SETS == 2 && (n & 1))
        rest(SETS - 1, n);
      else
        rest(0, n);
      flush(n);
    }
  }
}

// ---- gradients: one chunk of one key head, its value heads one after the other ------------------------------------------------
// 8 waves.  DK / 16 of them own 16 columns of dk each and all 64 rows of dQ, dKr and dKc; their operands over dv are S and dS' from
// memory (a wave's own rows) and Y = dO, X = beta Z, U = beta E of 32 columns of dv at a time from LDS.  dP = dO U^T and dX U^T:
// the ten 16 x 16 tiles on and below the diagonal, spread over the waves.
// 2 x 4096 tokens x 16 heads, bf16, 128 x 128: 235 us for 655 MB, 2.8 TB/s, 9 of them for d_g.  The slices wait for memory (a third of the time),
// the steps after them for LDS, where all waves read the whole C x C matrix; neither overlaps the other, since the registers leave one
// workgroup to a CU.  One that went on from chunk to chunk with the next one's first loads under way took as long.
// LDS of the slices, which a C x C matrix of three planes takes over
template <typename T>
constexpr size_t grads_room() {
  constexpr size_t slices = (Planes<T>::N + 6) * C * 40, square = 3 * C * (C + 8);
  return 2 * (slices > square ? slices : square);
}

// HEADS: what a workgroup takes of a key head -- its one value head; all, one after the other; one of several, leaving its dQ and dK in
// fp32 to delta_join_heads_kernel (where workgroups are few: 700 ragged tokens, 2 key heads, fp32: 53 -> 31 us with the joining)
enum { ALONE, GROUPED, APART };

template <typename T, int DK, int HEADS>
__global__ __launch_bounds__(512) void delta_grads_kernel(const Args a) {
  constexpr int N = Planes<T>::N, W = DK / 16, P = 40, PM = C + 8;
  constexpr int SL = C * P;                      // a plane of a slice
  extern __shared__ __align__(16) char smem[];
  __bf16* Y = reinterpret_cast<__bf16*>(smem);   // N planes
  __bf16* X = Y + N * SL;                        // 3
  __bf16* U = X + 3 * SL;                        // 3
  __bf16* M = reinterpret_cast<__bf16*>(smem);   // later: a C x C matrix, 3 planes
  f2* G = reinterpret_cast<f2*>(smem + grads_room<T>());
  float* read = reinterpret_cast<float*>(G + C);   // r and c of the header, 8 x C each: per wave
  float* written = read + 8 * C;
  float* ef = written + 8 * C;  // exp(G), exp(G_C - G): C each
  float* red = ef + 2 * C;      // 8
  float* rows_ = red + 8;       // sums over dP o P + dN o N, 16 each of its ten tiles: of rows (on the diagonal, of i >= t > j),
  float* cols_ = rows_ + 160;   // of columns,
  float* tiles_ = cols_ + 160;  // of all, 16
  float* db = tiles_ + 16;      // C
  constexpr bool TILES = !(HEADS == GROUPED && sizeof(T) == 4);   // K and Q in LDS, where they fit
  constexpr int PV = 16 / sizeof(T), PK = DK + PV;
  T* Kt = reinterpret_cast<T*>(db + C);
  T* Qt = Kt + (TILES ? C * PK : 0);
  f4* sums = reinterpret_cast<f4*>(Qt + (TILES ? C * PK : 0));   // GROUPED: dQ and dK over the value heads so far, 8 per thread
  const int heads = HEADS == APART ? a.d.value_heads : a.d.key_heads, head = blockIdx.x % heads, slot = blockIdx.x / heads;
  const int hk = HEADS == APART ? head / a.group : head;
  int s, t0, len;
  a.p.locate(slot, s, t0, len);
  if (len == 0) return;
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const long row = a.p.row(s), atk = (long)slot * a.d.key_heads + hk;
  const bool own = wave < W;
  // 4 values of dO and of d_v at a time
  const long dmask = a.do_st.bs | a.do_st.rs | a.do_st.cs;
  const bool wide = (a.d.dv & 3) == 0 && (dmask & 3) == 0 && ((reinterpret_cast<uintptr_t>(a.d_o) | reinterpret_cast<uintptr_t>(a.d_v)) & 15) == 0;
  // rows of d_q and d_k 16 bytes at a time
  const bool whole = TILES && HEADS != APART && a.d.dk % PV == 0 && ((reinterpret_cast<uintptr_t>(a.d_q) | reinterpret_cast<uintptr_t>(a.d_k)) & 15) == 0;
  const int group = HEADS == GROUPED ? a.group : 1;
  if (TILES) {
    const T* Kg = reinterpret_cast<const T*>(a.d.k) + row * a.d.k_st.bs + t0 * a.d.k_st.rs + hk * a.d.k_st.cs;
    const T* Qg = reinterpret_cast<const T*>(a.d.q) + row * a.d.q_st.bs + t0 * a.d.q_st.rs + hk * a.d.q_st.cs;
    constexpr int IT = C * DK / 512;
    T k[IT], q[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = min((i * 512 + t) / DK, len - 1), c = min((i * 512 + t) % DK, a.d.dk - 1);
      k[i] = Kg[r * a.d.k_st.rs + c];
      q[i] = Qg[r * a.d.q_st.rs + c];
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = (i * 512 + t) / DK, c = (i * 512 + t) % DK;
      const bool live = r < len && c < a.d.dk;
      Kt[r * PK + c] = live ? k[i] : T(0);
      Qt[r * PK + c] = live ? q[i] : T(0);
    }
  }
#pragma unroll 1
  for (int m = 0; m < group; ++m) {
    // Opaque, so that neither loads nor addresses of one head's work are kept in registers for the next head
    int tt = threadIdx.x;
    asm volatile("" : "+v"(tt)::"memory");
    const int t = tt, lane = t & 63, r4 = (lane >> 4) * 4, col = lane & 15, g8 = (lane >> 4) * 8;
    const int kc0 = wave * 16 + col;   // this lane's column of dk
    const int sr = t >> 3, sc = (t & 7) * 4;   // a thread's place in a slice: four columns of one row
    const int hv = HEADS == APART ? head : hk * group + m;
    const long at = (long)slot * a.d.value_heads + hv;
    __syncthreads();
    if (wave == 0) {
      G[lane] = a.G[at * C + lane];
      ef[lane] = a.fac[at * FACS + lane];
      ef[C + lane] = a.fac[at * FACS + 4 * C + lane];
    }
    const float keep = a.fac[at * FACS + 3 * C];
    const float bt = a.fac[at * FACS + C + sr];
    f4 q1[4], kr[4], kc[4], dp[2], da[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) q1[i] = kr[i] = kc[i] = f4{0, 0, 0, 0};
    dp[0] = dp[1] = da[0] = da[1] = f4{0, 0, 0, 0};
    float ss = 0.f, dbeta = 0.f;
    const T* dO = reinterpret_cast<const T*>(a.d_o) + row * a.do_st.bs + (t0 + min(sr, len - 1)) * a.do_st.rs + hv * a.do_st.cs;
    T* dv = reinterpret_cast<T*>(a.d_v) + ((row * a.d.tokens + t0 + sr) * a.d.value_heads + hv) * (long)a.d.dv;
    f4 ev, zv, sv[2], tv[2];
    T yv[4];
    // a slice's values, loaded while the slice before it is multiplied (two workgroups on a CU instead, with 128 registers
    // and 56 of them spilled: 330 us for 270)
    auto load_slice = [&](int c0) {
      const long eo = at * (C * a.dvp) + (long)(c0 + (sc & 16)) * C + sr * 16 + (sc & 15);
      ev = *reinterpret_cast<const f4*>(a.Erow + eo);
      zv = *reinterpret_cast<const f4*>(a.Z + eo);
      if (wide) {
        __builtin_memcpy(yv, __builtin_assume_aligned(dO + min(c0 + sc, a.d.dv - 4), 4 * sizeof(T)), sizeof(yv));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) yv[e] = dO[min(c0 + sc + e, a.d.dv - 1)];
      }
      const long so = at * (DK * a.dvp) + (long)(c0 + (g8 & 16)) * DK + min(kc0, DK - 1) * 16 + (g8 & 15);
      const f4* p = reinterpret_cast<const f4*>(a.Srow + so);
      const f4* q = reinterpret_cast<const f4*>(a.dS + so);
      sv[0] = p[0];
      sv[1] = p[1];
      tv[0] = q[0];
      tv[1] = q[1];
    };
    load_slice(0);
    for (int c0 = 0; c0 < a.dvp; c0 += 32) {
      float x[4], u[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool live = sr < len && c0 + sc + e < a.d.dv;
        y[e] = live ? (float)yv[e] : 0.f;
        x[e] = bt * zv[e];
        u[e] = bt * ev[e];
        dbeta = fmaf(ev[e], zv[e], dbeta);
        if (live && !wide) dv[c0 + sc + e] = (T)x[e];
      }
      if (wide && sr < len && c0 + sc < a.d.dv) {
        struct __align__(sizeof(T) * 4) Four { T x[4]; } w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w.x[e] = (T)x[e];
        *reinterpret_cast<Four*>(dv + c0 + sc) = w;
      }
      b8 sb[3], db_[3];
      {
        float sx[8], dx[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sx[e] = sv[e >> 2][e & 3];
          dx[e] = tv[e >> 2][e & 3];
          ss = own ? fmaf(sx[e], dx[e], ss) : 0.f;
        }
        split<8, 3>(sx, sb);
        split<8, 3>(dx, db_);
      }
      b4 yp[N], xp[3], up[3];
      split<4, N>(y, yp);
      split<4, 3>(x, xp);
      split<4, 3>(u, up);
      __syncthreads();   // the slice before this one, or M and MT, are done with
#pragma unroll
      for (int k = 0; k < N; ++k) *reinterpret_cast<b4*>(Y + k * SL + sr * P + sc) = yp[k];
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        *reinterpret_cast<b4*>(X + k * SL + sr * P + sc) = xp[k];
        *reinterpret_cast<b4*>(U + k * SL + sr * P + sc) = up[k];
      }
      __syncthreads();
      load_slice(min(c0 + 32, a.dvp - 32));
      auto rows = [&](const __bf16* base, int rb) { return *reinterpret_cast<const b8*>(base + (rb * 16 + col) * P + g8); };
      if (own) {
#pragma unroll
        for (int rb = 0; rb < 4; ++rb) {
          b8 yy[N], xx[3], uu[3];
#pragma unroll
          for (int k = 0; k < N; ++k) yy[k] = rows(Y + k * SL, rb);
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            xx[k] = rows(X + k * SL, rb);
            uu[k] = rows(U + k * SL, rb);
          }
          q1[rb] = planes_mma<N, 3, 3>(yy, sb, q1[rb]);
          kr[rb] = planes_mma<3, 3, 3>(xx, sb, kr[rb]);
          kc[rb] = planes_mma<3, 3, 3>(uu, db_, kc[rb]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int tile = wave + 8 * h;   // of the ten
        if (tile < 10) {
          const int rb = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, cb = tile - rb * (rb + 1) / 2;
          b8 yy[N], xx[3], uu[3];
#pragma unroll
          for (int k = 0; k < N; ++k) yy[k] = rows(Y + k * SL, rb);
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            xx[k] = rows(X + k * SL, rb);
            uu[k] = rows(U + k * SL, cb);
          }
          dp[h] = planes_mma<N, 3, 3>(yy, uu, dp[h]);
          da[h] = planes_mma<3, 3, 3>(xx, uu, da[h]);
        }
      }
    }
    // row factors; what tokens read of S and leave in S'
    const T* Kg = reinterpret_cast<const T*>(a.d.k) + row * a.d.k_st.bs + t0 * a.d.k_st.rs + hk * a.d.k_st.cs + min(kc0, a.d.dk - 1);
    const T* Qg = reinterpret_cast<const T*>(a.d.q) + row * a.d.q_st.bs + t0 * a.d.q_st.rs + hk * a.d.q_st.cs + min(kc0, a.d.dk - 1);
    auto element = [&](const T* tile, const T* p, const gpx_strided& st_, int r) {
      if (TILES) return (float)tile[r * PK + kc0];
      return r < len && kc0 < a.d.dk ? (float)p[min(r, len - 1) * st_.rs] : 0.f;
    };
    // K^T and Q^T, from here on under way
    b8 kt[2][N], qt[2][N];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const long o = (atk * N + k) * (DK * C) + (min(wave, W - 1) * 2 + ks) * 512;
        kt[ks][k] = ld_frag(a.KTf + o, lane * 16);
        qt[ks][k] = ld_frag(a.QTf + o, lane * 16);
      }
    if (own) {
#pragma unroll
      for (int rb = 0; rb < 4; ++rb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = rb * 16 + r4 + e;
          const float eg = ef[r], kv = element(Kt, Kg, a.d.k_st, r), qv = element(Qt, Qg, a.d.q_st, r);
          q1[rb][e] *= a.scale * eg;
          kr[rb][e] *= -eg;
          kc[rb][e] *= ef[C + r];
          const float x = row_sum(fmaf(qv, q1[rb][e], kv * kr[rb][e])), y = row_sum(kv * kc[rb][e]);
          if (col == 0) {
            read[wave * C + r] = x;
            written[wave * C + r] = y;
          }
        }
    }
    ss = row_sum(ss);
    for (int o = 16; o < 64; o <<= 1) ss += __shfl_xor(ss, o);
    if (lane == 0) red[wave] = keep * ss;
    for (int o = 1; o < 8; o <<= 1) dbeta += __shfl_xor(dbeta, o);
    if ((t & 7) == 0) db[sr] = dbeta;
    // dP o D, dN o D, and the sums of dP o P + dN o N.  K K^T and Q K^T again, as in the chunk kernel; where K and Q are not in LDS, K's
    // fragments and P^T's
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int tile = wave + 8 * h;
      if (tile < 10) {
        const int rb = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, cb = tile - rb * (rb + 1) / 2, c = cb * 16 + col;
        f4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
        if constexpr (TILES) {
          auto planes_of = [&](const T* m, int r, int c, b8* p) {
            T v[8];
            __builtin_memcpy(v, __builtin_assume_aligned(m + r * PK + c, 16), sizeof(v));
            if constexpr (N == 1) {
              __builtin_memcpy(p, v, sizeof(v));
            } else {
              float x[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
              split<8, N>(x, p);
            }
          };
#pragma unroll
          for (int ks = 0; ks < DK / 32; ++ks) {
            b8 x[N], y[N], z[N];
            planes_of(Kt, rb * 16 + col, ks * 32 + g8, x);
            planes_of(Qt, rb * 16 + col, ks * 32 + g8, y);
            planes_of(Kt, cb * 16 + col, ks * 32 + g8, z);
            kk = planes_mma<N, N, 3>(x, z, kk);
            qk = planes_mma<N, N, 3>(y, z, qk);
          }
        } else {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            b8 x[N], z[N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
              const __bf16* f = a.Kf + (atk * N + k) * KF + w * 512;
              x[k] = ld_frag(f + rb * 4 * 512, lane * 16);
              z[k] = ld_frag(f + cb * 4 * 512, lane * 16);
            }
            kk = planes_mma<N, N, 3>(x, z, kk);
          }
          const __bf16* f = a.PTf + at * 3 * TF + ((cb * 2 + (rb >> 1)) * 64 + ((rb & 1) * 2 + (lane >> 5)) * 16 + col) * 8 + (lane >> 4 & 1) * 4;
#pragma unroll
          for (int k = 2; k >= 0; --k) {
            const b4 v = *reinterpret_cast<const b4*>(f + k * TF);
#pragma unroll
            for (int e = 0; e < 4; ++e) qk[e] += (float)v[e];
          }
        }
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = rb * 16 + r4 + e;
          const float D = r >= c ? decay(G[r], G[c]) : 0.f, y = a.scale * dp[h][e], P = TILES ? qk[e] * D : qk[e];
          dp[h][e] = y * D;
          da[h][e] = r > c ? -da[h][e] * D : 0.f;
          w[e] = r > c ? fmaf(da[h][e], kk[e], y * P) : 0.f;
        }
        if (rb == cb) {
          // w[e]: the sum of its column from its row on
#pragma unroll
          for (int e = 2; e >= 0; --e) w[e] += w[e + 1];
          const float a1 = __shfl_down(w[0], 16), a2 = __shfl_down(w[0], 32), a3 = __shfl_down(w[0], 48);
          const float below = (lane < 48 ? a1 : 0.f) + (lane < 32 ? a2 : 0.f) + (lane < 16 ? a3 : 0.f);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = row_sum(col < r4 + e ? w[e] + below : 0.f);
            if (col == 0) rows_[tile * 16 + r4 + e] = x;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = row_sum(w[e]);
            if (col == 0) rows_[tile * 16 + r4 + e] = x;
          }
          float x = (w[0] + w[1]) + (w[2] + w[3]);
          x += __shfl_xor(x, 16);
          x += __shfl_xor(x, 32);
          if (lane < 16) cols_[tile * 16 + col] = x;
          x = row_sum(x);
          if (lane == 0) tiles_[tile] = x;
        }
      }
    }
    // dP o D with K, its transpose with Q; then dN o D and its transpose with K
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const bool tr = w & 1;
      __syncthreads();
      // of the tiles that hold zeros only two are read
      {
        const int z = t >> 8, r = t >> 4 & 15, c = t & 15, rb = z * 2 + (tr ? 1 : 0), cb = z * 2 + (tr ? 0 : 1);
#pragma unroll
        for (int k = 0; k < 3; ++k) M[(k * C + rb * 16 + r) * PM + cb * 16 + c] = (__bf16)0.f;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int tile = wave + 8 * h;
        if (tile < 10) {
          const int rb = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, cb = tile - rb * (rb + 1) / 2, c = cb * 16 + col;
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = w < 2 ? dp[h][e] : da[h][e];
          b4 xp[3];
          split<4, 3>(x, xp);
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            if (tr) {
              *reinterpret_cast<b4*>(M + (k * C + c) * PM + rb * 16 + r4) = xp[k];
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) M[(k * C + rb * 16 + r4 + e) * PM + c] = xp[k][e];
            }
          }
        }
      }
      __syncthreads();
      if (own) {
#pragma unroll
        for (int rb = 0; rb < 4; ++rb)
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            if (tr ? ks * 2 + 1 < rb : ks * 2 > rb) continue;   // zeros
            b8 mm_[3];
#pragma unroll
            for (int k = 0; k < 3; ++k) mm_[k] = *reinterpret_cast<const b8*>(M + (k * C + rb * 16 + col) * PM + ks * 32 + g8);
            if (w == 0) q1[rb] = planes_mma<3, N, 3>(mm_, kt[ks], q1[rb]);
            if (w == 1) kc[rb] = planes_mma<3, N, 3>(mm_, qt[ks], kc[rb]);
            if (w == 2) kr[rb] = planes_mma<3, N, 3>(mm_, kt[ks], kr[rb]);
            if (w == 3) kc[rb] = planes_mma<3, N, 3>(mm_, kt[ks], kc[rb]);
          }
      }
    }
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) {
      kr[rb] += kc[rb];
      if (HEADS == GROUPED) {
        if (m > 0) {
          q1[rb] += sums[rb * 512 + t];
          kr[rb] += sums[(4 + rb) * 512 + t];
        }
        if (m + 1 < group) {
          sums[rb * 512 + t] = q1[rb];
          sums[(4 + rb) * 512 + t] = kr[rb];
        }
      }
      if (m + 1 == group && own && kc0 < a.d.dk) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = rb * 16 + r4 + e;
          if (HEADS == APART) {
            a.d_q_part[(at * C + r) * DK + kc0] = q1[rb][e];
            a.d_k_part[(at * C + r) * DK + kc0] = kr[rb][e];
          } else if (whole) {   // in place of Q and K, which this lane alone has read here
            Qt[r * PK + kc0] = (T)q1[rb][e];
            Kt[r * PK + kc0] = (T)kr[rb][e];
          } else if (r < len) {
            const long p = ((row * a.d.tokens + t0 + r) * a.d.key_heads + hk) * (long)a.d.dk + kc0;
            st<T>(a.d_q, p, q1[rb][e]);
            st<T>(a.d_k, p, kr[rb][e]);
          }
        }
      }
    }
    __syncthreads();
    if (whole && m + 1 == group) {
      const long p = ((row * a.d.tokens + t0) * a.d.key_heads + hk) * (long)a.d.dk, pitch = (long)a.d.key_heads * a.d.dk;
#pragma unroll
      for (int i = t; i < C * DK / PV; i += 512) {
        const int r = i / (DK / PV), c = i % (DK / PV) * PV;
        if (r >= len || c >= a.d.dk) continue;
        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.d_q) + p + r * pitch + c) = *reinterpret_cast<const uint4*>(Qt + r * PK + c);
        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.d_k) + p + r * pitch + c) = *reinterpret_cast<const uint4*>(Kt + r * PK + c);
      }
    }
    if (wave == 0) {
      const int tb = lane >> 4, n = lane & 15;
      float behind = 0.f, before = 0.f, all = 0.f;   // of all tokens
#pragma unroll
      for (int i = 0; i < W; ++i) {
        behind += read[i * C + lane];
        before += written[i * C + lane];
        all += red[i];
      }
      float x = 0.f, y = 0.f;   // rows of this token's block left of the diagonal, columns under it
#pragma unroll
      for (int rb = 1; rb < 4; ++rb)
#pragma unroll
        for (int cb = 0; cb < rb; ++cb) {
          const int tile = rb * (rb + 1) / 2 + cb;
          if (rb == tb) x += rows_[tile * 16 + n];
          if (cb == tb) y += cols_[tile * 16 + n];
          if (rb > tb && cb < tb) all += tiles_[tile];
        }
      before = __shfl_up(before, 1);   // sums before this token: none of them over it
      y = __shfl_up(y, 1);
      if (lane == 0) before = 0.f;
      if (n == 0) y = 0.f;
      for (int o = 1; o < 64; o <<= 1) {
        const float u = __shfl_down(behind, o), w = __shfl_up(before, o), x1 = __shfl_down(x, o), y1 = __shfl_up(y, o);
        if (lane + o < 64) behind += u;
        if (lane >= o) before += w;
        if (n + o < 16) x += x1;
        if (n >= o) y += y1;
      }
      const float v = (behind + before) + (x + y) + (all + rows_[tb * (tb + 3) / 2 * 16 + n]);
      if (lane < len) {
        const long p = (row * a.d.tokens + t0 + lane) * a.d.value_heads + hv;
        a.d_g[p] = v;
        a.d_beta[p] = db[lane];
      }
    }
  }
}

// dQ and dK of a chunk and key head: the sums over its value heads, in their order; 8 rows a workgroup
template <typename T, int DK>
__global__ __launch_bounds__(256) void delta_join_heads_kernel(const Args a) {
  const int r0 = blockIdx.x % 8 * 8, hk = blockIdx.x / 8 % a.d.key_heads, slot = blockIdx.x / 8 / a.d.key_heads;
  int s, t0, len;
  a.p.locate(slot, s, t0, len);
  if (r0 >= len) return;
  const long row = a.p.row(s), at = (long)slot * a.d.value_heads + hk * a.group;
  constexpr int IT = 8 * DK / 256;
  float q[IT], k[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) q[i] = k[i] = 0.f;
#pragma unroll 2
  for (int m = 0; m < a.group; ++m)
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const long p = ((at + m) * C + r0) * DK + i * 256 + threadIdx.x;
      q[i] += a.d_q_part[p];
      k[i] += a.d_k_part[p];
    }
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int r = r0 + (i * 256 + threadIdx.x) / DK, c = (i * 256 + threadIdx.x) % DK;
    if (r >= len || c >= a.d.dk) continue;
    const long p = ((row * a.d.tokens + t0 + r) * a.d.key_heads + hk) * (long)a.d.dk + c;
    st<T>(a.d_q, p, q[i]);
    st<T>(a.d_k, p, k[i]);
  }
}

// ---- the recurrence itself ---------------------------------------------------------------------------------------------
// 64 columns of a state per workgroup: thread = 4 columns x RPT rows, in registers for all of its tokens.  One
// reduction per token, since o = scale (q^T Sbar + (q . k) beta e).  A step of 64 users is bound by the states, 268 MB there and back
// in 44.6 us (6.0 TB/s, a large copy's 5.2 to 5.8); one user's takes a launch (5.6 us, 8 states of 64 x 64).
struct StepArgs {
  Args a;
  const int* slot;   // step: the state of each row
  int slots;
  int step;
};

template <typename T, int DK>
__global__ __launch_bounds__(256) void delta_recurrent_kernel(const StepArgs x) {
  constexpr int RPT = DK / 16;
  const Args& a = x.a;
  __shared__ float sm[2][4][2][64];   // parity, wave, k S / q S, column
  __shared__ float qk[2][2][DK];      // parity, k / q
  const int slices = (a.d.dv + 63) / 64, heads = a.d.value_heads;
  const int slice = blockIdx.x % slices, hv = blockIdx.x / slices % heads, s = blockIdx.x / slices / heads;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, hk = hv / a.group;
  const int cc = (lane & 15) * 4, c0 = slice * 64 + cc, r0 = (wave * 4 + (lane >> 4)) * RPT;
  const bool vec = (a.d.dv & 3) == 0 && ((reinterpret_cast<uintptr_t>(a.state) | reinterpret_cast<uintptr_t>(a.state_out)) & 15) == 0;
  int own = s, tok, end;
  long row = 0;
  if (x.step) {
    if (x.slot != nullptr) {
      own = x.slot[s];
      if (own < 0 || own >= x.slots) return;
      bool first = true;   // an earlier row of this slot takes this one too
      for (int b = 0; b < s; b += 64) first = first && !__any(b + lane < s && x.slot[b + lane] == own);
      if (!first) return;
    }
    tok = s;
    end = a.d.batch;
  } else {
    row = a.p.row(s);
    tok = a.p.begin(s);
    end = a.p.end(s);
  }
  const long base = ((long)own * heads + hv) * a.d.dk * (long)a.d.dv;
  float S[RPT][4];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = r0 + i;
#pragma unroll
    for (int j = 0; j < 4; ++j) S[i][j] = 0.f;
    if (a.state != nullptr && r < a.d.dk) {
      const float* p = a.state + base + (long)r * a.d.dv + c0;
      if (vec && c0 < a.d.dv) {
        const f4 v = *reinterpret_cast<const f4*>(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) S[i][j] = v[j];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c0 + j < a.d.dv) S[i][j] = p[j];
      }
    }
  }
  for (int par = 0; tok < end; par ^= 1) {
    // element offsets of this token: rows are the batch when stepping
    const long br = x.step ? tok : row, tr = x.step ? 0 : tok;
    for (int i = t; i < 2 * DK; i += 256) {
      const int c = i % DK;
      float v = 0.f;
      if (c < a.d.dk)
        v = i < DK ? ld<T>(a.d.k, br * a.d.k_st.bs + tr * a.d.k_st.rs + hk * a.d.k_st.cs + c)
                   : ld<T>(a.d.q, br * a.d.q_st.bs + tr * a.d.q_st.rs + hk * a.d.q_st.cs + c);
      qk[par][i / DK][c] = v;
    }
    const float decay = expf(a.d.g[br * a.d.g_st.bs + tr * a.d.g_st.rs + hv * a.d.g_st.cs]);
    const float beta = a.d.beta[br * a.d.beta_st.bs + tr * a.d.beta_st.rs + hv * a.d.beta_st.cs];
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = c0 + j < a.d.dv ? ld<T>(a.d.v, br * a.d.v_st.bs + tr * a.d.v_st.rs + hv * a.d.v_st.cs + c0 + j) : 0.f;
    __syncthreads();
    float ks[4] = {0, 0, 0, 0}, qs[4] = {0, 0, 0, 0}, dot = 0.f;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const float kv = qk[par][0][r0 + i], qv = qk[par][1][r0 + i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        S[i][j] *= decay;
        ks[j] = fmaf(kv, S[i][j], ks[j]);
        qs[j] = fmaf(qv, S[i][j], qs[j]);
      }
    }
    for (int i = lane; i < DK; i += 64) dot = fmaf(qk[par][0][i], qk[par][1][i], dot);
    for (int o = 1; o < 64; o <<= 1) dot += __shfl_xor(dot, o);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      ks[j] += __shfl_xor(ks[j], 16);
      qs[j] += __shfl_xor(qs[j], 16);
      ks[j] += __shfl_xor(ks[j], 32);
      qs[j] += __shfl_xor(qs[j], 32);
      if (lane < 16) {
        sm[par][wave][0][cc + j] = ks[j];
        sm[par][wave][1][cc + j] = qs[j];
      }
    }
    __syncthreads();
    float u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float k4 = (sm[par][0][0][cc + j] + sm[par][1][0][cc + j]) + (sm[par][2][0][cc + j] + sm[par][3][0][cc + j]);
      u[j] = beta * (v[j] - k4);
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const float kv = qk[par][0][r0 + i];
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = fmaf(kv, u[j], S[i][j]);
    }
    if (t < 16) {
      const long p = (x.step ? ((long)tok * heads + hv) : ((row * a.d.tokens + tok) * heads + hv)) * (long)a.d.dv + c0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float q4 = (sm[par][0][1][cc + j] + sm[par][1][1][cc + j]) + (sm[par][2][1][cc + j] + sm[par][3][1][cc + j]);
        if (c0 + j < a.d.dv) st<T>(a.o, p + j, a.scale * fmaf(dot, u[j], q4));
      }
    }
    if (!x.step) {
      ++tok;
    } else if (x.slot == nullptr) {
      break;
    } else {   // the next row of the same slot
      int next = end;
      for (int b = tok + 1; b < end && next == end; b += 64) {
        const unsigned long long hit = __ballot(b + lane < end && x.slot[min(b + lane, end - 1)] == own);
        if (hit) next = b + __ffsll(hit) - 1;
      }
      tok = next;
    }
  }
  if (a.state_out == nullptr) return;
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = r0 + i;
    if (r >= a.d.dk) continue;
    float* p = a.state_out + base + (long)r * a.d.dv + c0;
    if (vec && c0 < a.d.dv) {
      // past the caches: 64 users' states of 32 x 128 x 128 are 268 MB there and back, 49.7 us with plain stores, 44.6 with these
      __builtin_nontemporal_store(f4{S[i][0], S[i][1], S[i][2], S[i][3]}, reinterpret_cast<f4*>(p));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c0 + j < a.d.dv) p[j] = S[i][j];
    }
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------
constexpr int RECURRENT_MAX = 16;   // longest input (tokens per row, or packed tokens) that takes the recurrence

int sequences_of(const gpx_delta* d) { return d->sequences > 0 ? d->sequences : d->batch; }
long slots_of(const gpx_delta* d) {
  return d->sequences > 0 ? d->tokens / C + (long)d->sequences : (long)d->batch * ((d->tokens + C - 1) / C);
}
size_t up256(size_t x) { return (x + 255) / 256 * 256; }

bool recurrent(const gpx_delta* d, int save) { return !save && d->tokens <= RECURRENT_MAX; }

// gradients: value heads that share a key head on workgroups of their own
bool apart(const gpx_delta* d) { return d->value_heads > d->key_heads && slots_of(d) * d->value_heads <= 256; }

// Parts of a workspace, in this order; nullptr base: sizes only.
enum { WORK = 0, SAVED = 1, SCRATCH = 2, WORK_SAVING = 3 };
size_t lay_out(const gpx_delta* d, int use, char* base, Args* a, int** off) {
  const size_t dkp = d->dk <= 64 ? 64 : 128, dvp = (size_t)(d->dv + DVT - 1) / DVT * DVT;
  const size_t heads = (size_t)slots_of(d) * d->value_heads, kheads = (size_t)slots_of(d) * d->key_heads;
  const size_t n = d->dtype == GPX_F32 ? 3 : d->dtype == GPX_F16 ? 2 : 1, no = d->dtype == GPX_BF16 ? 2 : 3;
  size_t at = 0;
  Args dummy;
  Args& x = a != nullptr ? *a : dummy;
  auto part = [&](auto*& p, size_t bytes) {
    p = base == nullptr ? nullptr : reinterpret_cast<std::remove_reference_t<decltype(p)>>(base + at);
    at += up256(bytes);
  };
  if ((use == WORK || use == SAVED) && d->sequences > 0) {
    int* p;
    part(p, (size_t)(2 * d->sequences + 1) * 4);
    if (off != nullptr) *off = p;
  }
  if (use == WORK && recurrent(d, 0)) return at;
  if (use == WORK || use == SAVED) {
    part(x.G, heads * C * 8);
    part(x.fac, heads * FACS * 4);
    part(x.Kf, kheads * n * KF * 2);
    part(x.KTf, kheads * n * dkp * C * 2);
  }
  if (use == SAVED) {
    part(x.QTf, kheads * n * dkp * C * 2);
    part(x.T2f, heads * 3 * TF * 2);
    part(x.PTf, heads * 3 * TF * 2);
    part(x.Erow, heads * C * dvp * 4);
    part(x.Srow, heads * dkp * dvp * 4);
  }
  if (use == WORK || use == WORK_SAVING) {
    part(x.Qf, kheads * n * KF * 2);
    part(x.Tf, heads * 3 * TF * 2);
    part(x.Pf, heads * no * TF * 2);
  }
  if (use == SCRATCH) {
    part(x.Z, heads * C * dvp * 4);
    part(x.dS, heads * dkp * dvp * 4);
    if (apart(d)) {
      part(x.d_q_part, heads * C * dkp * 4);
      part(x.d_k_part, heads * C * dkp * 4);
    }
  }
  return at;
}

int check_delta(const gpx_delta* d, const char* what) {
  GPX_REQUIRE(d != nullptr, "%s: null description", what);
  GPX_REQUIRE(d->dtype == GPX_F32 || d->dtype == GPX_F16 || d->dtype == GPX_BF16, "%s: unknown element type %d", what, d->dtype);
  GPX_REQUIRE(d->batch >= 0 && d->tokens >= 0 && d->sequences >= 0, "%s: negative size", what);
  GPX_REQUIRE(d->key_heads >= 1 && d->value_heads >= 1 && d->value_heads % d->key_heads == 0,
              "%s: %d value heads are not a multiple of %d key heads", what, d->value_heads, d->key_heads);
  GPX_REQUIRE(d->dk >= 1 && d->dk <= 128, "%s: dk = %d is outside [1, 128]", what, d->dk);
  GPX_REQUIRE(d->dv >= 1 && d->dv <= 1024, "%s: dv = %d is outside [1, 1024]", what, d->dv);
  GPX_REQUIRE(d->tokens <= (1 << 30) && d->batch <= (1 << 24) && d->sequences <= (1 << 24), "%s: size out of range", what);
  GPX_REQUIRE(d->sequences == 0 || (d->batch == 1 && d->offsets != nullptr), "%s: packed sequences need batch == 1 and offsets", what);
  GPX_REQUIRE(std::isfinite(d->scale), "%s: scale is not finite", what);
  for (const gpx_strided* s : {&d->q_st, &d->k_st, &d->v_st, &d->g_st, &d->beta_st})
    GPX_REQUIRE(s->bs >= 0 && s->rs >= 0 && s->cs >= 0, "%s: negative stride", what);
  GPX_REQUIRE(d->v_st.rs <= (1 << 22), "%s: token stride of v beyond 2^22", what);   // 32-bit offsets inside a chunk
  if (d->batch > 0 && d->tokens > 0)
    GPX_REQUIRE(d->q && d->k && d->v && d->g && d->beta, "%s: null input", what);
  return 0;
}

// threads of a launch have 32 bits
int check_grid(const gpx_delta* d, bool rec, const char* what) {
  const double scan = (sequences_of(d) * (double)d->value_heads + 7) * ((d->dv + DVT - 1) / DVT * DVT / 16) * 512;
  const double steps = (double)sequences_of(d) * d->value_heads * ((d->dv + 63) / 64) * 256;
  const double chunks = (double)slots_of(d) * d->key_heads * 512;
  GPX_REQUIRE((rec ? steps : std::max(scan, chunks)) < 4.2e9, "%s: too many sequences, heads and chunks for one call", what);
  return 0;
}

Args make_args(const gpx_delta* d) {
  Args a = {};
  a.d = *d;
  a.group = d->value_heads / d->key_heads;
  a.parts = slots_of(d) * d->value_heads <= 512 ? a.group : 1;
  a.dvp = (d->dv + DVT - 1) / DVT * DVT;
  a.scale = (float)d->scale;
  a.p.sequences = sequences_of(d);
  a.p.tokens = d->tokens;
  a.p.chunks_per_row = (d->tokens + C - 1) / C;
  a.p.off = nullptr;
  return a;
}

// once per thread, kernel and device
template <auto Kernel>
int allow_lds(size_t bytes) {
  static thread_local bool done[GPX_MAX_DEVICES] = {};
  int dev = 0;
  GPX_HIP(hipGetDevice(&dev));
  if (dev < GPX_MAX_DEVICES && done[dev]) return 0;
  GPX_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  if (dev < GPX_MAX_DEVICES) done[dev] = true;
  return 0;
}

#define DELTA_TRY(...)        \
  do {                        \
    int rc_ = (__VA_ARGS__);  \
    if (rc_ != 0) return rc_; \
  } while (0)

unsigned chain_grid(const Args& a) {
  const unsigned heads = (unsigned)a.p.sequences * a.d.value_heads;
  return (heads + 7) / 8 * 8 * (a.dvp / 16);
}

// More workgroups than compute units: two at a time on each, in 128 registers a wave, which only bf16 has next to no spills in
// (512 workgroups, training: 201 -> 176 us, 1024, forward: 143 -> 117; 256 of them: 200 -> 205)
template <typename T, int DK, bool BACK>
int run_chain(hipStream_t s, const Args& a) {
  const unsigned grid = chain_grid(a);
  if constexpr (Planes<T>::N == 1) {
    if (grid > 256) {
      hipLaunchKernelGGL((delta_chain_kernel<T, DK, BACK, true>), dim3(grid), dim3(512), 0, s, a);
      GPX_HIP(hipGetLastError());
      return 0;
    }
  }
  hipLaunchKernelGGL((delta_chain_kernel<T, DK, BACK, false>), dim3(grid), dim3(512), 0, s, a);
  GPX_HIP(hipGetLastError());
  return 0;
}

template <typename T, int DK>
int run_forward(hipStream_t s, const Args& a, int rec) {
  if (rec) {
    StepArgs x = {a, nullptr, 0, 0};
    const unsigned grid = (unsigned)a.p.sequences * a.d.value_heads * ((a.d.dv + 63) / 64);
    hipLaunchKernelGGL((delta_recurrent_kernel<T, DK>), dim3(grid), dim3(256), 0, s, x);
    GPX_HIP(hipGetLastError());
    return 0;
  }
  constexpr size_t lds = chunk_room<T, DK>() + C * 8 + C * 4;
  static_assert(lds <= 160 * 1024, "LDS");
  DELTA_TRY(allow_lds<&delta_chunk_kernel<T, DK, false>>(lds));
  DELTA_TRY(allow_lds<&delta_chunk_kernel<T, DK, true>>(lds));
  const long slots = slots_of(&a.d);
  if (slots > 0) {
    const dim3 grid((unsigned)(slots * a.d.key_heads * a.parts));
    if (a.save && slots * a.d.value_heads > 512) hipLaunchKernelGGL((delta_chunk_kernel<T, DK, true>), grid, dim3(256), lds, s, a);
    else hipLaunchKernelGGL((delta_chunk_kernel<T, DK, false>), grid, dim3(256), lds, s, a);
    GPX_HIP(hipGetLastError());
  }
  return run_chain<T, DK, false>(s, a);
}

template <typename T, int DK>
int run_backward(hipStream_t s, const Args& a) {
  constexpr size_t tiles = 2 * C * (DK + 16 / sizeof(T)) * sizeof(T), base = grads_room<T>() + C * 8 + (16 * C + 2 * C + 8 + 336 + C) * 4;
  constexpr size_t lds = base + tiles, grouped = base + (sizeof(T) == 4 ? 0 : tiles) + 8 * 512 * 16;
  static_assert(lds <= 160 * 1024 && grouped <= 160 * 1024 && lds % 16 == 0, "LDS");
  DELTA_TRY(allow_lds<&delta_grads_kernel<T, DK, ALONE>>(lds));
  DELTA_TRY(allow_lds<&delta_grads_kernel<T, DK, GROUPED>>(grouped));
  DELTA_TRY(allow_lds<&delta_grads_kernel<T, DK, APART>>(lds));
  const long slots = slots_of(&a.d);
  DELTA_TRY((run_chain<T, DK, true>(s, a)));
  if (slots > 0) {
    const dim3 grid((unsigned)(slots * a.d.key_heads));
    if (a.group == 1) {
      hipLaunchKernelGGL((delta_grads_kernel<T, DK, ALONE>), grid, dim3(512), lds, s, a);
    } else if (apart(&a.d)) {
      hipLaunchKernelGGL((delta_grads_kernel<T, DK, APART>), dim3((unsigned)(slots * a.d.value_heads)), dim3(512), lds, s, a);
      GPX_HIP(hipGetLastError());
      hipLaunchKernelGGL((delta_join_heads_kernel<T, DK>), dim3(grid.x * 8), dim3(256), 0, s, a);
    } else {
      hipLaunchKernelGGL((delta_grads_kernel<T, DK, GROUPED>), grid, dim3(512), grouped, s, a);
    }
    GPX_HIP(hipGetLastError());
  }
  return 0;
}

#define DELTA_DISPATCH(fn, ...)                                                                             \
  (a.d.dk <= 64 ? (a.d.dtype == GPX_F32   ? fn<float, 64>(__VA_ARGS__)                                       \
                   : a.d.dtype == GPX_F16 ? fn<_Float16, 64>(__VA_ARGS__)                                    \
                                          : fn<__bf16, 64>(__VA_ARGS__))                                     \
                : (a.d.dtype == GPX_F32   ? fn<float, 128>(__VA_ARGS__)                                      \
                   : a.d.dtype == GPX_F16 ? fn<_Float16, 128>(__VA_ARGS__)                                   \
                                          : fn<__bf16, 128>(__VA_ARGS__)))

template <typename T, int DK>
int run_step(hipStream_t s, const Args& a, int slots, const int* slot) {
  StepArgs x = {a, slot, slots, 1};
  const unsigned grid = (unsigned)a.d.batch * a.d.value_heads * ((a.d.dv + 63) / 64);
  hipLaunchKernelGGL((delta_recurrent_kernel<T, DK>), dim3(grid), dim3(256), 0, s, x);
  GPX_HIP(hipGetLastError());
  return 0;
}

int plan(hipStream_t s, const gpx_delta* d, Args& a, int* off) {
  if (d->sequences == 0) return 0;
  hipLaunchKernelGGL(delta_plan_kernel, dim3(1), dim3(64), 0, s, d->offsets, d->sequences + 1, d->tokens, off);
  GPX_HIP(hipGetLastError());
  a.p.off = off;
  return 0;
}

int check_work(const gpx_delta* d, int use, const void* work, size_t work_bytes, const char* what) {
  const size_t need = lay_out(d, use, nullptr, nullptr, nullptr);
  GPX_REQUIRE(need == 0 || (work != nullptr && (reinterpret_cast<uintptr_t>(work) & 255) == 0), "%s: work null or misaligned", what);
  GPX_REQUIRE(work_bytes >= need, "%s: work holds %zu of %zu bytes", what, work_bytes, need);
  return 0;
}

}  // namespace

extern "C" {

size_t gpx_delta_work_bytes(const gpx_delta* d, int use) {
  if (use < 0 || use > 3 || check_delta(d, "delta_work_bytes") != 0) return 0;
  if (check_grid(d, use == WORK && recurrent(d, 0), "delta_work_bytes") != 0) return 0;
  return lay_out(d, use, nullptr, nullptr, nullptr);
}

int gpx_delta_forward(gpx_handle* h, const gpx_delta* d, const float* state, void* o, float* state_out, void* work,
                      size_t work_bytes, void* saved, size_t saved_bytes) {
  GPX_REQUIRE(h != nullptr, "null handle");
  DELTA_TRY(check_delta(d, "delta_forward"));
  if (sequences_of(d) == 0) return 0;
  GPX_REQUIRE(o != nullptr || d->tokens == 0, "delta_forward: null output");
  GPX_REQUIRE(state == nullptr || gpx_aligned16(state), "delta_forward: state must be 16-byte aligned");
  GPX_REQUIRE(state_out == nullptr || gpx_aligned16(state_out), "delta_forward: state_out must be 16-byte aligned");
  const int save = saved != nullptr;
  DELTA_TRY(check_grid(d, recurrent(d, save), "delta_forward"));
  DELTA_TRY(check_work(d, save ? WORK_SAVING : WORK, work, work_bytes, "delta_forward"));
  if (save) DELTA_TRY(check_work(d, SAVED, saved, saved_bytes, "delta_forward"));
  DeviceGuard dg(h->device);
  Args a = make_args(d);
  int* off = nullptr;
  lay_out(d, save ? WORK_SAVING : WORK, static_cast<char*>(work), &a, &off);
  if (save) lay_out(d, SAVED, static_cast<char*>(saved), &a, &off);
  DELTA_TRY(plan(h->stream, d, a, off));
  a.state = state;
  a.o = o;
  a.state_out = state_out;
  a.save = save;
  const int rec = recurrent(d, save);
  return DELTA_DISPATCH(run_forward, h->stream, a, rec);
}

int gpx_delta_backward(gpx_handle* h, const gpx_delta* d, const void* d_o, const gpx_strided* d_o_st, const float* d_state_out,
                       void* d_q, void* d_k, void* d_v, float* d_g, float* d_beta, float* d_state, const void* saved, size_t saved_bytes,
                       void* scratch, size_t scratch_bytes) {
  GPX_REQUIRE(h != nullptr, "null handle");
  DELTA_TRY(check_delta(d, "delta_backward"));
  if (sequences_of(d) == 0) return 0;
  if (d->tokens > 0) {
    GPX_REQUIRE(d_o != nullptr && d_o_st != nullptr, "delta_backward: null gradient of o");
    GPX_REQUIRE(d_o_st->bs >= 0 && d_o_st->rs >= 0 && d_o_st->cs >= 0, "delta_backward: negative stride");
    GPX_REQUIRE(d_q && d_k && d_v && d_g && d_beta, "delta_backward: null output");
  }
  DELTA_TRY(check_grid(d, false, "delta_backward"));
  DELTA_TRY(check_work(d, SAVED, saved, saved_bytes, "delta_backward"));
  DELTA_TRY(check_work(d, SCRATCH, scratch, scratch_bytes, "delta_backward"));
  DeviceGuard dg(h->device);
  Args a = make_args(d);
  int* off = nullptr;
  lay_out(d, SAVED, static_cast<char*>(const_cast<void*>(saved)), &a, &off);
  lay_out(d, SCRATCH, static_cast<char*>(scratch), &a, nullptr);
  if (d->sequences > 0) a.p.off = off;   // the forward call's plan
  a.d_o = d_o;
  if (d_o_st != nullptr) a.do_st = *d_o_st;
  a.d_state_out = d_state_out;
  a.d_q = d_q;
  a.d_k = d_k;
  a.d_v = d_v;
  a.d_g = d_g;
  a.d_beta = d_beta;
  a.d_state = d_state;
  return DELTA_DISPATCH(run_backward, h->stream, a);
}

int gpx_delta_step(gpx_handle* h, const gpx_delta* d, int slots, const int* slot, const float* state, float* state_out, void* o) {
  GPX_REQUIRE(h != nullptr, "null handle");
  DELTA_TRY(check_delta(d, "delta_step"));
  GPX_REQUIRE(d->tokens == 1 && d->sequences == 0, "delta_step: one token per row");
  DELTA_TRY(check_grid(d, true, "delta_step"));
  GPX_REQUIRE(slots >= 0 && (slot != nullptr || slots == d->batch), "delta_step: %d states for %d rows", slots, d->batch);
  if (d->batch == 0 || slots == 0) return 0;   // no row has a state
  GPX_REQUIRE(o != nullptr && state_out != nullptr && state != nullptr, "delta_step: null state or output");
  GPX_REQUIRE(((reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(state_out)) & 3) == 0, "delta_step: misaligned state");
  DeviceGuard dg(h->device);
  Args a = make_args(d);
  a.state = state;
  a.state_out = state_out;
  a.o = o;
  return DELTA_DISPATCH(run_step, h->stream, a, slots, slot);
}

}  // extern "C"
