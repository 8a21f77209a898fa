// Orthogonalising updates by Newton-Schulz products:  X <- U / (|U|_F + eps),  then `steps` times
//     A = X X^T,   S = a I + b A + c A A,   X <- S X          (X has m rows of n >= m values; U^T where U is tall)
// which applies the odd polynomial a s + b s^3 + c s^5 to every singular value s.
//
// Numerics: the smallest singular values grow 3.44-fold per step, and rounding of X, A or S to 16 bits is carried along with them
// (2e-3 .. 3e-2 of the result's norm after five steps); operands are therefore kept as pairs of fp16 (nt_product.h), which reproduces an fp32
// iteration's error.  Everything is scaled by 2^12 in storage: |X|, |A| and |S| stay below 16 (the entry checks the polynomial for
// that), so nothing overflows fp16, and the low parts reach down to 2^-36.  The Frobenius norm is summed in fp64.
//
// Work per step: m^2 n + m^3 multiply-adds halved by symmetry + m^2 n: A and S are computed on and below the diagonal and stored twice.  Every
// product's second operand is wanted with its contraction index contiguous, so X is kept in both orientations (X for A, X^T for S X); the
// product that makes the next X stores both.  All matrices of a call (one model's filters) share each launch: 2, and 3 (4 where A's contraction is
// split) per step, whatever their number; where none has more than 64 rows, one per step (ns_narrow_step_kernel).  Matrices of up to 16 rows are done
// with the first two (ns_short_apply).
//
// Measured (five steps): 2048 x 8192 bf16 1.70 .. 1.78 ms, 970 TFLOP/s of matrix instructions where a large library product reaches 1430 -- per step S X 180 us
// (1145 TFLOP/s), A 106, its join 26, S 46 (560: 528 tiles of 64); 4096 x 1024 fp32 400 .. 425 us; 1000 x 1537 bf16 264 .. 285 us (tiles for 1.6 rounds of
// the chip and 15 us a product: latency); a U-Net's 23 filters fp32 186 us (22 launches of 6 .. 15 us); 64 x 576 fp32 71 us (7 of 9 .. 11 us).
#include <math.h>

#include "nt_product.h"

namespace {

constexpr int NS_MAX = 64;                       // matrices per launch (their descriptors travel as kernel arguments)
constexpr float NS_SCALE = 4096.f;
constexpr int NS_CHUNK = 8192;                   // elements per partial sum of squares

struct NsItem {
  const void* u;
  void* out;
  unsigned base;                                 // its place in the workspace, in 256 bytes
  int m, n, tall, dtype, split;                  // split: parts of A's contraction; 0: the short form
};
// Work items of a launch, by kind
enum { NS_SUMS, NS_PREP, NS_A, NS_JOIN, NS_S, NS_X, NS_NARROW, NS_SHORT, NS_KINDS };
// The call's matrices on the device, at the head of the workspace.  They travel once, as the first kernel's arguments; that kernel leaves them here
// and the others get a pointer: arguments of kilobytes cost the host some microseconds per launch.
struct NsTable {
  NsItem it[NS_MAX];
  int start[NS_KINDS][NS_MAX];                   // first work item of each matrix
};
struct NsArgs {
  char* ws;
  NsItem it[NS_MAX];
  int count, narrow, tile[3];
  float eps;
  int first[NS_MAX];                             // each matrix's first work item of the first launch
};
static_assert(sizeof(NsArgs) <= 4096, "kernel arguments");
struct NsCtl {
  char* ws;
  int count, cur, last;
  float ca, cb, cc, eps;
};
// the short form takes all steps in one launch, whose first `items` workgroups are the other matrices'
constexpr int NS_STEPS = 32;
struct NsAll {
  int items, steps;
  float c[3 * NS_STEPS];
};

__device__ __host__ __forceinline__ int ns_pad(int v) { return (v + 31) & ~31; }
__device__ __host__ __forceinline__ int ns_sums(const NsItem& q) { return (int)(((long)q.m * q.n + NS_CHUNK - 1) / NS_CHUNK); }

// a matrix's part of the workspace: pair rows x [m][n], xt [n][m] twice (S X reads one and writes the other), a, s [m][m]; partial sums of
// squares; the partial tiles of a split A
struct NsMem {
  f16_t *x, *xt[2], *a, *s;
  double* sums;
  float* part;
  long bytes;
};
__device__ __host__ __forceinline__ NsMem ns_mem(char* p, const NsItem& q) {
  const long mp = ns_pad(q.m), np = ns_pad(q.n);
  const long bx = (4L * q.m * np + 255) & ~255L, bt = (4L * q.n * mp + 255) & ~255L, ba = (4L * q.m * mp + 255) & ~255L, bs = (8L * ns_sums(q) + 255) & ~255L;
  NsMem r;
  r.x = (f16_t*)p, p += bx;
  r.xt[0] = (f16_t*)p, p += bt;
  r.xt[1] = (f16_t*)p, p += bt;
  r.a = (f16_t*)p, p += ba;
  r.s = (f16_t*)p, p += ba;
  r.sums = (double*)p, p += bs;
  r.part = (float*)p;
  r.bytes = bx + 2 * bt + 2 * ba + bs;
  return r;
}
__device__ __forceinline__ NsMem ns_mem(const NsCtl& g, const NsItem& q) { return ns_mem(g.ws + (long)q.base * 256, q); }

// the same for matrices of at most 64 rows, see further down
__device__ __host__ __forceinline__ int ns_chunks(int n) {
  const int tiles = (n + 63) / 64;
  int p = 1;
  while (p < tiles && p * p < 8 * tiles) ++p;
  const int ch = (tiles + p - 1) / p;
  return (tiles + ch - 1) / ch;
}
constexpr long NS_PART64 = 64 * 64;
// the workspace: xt pair rows [n][64], partial A's twice, partial sums of squares
struct NsNarrow {
  f16_t* xt;
  float* part[2];
  double* sums;
  long bytes;
};
__device__ __host__ __forceinline__ NsNarrow ns_narrow_mem(char* p, const NsItem& q) {
  const long bt = 256L * q.n, bp = 4 * NS_PART64 * ns_chunks(q.n), bs = (8L * ns_sums(q) + 255) & ~255L;
  NsNarrow r;
  r.sums = (double*)p, p += bs;
  r.xt = (f16_t*)p, p += bt;
  r.part[0] = (float*)p, p += bp;
  r.part[1] = (float*)p;
  r.bytes = bs + bt + 2 * bp;
  return r;
}

// matrices of at most 16 rows, see further down: columns per workgroup -- whole tiles of 64, at most 128 workgroups
__device__ __host__ __forceinline__ int ns_short_cols(int n) {
  const int per = ((n + 127) / 128 + 63) & ~63;
  return per < 256 ? 256 : per;
}

// how many work items of a kind a matrix has (T: the launch's tile)
__device__ __host__ __forceinline__ long ns_items(const NsItem& q, int kind, int T) {
  if (!q.split) return kind == NS_SUMS || kind == NS_SHORT ? (q.n + ns_short_cols(q.n) - 1) / ns_short_cols(q.n) : 0;
  if (kind == NS_SHORT) return 0;
  const long mt = (q.m + T - 1) / T, nt = (q.n + T - 1) / T, tri = mt * (mt + 1) / 2;
  return kind == NS_SUMS ? ns_sums(q) : kind == NS_A ? tri * q.split : kind == NS_JOIN ? (q.split > 1 ? tri : 0)
         : kind == NS_S ? tri : kind == NS_NARROW ? ns_chunks(q.n) : mt * nt;
}
__device__ __host__ __forceinline__ int ns_side(int tile) { return tile < 64 ? 64 : tile; }
__device__ __host__ __forceinline__ int ns_side_of(const NsArgs& g, int kind) {
  return ns_side(kind == NS_A || kind == NS_JOIN ? g.tile[0] : kind == NS_S ? g.tile[1] : kind == NS_X ? g.tile[2] : 64);
}
__device__ __forceinline__ const NsTable* ns_table(const char* ws) { return (const NsTable*)ws; }
// the last matrix that starts at or before work item w: a lane each (64 matrices at most)
__device__ __forceinline__ int ns_find(const NsCtl& g, int kind, int w, int& first) {
  const int l = threadIdx.x & 63, v = l < g.count ? ns_table(g.ws)->start[kind][l] : 0x7fffffff;
  const int k = 63 - __builtin_clzll(__ballot(v <= w));
  first = __builtin_amdgcn_readlane(v, k);
  return __builtin_amdgcn_readfirstlane(k);
}
__device__ __forceinline__ float ns_load(const void* p, int dtype, long i) {
  return dtype == FI_F32 ? ((const float*)p)[i] : dtype == FI_BF16 ? (float)((const bf16_t*)p)[i] : (float)((const f16_t*)p)[i];
}
__device__ __forceinline__ void ns_tri(int t, int& i, int& j) {               // t = i (i + 1) / 2 + j, j <= i
  i = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
  while ((i + 1) * (i + 2) / 2 <= t) ++i;
  while (i * (i + 1) / 2 > t) --i;
  j = t - i * (i + 1) / 2;
}

template <typename T>
__device__ __forceinline__ double ns_squares(const T* p, long n) {
  constexpr int VG = DT<T>::VG;
  const long head = ((16 - ((uintptr_t)p & 15)) & 15) / sizeof(T);            // up to the first aligned vector
  const long h = head < n ? head : n, vecs = (n - h) / VG, tail = h + vecs * VG;
  double acc = 0.0;
  for (long i = threadIdx.x; i < vecs; i += 256) {
    float f[VG];
    VecWords<T>::unpack(((const typename DT<T>::vec_t*)(p + h))[i], f);
#pragma unroll
    for (int t = 0; t < VG; ++t) acc += (double)f[t] * (double)f[t];
  }
  if ((long)threadIdx.x < h + n - tail) {
    const double v = (double)to_f32(p[(long)threadIdx.x < h ? (long)threadIdx.x : tail + threadIdx.x - h]);
    acc += v * v;
  }
  return acc;
}
// ---- matrices of at most 16 rows -------------------------------------------------------------------------------------------------------
// The steps' matrices are all polynomials of G = U U^T and commute, so X after the last step is P X0 with a 16 x 16 matrix P:
//     A <- G / (sqrt(trace G) + eps)^2,  P <- I;   per step  S = a I + b A + c A A,  P <- S P,  A <- S A S.
// Squaring U loses half its digits and P's entries reach 3.4^steps, so all of it is fp64, for which 16 rows are little work: the result is off by its
// rounding to fp32, where pairs are off by their 22 bits (and short sums show every rounding).  Two launches for any number of steps, both shared
// with the other matrices of the call: G in parts of 256 columns or more, and P -- by every workgroup for itself, some 4 us for five steps -- with its
// product with the workgroup's columns.
constexpr int NS_SHORT_ROWS = 16, NS_SHORT_LDS = 4 * 16 * 18 * 8;
constexpr int NS_GRAM_LD = 260;
__device__ __forceinline__ void ns_short_gram(char* ws, const NsItem& q, int chunk, float* xs) {       // xs: [16][NS_GRAM_LD]
  const int per = ns_short_cols(q.n), lo = chunk * per, hi = lo + per < q.n ? lo + per : q.n, tid = threadIdx.x, i = tid >> 4, j = tid & 15;
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  for (int t = lo; t < hi; t += 256) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int e = k * 256 + tid, r = q.tall ? e & 15 : k, c = q.tall ? e >> 4 : tid;
      xs[r * NS_GRAM_LD + c] = r < q.m && t + c < hi ? ns_load(q.u, q.dtype, q.tall ? (long)(t + c) * q.m + r : (long)r * q.n + t + c) : 0.f;
    }
    __syncthreads();
#pragma unroll 4
    for (int c = 0; c < 256; c += 4) {
      const float4 x = *(const float4*)(xs + i * NS_GRAM_LD + c), y = *(const float4*)(xs + j * NS_GRAM_LD + c);
      acc[0] += (double)x.x * (double)y.x;
      acc[1] += (double)x.y * (double)y.y;
      acc[2] += (double)x.z * (double)y.z;
      acc[3] += (double)x.w * (double)y.w;
    }
  }
  ((double*)(ws + (long)q.base * 256))[chunk * 256 + tid] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
}
// (the matrices are symmetric: a product's element is that of two rows, which are read in vectors)
typedef double NsRow[18];
__device__ __forceinline__ void ns_row16(const NsRow& a, double (&v)[16]) {
#pragma unroll
  for (int d = 0; d < 16; d += 2) {
    const double2 x = *(const double2*)(a + d);
    v[d] = x.x, v[d + 1] = x.y;
  }
}
__device__ __forceinline__ double ns_dot16(const double (&a)[16], const double (&b)[16]) {
  double v[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
  for (int d = 0; d < 16; ++d) v[d & 3] += a[d] * b[d];
  return (v[0] + v[1]) + (v[2] + v[3]);
}
template <typename T>
__device__ __forceinline__ void ns_short_columns(const NsItem& q, int lo, int hi, const NsRow* P) {
  const T* const u = (const T*)q.u;
  T* const out = (T*)q.out;
  const long sr = q.tall ? 1 : q.n, sc = q.tall ? q.m : 1;              // strides of X's rows and columns
  for (int c = lo + (int)threadIdx.x; c < hi; c += 256) {               // (a column is read whole before it is written: out may be u)
    double x[16];
#pragma unroll
    for (int d = 0; d < 16; ++d) x[d] = d < q.m ? (double)to_f32(u[d * sr + c * sc]) : 0.0;
    for (int r = 0; r < q.m; ++r) {
      double v = 0.0;
#pragma unroll
      for (int d = 0; d < 16; ++d) v += P[r][d] * x[d];
      out[r * sr + c * sc] = (T)(float)v;
    }
  }
}
__device__ __forceinline__ void ns_short_apply(const NsCtl& g, const NsAll& all, int w, char* lds) {
  NsRow *const A = (NsRow*)lds, *const S = A + 16, *const P = A + 32, *const B = A + 48;
  int first;
  const int k = ns_find(g, NS_SHORT, w, first), tid = threadIdx.x, i = tid >> 4, j = tid & 15;
  const NsItem q = ns_table(g.ws)->it[k];
  const int per = ns_short_cols(q.n), parts = (q.n + per - 1) / per, lo = (w - first) * per, hi = lo + per < q.n ? lo + per : q.n;
  const double* const part = (const double*)(g.ws + (long)q.base * 256) + tid;
  double v = 0.0, trace = 0.0;
  for (int p = 0; p < parts; ++p) v += part[p * 256];
  A[i][j] = v;
  __syncthreads();
#pragma unroll
  for (int d = 0; d < 16; ++d) trace += A[d][d];
  const double norm = sqrt(trace) + (double)g.eps, inv = norm == 0.0 ? 0.0 : 1.0 / norm;
  __syncthreads();
  A[i][j] = v * inv * inv;
  P[i][j] = i == j ? inv : 0.0;
  double a[16], f[16], x[16];
  for (int s = 0; s < all.steps; ++s) {
    __syncthreads();
    ns_row16(A[i], a), ns_row16(A[j], x);
    S[i][j] = (i == j ? (double)all.c[3 * s] : 0.0) + (double)all.c[3 * s + 1] * A[i][j] + (double)all.c[3 * s + 2] * ns_dot16(a, x);
    __syncthreads();
    ns_row16(S[j], x);
    B[i][j] = ns_dot16(a, x);
    ns_row16(S[i], f), ns_row16(P[j], x);
    const double p = ns_dot16(f, x);
    __syncthreads();
    ns_row16(B[j], x);
    P[i][j] = p;
    A[i][j] = ns_dot16(f, x);
  }
  __syncthreads();
  if (q.dtype == FI_F32)
    ns_short_columns<float>(q, lo, hi, P);
  else if (q.dtype == FI_BF16)
    ns_short_columns<bf16_t>(q, lo, hi, P);
  else
    ns_short_columns<f16_t>(q, lo, hi, P);
}

// the sums of squares (the short form's G); the first workgroup also leaves the table for the kernels behind
// (SHORT, here and below: with matrices of few rows among the others, whose form needs registers that would halve the others' waves: the next kernel
// takes 54 us instead of 39 at 2048 x 8192)
template <bool SHORT>
__global__ __launch_bounds__(256) void ns_norm_kernel(NsArgs g) {
  __shared__ double sm[4];
  __shared__ __attribute__((aligned(16))) float xs[SHORT ? 16 * NS_GRAM_LD : 1];
  const int at = (int)(threadIdx.x & 63) < g.count ? g.first[threadIdx.x & 63] : 0x7fffffff;
  const int k = 63 - __builtin_clzll(__ballot(at <= (int)blockIdx.x)), w = (int)blockIdx.x - __builtin_amdgcn_readlane(at, k);
  const NsItem& q = g.it[k];
  if (blockIdx.x == 0 && threadIdx.x < 64) {
    NsTable* const t = (NsTable*)g.ws;
    const int l = threadIdx.x;
    if (l < g.count) t->it[l] = g.it[l];
    for (int kind = 0; kind < NS_KINDS; ++kind) {
      int n = l < g.count ? (int)ns_items(g.it[l], kind, ns_side_of(g, kind)) : 0, sum = n;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(sum, o, 64);
        sum += l >= o ? up : 0;
      }
      t->start[kind][l] = sum - n;
    }
  }
  if (SHORT && !q.split) {
    ns_short_gram(g.ws, q, w, xs);
    return;
  }
  const long total = (long)q.m * q.n, lo = (long)w * NS_CHUNK, n = total - lo < NS_CHUNK ? total - lo : NS_CHUNK;
  double acc = q.dtype == FI_F32 ? ns_squares((const float*)q.u + lo, n) : q.dtype == FI_BF16 ? ns_squares((const bf16_t*)q.u + lo, n)
                                                                                           : ns_squares((const f16_t*)q.u + lo, n);
  acc = wave_sum(acc);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = acc;
  __syncthreads();
  char* const p = g.ws + (long)q.base * 256;
  double* const sums = g.narrow ? ns_narrow_mem(p, q).sums : ns_mem(p, q).sums;
  if (threadIdx.x == 0) sums[w] = sm[0] + sm[1] + sm[2] + sm[3];
}

// storage's scale / (|U| + eps) as x * y (y = 1 but past fp32's range, where eps is zero and |U| next to it); a zero matrix stays one where eps is zero too
__device__ __forceinline__ float2 ns_inverse(double squares, float eps) {
  const double norm = sqrt(squares) + (double)eps, inv = norm == 0.0 ? 0.0 : (double)NS_SCALE / norm;
  return inv > 0x1p100 ? make_float2((float)(inv * 0x1p-80), 0x1p80f) : make_float2((float)inv, 1.f);
}

// U, normalised, as pair rows in both orientations: one 64 x 64 block of U per workgroup
template <bool SHORT>
__global__ __launch_bounds__(256) void ns_prep_kernel(NsCtl g, NsAll all) {
  __shared__ __attribute__((aligned(16))) float tile[64][65];
  __shared__ double sm[4];
  __shared__ float2 s_inv;
  static_assert(sizeof(tile) >= NS_SHORT_LDS, "LDS");
  if (SHORT && (int)blockIdx.x >= all.items) {
    ns_short_apply(g, all, (int)blockIdx.x - all.items, (char*)tile);
    return;
  }
  int first;
  const int w = (int)blockIdx.x, k = ns_find(g, NS_PREP, w, first), tid = threadIdx.x;
  const NsItem q = ns_table(g.ws)->it[k];
  const NsMem mem = ns_mem(g, q);
  double acc = 0.0;
  for (int i = tid, n = ns_sums(q); i < n; i += 256) acc += mem.sums[i];
  acc = wave_sum(acc);
  if ((tid & 63) == 0) sm[tid >> 6] = acc;
  __syncthreads();
  if (tid == 0) s_inv = ns_inverse(sm[0] + sm[1] + sm[2] + sm[3], g.eps);
  __syncthreads();
  const float2 inv = s_inv;
  const int rows = q.tall ? q.n : q.m, cols = q.tall ? q.m : q.n;
  const int nb = (cols + 63) / 64, t = w - first, r0 = (t / nb) * 64, c0 = (t % nb) * 64;
  for (int e = tid; e < 64 * 64; e += 256) {
    const int r = r0 + (e >> 6), c = c0 + (e & 63);
    tile[e >> 6][e & 63] = r < rows && c < cols ? ns_load(q.u, q.dtype, (long)r * cols + c) * inv.y * inv.x : 0.f;
  }
  __syncthreads();
  f16_t* const same = q.tall ? mem.xt[0] : mem.x;          // U's own orientation
  f16_t* const turned = q.tall ? mem.x : mem.xt[0];
  const int cpad = ns_pad(cols), rpad = ns_pad(rows);
  for (int e = tid; e < 64 * 8; e += 256) {
    const int r = e >> 3, c = (e & 7) * 8;
    float v[8];
    if (r0 + r < rows && c0 + c < cpad) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = tile[r][c + i];
      nt_store_pair(same + (long)(r0 + r) * 2 * cpad, c0 + c, v);
    }
    if (c0 + r < cols && r0 + c < rpad) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = tile[c + i][r];
      nt_store_pair(turned + (long)(c0 + r) * 2 * rpad, r0 + c, v);
    }
  }
}

// (32 stands for tiles of 64 whose sums are kept apart)
template <int TILE>
struct NsTile;
template <> struct NsTile<32> { typedef NtCore<f16_t, 2, 64, 64, 32, 32, 3, true> Core; };
template <> struct NsTile<64> { typedef NtCore<f16_t, 2, 64, 64, 32, 32, 3> Core; };
template <> struct NsTile<128> { typedef NtCore<f16_t, 2, 128, 128, 64, 32, 2> Core; };
template <> struct NsTile<256> { typedef NtCore<f16_t, 2, 256, 256, 64, 64> Core; };

__device__ __forceinline__ void ns_put(void* out, int dtype, long at, const float (&v)[8], int n) {
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    if (t < n) {
      if (dtype == FI_F32)
        ((float*)out)[at + t] = v[t];
      else if (dtype == FI_BF16)
        ((bf16_t*)out)[at + t] = (bf16_t)v[t];
      else
        ((f16_t*)out)[at + t] = (f16_t)v[t];
    }
  }
}

// what becomes of a tile of PHASE 0 (A), 1 (S) or 2 (X)
template <int PHASE, class Core>
__device__ __forceinline__ void ns_store(const NsCtl& g, const NsItem& q, const NsMem& mem, const Core& c, int ti, int tj, int wave, char* scratch) {
  constexpr int SB = Core::BLOCK, T = Core::BM;
  const NtBlock<SB, SB> blk{(float*)scratch};
  const int m = q.m, N = PHASE == 2 ? q.n : q.m;
  const int mpad = ns_pad(m), npad = ns_pad(N);
  f16_t* const direct = PHASE == 0 ? mem.a : PHASE == 1 ? mem.s : mem.x;
  f16_t* const turned = PHASE == 2 ? mem.xt[g.cur ^ 1] : direct;
  const bool out = PHASE == 2 && g.last;
  const bool do_rows = !out || !q.tall, do_cols = out ? q.tall != 0 : PHASE == 2 || ti != tj;      // (a diagonal tile is its own mirror image)
#pragma unroll
  for (int bi = 0; bi < Core::WM / SB; ++bi)
#pragma unroll
    for (int bj = 0; bj < Core::WN / SB; ++bj) {
      const int gi = ti * T + Core::row0(wave) + bi * SB, gj = tj * T + Core::col0(wave) + bj * SB;
      blk.put(c, bi, bj, 1.f / NS_SCALE);
      if (do_rows || PHASE == 1) {
        blk.template rows<PHASE == 1>([&](int i, int j0, float (&v)[8]) {
          const int r = gi + i, k = gj + j0;
          if (r >= m || k >= npad) return;
          if constexpr (PHASE == 1) {
            float a[8];
            nt_load_pair(mem.a + (long)r * 2 * mpad, k, a);
#pragma unroll
            for (int t = 0; t < 8; ++t) v[t] = g.cc * v[t] + g.cb * a[t] + (r == k + t ? g.ca * NS_SCALE : 0.f);
          }
          if (out) {
#pragma unroll
            for (int t = 0; t < 8; ++t) v[t] *= 1.f / NS_SCALE;
            ns_put(q.out, q.dtype, (long)r * N + k, v, N - k);
          } else {
#pragma unroll
            for (int t = 0; t < 8; ++t) v[t] = k + t < N ? v[t] : 0.f;
            nt_store_pair(direct + (long)r * 2 * npad, k, v);
          }
        });
      }
      nt_wave_lds_fence();
      if (do_cols) {
        blk.cols([&](int j, int i0, float (&v)[8]) {
          const int r = gj + j, k = gi + i0;
          if (r >= N || k >= mpad) return;
          if (out) {
#pragma unroll
            for (int t = 0; t < 8; ++t) v[t] *= 1.f / NS_SCALE;
            ns_put(q.out, q.dtype, (long)r * m + k, v, m - k);
          } else {
#pragma unroll
            for (int t = 0; t < 8; ++t) v[t] = k + t < m ? v[t] : 0.f;
            nt_store_pair(turned + (long)r * 2 * mpad, k, v);
          }
        });
      }
    }
}

template <int PHASE, int TILE>
__global__ __launch_bounds__(NsTile<TILE>::Core::THREADS) void ns_product_kernel(NsCtl g, int items) {
  typedef typename NsTile<TILE>::Core Core;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int w = nt_xcd_item((int)blockIdx.x, (int)gridDim.x, items);
  if (w < 0) return;
  int first;
  const int k = ns_find(g, PHASE == 0 ? NS_A : PHASE == 1 ? NS_S : NS_X, w, first);
  const NsItem q = ns_table(g.ws)->it[k];
  const NsMem mem = ns_mem(g, q);
  constexpr int SIDE = Core::BM;
  const int mt = (q.m + SIDE - 1) / SIDE, mpad = ns_pad(q.m), npad = ns_pad(q.n);
  int t = w - first, sp = 0, ti, tj;
  if (PHASE == 0) {                               // (workgroups that run together share a part of the contraction)
    const int tri = mt * (mt + 1) / 2;
    sp = t / tri;
    t -= sp * tri;
  }
  if (PHASE == 2)
    ti = t % mt, tj = t / mt;
  else
    ns_tri(t, ti, tj);
  const f16_t* a = PHASE == 0 ? mem.x : PHASE == 1 ? mem.a : mem.s;
  const f16_t* b = PHASE == 0 ? mem.x : PHASE == 1 ? mem.a : mem.xt[g.cur];
  const long ld = 2L * (PHASE == 0 ? npad : mpad);
  const int stages = (PHASE == 0 ? npad : mpad) / 32;
  const int per = PHASE == 0 ? (stages + q.split - 1) / q.split : stages;
  const int s0 = sp * per, s1 = s0 + per < stages ? s0 + per : stages;
  Core c;
  c.clear();
  c.run(a + (long)ti * SIDE * ld, ld, q.m - ti * SIDE, b + (long)tj * SIDE * ld, ld, (PHASE == 2 ? q.n : q.m) - tj * SIDE, s0, s1, smem);
  if (PHASE == 0 && q.split > 1) {
    f32x4* p = (f32x4*)(mem.part + ((long)t * q.split + sp) * Core::BM * Core::BM) + (long)Core::wave() * Core::TI * Core::TJ * 64 + Core::lane();
#pragma unroll
    for (int i = 0; i < Core::TI; ++i)
#pragma unroll
      for (int j = 0; j < Core::TJ; ++j) p[(i * Core::TJ + j) * 64] = c.acc[i][j];
    return;
  }
  constexpr int SB = Core::BLOCK;
  ns_store<PHASE>(g, q, mem, c, ti, tj, Core::wave(), smem + Core::wave() * NtBlock<SB, SB>::BYTES);
}

// joins the partial tiles of a split A = X X^T, in their order: one wave per workgroup, for one wave's share of a tile
template <int TILE>
__global__ __launch_bounds__(64) void ns_join_kernel(NsCtl g) {
  typedef typename NsTile<TILE>::Core Core;
  constexpr int SB = Core::BLOCK;
  __shared__ __attribute__((aligned(16))) char scratch[NtBlock<SB, SB>::BYTES];
  int first;
  const int w = (int)blockIdx.x / Core::NW, wave = (int)blockIdx.x % Core::NW, k = ns_find(g, NS_JOIN, w, first);
  const NsItem q = ns_table(g.ws)->it[k];
  const NsMem mem = ns_mem(g, q);
  const int t = w - first;
  int ti, tj;
  ns_tri(t, ti, tj);
  Core c;
  c.clear();
  const f32x4* p = (const f32x4*)(mem.part + (long)t * q.split * Core::BM * Core::BM) + (long)wave * Core::TI * Core::TJ * 64 + Core::lane();
  for (int s = 0; s < q.split; ++s, p += Core::BM * Core::BM / 4) {
#pragma unroll
    for (int i = 0; i < Core::TI; ++i)
#pragma unroll
      for (int j = 0; j < Core::TJ; ++j) c.acc[i][j] += p[(i * Core::TJ + j) * 64];
  }
  ns_store<0>(g, q, mem, c, ti, tj, wave, scratch);
}

// ---- matrices of at most 64 rows -------------------------------------------------------------------------------------------------------
// A and S fit a workgroup, so a step is one launch: every workgroup sums the partial A's, makes S for itself, takes its columns of X through
// S X -- in place, in the X^T orientation alone -- and leaves the partial A of what it made.  A chunk is CH tiles of 64 columns; with about
// sqrt(8 tiles) chunks the reading of all partial A's (16 KB each) and a chunk's own tiles take about as long.  Launches, not work, are what
// such a call costs: 2 + one per step.
// a 64 x 64 pair operand in LDS: [2 stages][64 rows][128 bytes], pieces swizzled as in the ring
struct NsPair64 {
  static constexpr int BYTES = 2 * 64 * 128;
  char* s;
  __device__ __forceinline__ char* at(int row, int k, int lo) const {    // k: a multiple of 8
    return s + (k >> 5) * 8192 + row * 128 + (((lo * 4 + ((k & 31) >> 3)) ^ (row & 7)) * 16);
  }
  __device__ __forceinline__ void put(int row, int k, const float (&v)[8]) const {
    uint4 hi, lo;
    nt_split8(v, hi, lo);
    *(uint4*)at(row, k, 0) = hi;
    *(uint4*)at(row, k, 1) = lo;
  }
};
// wave w's 32 x 32 quarter of a b^T, added to acc (coordinates as NtCore's; hi * lo + lo * hi summed apart, as there)
__device__ __forceinline__ void ns_mul64(const NsPair64& a, const NsPair64& b, f32x4 (&acc)[2][2]) {
  const int w = (int)(threadIdx.x >> 6), l = threadIdx.x & 63, r0 = (w >> 1) * 32 + (l & 15), c0 = (w & 1) * 32 + (l & 15), g = (l >> 4) * 8;
  f32x4 low[2][2] = {};
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    f16x8 bh[2], bl[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) bh[j] = *(const f16x8*)b.at(c0 + j * 16, s * 32 + g, 0), bl[j] = *(const f16x8*)b.at(c0 + j * 16, s * 32 + g, 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f16x8 ah = *(const f16x8*)a.at(r0 + i * 16, s * 32 + g, 0), al = *(const f16x8*)a.at(r0 + i * 16, s * 32 + g, 1);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        low[i][j] = mfma16(bl[j], al, low[i][j]);
        low[i][j] = mfma16(bh[j], al, low[i][j]);
        low[i][j] = mfma16(bl[j], ah, low[i][j]);
        acc[i][j] = mfma16(bh[j], ah, acc[i][j]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] += low[i >> 1][i & 1];
}
// fp32 64 x 64 in LDS, in NtBlock's arrangement, for the whole workgroup
typedef NtBlock<64, 64> NsF64;
__device__ __forceinline__ void ns_f64_put(const NsF64& f, const f32x4 (&acc)[2][2]) {
  const int w = (int)(threadIdx.x >> 6), l = threadIdx.x & 63, r0 = (w >> 1) * 32 + (l & 15), c0 = (w & 1) * 32 + 4 * (l >> 4);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) *(float4*)f.at(r0 + i * 16, c0 + j * 16) = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
}
__device__ __forceinline__ void ns_f64_row8(const NsF64& f, int i, int j, float (&v)[8]) {     // j: a multiple of 8
  const float4 x = ((const float4*)f.at(i, j))[0], y = ((const float4*)f.at(i, j))[1];
  v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
}
__device__ __forceinline__ void ns_part_put(float* part, const f32x4 (&acc)[2][2]) {
  f32x4* p = (f32x4*)part + threadIdx.x;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) p[(i * 2 + j) * 256] = acc[i][j];
}

// normalises U into xt and makes the first partial A
template <bool SHORT>
__global__ __launch_bounds__(256) void ns_narrow_prep_kernel(NsCtl g, NsAll all) {
  __shared__ __attribute__((aligned(16))) char pool[64 * 65 * 4 + NsPair64::BYTES];
  __shared__ double sm[4];
  __shared__ float2 s_inv;
  static_assert(sizeof(pool) >= NS_SHORT_LDS, "LDS");
  if (SHORT && (int)blockIdx.x >= all.items) {
    ns_short_apply(g, all, (int)blockIdx.x - all.items, pool);
    return;
  }
  float* const tile = (float*)pool;                                     // [row of X][65]
  const NsPair64 xa{pool + ((64 * 65 * 4 + 127) & ~127)};
  int first;
  const int w = (int)blockIdx.x, k = ns_find(g, NS_NARROW, w, first), tid = threadIdx.x, chunk = w - first;
  const NsItem q = ns_table(g.ws)->it[k];
  const NsNarrow mem = ns_narrow_mem(g.ws + (long)q.base * 256, q);
  double sum = 0.0;
  for (int i = tid, n = ns_sums(q); i < n; i += 256) sum += mem.sums[i];
  sum = wave_sum(sum);
  if ((tid & 63) == 0) sm[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) s_inv = ns_inverse(sm[0] + sm[1] + sm[2] + sm[3], g.eps);
  __syncthreads();
  const float2 inv = s_inv;
  const int tiles = (q.n + 63) / 64, P = ns_chunks(q.n), ch = (tiles + P - 1) / P;
  f32x4 acc[2][2] = {};
  for (int t = chunk * ch; t < tiles && t < chunk * ch + ch; ++t) {
    const int c0 = t * 64;
    __syncthreads();
    for (int e = tid; e < 64 * 64; e += 256) {
      const int i = q.tall ? e & 63 : e >> 6, j = q.tall ? e >> 6 : e & 63;                    // X's row and column; along U's rows either way
      tile[i * 65 + j] = i < q.m && c0 + j < q.n ? ns_load(q.u, q.dtype, q.tall ? (long)(c0 + j) * q.m + i : (long)i * q.n + c0 + j) * inv.y * inv.x : 0.f;
    }
    __syncthreads();
    for (int e = tid; e < 64 * 8; e += 256) {
      const int r = e >> 3, c = (e & 7) * 8;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = tile[r * 65 + c + i];
      xa.put(r, c, v);
      if (c0 + r < q.n) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = tile[(c + i) * 65 + r];
        nt_store_pair(mem.xt + (long)(c0 + r) * 128, c, v);
      }
    }
    __syncthreads();
    ns_mul64(xa, xa, acc);
  }
  ns_part_put(mem.part[0] + NS_PART64 * chunk, acc);
}

__global__ __launch_bounds__(256) void ns_narrow_step_kernel(NsCtl g) {
  __shared__ __attribute__((aligned(128))) char pool[NsF64::BYTES + 2 * NsPair64::BYTES];
  const NsF64 f{(float*)pool};
  const NsPair64 sp{pool + NsF64::BYTES}, xp{pool + NsF64::BYTES + NsPair64::BYTES};           // S; X^T's rows, then X's
  int first;
  const int w = (int)blockIdx.x, k = ns_find(g, NS_NARROW, w, first), tid = threadIdx.x, chunk = w - first;
  const NsItem q = ns_table(g.ws)->it[k];
  const NsNarrow mem = ns_narrow_mem(g.ws + (long)q.base * 256, q);
  const int tiles = (q.n + 63) / 64, P = ns_chunks(q.n), ch = (tiles + P - 1) / P;
  // A: the parts in their order, in the accumulators' own arrangement
  f32x4 a[2][2] = {}, acc[2][2] = {};
  {
    const f32x4* p = (const f32x4*)mem.part[g.cur] + tid;
#pragma unroll 4
    for (int s = 0; s < P; ++s, p += NS_PART64 / 4)
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i >> 1][i & 1] += p[i * 256];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i >> 1][i & 1] *= 1.f / NS_SCALE;
  ns_f64_put(f, a);
  __syncthreads();
  for (int e = tid; e < 64 * 8; e += 256) {
    float v[8];
    ns_f64_row8(f, e >> 3, (e & 7) * 8, v);
    xp.put(e >> 3, (e & 7) * 8, v);
  }
  __syncthreads();
  ns_mul64(xp, xp, acc);
  {
    const int l = tid & 63, r0 = (tid >> 7) * 32 + (l & 15), c0 = ((tid >> 6) & 1) * 32 + 4 * (l >> 4);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          // (A as its square saw it: b and c then act on the same eigenvalues, and their roundings' effects largely cancel)
          const f16_t hi = (f16_t)a[i][j][r], lo = (f16_t)(a[i][j][r] - (float)hi);
          a[i][j][r] = (float)hi + (float)lo;
          acc[i][j][r] = g.cc * (acc[i][j][r] * (1.f / NS_SCALE)) + g.cb * a[i][j][r] + (r0 + i * 16 == c0 + j * 16 + r ? g.ca * NS_SCALE : 0.f);
        }
  }
  ns_f64_put(f, acc);                                                   // (every wave has read A's copy: the barrier above)
  __syncthreads();
  for (int e = tid; e < 64 * 8; e += 256) {
    float v[8];
    ns_f64_row8(f, e >> 3, (e & 7) * 8, v);
    sp.put(e >> 3, (e & 7) * 8, v);
  }
  f32x4 next[2][2] = {};
  for (int t = chunk * ch; t < tiles && t < chunk * ch + ch; ++t) {
    const int c0 = t * 64;
    __syncthreads();
    for (int e = tid; e < 64 * 16; e += 256) {                          // X^T's 64 rows of 256 bytes
      const int r = e >> 4, piece = e & 15;
      const uint4 v = c0 + r < q.n ? *(const uint4*)(mem.xt + (long)(c0 + r) * 128 + piece * 8) : make_uint4(0, 0, 0, 0);
      *(uint4*)(xp.s + (piece >> 3) * 8192 + r * 128 + (((piece & 7) ^ (r & 7)) * 16)) = v;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = f32x4{0.f, 0.f, 0.f, 0.f};
    ns_mul64(sp, xp, acc);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] *= 1.f / NS_SCALE;
    ns_f64_put(f, acc);
    __syncthreads();
    for (int e = tid; e < 64 * 8; e += 256) {
      const int r = e >> 3, c = (e & 7) * 8;
      float v[8];
      if (g.last) {
        if (!q.tall) {
          ns_f64_row8(f, r, c, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] *= 1.f / NS_SCALE;
          if (r < q.m && c0 + c < q.n) ns_put(q.out, q.dtype, (long)r * q.n + c0 + c, v, q.n - c0 - c);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = *f.at(c + i, r) * (1.f / NS_SCALE);
          if (c0 + r < q.n && c < q.m) ns_put(q.out, q.dtype, (long)(c0 + r) * q.m + c, v, q.m - c);
        }
      } else {
        ns_f64_row8(f, r, c, v);
        xp.put(r, c, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = *f.at(c + i, r);
        if (c0 + r < q.n) nt_store_pair(mem.xt + (long)(c0 + r) * 128, c, v);
      }
    }
    if (!g.last) {
      __syncthreads();
      ns_mul64(xp, xp, next);
    }
  }
  if (!g.last) ns_part_put(mem.part[g.cur ^ 1] + NS_PART64 * chunk, next);
}

// ---- host side ------------------------------------------------------------------------------------------------------------------
// One tile size serves all matrices of a launch.  A workgroup's stage takes about CYC cycles where it shares a CU with others (the matrix pipe and
// LDS are then busy) and at least LAT where it is alone; 256-wide tiles move the fewest bytes per product, smaller ones reach more CUs.
struct NsPlan {
  int tile[3], split;                            // per phase; parts of A's contraction
  bool narrow;                                   // no matrix has more than 64 rows
};
constexpr int NS_TILES[3] = {256, 128, 64};
constexpr double NS_CYC[3] = {5200, 1500, 480}, NS_LAT[3] = {5200, 1900, 700}, NS_LAUNCH = 9000;

NsPlan ns_plan(const FiNsMat* const* mats, int count) {
  NsPlan p = {};
  p.split = 1, p.narrow = true;
  for (int i = 0; i < count; ++i) p.narrow = p.narrow && (mats[i]->rows <= 64 || mats[i]->cols <= 64);
  if (p.narrow) return p;
  for (int phase = 0; phase < 3; ++phase) {
    double best = 0;
    for (int k = 0; k < 3; ++k) {
      const int T = NS_TILES[k];
      for (int split = 1; split <= (phase == 0 ? 32 : 1); split *= 2) {
        double wgs = 0, longest = 0;
        for (int i = 0; i < count; ++i) {
          const int m = mats[i]->rows < mats[i]->cols ? mats[i]->rows : mats[i]->cols, n = mats[i]->rows < mats[i]->cols ? mats[i]->cols : mats[i]->rows;
          const double mt = (m + T - 1) / T, nt = (n + T - 1) / T, stages = (ns_pad(phase == 0 ? n : m) / 32 + split - 1) / split;
          wgs += phase == 2 ? mt * nt : mt * (mt + 1) / 2 * split;
          if (stages > longest) longest = stages;
        }
        const double rounds = (double)((long)(wgs + 255) / 256);
        double cost = longest * (rounds * NS_CYC[k] > NS_LAT[k] ? rounds * NS_CYC[k] : NS_LAT[k]);
        if (split > 1) cost += NS_LAUNCH + split * T * T / 12.0;       // the joining launch, its partial tiles read by one workgroup each
        if (best == 0 || cost < best) best = cost, p.tile[phase] = T, p.split = phase == 0 ? split : p.split;
      }
    }
  }
  // small matrices are held to an fp32 iteration's error: where no larger one shares their launches, their tiles keep the low parts' sums apart (17 .. 64 rows: 6.2e-7 ..
  // 9.0e-7 of the result off by themselves, 7.7e-7 .. 1.04e-6 beside a matrix of 300 or 1000 rows, 7.9e-7 .. 1.2e-6 by fp32 products)
  int most = 0;
  for (int i = 0; i < count; ++i) {
    const int m = mats[i]->rows < mats[i]->cols ? mats[i]->rows : mats[i]->cols;
    if (m > most) most = m;
  }
  for (int phase = 0; phase < 3 && most <= 256; ++phase)
    if (p.tile[phase] == 64) p.tile[phase] = 32;
  return p;
}

// Fills in the matrices of a launch group; returns their workspace's size.
long ns_layout(const FiNsMat* const* mats, int count, const NsPlan& plan, bool shorts, NsArgs& g) {
  long at = (sizeof(NsTable) + 255) & ~255L;
  g.count = count, g.narrow = plan.narrow;
  for (int k = 0; k < 3; ++k) g.tile[k] = plan.narrow ? 64 : plan.tile[k];
  for (int i = 0; i < count; ++i) {
    NsItem& q = g.it[i];
    q.u = mats[i]->u, q.out = mats[i]->out, q.dtype = mats[i]->dtype;
    q.tall = mats[i]->rows > mats[i]->cols;
    q.m = q.tall ? mats[i]->cols : mats[i]->rows;
    q.n = q.tall ? mats[i]->rows : mats[i]->cols;
    const int stages = ns_pad(q.n) / 32, per = (stages + plan.split - 1) / plan.split;
    q.split = (stages + per - 1) / per;          // (no part is empty)
    q.base = (unsigned)(at >> 8);
    const long side = ns_side(plan.tile[0]), mt = (q.m + side - 1) / side, own = plan.narrow ? ns_narrow_mem(nullptr, q).bytes : ns_mem(nullptr, q).bytes;
    const long few = q.m <= NS_SHORT_ROWS ? 2048L * ((q.n + ns_short_cols(q.n) - 1) / ns_short_cols(q.n)) : 0;      // (whichever form the steps' number allows)
    at += own > few ? own : few;
    if (!plan.narrow && q.split > 1) at += 4L * (mt * (mt + 1) / 2) * q.split * side * side;
    if (shorts && q.m <= NS_SHORT_ROWS) q.split = 0;
  }
  return at;
}

int ns_check_polynomial(int steps, const float* coeffs) {
  // every singular value starts in [0, 1]: the polynomial must keep X, A and S inside the storage's range (16 / 2^-12)
  for (int i = 0; i <= 1024; ++i) {
    double s = i / 1024.0;
    for (int k = 0; k < steps; ++k) {
      const double l = s * s, f = coeffs[3 * k] + coeffs[3 * k + 1] * l + coeffs[3 * k + 2] * l * l;
      if (!(fabs(f) < 15.0)) return FI_ERR_UNSUPPORTED;
      s = f * s;
      if (!(fabs(s) < 3.75)) return FI_ERR_UNSUPPORTED;
    }
  }
  return 0;
}

int ns_check(const FiNsMat* mats, int count, int steps, const float* coeffs) {
  if (!mats || !coeffs) return FI_ERR_NULL;
  if (count < 1 || steps < 1) return FI_ERR_SHAPE;
  for (int i = 0; i < count; ++i) {
    const FiNsMat& q = mats[i];
    if (q.dtype != FI_F32 && q.dtype != FI_BF16 && q.dtype != FI_F16) return FI_ERR_DTYPE;
    if (q.rows < 1 || q.cols < 1 || q.rows > (1 << 20) || q.cols > (1 << 20)) return FI_ERR_SHAPE;
    const int m = q.rows < q.cols ? q.rows : q.cols;
    if (m > 32768) return FI_ERR_SHAPE;
  }
  return ns_check_polynomial(steps, coeffs);
}

int ns_total(const NsArgs& g, int kind) {
  long n = 0;
  for (int i = 0; i < g.count; ++i) n += ns_items(g.it[i], kind, ns_side_of(g, kind));
  return n < (1L << 30) ? (int)n : -1;
}
template <int PHASE, int TILE>
int ns_product(const NsCtl& c, int items, int joins, hipStream_t st) {
  typedef typename NsTile<TILE>::Core Core;
  static NtLdsDevices allowed;
  if (!nt_allow_lds((const void*)ns_product_kernel<PHASE, TILE>, allowed)) return FI_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((ns_product_kernel<PHASE, TILE>), dim3((items + 7) & ~7), dim3(Core::THREADS), Core::LDS, st, c, items);
  FI_CHECK_LAUNCH();
  if (PHASE == 0 && joins) {
    hipLaunchKernelGGL((ns_join_kernel<TILE>), dim3(joins * Core::NW), dim3(64), 0, st, c);
    FI_CHECK_LAUNCH();
  }
  return 0;
}
template <int PHASE>
int ns_product(const NsCtl& c, int tile, int items, int joins, hipStream_t st) {
  return tile == 32 ? ns_product<PHASE, 32>(c, items, joins, st) : tile == 64 ? ns_product<PHASE, 64>(c, items, joins, st) : tile == 128 ? ns_product<PHASE, 128>(c, items, joins, st)
                                                                               : ns_product<PHASE, 256>(c, items, joins, st);
}

int ns_run(NsArgs& g, int steps, const float* coeffs, float eps, hipStream_t st) {
  int n[NS_KINDS];
  for (int k = 0; k < NS_KINDS; ++k)
    if ((n[k] = ns_total(g, k)) < 0) return FI_ERR_SHAPE;
  g.eps = eps;
  for (int i = 0, at = 0; i < g.count; ++i) g.first[i] = at, at += (int)ns_items(g.it[i], NS_SUMS, 64);
  NsCtl c = {g.ws, g.count, 0, 0, 0.f, 0.f, 0.f, eps};
  NsAll all = {n[g.narrow ? NS_NARROW : NS_PREP], steps, {}};
  for (int k = 0; k < 3 * steps && k < 3 * NS_STEPS; ++k) all.c[k] = coeffs[k];
  hipLaunchKernelGGL(n[NS_SHORT] ? ns_norm_kernel<true> : ns_norm_kernel<false>, dim3(n[NS_SUMS]), dim3(256), 0, st, g);
  FI_CHECK_LAUNCH();
  auto* const prep = n[NS_SHORT] ? (g.narrow ? ns_narrow_prep_kernel<true> : ns_prep_kernel<true>) : g.narrow ? ns_narrow_prep_kernel<false> : ns_prep_kernel<false>;
  hipLaunchKernelGGL(prep, dim3(all.items + n[NS_SHORT]), dim3(256), 0, st, c, all);
  FI_CHECK_LAUNCH();
  for (int k = 0; k < steps && all.items; ++k) {
    c.ca = coeffs[3 * k], c.cb = coeffs[3 * k + 1], c.cc = coeffs[3 * k + 2];
    c.cur = k & 1, c.last = k + 1 == steps;
    if (g.narrow) {
      hipLaunchKernelGGL(ns_narrow_step_kernel, dim3(n[NS_NARROW]), dim3(256), 0, st, c);
      FI_CHECK_LAUNCH();
      continue;
    }
    int rc = ns_product<0>(c, g.tile[0], n[NS_A], n[NS_JOIN], st);
    if (!rc) rc = ns_product<1>(c, g.tile[1], n[NS_S], 0, st);
    if (!rc) rc = ns_product<2>(c, g.tile[2], n[NS_X], 0, st);
    if (rc) return rc;
  }
  return 0;
}

// f(arguments) for every launch group; the workspace is used again by each.  Returns its size, or an error (positive ones as -1000 - error).
template <class F>
long ns_groups(const FiNsMat* mats, int count, int steps, char* ws, F f) {
  long most = 0;
  for (int lo = 0; lo < count; lo += NS_MAX) {
    const FiNsMat* pick[NS_MAX];
    const int n = count - lo < NS_MAX ? count - lo : NS_MAX;
    for (int i = 0; i < n; ++i) pick[i] = &mats[lo + i];
    const NsPlan plan = ns_plan(pick, n);
    NsArgs g = {};
    g.ws = ws;
    const long bytes = ns_layout(pick, n, plan, steps <= NS_STEPS, g);
    if (bytes >> 40) return FI_ERR_SHAPE;
    if (bytes > most) most = bytes;
    const int rc = f(g);
    if (rc) return rc < 0 ? rc : -1000 - rc;
  }
  return most;
}

}  // namespace

extern "C" long fi_newton_schulz_workspace(const FiNsMat* mats, int count) {
  const float c[3] = {0.f, 0.f, 0.f};
  const int rc = ns_check(mats, count, 1, c);
  if (rc) return rc;
  return ns_groups(mats, count, 1, nullptr, [](NsArgs&) { return 0; });
}

extern "C" int fi_newton_schulz(const FiNsMat* mats, int count, int steps, const float* coeffs, float eps, void* workspace, void* stream) {
  const int rc = ns_check(mats, count, steps, coeffs);
  if (rc) return rc;
  if (!workspace) return FI_ERR_NULL;
  for (int i = 0; i < count; ++i)
    if (!mats[i].u || !mats[i].out) return FI_ERR_NULL;
  hipStream_t st = (hipStream_t)stream;
  const long got = ns_groups(mats, count, steps, (char*)workspace, [&](NsArgs& g) { return ns_run(g, steps, coeffs, eps, st); });
  return got >= 0 ? 0 : got > -1000 ? (int)got : (int)(-1000 - got);
}

// ---- the optimizer step around it ---------------------------------------------------------------------------------------------------------
namespace {

struct MuonArgs {
  FiMuonMat it[NS_MAX];
  int start[NS_MAX + 1];                         // first block of NS_CHUNK values of each matrix
  int count, nesterov;
  float momentum, wd;
  const double* lr;
  const float* skip;
  float* u;                                      // the updates, each from a multiple of NS_CHUNK values on
};
static_assert(sizeof(MuonArgs) <= 4096, "kernel arguments");

__device__ __forceinline__ int muon_find(const MuonArgs& a, int w) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.start[mid] <= w)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}
__host__ __device__ __forceinline__ long muon_size(const FiMuonMat& q) { return (long)q.rows * q.cols; }

// buf <- momentum buf + (1 - momentum) g;  u = (1 - momentum) g + momentum buf (Nesterov) or buf
__global__ __launch_bounds__(256) void muon_momentum_kernel(MuonArgs a) {
  const int k = muon_find(a, (int)blockIdx.x);
  const FiMuonMat& q = a.it[k];
  const long n = muon_size(q), lo = (long)((int)blockIdx.x - a.start[k]) * NS_CHUNK, hi = lo + NS_CHUNK < n ? lo + NS_CHUNK : n;
  const bool skip = a.skip && a.skip[0] != 0.f;
  float* const u = a.u + (long)a.start[k] * NS_CHUNK;
  for (long i = lo + threadIdx.x; i < hi; i += 256) {
    const float g = q.grad[i], b = __builtin_fmaf(a.momentum, q.buf[i] - g, g);
    u[i] = a.nesterov ? __builtin_fmaf(a.momentum, b - g, g) : b;
    if (!skip) q.buf[i] = b;
  }
}
// p <- (1 - lr wd) p - lr scale u
__global__ __launch_bounds__(256) void muon_apply_kernel(MuonArgs a) {
  if (a.skip && a.skip[0] != 0.f) return;
  const int k = muon_find(a, (int)blockIdx.x);
  const FiMuonMat& q = a.it[k];
  const long n = muon_size(q), lo = (long)((int)blockIdx.x - a.start[k]) * NS_CHUNK, hi = lo + NS_CHUNK < n ? lo + NS_CHUNK : n;
  const double lr = a.lr[0];
  const float keep = (float)(1.0 - lr * (double)a.wd), step = (float)(lr * (double)q.scale);
  const float* const u = a.u + (long)a.start[k] * NS_CHUNK;
  for (long i = lo + threadIdx.x; i < hi; i += 256) q.param[i] = q.param[i] * keep - step * u[i];
}

// the step's groups of at most NS_MAX matrices: f(arguments, their matrices as the iteration takes them, count, blocks)
template <class F>
long muon_groups(const FiMuonMat* mats, int count, float* u, F f) {
  long most = 0;
  for (int lo = 0; lo < count; lo += NS_MAX) {
    MuonArgs a = {};
    FiNsMat ns[NS_MAX];
    a.count = count - lo < NS_MAX ? count - lo : NS_MAX;
    a.u = u;
    long n = 0;
    for (int i = 0; i < a.count; ++i) {
      a.it[i] = mats[lo + i];
      a.start[i] = (int)n;
      float* const at = u + n * NS_CHUNK;
      ns[i] = FiNsMat{at, at, FI_F32, mats[lo + i].rows, mats[lo + i].cols};
      n += (muon_size(mats[lo + i]) + NS_CHUNK - 1) / NS_CHUNK;
    }
    a.start[a.count] = (int)n;
    if (n >= (1L << 30)) return FI_ERR_SHAPE;
    if (n * NS_CHUNK * 4 > most) most = n * NS_CHUNK * 4;
    const long rc = f(a, ns, (int)n);
    if (rc) return rc;
  }
  return most;
}

}  // namespace

extern "C" long fi_muon_step_workspace(const FiMuonMat* mats, int count) {
  if (!mats) return FI_ERR_NULL;
  if (count < 1) return FI_ERR_SHAPE;
  long most = 0;
  const long u = muon_groups(mats, count, (float*)256, [&](MuonArgs& a, const FiNsMat* ns, int) {
    const long b = fi_newton_schulz_workspace(ns, a.count);
    if (b < 0) return b;
    if (b > most) most = b;
    return 0L;
  });
  return u < 0 ? u : u + most;
}

extern "C" int fi_muon_step(const FiMuonMat* mats, int count, const double* lr, float momentum, int nesterov, float weight_decay, int steps,
                            const float* coeffs, float eps, const float* skip, void* workspace, void* stream) {
  const long total = fi_muon_step_workspace(mats, count);
  if (total < 0) return (int)total;
  if (!lr || !coeffs || !workspace) return FI_ERR_NULL;
  if (steps < 1) return FI_ERR_SHAPE;
  const int rc0 = ns_check_polynomial(steps, coeffs);                   // (before the momentum moves: an error leaves everything as it was)
  if (rc0) return rc0;
  for (int i = 0; i < count; ++i)
    if (!mats[i].param || !mats[i].grad || !mats[i].buf) return FI_ERR_NULL;
  hipStream_t st = (hipStream_t)stream;
  const long u = muon_groups(mats, count, (float*)workspace, [](MuonArgs&, const FiNsMat*, int) { return 0L; });
  const long rc = muon_groups(mats, count, (float*)workspace, [&](MuonArgs& a, const FiNsMat* ns, int blocks) -> long {
    a.lr = lr, a.momentum = momentum, a.nesterov = nesterov, a.wd = weight_decay, a.skip = skip;
    hipLaunchKernelGGL(muon_momentum_kernel, dim3(blocks), dim3(256), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return -1000 - (long)e;
    const int r = fi_newton_schulz(ns, a.count, steps, coeffs, eps, (char*)workspace + u, stream);
    if (r) return r < 0 ? r : -1000 - (long)r;
    hipLaunchKernelGGL(muon_apply_kernel, dim3(blocks), dim3(256), 0, st, a);
    e = hipGetLastError();
    return e != hipSuccess ? -1000 - (long)e : 0;
  });
  return rc >= 0 ? 0 : rc > -1000 ? (int)rc : (int)(-1000 - rc);
}
