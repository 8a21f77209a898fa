// Softmax cross entropy of a linear head over many classes, without its logits:  z = x W^T + b,
//     loss_t = log sum_v exp z_tv - z_{t, label_t},        G_tv = g_t (exp(z_tv) / sum_v exp z_tv - [v = label_t]),
//     dx = G W,   dW = G^T x,   db = sum_t G_t            (g_t: the gradient of row t's loss; ignored rows take no part)
//
// Forward: one product whose epilogue turns each tile of logits into the row's maximum and sum of exponentials over the tile's
// classes and picks the label's logit; a second pass over those (8 bytes per row and tile) joins them.  Backward: the product is made
// again, a piece of rows x classes at a time, its epilogue writes G in 16 bits in both orientations, and two products take it from there.
// The logits never exist in memory, G only a piece at a time -- and with up to 128 features not at all (ce_fused_kernel).
//
// Only labelled rows take part: their numbers are gathered first (stable, no atomics), x is packed through that list, and every
// kernel takes the number of rows from the device -- nine pixels of ten unlabelled cost a tenth.
//
// Types: fp32 operands and their G go to the matrix pipe as triples of bf16 (nt_product.h): exactly, whatever their sizes (from 8e-34 on), so that no row, class or feature costs
// another its bits; short products of fp16 as triples too, for G's sake (ce_shape).  Other 16-bit x and W go as they are.  Their G is fp16, which keeps 11 bits
// where bf16 would keep 8, and so are x and W in its products: bf16 ones under a power-of-two scale per tensor, exact down to 2^-31 of the tensor's largest value and
// lost below 2^-39.  For dx a row of G is made with a factor of one, at 2^14, for dW with its own, the largest |g_t| at 2^14; what lies below 2^-39 of that is
// lost.  Row statistics, sums and db are fp32 (joins in fp64).
//
// Measured at 7370 labelled rows x 50000 x 1024 bf16: forward 691 us (1092 TFLOP/s), and per half of the classes G 503 (750: its stores) and each
// gradient 392 (963), where a large library product reaches 1430 and one of a gradient's size 1068.  Bound by the fill of LDS from L2 and by its
// reads: without any fill the product of 7370 x 1024 x 16384 takes 158 us where it takes 221.  4001 x 8003 x 384 fp32 (triples): forward 144 us (1020 TFLOP/s of
// matrix instructions), G 197, each gradient 173.
#include "nt_product.h"

namespace {

typedef int64_t i64;
constexpr float CE_LOG2E = 1.4426950408889634f;
constexpr int CE_ROWS = 2048;                   // rows per workgroup of the gathering passes
constexpr int CE_PARTS = 1024;                  // partial results of the max passes
constexpr int CE_LOSS_WGS = 512;

// kept from the forward to the backward pass, at the head of the caller's `saved` buffer; T = rows
//   int count (labelled rows) | ... 64 bytes | int idx[T] | int label[T] | float2 stat[T] (row maximum, 1 / sum)
struct CeSaved {
  int* count;
  int* idx;
  int* lab;
  float2* stat;
};
__host__ __device__ __forceinline__ i64 ce_up(i64 v, i64 a) { return (v + a - 1) / a * a; }
CeSaved ce_saved(void* p, i64 T) {
  char* c = (char*)p;
  const i64 n = ce_up(4 * T, 64);
  return CeSaved{(int*)c, (int*)(c + 64), (int*)(c + 64 + n), (float2*)(c + 64 + 2 * n)};
}

// the backward pass's scalars on the device: [0] / [1] the scale of bf16 x / W as fp16, [2] / [3] their reciprocals, [4] 1 / (scale of G)
enum { SC_X = 0, SC_W = 1, SC_RX = 2, SC_RW = 3, SC_RG = 4, SC_N = 8 };

__device__ __forceinline__ float ce_load(const void* p, int dtype, i64 i) {
  return dtype == FI_F32 ? ((const float*)p)[i] : dtype == FI_BF16 ? (float)((const bf16_t*)p)[i] : (float)((const f16_t*)p)[i];
}
__device__ __forceinline__ i64 ce_label(const void* p, int ltype, i64 i) {
  return ltype == FI_LABEL_U8 ? (i64)((const uint8_t*)p)[i] : ltype == FI_LABEL_I32 ? (i64)((const int*)p)[i] : ((const i64*)p)[i];
}
__device__ __forceinline__ float ce_pow2_scale(float amax) {          // s with amax * s in [2^14, 2^15); 1 where there is nothing to scale
  if (!(amax > 0.f) || !(amax < INFINITY)) return 1.f;
  int e = (int)((__float_as_uint(amax) >> 23) & 255) - 127;
  e = 14 - e;
  e = e > 126 ? 126 : e < -126 ? -126 : e;
  return __uint_as_float((unsigned)(e + 127) << 23);
}

// ---- gathering the labelled rows ----------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void ce_count_kernel(const void* labels, int ltype, i64 T, i64 ignore, int* cnt) {
  __shared__ int sm[4];
  const i64 r0 = (i64)blockIdx.x * CE_ROWS;
  int n = 0;
  for (int k = threadIdx.x; k < CE_ROWS; k += 256)
    if (r0 + k < T && ce_label(labels, ltype, r0 + k) != ignore) ++n;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) cnt[blockIdx.x] = sm[0] + sm[1] + sm[2] + sm[3];
}

// the workgroups' counts -> the number of rows before each, in place: one workgroup, a run of counts per thread
// (from CE_SCAN workgroups on: 134e6 rows 590 -> 252 us with the gathering; 17e6 rows 26 -> 30, where every workgroup sums those before it instead)
constexpr int CE_SCAN = 16384;
__global__ __launch_bounds__(1024) void ce_scan_kernel(int* cnt, int nb) {
  __shared__ int sm[1024];
  const int tid = threadIdx.x, per = (nb + 1023) / 1024, lo = tid * per < nb ? tid * per : nb, hi = lo + per < nb ? lo + per : nb;
  int n = 0;
  for (int k = lo; k < hi; ++k) n += cnt[k];
  sm[tid] = n;
  __syncthreads();
  for (int o = 1; o < 1024; o <<= 1) {                                 // inclusive scan
    const int v = tid >= o ? sm[tid - o] : 0;
    __syncthreads();
    sm[tid] += v;
    __syncthreads();
  }
  int at = sm[tid] - n;
  for (int k = lo; k < hi; ++k) {
    const int c = cnt[k];
    cnt[k] = at;
    at += c;
  }
}

// each thread owns 8 consecutive rows; cnt: the workgroups' counts, or (scanned) the rows before each
__global__ __launch_bounds__(256) void ce_gather_kernel(const void* labels, int ltype, i64 T, i64 ignore, int V, const int* cnt, int scanned, CeSaved s,
                                                        float* zt, float* rows_out, const float* bias, float* bias_pad) {
  __shared__ int sm[256], base_sm[4];
  const int tid = threadIdx.x;
  if (bias_pad)                                                         // (the streamed form reads it in whole tiles of 64 classes)
    for (i64 v = (i64)blockIdx.x * 256 + tid; v < ((V + 63) & ~63); v += (i64)gridDim.x * 256) bias_pad[v] = bias && v < V ? bias[v] : 0.f;
  int before = scanned && tid == 0 ? cnt[blockIdx.x] : 0;
  for (int k = tid; k < (int)blockIdx.x && !scanned; k += 256) before += cnt[k];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o, 64);
  if ((tid & 63) == 0) base_sm[tid >> 6] = before;
  const i64 r0 = (i64)blockIdx.x * CE_ROWS + tid * 8;
  i64 lab[8];
  int n = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    lab[k] = r0 + k < T ? ce_label(labels, ltype, r0 + k) : ignore;
    n += lab[k] != ignore;
  }
  sm[tid] = n;
  __syncthreads();
  for (int o = 1; o < 256; o <<= 1) {                                  // inclusive scan
    const int v = tid >= o ? sm[tid - o] : 0;
    __syncthreads();
    sm[tid] += v;
    __syncthreads();
  }
  int at = base_sm[0] + base_sm[1] + base_sm[2] + base_sm[3] + sm[tid] - n;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (lab[k] != ignore) {
      s.idx[at] = (int)(r0 + k);
      s.lab[at] = lab[k] >= 0 && lab[k] < V ? (int)lab[k] : -1;
      zt[at] = __uint_as_float(0x7fc00000u);                           // (a label that is no class leaves NaN behind)
      ++at;
    } else if (rows_out && r0 + k < T) {
      rows_out[r0 + k] = 0.f;
    }
  }
  if (blockIdx.x == gridDim.x - 1 && tid == 255) s.count[0] = at;
}

// ---- the largest finite magnitude of x's labelled rows and of W ------------------------------------------------------------------------
struct CeAmax {
  const void* p;
  int dtype, D, vec;       // vec: rows are aligned for 16-byte loads
  i64 ld, rows;
  const int *idx, *count;  // row list and its length, or NULL
  float* part;             // [CE_PARTS]
  i64 tail;                // values behind the last row
};
template <typename T>
__device__ __forceinline__ float ce_amax_rows(const CeAmax& a, i64 rows) {
  constexpr int VG = DT<T>::VG;
  const int l = threadIdx.x & 63, per = a.vec ? (a.D + VG - 1) / VG : a.D;
  int lanes = 64;                                                       // per row
  while (lanes > 1 && lanes / 2 >= per) lanes >>= 1;
  const int sub = l & (lanes - 1), nr = 64 / lanes, dv = a.vec ? a.D / VG : 0;
  float m = 0.f;
  for (i64 r = ((i64)blockIdx.x * 4 + (threadIdx.x >> 6)) * nr + l / lanes; r < rows; r += (i64)gridDim.x * 4 * nr) {
    const T* q = (const T*)a.p + (a.idx ? (i64)a.idx[r] : r) * a.ld;
    for (int c = sub; c < dv; c += lanes) {
      float f[VG];
      VecWords<T>::unpack(((const typename DT<T>::vec_t*)q)[c], f);
#pragma unroll
      for (int t = 0; t < VG; ++t) m = fabsf(f[t]) < INFINITY ? fmaxf(m, fabsf(f[t])) : m;
    }
    for (int c = dv * VG + sub; c < a.D; c += lanes) {
      const float v = fabsf(to_f32(q[c]));
      if (v < INFINITY) m = fmaxf(m, v);
    }
  }
  for (i64 c = (i64)blockIdx.x * 256 + threadIdx.x; c < a.tail; c += (i64)gridDim.x * 256) {
    const float v = fabsf(to_f32(((const T*)a.p)[rows * a.ld + c]));
    if (v < INFINITY) m = fmaxf(m, v);
  }
  return m;
}
__device__ __forceinline__ float ce_block_max(float m, float* sm) {       // 256 threads; the result in all of them
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = m;
  __syncthreads();
  return fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
}
__global__ __launch_bounds__(256) void ce_amax_kernel(CeAmax x, CeAmax w) {
  __shared__ float sm[4];
  const CeAmax& a = blockIdx.y ? w : x;
  const i64 rows = a.count ? (i64)a.count[0] : a.rows;
  const float m = ce_block_max(a.dtype == FI_F32 ? ce_amax_rows<float>(a, rows) : a.dtype == FI_BF16 ? ce_amax_rows<bf16_t>(a, rows) : ce_amax_rows<f16_t>(a, rows), sm);
  if (threadIdx.x == 0) a.part[blockIdx.x] = m;
}

// ---- the backward pass's rows --------------------------------------------------------------------------------------------------------------
// dx of the rows that take no part: a lane looks at a label, the wave clears the rows it finds
__device__ __forceinline__ void ce_zero_rows(const void* labels, int ltype, i64 T, i64 ignore, char* dx, i64 row_bytes) {
  const int l = threadIdx.x & 63;
  const i64 r0 = ((i64)blockIdx.x * 4 + (threadIdx.x >> 6)) * 64;
  const bool mine = r0 + l < T && ce_label(labels, ltype, r0 + l) == ignore;
  unsigned long long todo = __ballot(mine);
  const bool vec = row_bytes % 16 == 0 && ((uintptr_t)dx & 15) == 0;
  if (vec && row_bytes <= 512) {                                        // several rows at a time
    const int per = (int)(row_bytes / 16), rows = 64 / per;
    if (todo)
      for (int i = 0; i < 64; i += rows) {
        const int r = i + l / per;
        if (l / per < rows && r < 64 && (todo >> r & 1)) ((uint4*)(dx + (r0 + r) * row_bytes))[l % per] = make_uint4(0, 0, 0, 0);
      }
    return;
  }
  while (todo) {
    const int r = __builtin_ctzll(todo);
    todo &= todo - 1;
    char* p = dx + (r0 + r) * row_bytes;
    if (vec)
      for (i64 c = l; c < row_bytes / 16; c += 64) ((uint4*)p)[c] = make_uint4(0, 0, 0, 0);
    else
      for (i64 c = l; c < row_bytes / 2; c += 64) ((uint16_t*)p)[c] = 0;
  }
}

// G is made with CE_UNIT in the factors' place (triples: with one).  These are the rows' factors g_t * scale over that (reduction 0: one upstream gradient per row;
// 1 mean, 2 sum: one for all); zeros for dx's other rows
constexpr float CE_UNIT = 16384.f;
struct CeFactors {
  const float* g;          // upstream gradient
  int reduction;
  const float* part;       // reduction 0: maxima of |g|
  CeSaved s;
  int triple;
  float *scal, *out;
  float4* meta;
  const float* bias;
  float* bias_pad;
  const void* labels;
  int ltype, V;
  i64 T, ignore;
  char* dx;
  i64 row_bytes;
};
__device__ __forceinline__ void ce_factors(const CeFactors& a, float* sm) {
  const CeSaved& s = a.s;
  const float* const g = a.g;
  const int reduction = a.reduction, triple = a.triple, V = a.V, n = s.count[0], tid = threadIdx.x;
  const float *const part = a.part, *const bias = a.bias;
  float *const scal = a.scal, *const out = a.out, *const bias_pad = a.bias_pad;
  float4* const meta = a.meta;
  if (a.dx) ce_zero_rows(a.labels, a.ltype, a.T, a.ignore, a.dx, a.row_bytes);
  const float one = reduction == 1 ? (float)((double)g[0] / (double)n) : reduction == 2 ? g[0] : 0.f;
  float m = fabsf(one);
  if (reduction == 0 && !triple)
    for (int k = tid; k < CE_PARTS; k += 256) m = fmaxf(m, part[k]);
  // The largest factor of 16-bit G is at 2^14 exactly: a label's entry, -g (1 - p), mostly the largest of its row, then lies right below 2^14, where
  // fp16 is finest for its size (1.4e-4 of it, 2.1e-4 on average elsewhere).  Triples need no scale.
  const float top = triple ? 1.f : ce_block_max(m, sm);
  const float sc = triple ? 1.f : !(top > 1e-30f && top < INFINITY) ? 0.5f * ce_pow2_scale(top) : CE_UNIT / top;
  if (blockIdx.x == 0 && tid == 0) scal[SC_RG] = 1.f / sc;
  for (i64 r = (i64)blockIdx.x * 256 + tid; r < n; r += (i64)gridDim.x * 256) {
    const float f = reduction == 0 ? g[s.idx[r]] : one;
    out[r] = s.lab[r] < 0 ? __uint_as_float(0x7fc00000u) : f * (sc / (triple ? 1.f : CE_UNIT));
  }
  if (!meta) return;
  // the fused form's row table, whole tiles of 64 rows long (a row behind the last one: exp2(-inf) * 0), and its bias likewise
  for (i64 r = (i64)blockIdx.x * 256 + tid; r < ((n + 63) & ~63); r += (i64)gridDim.x * 256) {
    float4 m = make_float4(INFINITY, 0.f, 0.f, __int_as_float(-1));
    if (r < n) {
      const float2 st = s.stat[r];
      const float f = s.lab[r] < 0 ? __uint_as_float(0x7fc00000u) : (reduction == 0 ? g[s.idx[r]] : one) * sc;
      m = make_float4(st.x, f * st.y, f, __int_as_float(s.lab[r]));
    }
    meta[r] = m;
  }
  for (i64 v = (i64)blockIdx.x * 256 + tid; v < ((V + 63) & ~63); v += (i64)gridDim.x * 256) bias_pad[v] = bias && v < V ? bias[v] : 0.f;
}
__global__ __launch_bounds__(256) void ce_factors_kernel(CeFactors a) {
  __shared__ float sm[4];
  ce_factors(a, sm);
}

// ---- packing an operand ---------------------------------------------------------------------------------------------------------------
struct CePack {
  const void* src;         // [rows][D], leading dimension ld, storage `dtype`
  int dtype, D, vec;       // vec: rows are aligned for 16-byte loads
  int round;               // fp32 values are rounded to this type first (FI_F32: kept)
  i64 ld, rows, begin;     // rows [begin, begin + rows) of the source (of the list); same and turned start there
  const int* idx;          // row list (x) or NULL
  const int* count;        // rows from the device, or NULL
  const float* part;       // CE_PARTS maxima that the scale of fp16 made of bf16 comes from
  const float* scale;      // or the scale itself; neither: 1
  float *put, *rput;       // where the scale and its reciprocal go (with part)
  void* same;              // [rows][K] operand rows, or NULL
  i64 ld_same;
  int same_k;              // its padded width: whole stages, a multiple of 8
  int same_kind;           // 0 bf16, 1 fp16, 2 triples
  void* turned;            // [D][rows] operand rows (fp16, scaled, or triples), or NULL
  i64 ld_turned;
  int turned_triple;
};
template <typename T>
__device__ __forceinline__ void ce_load8(const T* q, int left, int vec, float (&v)[8]) {
  if (vec && left >= 8) {
    if constexpr (sizeof(T) == 4) {
      const float4 x = ((const float4*)q)[0], y = ((const float4*)q)[1];
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    } else {
      VecWords<T>::unpack(*(const uint4*)q, v);
    }
    return;
  }
#pragma unroll
  for (int t = 0; t < 8; ++t) v[t] = t < left ? to_f32(q[t]) : 0.f;
}
// one 64 x 64 block of the source per workgroup (blockIdx.x: rows, .y: columns, .z: which operand); pads are written as zeros
// (the last slice of a launch with f.g: the rows' factors, which need nothing of the operands)
// LOOSE: some rows are not aligned for vectors; they come by a value per lane, through the tile (122 x 72099 x 1730 fp32: 528 -> 427 us a launch, whose
// registers cost aligned operands a third: 15 -> 20 us at 524288 x 16)
template <bool LOOSE>
__global__ __launch_bounds__(256) void ce_pack_kernel(CePack px, CePack pw, CeFactors f) {
  __shared__ float tile[64][65];
  __shared__ float sm[4];
  if (f.g && blockIdx.z == gridDim.z - 1) {
    if (blockIdx.y == 0) ce_factors(f, sm);
    return;
  }
  const CePack& a = blockIdx.z ? pw : px;
  const i64 have = a.count ? (i64)a.count[0] - a.begin : a.rows, rows = have < a.rows ? have : a.rows;
  const i64 r0 = (i64)blockIdx.x * 64;
  const int c0 = (int)blockIdx.y * 64, tid = threadIdx.x;
  float sc = a.scale ? a.scale[0] : 1.f;
  if (a.part && (r0 < rows || blockIdx.x == 0)) {
    float m = 0.f;
    for (int k = tid; k < CE_PARTS; k += 256) m = fmaxf(m, a.part[k]);
    sc = ce_pow2_scale(ce_block_max(m, sm));
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) a.put[0] = sc, a.rput[0] = 1.f / sc;
  }
  if (r0 >= rows || c0 >= (a.same && a.same_k > a.D ? a.same_k : a.D)) return;
  // 8 columns a lane, as many lanes a row as the block has columns for (a power of two)
  const int cols = (a.same && a.same_k > a.D ? a.same_k : a.D) - c0, sh = cols > 32 ? 3 : cols > 16 ? 2 : cols > 8 ? 1 : 0;
  const bool by_one = LOOSE && !a.vec && a.D - c0 >= 16;
  if (by_one) {
    const auto stage = [&](const auto* src) {
      const int c = c0 + (tid & 63);
      float v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const i64 r = r0 + k * 4 + (tid >> 6);
        v[k] = r < rows && c < a.D ? to_f32(src[(a.idx ? (i64)a.idx[a.begin + r] : r) * a.ld + c]) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 16; ++k) tile[k * 4 + (tid >> 6)][tid & 63] = v[k];
    };
    if (a.dtype == FI_F32)
      stage((const float*)a.src);
    else if (a.dtype == FI_BF16)
      stage((const bf16_t*)a.src);
    else
      stage((const f16_t*)a.src);
    __syncthreads();
  }
  for (int e = tid; e < 64 << sh; e += 256) {
    const int er = e >> sh, ec = (e & ((1 << sh) - 1)) * 8;
    const i64 r = r0 + er;
    const int c = c0 + ec, left = r < rows ? a.D - c : 0;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (by_one) {
#pragma unroll
      for (int t = 0; t < 8; ++t) v[t] = tile[er][ec + t];
    } else if (left > 0) {
      const i64 at = (a.idx ? (i64)a.idx[a.begin + r] : r) * a.ld + c;
      if (a.dtype == FI_F32)
        ce_load8((const float*)a.src + at, left, a.vec, v);
      else if (a.dtype == FI_BF16)
        ce_load8((const bf16_t*)a.src + at, left, a.vec, v);
      else
        ce_load8((const f16_t*)a.src + at, left, a.vec, v);
    }
    if (a.round != a.dtype) {
#pragma unroll
      for (int t = 0; t < 8; ++t) v[t] = a.round == FI_BF16 ? (float)(bf16_t)v[t] : (float)(f16_t)v[t];
    }
    if (a.same && r < rows && c < a.same_k) {
      char* row = (char*)a.same + r * a.ld_same * 2;
      if (a.same_kind == 2) {
        nt_store_triple((bf16_t*)row, c, v);
      } else if (a.same_kind == 1) {
        *(uint4*)((f16_t*)row + c) = VecWords<f16_t>::pack(v);
      } else {
        *(uint4*)((bf16_t*)row + c) = VecWords<bf16_t>::pack(v);
      }
    }
    if (a.turned) {
#pragma unroll
      for (int t = 0; t < 8; ++t) tile[er][ec + t] = v[t] * sc;
    }
  }
  if (!a.turned) return;
  __syncthreads();
  for (int e = tid; e < 64 * 8; e += 256) {
    const int r = e >> 3, c = (e & 7) * 8;
    if (c0 + r >= a.D) break;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = tile[c + i][r];
    uint16_t* row = (uint16_t*)a.turned + (i64)(c0 + r) * a.ld_turned;
    if (a.turned_triple)
      nt_store_triple((bf16_t*)row, r0 + c, v);
    else
      *(uint4*)(row + r0 + c) = VecWords<f16_t>::pack(v);
  }
}

// ---- the logits' product --------------------------------------------------------------------------------------------------------------
struct CeLogits {
  const void* x;           // packed rows
  const void* w;           // operand rows [V]
  i64 ldx, ldw;
  int stages, V;
  const float* bias;
  CeSaved s;
  // forward
  float2* part;            // [row][ntj]
  float* zt;
  int ntj;
  // backward: rows [t0, t0 + Tc), classes [v0, v0 + Vc)
  i64 t0, Tc;
  int v0, Vc;
  const float* g;          // row factors
  uint16_t *dl, *dlt;
  i64 ld_dl, ld_dlt;
  float* db;               // [row tile][V] partial column sums, or NULL
  float* db_out;           // or, where one row tile holds every row, the sums themselves
  int db_add;
  const float* rg;
};

// item -> tile, groups of 8 row tiles walking the classes together so that an XCD's workgroups share both operands in its L2
__device__ __forceinline__ bool ce_tile(int nti, int ntj, int& ti, int& tj) {
  const unsigned total = (unsigned)nti * (unsigned)ntj, per = (total + 7) >> 3;
  const unsigned k = blockIdx.x >> 3, t = (blockIdx.x & 7) * per + k;
  if (k >= per || t >= total) return false;
  const unsigned grp = t / (8u * (unsigned)ntj), in = t - grp * 8u * (unsigned)ntj;
  const unsigned gm = (unsigned)nti - grp * 8u < 8u ? (unsigned)nti - grp * 8u : 8u;
  ti = (int)(grp * 8u + in % gm);
  tj = (int)(in / gm);
  return true;
}

// exp(z - m).  The difference comes first: one fma of z, log2 e and -m log2 e would save an operation, but is not zero at z = m -- it is the
// rounding of m log2 e, which overflows the exponential where every class of a lane is ruled out by a bias of -1e10 or less.
__device__ __forceinline__ float ce_exp(float z, float m) { return __builtin_amdgcn_exp2f((z - m) * CE_LOG2E); }

// The bias of a lane's columns: 16-bit operands start from it, triples get it behind their sum (a rounding instead of one per instruction).
template <class Core>
__device__ __forceinline__ void ce_begin(Core& c, const CeLogits& a, int c0) {
  c.clear();
  if (Core::PARTS == 3 || !a.bias) return;
  const int j0 = c0 + Core::col0() + 4 * (Core::lane() >> 4);
#pragma unroll
  for (int j = 0; j < Core::TJ; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float b = j0 + j * 16 + r < a.V ? a.bias[j0 + j * 16 + r] : 0.f;
#pragma unroll
      for (int i = 0; i < Core::TI; ++i) c.acc[i][j][r] = b;
    }
}
template <class Core>
__device__ __forceinline__ void ce_finish(Core& c, const CeLogits& a, int c0) {
  if (Core::PARTS == 3 && a.bias) {
    const int j0 = c0 + Core::col0() + 4 * (Core::lane() >> 4);
#pragma unroll
    for (int j = 0; j < Core::TJ; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float b = j0 + j * 16 + r < a.V ? a.bias[j0 + j * 16 + r] : 0.f;
#pragma unroll
        for (int i = 0; i < Core::TI; ++i) c.acc[i][j][r] += b;
      }
  }
}

template <class Core, typename T>
__global__ __launch_bounds__(Core::THREADS) void ce_fwd_kernel(CeLogits a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int n = a.s.count[0];
  int ti, tj;
  if (!ce_tile((n + Core::BM - 1) / Core::BM, a.ntj, ti, tj)) return;
  const int r0 = ti * Core::BM, c0 = tj * Core::BN;
  Core c;
  ce_begin(c, a, c0);
  c.run((const T*)a.x + (i64)r0 * a.ldx, a.ldx, n - r0, (const T*)a.w + (i64)c0 * a.ldw, a.ldw, a.V - c0, 0, a.stages, smem);
  ce_finish(c, a, c0);
  const int l = Core::lane(), j0 = c0 + Core::col0() + 4 * (l >> 4);
  if (c0 + Core::BN > a.V) {
#pragma unroll
    for (int j = 0; j < Core::TJ; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (j0 + j * 16 + r >= a.V) {
#pragma unroll
          for (int i = 0; i < Core::TI; ++i) c.acc[i][j][r] = -INFINITY;
        }
  }
  // a lane's 4 TJ columns of a row first, each with its own maximum; 4 NWN such pairs per row meet in LDS
  float2* red = (float2*)smem;                                          // [4 NWN][BM]
  const int q0 = (Core::wave() % Core::NWN) * 4 + (l >> 4);
#pragma unroll
  for (int i = 0; i < Core::TI; ++i) {
    const int row = Core::row0() + i * 16 + (l & 15);
    const int lab = r0 + row < n ? a.s.lab[r0 + row] - (c0 + Core::col0()) : -1;
    if ((unsigned)lab < (unsigned)Core::WN) {
#pragma unroll
      for (int j = 0; j < Core::TJ; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (lab == j * 16 + 4 * (l >> 4) + r) a.zt[r0 + row] = c.acc[i][j][r];
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < Core::TJ; ++j)
      m = fmaxf(fmaxf(m, fmaxf(c.acc[i][j][0], c.acc[i][j][1])), fmaxf(c.acc[i][j][2], c.acc[i][j][3]));
    const float safe = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < Core::TJ; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) sum += ce_exp(c.acc[i][j][r], safe);
    red[q0 * Core::BM + row] = make_float2(m, sum);
  }
  __syncthreads();
  for (int row = threadIdx.x; row < Core::BM; row += Core::THREADS) {
    if (r0 + row >= n) continue;
    float m = -INFINITY, sum = 0.f;
#pragma unroll
    for (int q = 0; q < 4 * Core::NWN; ++q) m = fmaxf(m, red[q * Core::BM + row].x);
    const float safe = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int q = 0; q < 4 * Core::NWN; ++q) {
      const float2 o = red[q * Core::BM + row];
      sum += o.y * ce_exp(o.x, safe);
    }
    a.part[(i64)(r0 + row) * a.ntj + tj] = make_float2(m, sum);
  }
}

// joins a row's tiles: LANES lanes per row
template <int LANES>
__global__ __launch_bounds__(256) void ce_rows_kernel(const float2* part, int ntj, const float* zt, CeSaved s, float* rows_out, double* sums, int mean, float* loss) {
  __shared__ double sm[4];
  const int n = s.count[0], sub = threadIdx.x % LANES;
  double acc = 0.0;
  for (i64 r0 = (i64)blockIdx.x * (256 / LANES); r0 < n; r0 += (i64)gridDim.x * (256 / LANES)) {
    const i64 r = r0 + threadIdx.x / LANES;
    float m = -INFINITY;
    double sum = 0.0;
    if (r < n) {
      for (int k = sub; k < ntj; k += LANES) m = fmaxf(m, part[r * ntj + k].x);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    const float safe = m == -INFINITY ? 0.f : m;
    if (r < n) {
      for (int k = sub; k < ntj; k += LANES) {
        const float2 p = part[r * ntj + k];
        sum += (double)(p.y * ce_exp(p.x, safe));
      }
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (r < n && sub == 0) {
      const float loss = (float)((double)(safe - zt[r]) + log(sum));
      s.stat[r] = make_float2(safe, (float)(1.0 / sum));
      if (rows_out) rows_out[s.idx[r]] = loss;
      acc += (double)loss;
    }
  }
  acc = wave_sum(acc);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    acc = sm[0] + sm[1] + sm[2] + sm[3];
    sums[blockIdx.x] = acc;
    if (loss) loss[0] = (float)(mean ? acc / (double)n : acc);          // (a lone workgroup)
  }
}
__global__ __launch_bounds__(256) void ce_loss_kernel(const double* sums, int nsums, const int* count, int mean, float* loss) {
  __shared__ double sm[4];
  double acc = 0.0;
  for (int k = threadIdx.x; k < nsums; k += 256) acc += sums[k];
  acc = wave_sum(acc);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    acc = sm[0] + sm[1] + sm[2] + sm[3];
    loss[0] = (float)(mean ? acc / (double)count[0] : acc);            // (no labelled row: NaN, as fi_ce_finalize)
  }
}

// ---- backward ---------------------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void ce_gmax_kernel(const float* g, const int* idx, const int* count, float* part) {
  __shared__ float sm[4];
  const int n = count[0];
  float m = 0.f;
  for (i64 r = (i64)blockIdx.x * 256 + threadIdx.x; r < n; r += (i64)gridDim.x * 256) {
    const float v = fabsf(g[idx[r]]);
    if (v < INFINITY) m = fmaxf(m, v);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
}
template <class Core>
__device__ __forceinline__ int ce_kpad(int n) { return Core::PARTS == 3 ? (n + 31) & ~31 : (n + 63) & ~63; }
template <class Core>
__device__ __forceinline__ void ce_store_g(uint16_t* row, long k, const float (&v)[8]) {
  if constexpr (Core::PARTS == 3)
    nt_store_triple((bf16_t*)row, k, v);
  else
    *(uint4*)(row + k) = VecWords<f16_t>::pack(v);
}

// G of a piece, in both orientations.  A row of dx is its own factor times what it would be with a factor of one: the rows that dx's product reads are made
// with CE_UNIT in the factor's place, which its epilogue puts right, and only the columns that dW's sum over rows reads carry the factors.
template <class Core, typename T>
__global__ __launch_bounds__(Core::THREADS) void ce_dlogits_kernel(CeLogits a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr float UNIT = Core::PARTS == 3 ? 1.f : CE_UNIT;
  constexpr int SB = Core::BLOCK, EXTRA = Core::NW * NtBlock<SB, SB>::BYTES;
  const i64 left = (i64)a.s.count[0] - a.t0;
  const int n = (int)(left < 0 ? 0 : left < a.Tc ? left : a.Tc);       // rows of this piece
  int ti, tj;
  if (!ce_tile((n + Core::BM - 1) / Core::BM, (a.Vc + Core::BN - 1) / Core::BN, ti, tj)) {
    if (n == 0 && a.db_out && !a.db_add)
      for (i64 v = (i64)blockIdx.x * Core::THREADS + threadIdx.x; v < a.V; v += (i64)gridDim.x * Core::THREADS) a.db_out[v] = 0.f;
    return;
  }
  const int r0 = ti * Core::BM, c0 = tj * Core::BN;
  const i64 rg = a.t0 + r0;
  const int cg = a.v0 + c0;
  Core c;
  ce_begin(c, a, cg);
  c.run((const T*)a.x + rg * a.ldx, a.ldx, n - r0, (const T*)a.w + (i64)cg * a.ldw, a.ldw, a.V - cg, 0, a.stages, smem);
  ce_finish(c, a, cg);
  float4* meta = (float4*)(smem + EXTRA);                               // [BM]: maximum, UNIT / sum, factor, label
  float* fac = (float*)(smem + EXTRA + Core::BM * 16);                  // [BM]: the factors alone, for vectors of rows
  float* colsum = fac + Core::BM;                                      // [BM / WM][BN]
  for (int row = threadIdx.x; row < Core::BM; row += Core::THREADS) {
    float4 m = make_float4(INFINITY, 0.f, 0.f, __int_as_float(-1));    // (rows behind the last one: exp2(-inf) = 0)
    if (r0 + row < n) {
      const float2 st = a.s.stat[rg + row];
      m = make_float4(st.x, UNIT * st.y, a.g[rg + row], __int_as_float(a.s.lab[rg + row]));
    }
    meta[row] = m;
    fac[row] = m.z;
  }
  __syncthreads();
  const int l = Core::lane(), j0 = cg + Core::col0() + 4 * (l >> 4);
  float mine[Core::TI];
#pragma unroll
  for (int i = 0; i < Core::TI; ++i) {
    const float4 m = meta[Core::row0() + i * 16 + (l & 15)];
    mine[i] = m.z;
#pragma unroll
    for (int j = 0; j < Core::TJ; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) c.acc[i][j][r] = ce_exp(c.acc[i][j][r], m.x) * m.y;
    const int lab = __float_as_int(m.w) - (cg + Core::col0());
    if ((unsigned)lab < (unsigned)Core::WN) {
#pragma unroll
      for (int j = 0; j < Core::TJ; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) c.acc[i][j][r] -= lab == j * 16 + 4 * (l >> 4) + r ? UNIT : 0.f;
    }
  }
  if (cg + Core::BN > a.V) {
#pragma unroll
    for (int j = 0; j < Core::TJ; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (j0 + j * 16 + r >= a.V) {
#pragma unroll
          for (int i = 0; i < Core::TI; ++i) c.acc[i][j][r] = 0.f;
        }
  }
  if (a.db || a.db_out) {
#pragma unroll
    for (int j = 0; j < Core::TJ; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < Core::TI; ++i) v += c.acc[i][j][r] * mine[i];
        v = fi_row16_sum(v);
        if ((l & 15) == 0) colsum[(Core::wave() / Core::NWN) * Core::BN + Core::col0() + j * 16 + 4 * (l >> 4) + r] = v;
      }
    __syncthreads();
    for (int j = threadIdx.x; j < Core::BN; j += Core::THREADS) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < Core::BM / Core::WM; ++q) v += colsum[q * Core::BN + j];
      if (cg + j < a.V) {
        if (a.db_out)
          a.db_out[cg + j] = (a.db_add ? a.db_out[cg + j] : 0.f) + v * a.rg[0];
        else
          a.db[(rg / Core::BM) * a.V + cg + j] = v;
      }
    }
  }
  const NtBlock<SB, SB> blk{(float*)(smem + Core::wave() * NtBlock<SB, SB>::BYTES)};
  const int vcols = a.V - a.v0 < a.Vc ? a.V - a.v0 : a.Vc, vpad = ce_kpad<Core>(vcols), npad = ce_kpad<Core>(n);
#pragma unroll
  for (int bi = 0; bi < Core::WM / SB; ++bi)
#pragma unroll
    for (int bj = 0; bj < Core::WN / SB; ++bj) {
      const int gi = r0 + Core::row0() + bi * SB, gj = c0 + Core::col0() + bj * SB;
      blk.put(c, bi, bj, 1.f);
      if (a.dl) {
        blk.template rows<false>([&](int i, int j0, float (&v)[8]) {
          if (gi + i >= n || gj + j0 >= vpad) return;
          ce_store_g<Core>(a.dl + (i64)(gi + i) * a.ld_dl, gj + j0, v);
        });
      }
      if (a.dlt) {
        blk.cols([&](int j, int i0, float (&v)[8]) {
          if (gj + j >= vcols || gi + i0 >= npad) return;
          const float4 lo = *(const float4*)(fac + gi - r0 + i0), hi = *(const float4*)(fac + gi - r0 + i0 + 4);
          v[0] *= lo.x, v[1] *= lo.y, v[2] *= lo.z, v[3] *= lo.w, v[4] *= hi.x, v[5] *= hi.y, v[6] *= hi.z, v[7] *= hi.w;
          ce_store_g<Core>(a.dlt + (i64)(gj + j) * a.ld_dlt, gi + i0, v);
        });
      }
    }
}

// dx (A = G rows, B = W^T rows) or dW (A = G^T rows, B = x^T rows)
struct CeGrad {
  const uint16_t *a, *b;
  i64 lda, ldb;
  int M, N;                // upper bound of the output's rows; columns (D)
  i64 K;                   // upper bound of the contraction (values)
  const int* count;        // labelled rows
  i64 t0, Tc;              // the piece's rows
  int rows_are_tokens;     // dx: M comes from the device; else K does
  int splits, first;       // first piece of the output: store, else add
  float* part;             // [split][M][N] fp32, or NULL: `out` is written straight away
  // the output
  void* out;
  int out_dtype, accumulate, vec;
  i64 ldo;
  const int* idx;          // dx: where a row belongs, else NULL
  const float* rowf;       // dx: the rows' factors, where G was made without them, else NULL
  const float* scal;
  int rscale;              // index of the reciprocal of b's scale, -1: none
};

__device__ __forceinline__ void ce_put(const CeGrad& a, i64 row, int col, const float (&v)[8], int nv) {
  const i64 at = row * a.ldo + col;
  if (a.vec && !a.accumulate) {                                         // (every vector of 8 is whole and 16-byte aligned)
    if (a.out_dtype == FI_F32) {
      float4* p = (float4*)((float*)a.out + at);
      p[0] = make_float4(v[0], v[1], v[2], v[3]);
      p[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *(uint4*)((uint16_t*)a.out + at) = a.out_dtype == FI_BF16 ? VecWords<bf16_t>::pack(v) : VecWords<f16_t>::pack(v);
    }
    return;
  }
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    if (t < nv) {
      if (a.out_dtype == FI_F32)
        ((float*)a.out)[at + t] = a.accumulate ? ((float*)a.out)[at + t] + v[t] : v[t];
      else if (a.out_dtype == FI_BF16)
        ((bf16_t*)a.out)[at + t] = (bf16_t)v[t];
      else
        ((f16_t*)a.out)[at + t] = (f16_t)v[t];
    }
  }
}
__device__ __forceinline__ float ce_row_factor(const CeGrad& a, i64 r) { return a.rowf ? a.rowf[a.t0 + r] : 1.f; }
__device__ __forceinline__ float ce_rscale(const CeGrad& a) { return a.rscale >= 0 ? a.scal[a.rscale] : 1.f; }

template <class Core, typename T>
__global__ __launch_bounds__(Core::THREADS) void ce_grad_kernel(CeGrad a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const i64 left = (i64)a.count[0] - a.t0;
  const int n = (int)(left < 0 ? 0 : left < a.Tc ? left : a.Tc);
  const int M = a.rows_are_tokens ? n : a.M;
  const i64 K = a.rows_are_tokens ? a.K : n;
  const int nti = (M + Core::BM - 1) / Core::BM, ntj = (a.N + Core::BN - 1) / Core::BN;
  int ti, tj;
  if (!ce_tile(nti, ntj * a.splits, ti, tj)) return;
  const int sp = tj / ntj;                                              // (workgroups that run together share a part of the contraction)
  tj -= sp * ntj;
  const int stages = (int)((K + (Core::PARTS == 3 ? 31 : 63)) / (Core::PARTS == 3 ? 32 : 64)), per = (stages + a.splits - 1) / a.splits;
  const int s0 = sp * per < stages ? sp * per : stages, s1 = s0 + per < stages ? s0 + per : stages;
  Core c;
  c.clear();
  c.run((const T*)a.a + (i64)ti * Core::BM * a.lda, a.lda, M - ti * Core::BM, (const T*)a.b + (i64)tj * Core::BN * a.ldb, a.ldb, a.N - tj * Core::BN, s0, s1, smem);
  constexpr int SB = Core::BLOCK;
  const NtBlock<SB, SB> blk{(float*)(smem + Core::wave() * NtBlock<SB, SB>::BYTES)};
  const float rg = a.scal[SC_RG], rb = ce_rscale(a);
#pragma unroll
  for (int bi = 0; bi < Core::WM / SB; ++bi)
#pragma unroll
    for (int bj = 0; bj < Core::WN / SB; ++bj) {
      const int gi = ti * Core::BM + Core::row0() + bi * SB, gj = tj * Core::BN + Core::col0() + bj * SB;
      blk.put(c, bi, bj, 1.f);
      if (a.part ? (a.N & 7) != 0 : !a.vec || a.accumulate) {
        blk.each([&](int i, int j, float v) {
          const int r = gi + i, k = gj + j;
          if (r >= M || k >= a.N) return;
          if (a.part) {
            float* p = a.part + ((i64)sp * a.M + r) * a.N + k;
            *p = a.first ? v : *p + v;
          } else {
            const float one[8] = {v * rg * rb * ce_row_factor(a, r)};
            ce_put(a, a.idx ? (i64)a.idx[a.t0 + r] : (i64)r, k, one, 1);
          }
        });
        continue;
      }
      blk.template rows<false>([&](int i, int j0, float (&v)[8]) {
        const int r = gi + i, k = gj + j0;
        if (r >= M || k >= a.N) return;
        if (a.part) {
          float* p = a.part + ((i64)sp * a.M + r) * a.N + k;
          float4 lo = make_float4(v[0], v[1], v[2], v[3]), hi = make_float4(v[4], v[5], v[6], v[7]);
          if (!a.first) {
            const float4 x = ((const float4*)p)[0], y = ((const float4*)p)[1];
            lo.x += x.x, lo.y += x.y, lo.z += x.z, lo.w += x.w, hi.x += y.x, hi.y += y.y, hi.z += y.z, hi.w += y.w;
          }
          ((float4*)p)[0] = lo, ((float4*)p)[1] = hi;
        } else {
          const float f = ce_row_factor(a, r);
#pragma unroll
          for (int t = 0; t < 8; ++t) v[t] = v[t] * rg * rb * f;
          ce_put(a, a.idx ? (i64)a.idx[a.t0 + r] : (i64)r, k, v, 8);
        }
      });
    }
}

// joins the split parts of an output: SUB lanes per 8 values, each over its share of the parts, then over the lanes -- a fixed order
template <int SUB>
__global__ __launch_bounds__(256) void ce_join_kernel(CeGrad a) {
  const i64 left = (i64)a.count[0] - a.t0;
  const i64 M = a.rows_are_tokens ? (left < 0 ? 0 : left < a.Tc ? left : a.Tc) : a.M;
  const i64 nv = (a.N + 7) / 8, total = M * nv;
  const float rg = a.scal[SC_RG], rb = ce_rscale(a);
  const int sub = threadIdx.x % SUB;
  for (i64 e0 = (i64)blockIdx.x * (256 / SUB); e0 < total; e0 += (i64)gridDim.x * (256 / SUB)) {
    const i64 e = e0 + threadIdx.x / SUB, r = e / nv;
    const int k = (int)(e - r * nv) * 8, n = a.N - k < 8 ? a.N - k : 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (e < total) {
      for (int s = sub; s < a.splits; s += SUB) {
        const float* p = a.part + ((i64)s * a.M + r) * a.N + k;
        if ((a.N & 7) == 0) {
          const float4 x = ((const float4*)p)[0], y = ((const float4*)p)[1];
          v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
        } else {
#pragma unroll
          for (int t = 0; t < 8; ++t)
            if (t < n) v[t] += p[t];
        }
      }
    }
#pragma unroll
    for (int o = SUB / 2; o > 0; o >>= 1)
#pragma unroll
      for (int t = 0; t < 8; ++t) v[t] += __shfl_xor(v[t], o, 64);
    if (e < total && sub == 0) {
      const float f = ce_row_factor(a, r);
#pragma unroll
      for (int t = 0; t < 8; ++t) v[t] = v[t] * rg * rb * f;
      ce_put(a, a.idx ? (i64)a.idx[a.t0 + r] : r, k, v, n);
    }
  }
}

// db: column sums over the row tiles (or over `parts` partial sums), in fp64: 16 columns per workgroup, 64 lanes' worth of row tiles each
__global__ __launch_bounds__(1024) void ce_dbias_kernel(const float* part, int tile, int parts, int V, const int* count, const float* scal, float* db, int accumulate) {
  __shared__ double sm[64][17];
  const int col = threadIdx.x & 15, q = threadIdx.x >> 4, v = blockIdx.x * 16 + col;
  const int nt = parts ? parts : (count[0] + tile - 1) / tile;
  double acc = 0.0;
  if (v < V)
    for (int t = q; t < nt; t += 64) acc += (double)part[(i64)t * V + v];
  sm[q][col] = acc;
  __syncthreads();
  for (int o = 32; o > 0; o >>= 1) {
    if (q < o) sm[q][col] += sm[q + o][col];
    __syncthreads();
  }
  if (q == 0 && v < V) {
    acc = sm[0][col] * (double)scal[SC_RG];
    db[v] = accumulate ? db[v] + (float)acc : (float)acc;
  }
}

// ---- narrow operands: logits and G stay in registers -------------------------------------------------------------------------------------
// With up to 128 features the two gradient products do less work per value of G than writing and reading it costs (2 x 4 bytes against 4 D
// operations), so each makes its own G.  A wave owns 32 rows -- tokens for dx, classes for dW (DW) -- whose operand fragments stay in registers; the
// other side is streamed through LDS in tiles of 64, once as rows [64][K] for the logits and once turned, [D][64], for the product with G.
// G never leaves the lane that made it: the matrix instruction returns 4 consecutive rows of its first operand per lane, so if fragment row i of
// tile j is taken from streamed row 32 (j / 2) + 8 (i / 4) + 4 (j % 2) + i % 4, a lane's results of two tiles are 8 consecutive streamed rows
// -- exactly the fragment that the next product wants from it.  (Pieces of a row are swizzled by (row & 3) | (row / 8 & 1) * 4, which is free of
// bank conflicts under that order.)  The forward pass of such operands streams the classes the same way and keeps each row's running maximum and sum.
// Rows are packed to a multiple of 8 features only; the rest of a stage is masked in the load (its offset lies beyond the resource: zeros).
// Measured: 16384 x 65536 x 128 bf16 dx 584 us, dW 625, forward 351: half the matrix rate, the exponential, scaling and conversion of every value of
// G sharing the issue port with the products; 524288 x 105 x 16 bf16 33, 38 and 29 us.
struct CeFused {
  CeGrad out;
  CeSaved s;
  const void *own, *tile;  // rows in registers, streamed rows: packed operands
  i64 ld_own, ld_tile;
  const uint16_t* turned;  // the streamed side turned, [D][..]
  i64 ld_turned;
  const float4* meta;      // per token: maximum, factor / sum, factor, label
  const float* bias;       // padded to 64 classes (zeros without a bias)
  float* db;               // DW: [split][V] partial sums, or NULL
  float2* part;            // FWD: [row][split] maximum and sum
  float* zt;               // FWD: the label's logit
  int V;
};

__device__ __forceinline__ void ce_put4(const CeGrad& a, i64 row, int col, const float (&v)[4], int nv) {
  const i64 at = row * a.ldo + col;
  if (a.vec && !a.accumulate) {
    if (a.out_dtype == FI_F32)
      *(float4*)((float*)a.out + at) = make_float4(v[0], v[1], v[2], v[3]);
    else
      *(uint2*)((uint16_t*)a.out + at) = a.out_dtype == FI_BF16 ? make_uint2(__builtin_bit_cast(unsigned, bf16x2_t{(bf16_t)v[0], (bf16_t)v[1]}), __builtin_bit_cast(unsigned, bf16x2_t{(bf16_t)v[2], (bf16_t)v[3]}))
                                                                : make_uint2(__builtin_bit_cast(unsigned, f16x2_t{(f16_t)v[0], (f16_t)v[1]}), __builtin_bit_cast(unsigned, f16x2_t{(f16_t)v[2], (f16_t)v[3]}));
    return;
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if (t < nv) {
      if (a.out_dtype == FI_F32)
        ((float*)a.out)[at + t] = a.accumulate ? ((float*)a.out)[at + t] + v[t] : v[t];
      else if (a.out_dtype == FI_BF16)
        ((bf16_t*)a.out)[at + t] = (bf16_t)v[t];
      else
        ((f16_t*)a.out)[at + t] = (f16_t)v[t];
    }
  }
}

enum { CE_DX, CE_DW, CE_FWD };
template <typename T, int KD, int MODE>                                 // KD: 32 features each
__global__ __launch_bounds__(512) void ce_fused_kernel(CeFused a) {
  constexpr bool DW = MODE == CE_DW, FWD = MODE == CE_FWD;
  constexpr int S_BYTES = KD * 4096, T_BYTES = FWD ? 0 : KD * 4096, X_BYTES = 1024, SLOT = S_BYTES + T_BYTES + X_BYTES;   // rows, turned, table or bias
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typedef __attribute__((address_space(3))) char* lds_ptr_t;
  typedef typename DT<T>::frag_t frag_t;
  const unsigned lds0 = (unsigned)(uintptr_t)(lds_ptr_t)smem;
  const int n = a.s.count[0], M = DW ? a.V : n, S = DW ? n : a.V, D = a.out.N, width = (D + 7) & ~7;
  int ti, sp;
  if (!ce_tile((M + 255) / 256, a.out.splits, ti, sp)) return;
  const int tiles = (S + 63) / 64, per = (tiles + a.out.splits - 1) / a.out.splits, t0 = sp * per < tiles ? sp * per : tiles, t1 = t0 + per < tiles ? t0 + per : tiles;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), l = threadIdx.x & 63, lr = l & 15, g = l >> 4;
  const int o0 = ti * 256 + w * 32;

  // DMA: waves 0 .. 3 fetch the rows (8 rows of 128 bytes per instruction), 4 .. 7 the turned ones, wave 0 also the table's 1 KB (the bias' 256 bytes)
  // (forward: all eight the rows)
  constexpr int Q = FWD ? KD / 2 : KD;
  const bool isT = !FWD && w >= 4;
  const int wq = FWD ? w : w & 3;
  unsigned voff[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int id = wq * Q + q;
    if (isT) {
      const int r = id * 8 + (l >> 3);
      voff[q] = (unsigned)(r < D ? r : D - 1) * (unsigned)(a.ld_turned * 2) + (unsigned)(((l & 7) ^ (l >> 3)) * 16);
    } else {
      const int r = (id & 7) * 8 + (l >> 3);
      const int c = (id >> 3) * 64 + ((l & 7) ^ (((l >> 3) & 3) | ((id & 1) << 2))) * 8;
      voff[q] = c < width ? (unsigned)r * (unsigned)(a.ld_tile * 2) + (unsigned)(c * 2) : 0x80000000u;       // (behind a row's end: beyond the resource)
    }
  }
  auto fetch = [&](int t, int slot) {
    const unsigned base = lds0 + (unsigned)(slot * SLOT);
    if (isT) {
      const nt_v4i rs = nt_rsrc(a.turned + (i64)t * 64, ((unsigned long long)(D - 1) * a.ld_turned + 64) * 2);
#pragma unroll
      for (int q = 0; q < Q; ++q) nt_dma16(rs, base + (unsigned)(S_BYTES + (wq * Q + q) * 1024), voff[q], 0u);
    } else {
      // (rows behind the last one lie beyond the resource, which stays below 2^31 bytes: zeros)
      const int rows = S - t * 64 < 64 ? S - t * 64 : 64;
      const nt_v4i rs = nt_rsrc((const T*)a.tile + (i64)t * 64 * a.ld_tile, ((unsigned long long)(rows - 1) * a.ld_tile + width) * 2);
#pragma unroll
      for (int q = 0; q < Q; ++q) nt_dma16(rs, base + (unsigned)((wq * Q + q) * 1024), voff[q], 0u);
      if (w == 0) {
        const nt_v4i rx = DW ? nt_rsrc(a.meta + (i64)t * 64, 1024) : nt_rsrc(a.bias + (i64)t * 64, 256);
        nt_dma16(rx, base + (unsigned)(S_BYTES + T_BYTES), (unsigned)(l * 16), 0u);
      }
    }
  };
  if (t0 < t1) fetch(t0, 0);

  // own rows
  frag_t own[2][KD];
  float mx[2], y[2], gg[2], b[2], cs[2] = {0.f, 0.f};
  int lab[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int o = o0 + i * 16 + lr, oc = o < M ? o : M - 1;
#pragma unroll
    for (int k = 0; k < KD; ++k) own[i][k] = k * 32 + g * 8 < width ? *(const frag_t*)((const T*)a.own + (i64)oc * a.ld_own + k * 32 + g * 8) : frag_t{};
    mx[i] = y[i] = gg[i] = b[i] = 0.f, lab[i] = -1;
    if constexpr (DW) {
      b[i] = a.bias[oc];
    } else if constexpr (FWD) {
      lab[i] = o < M ? a.s.lab[oc] : -1;
      mx[i] = -INFINITY;                                                // the running maximum; y: the running sum
    } else {
      // (dx takes every row's own factor out of the sum: G is made with CE_UNIT in its place, where its label's entry is rounded least)
      const float4 m = a.meta[oc];
      mx[i] = m.x, y[i] = CE_UNIT * a.s.stat[oc].y, gg[i] = CE_UNIT, b[i] = m.z * (1.f / CE_UNIT), lab[i] = __float_as_int(m.w);
    }
  }
  f32x4 acc[2][2 * KD];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int d = 0; d < 2 * KD; ++d) acc[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int t = t0; t < t1; ++t) {
    const int slot = (t - t0) & 1;
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (t + 1 < t1) fetch(t + 1, slot ^ 1);
    if (o0 >= M) continue;                                              // (a wave without rows only fetches)
    const char* const sm = smem + slot * SLOT;
    const float4* const xm = (const float4*)(sm + S_BYTES + T_BYTES);
    f32x4 z[2][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DW) {
#pragma unroll
        for (int i = 0; i < 2; ++i) z[i][j] = f32x4{b[i], b[i], b[i], b[i]};
      } else {
        const float4 c = xm[8 * (j >> 1) + 2 * g + (j & 1)];              // classes 32 (j / 2) + 8 g + 4 (j % 2) ..
#pragma unroll
        for (int i = 0; i < 2; ++i) z[i][j] = f32x4{c.x, c.y, c.z, c.w};
      }
    }
#pragma unroll
    for (int k = 0; k < KD; ++k) {
      if (KD == 2 && k == 1 && width <= 32) break;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 32 * (j >> 1) + 8 * (lr >> 2) + 4 * (j & 1) + (lr & 3), c = (k & 1) * 4 + g;
        const frag_t f = *(const frag_t*)(sm + (k >> 1) * 8192 + r * 128 + ((c ^ ((r & 3) | ((r >> 1) & 4))) * 16));
#pragma unroll
        for (int i = 0; i < 2; ++i) z[i][j] = mfma16(f, own[i][k], z[i][j]);
      }
    }
    if constexpr (FWD) {
      if (t * 64 + 64 > S) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (t * 64 + 32 * (j >> 1) + 8 * g + 4 * (j & 1) + r >= S) z[0][j][r] = z[1][j][r] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = lab[i] - t * 64;
        if ((unsigned)c < 64u) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (c == 32 * (j >> 1) + 8 * g + 4 * (j & 1) + r) a.zt[o0 + i * 16 + lr] = z[i][j][r];
        }
        float top = mx[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) top = fmaxf(fmaxf(top, fmaxf(z[i][j][0], z[i][j][1])), fmaxf(z[i][j][2], z[i][j][3]));
        // (the sum so far is multiplied by exactly one where the maximum stays, however many tiles there are; a tile's own sum first, so that the
        // running one is rounded once per tile)
        const float safe = top == -INFINITY ? 0.f : top, keep = ce_exp(mx[i], safe);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) sum += ce_exp(z[i][j][r], safe);
        mx[i] = top, y[i] = __builtin_fmaf(y[i], keep, sum);
      }
      continue;
    } else if constexpr (DW) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float4 m = xm[32 * (j >> 1) + 8 * g + 4 * (j & 1) + r];
          const int cls = __float_as_int(m.w) - o0 - lr;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float v = ce_exp(z[i][j][r], m.x) * m.y;
            v -= cls == i * 16 ? m.z : 0.f;
            cs[i] += v;
            z[i][j][r] = v;
          }
        }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) z[i][j][r] = ce_exp(z[i][j][r], mx[i]) * y[i];
        const int c = lab[i] - t * 64;
        if ((unsigned)c < 64u) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) z[i][j][r] -= c == 32 * (j >> 1) + 8 * g + 4 * (j & 1) + r ? gg[i] : 0.f;
        }
      }
      if (t * 64 + 64 > S) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (t * 64 + 32 * (j >> 1) + 8 * g + 4 * (j & 1) + r >= S) z[0][j][r] = z[1][j][r] = 0.f;
      }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      f16x8 gf[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) gf[i][e] = (f16_t)z[i][2 * q][e], gf[i][4 + e] = (f16_t)z[i][2 * q + 1][e];
#pragma unroll
      for (int d = 0; d < 2 * KD; ++d) {
        if (KD == 2 && d * 16 >= D) break;
        const int r = d * 16 + lr;
        const f16x8 f = *(const f16x8*)(sm + S_BYTES + r * 128 + (((q * 4 + g) ^ (r & 7)) * 16));
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[i][d] = mfma16(f, gf[i], acc[i][d]);
      }
    }
  }

  if constexpr (FWD) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float m = fmaxf(mx[i], __shfl_xor(mx[i], 16, 64));
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const float safe = m == -INFINITY ? 0.f : m;
      float sum = y[i] * ce_exp(mx[i], safe);
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      const int o = o0 + i * 16 + lr;
      if (g == 0 && o < M) a.part[(i64)o * a.out.splits + sp] = make_float2(m, sum);
    }
    return;
  }
  const float rg = a.out.scal[SC_RG], rb = ce_rscale(a.out);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int o = o0 + i * 16 + lr;
    if constexpr (DW) {
      cs[i] += __shfl_xor(cs[i], 16, 64);
      cs[i] += __shfl_xor(cs[i], 32, 64);
      if (a.db && g == 0 && o < M) a.db[(i64)sp * a.V + o] = cs[i];
      if (!a.out.out) continue;
    }
    if (o >= M) continue;
    if constexpr (!DW) {
#pragma unroll
      for (int d = 0; d < 2 * KD; ++d) acc[i][d] *= b[i];
    }
    const i64 row = a.out.idx ? (i64)a.out.idx[o] : (i64)o;
#pragma unroll
    for (int d = 0; d < 2 * KD; ++d) {
      const int c = d * 16 + 4 * g, nv = D - c < 4 ? D - c : 4;
      if (nv <= 0) continue;
      if (a.out.part) {
        float* p = a.out.part + ((i64)sp * a.out.M + o) * D + c;
        if ((D & 3) == 0) {
          *(float4*)p = make_float4(acc[i][d][0], acc[i][d][1], acc[i][d][2], acc[i][d][3]);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (r < nv) p[r] = acc[i][d][r];
        }
      } else {
        const float v[4] = {acc[i][d][0] * rg * rb, acc[i][d][1] * rg * rb, acc[i][d][2] * rg * rb, acc[i][d][3] * rg * rb};
        ce_put4(a.out, row, c, v, nv);
      }
    }
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------------------
struct Carve {
  char* base;
  i64 at = 0;
  template <typename P>
  P* take(i64 n) {
    P* p = base ? (P*)(base + at) : nullptr;
    at += ce_up(n * (i64)sizeof(P), 256);
    return p;
  }
};

struct CeShape {
  bool triple, fused;
  int tile;                // of the logits' product, see CE_BM
  int ku;                  // values per stage
  int kp;                  // D padded to stages
  int kw;                  // packed rows' width: kp; in the fused form, which masks the rest of a stage, a multiple of 8
  i64 ldx;                 // packed operand rows, elements
  bool w_direct;           // W is used where it lies
  i64 ldw;
  bool scaled;             // scales are computed (fp16 made of bf16)
};
// tiles of the logits' product: 256 x 256, of triples, whose two stages would not fit the LDS, 128 x 256; 64 rows where there are no more (the classes are then
// streamed once, and three quarters of a tall tile would repeat the last row), 128 likewise (122 x 72099 x 1730 bf16: G 126 -> 116 us, forward 105 -> 100); 64
// or 128 classes too
int ce_logits_tile(const FiLinearCe& d, bool triple) { return d.T <= 64 ? 1 : d.V <= 64 ? 2 : d.V <= 128 ? 3 : d.T <= 128 || triple ? 4 : 0; }
constexpr int CE_BM[5] = {256, 64, 256, 256, 128}, CE_BN[5] = {256, 256, 64, 128, 256};

// Logits and G stay in registers (ce_fused_kernel) for 16-bit operands of up to 128 features; rows up to where a turned operand's offsets fit 32 bits
// (forward pass of up to 64 rows: the 64 x 256 tiles of the general product read the classes with more workgroups)
CeShape ce_shape(const FiLinearCe& d, const void* w, bool fwd) {
  CeShape s;
  // Half precision keeps 11 bits, as many as G does: up to 2^28 multiply-adds, where six products cost little more than one, it goes as triples too, and
  // its gradients are rounded once (over 80 sizes, those more than 1.5 times an fp32 product's error off fell from 10 to none)
  s.triple = d.dtype == FI_F32 || (d.dtype == FI_F16 && (double)d.T * d.V * d.D <= (double)(1 << 28));
  s.ku = s.triple ? 32 : 64;
  s.kp = (int)ce_up(d.D, s.ku);
  s.fused = !s.triple && s.kp <= 128 && d.T <= (1 << 23) && !(fwd && d.T <= 64);
  s.tile = ce_logits_tile(d, s.triple);
  s.kw = s.fused ? (int)ce_up(d.D, 8) : s.kp;
  s.ldx = s.triple ? 3L * s.kw : s.kw;
  // 16-bit weights whose rows need no padding and are 16-byte aligned are read in place
  s.w_direct = !s.triple && d.wdtype == d.dtype && d.D == s.kw && d.ldw % 8 == 0 && ((uintptr_t)w & 15) == 0;
  s.ldw = s.w_direct ? d.ldw : s.ldx;
  s.scaled = d.dtype == FI_BF16;
  return s;
}

int ce_check(const FiLinearCe* d) {
  if (!d) return FI_ERR_NULL;
  if (d->dtype != FI_F32 && d->dtype != FI_BF16 && d->dtype != FI_F16) return FI_ERR_DTYPE;
  if (d->wdtype != d->dtype && d->wdtype != FI_F32) return FI_ERR_DTYPE;
  if (d->ltype != FI_LABEL_U8 && d->ltype != FI_LABEL_I32 && d->ltype != FI_LABEL_I64) return FI_ERR_DTYPE;
  if (d->reduction < 0 || d->reduction > 2) return FI_ERR_SHAPE;
  if (d->T < 1 || d->V < 1 || d->D < 1 || d->T >= (1LL << 30) || d->V > (1 << 20) || d->D > (1 << 16)) return FI_ERR_SHAPE;
  if (d->ldx < d->D || d->ldw < d->D || d->ldw > (1 << 22)) return FI_ERR_SHAPE;
  return 0;
}

// (the same tile by 16 waves of 64 x 64 in the forward pass -- four per SIMD hide LDS and DMA latency: 845 -> 757 us at 7370 x 50000 x 1024 -- and by
// 8 of 128 x 64 for G, whose epilogue wants 64 x 64 blocks of scratch: 267 against 290 us a piece of 7370 x 16384)
template <typename T, int PARTS> struct CeCores {
  typedef NtCore<T, PARTS, 64, 256, 64, 32> C1;
  typedef NtCore<T, PARTS, 256, 64, 32, 64> C2;
  typedef NtCore<T, PARTS, 256, 128, 64, 64> C3;
  typedef NtCore<T, PARTS, 128, 256, 64, 64> C4;
};

template <class Core, typename T>
int ce_launch_fwd(const CeLogits& a, i64 T_rows, hipStream_t st) {
  static NtLdsDevices allowed;
  if (!nt_allow_lds((const void*)ce_fwd_kernel<Core, T>, allowed)) return FI_ERR_UNSUPPORTED;
  const i64 n = (T_rows + Core::BM - 1) / Core::BM * a.ntj;
  if (n > (1LL << 30)) return FI_ERR_SHAPE;
  hipLaunchKernelGGL((ce_fwd_kernel<Core, T>), dim3((unsigned)ce_up(n, 8)), dim3(Core::THREADS), Core::LDS, st, a);
  FI_CHECK_LAUNCH();
  return 0;
}
template <class Core, typename T>
int ce_launch_dlogits(const CeLogits& a, hipStream_t st) {
  static NtLdsDevices allowed;
  if (!nt_allow_lds((const void*)ce_dlogits_kernel<Core, T>, allowed)) return FI_ERR_UNSUPPORTED;
  constexpr int SB = Core::BLOCK, SCR = Core::NW * NtBlock<SB, SB>::BYTES;
  constexpr int need = SCR + Core::BM * 20 + Core::BM / Core::WM * Core::BN * 4, lds = need > Core::LDS ? need : Core::LDS;
  const i64 n = (a.Tc + Core::BM - 1) / Core::BM * ((a.Vc + Core::BN - 1) / Core::BN);
  hipLaunchKernelGGL((ce_dlogits_kernel<Core, T>), dim3((unsigned)ce_up(n, 8)), dim3(Core::THREADS), lds, st, a);
  FI_CHECK_LAUNCH();
  return 0;
}
template <typename T, int PARTS>
int ce_logits(const CeLogits& a, i64 T_rows, int tile, bool fwd, hipStream_t st) {
  typedef CeCores<T, PARTS> C;
  switch (tile) {
    case 1: return fwd ? ce_launch_fwd<typename C::C1, T>(a, T_rows, st) : ce_launch_dlogits<typename C::C1, T>(a, st);
    case 2: return fwd ? ce_launch_fwd<typename C::C2, T>(a, T_rows, st) : ce_launch_dlogits<typename C::C2, T>(a, st);
    case 3: return fwd ? ce_launch_fwd<typename C::C3, T>(a, T_rows, st) : ce_launch_dlogits<typename C::C3, T>(a, st);
    case 4: return fwd ? ce_launch_fwd<typename C::C4, T>(a, T_rows, st) : ce_launch_dlogits<typename C::C4, T>(a, st);
  }
  if constexpr (PARTS == 1) return fwd ? ce_launch_fwd<NtCore<T, 1, 256, 256, 64, 64>, T>(a, T_rows, st) : ce_launch_dlogits<NtCore<T, 1, 256, 256, 128, 64>, T>(a, st);
  return FI_ERR_UNSUPPORTED;
}
int ce_logits_any(const CeLogits& a, const FiLinearCe& d, const CeShape& s, bool fwd, hipStream_t st) {
  return s.triple ? ce_logits<bf16_t, 3>(a, d.T, s.tile, fwd, st) : d.dtype == FI_BF16 ? ce_logits<bf16_t, 1>(a, d.T, s.tile, fwd, st) : ce_logits<f16_t, 1>(a, d.T, s.tile, fwd, st);
}

// one or two operands in a launch (src == NULL: none)
int ce_pack(const CePack& x, const CePack& w, hipStream_t st, const CeFactors& f = CeFactors{}) {
  i64 gx = 0;
  int gy = 0;
  for (const CePack* p : {&x, &w}) {
    if (!p->src) continue;
    const int cols = p->same && p->same_k > p->D ? p->same_k : p->D;
    if ((p->rows + 63) / 64 > gx) gx = (p->rows + 63) / 64;
    if ((cols + 63) / 64 > gy) gy = (cols + 63) / 64;
  }
  if (!x.src && !w.src) return 0;
  const bool loose = (x.src && !x.vec) || (w.src && !w.vec);
  hipLaunchKernelGGL(loose ? ce_pack_kernel<true> : ce_pack_kernel<false>, dim3((unsigned)gx, (unsigned)gy, (x.src && w.src ? 2 : 1) + (f.g ? 1 : 0)), dim3(256), 0, st, x.src ? x : w, w, f);
  FI_CHECK_LAUNCH();
  return 0;
}
int ce_vec(const void* p, int dtype, i64 ld) { return ((uintptr_t)p & 15) == 0 && ld % (dtype == FI_F32 ? 4 : 8) == 0; }

int ce_amax(const FiLinearCe& d, const void* x, const void* w, const CeSaved& s, float* parts, hipStream_t st) {
  const CeAmax ax = {x, d.dtype, d.D, ce_vec(x, d.dtype, d.ldx), d.ldx, d.T, s.idx, s.count, parts, 0};
  CeAmax aw = {w, d.wdtype, d.D, ce_vec(w, d.wdtype, d.ldw), d.ldw, d.V, nullptr, nullptr, parts + CE_PARTS, 0};
  if (!aw.vec && d.ldw == d.D && ((uintptr_t)w & 15) == 0) {            // rows of any width that follow one another are as good as rows of 4096
    const i64 total = (i64)d.V * d.D;
    aw.vec = 1, aw.D = 4096, aw.ld = 4096, aw.rows = total / 4096, aw.tail = total % 4096;
  }
  hipLaunchKernelGGL(ce_amax_kernel, dim3(CE_PARTS, 2), dim3(256), 0, st, ax, aw);
  FI_CHECK_LAUNCH();
  return 0;
}

// parts of the streamed side: enough workgroups (of 256 own rows) to fill the chip twice, no fewer than 8 tiles of 64 each
int ce_fused_splits(i64 own, i64 streamed) {
  const i64 wgs = (own + 255) / 256, tiles = (streamed + 63) / 64;
  i64 s = 512 / wgs;
  if (s > tiles / 8) s = tiles / 8;
  if (s > 256) s = 256;
  return s < 1 ? 1 : (int)s;
}
template <typename T, int KD, int MODE>
int ce_launch_fused(const CeFused& a, hipStream_t st) {
  constexpr int lds = 2 * (KD * (MODE == CE_FWD ? 4096 : 8192) + 1024);
  static NtLdsDevices allowed;
  if (!nt_allow_lds((const void*)ce_fused_kernel<T, KD, MODE>, allowed)) return FI_ERR_UNSUPPORTED;
  const i64 n = (i64)((a.out.M + 255) / 256) * a.out.splits;
  hipLaunchKernelGGL((ce_fused_kernel<T, KD, MODE>), dim3((unsigned)ce_up(n, 8)), dim3(512), lds, st, a);
  FI_CHECK_LAUNCH();
  return 0;
}
template <int MODE>
int ce_fused(const CeFused& a, const FiLinearCe& d, int kp, hipStream_t st) {
  if (d.dtype == FI_BF16) return kp <= 64 ? ce_launch_fused<bf16_t, 2, MODE>(a, st) : ce_launch_fused<bf16_t, 4, MODE>(a, st);
  return kp <= 64 ? ce_launch_fused<f16_t, 2, MODE>(a, st) : ce_launch_fused<f16_t, 4, MODE>(a, st);
}

struct CeFwdWs {
  int* cnt;
  float *zt, *bias_pad;
  int nparts;              // of a row's statistics
  uint16_t *xc, *wc;
  float2* part;
  double* sums;
  i64 bytes;
};
CeFwdWs ce_fwd_ws(const FiLinearCe& d, const CeShape& s, void* p) {
  Carve c{(char*)p};
  CeFwdWs w;
  w.cnt = c.take<int>((d.T + CE_ROWS - 1) / CE_ROWS);
  w.zt = c.take<float>(d.T);
  w.sums = c.take<double>(CE_LOSS_WGS);
  w.xc = c.take<uint16_t>(d.T * s.ldx);
  w.wc = s.w_direct ? nullptr : c.take<uint16_t>((i64)d.V * s.ldx);
  const int bn = CE_BN[s.tile];
  w.nparts = s.fused ? ce_fused_splits(d.T, d.V) : (d.V + bn - 1) / bn;
  w.bias_pad = s.fused ? c.take<float>(ce_up(d.V, 64)) : nullptr;
  w.part = c.take<float2>(d.T * w.nparts);
  w.bytes = c.at;
  return w;
}

// scal: NULL, or where the scales are (parts == NULL) or go
CePack ce_pack_x(const FiLinearCe& d, const CeShape& s, const void* x, const CeSaved& sv, const float* parts, float* scal, uint16_t* xc) {
  CePack k = {};
  k.src = x, k.dtype = k.round = d.dtype, k.D = d.D, k.vec = ce_vec(x, d.dtype, d.ldx), k.ld = d.ldx, k.rows = d.T, k.idx = sv.idx, k.count = sv.count;
  if (scal) k.part = parts, k.scale = parts ? nullptr : scal + SC_X, k.put = scal + SC_X, k.rput = scal + SC_RX;
  k.same = xc, k.ld_same = s.ldx, k.same_k = s.kw, k.same_kind = s.triple ? 2 : d.dtype == FI_F16 ? 1 : 0;
  return k;
}
CePack ce_pack_w(const FiLinearCe& d, const CeShape& s, const void* w, const float* parts, float* scal, uint16_t* wc) {
  CePack k = {};
  k.src = w, k.dtype = d.wdtype, k.round = d.dtype, k.D = d.D, k.vec = ce_vec(w, d.wdtype, d.ldw), k.ld = d.ldw, k.rows = d.V;
  if (scal) k.part = parts + CE_PARTS, k.put = scal + SC_W, k.rput = scal + SC_RW;
  k.same = wc, k.ld_same = s.ldx, k.same_k = s.kw, k.same_kind = s.triple ? 2 : d.dtype == FI_F16 ? 1 : 0;
  return k;
}

// ---- the backward pass's plan
struct CeGradPlan {
  int tile, splits;
  bool part;
};
// Output tiles of 256 x 256 (of triples 128 x 256), 128 x 128 or 64 x 64 (columns or rows that few); a contraction is split where the tiles do not fill the chip.
CeGradPlan ce_grad_plan(i64 M, i64 N, i64 K, bool triple, bool pieces) {
  CeGradPlan p;
  const i64 least = M < N ? M : N, bm = triple ? 128 : 256, ku = triple ? 32 : 64;
  p.tile = least > 128 && (M + bm - 1) / bm * ((N + 255) / 256) >= 128 ? 0 : least > 64 ? 1 : 2;
  const i64 tm = p.tile == 0 ? bm : p.tile == 1 ? 128 : 64, tn = p.tile == 0 ? 256 : tm;
  const i64 tiles = (M + tm - 1) / tm * ((N + tn - 1) / tn), stages = (K + ku - 1) / ku;
  i64 s = 512 / tiles;
  if (s > stages / 8) s = stages / 8;
  if (s > 64) s = 64;
  if (stages < 64) s = 1;                        // (the join costs as much)
  if (s < 1) s = 1;
  p.splits = (int)s;
  p.part = p.splits > 1 || pieces;
  return p;
}
struct CeBwdWs {
  float *parts, *scal, *g, *db, *pdx, *pdw, *bias_pad;
  float4* meta;
  int sdx, sdw;
  uint16_t *xc, *wc, *xt, *wt, *dl, *dlt;
  i64 ld_xt, ld_wt, ld_dl, ld_dlt, Tc;
  int Vc;
  CeGradPlan dx, dw;
  i64 pdw_piece, bytes;
};
// values of G held at a time: two orientations of 16 bits, 1 GiB (3 GiB of triples).  Smaller pieces write dx's sums more often: 7370 x 50000 x 1024 takes 3486 us
// with 2^27, 3291 with 2^28, 3235 with 2^29
constexpr i64 CE_PIECE = 1LL << 28;
CeBwdWs ce_bwd_ws(const FiLinearCe& d, const CeShape& s, bool need_dx, bool need_dw, bool need_db, void* p) {
  Carve c{(char*)p};
  CeBwdWs w;
  const int f = s.triple ? 3 : 1;
  const i64 Tp = ce_up(d.T, 256), Vp = ce_up(d.V, 256);
  // a piece: all rows, if 256 classes of them fit, and as many classes as do
  w.Tc = Tp < CE_PIECE / 256 ? Tp : CE_PIECE / 256;
  const i64 vc = CE_PIECE / w.Tc / 256 * 256;
  w.Vc = (int)(vc < Vp ? vc : Vp);
  w.ld_xt = f * w.Tc, w.ld_wt = f * Vp, w.ld_dl = (i64)f * w.Vc, w.ld_dlt = f * w.Tc;
  w.parts = c.take<float>(3 * CE_PARTS);
  w.scal = c.take<float>(SC_N);
  w.g = c.take<float>(d.T);
  w.meta = nullptr, w.bias_pad = nullptr;
  if (s.fused) {
    w.sdx = ce_fused_splits(d.T, d.V), w.sdw = ce_fused_splits(d.V, d.T);
    w.ld_xt = Tp, w.ld_wt = Vp, w.Tc = Tp;
    w.meta = c.take<float4>(ce_up(d.T, 64));
    w.bias_pad = c.take<float>(ce_up(d.V, 64));
    w.db = need_db ? c.take<float>((i64)w.sdw * d.V) : nullptr;
    w.xc = c.take<uint16_t>(d.T * s.ldx);
    w.wc = s.w_direct ? nullptr : c.take<uint16_t>((i64)d.V * s.ldx);
    w.xt = need_dw || need_db ? c.take<uint16_t>(d.D * w.ld_xt) : nullptr;
    w.wt = need_dx ? c.take<uint16_t>(d.D * w.ld_wt) : nullptr;
    w.pdx = need_dx && w.sdx > 1 ? c.take<float>((i64)w.sdx * d.T * d.D) : nullptr;
    w.pdw = need_dw && w.sdw > 1 ? c.take<float>((i64)w.sdw * d.V * d.D) : nullptr;
    w.bytes = c.at;
    return w;
  }
  const int bm = CE_BM[s.tile];
  w.db = need_db ? c.take<float>((d.T + bm - 1) / bm * d.V) : nullptr;
  w.xc = c.take<uint16_t>(d.T * s.ldx);
  w.wc = s.w_direct ? nullptr : c.take<uint16_t>((i64)d.V * s.ldx);
  w.xt = need_dw ? c.take<uint16_t>(d.D * w.ld_xt) : nullptr;
  w.wt = need_dx ? c.take<uint16_t>(d.D * w.ld_wt) : nullptr;
  w.dl = need_dx ? c.take<uint16_t>(w.Tc * w.ld_dl) : nullptr;
  w.dlt = need_dw ? c.take<uint16_t>((i64)w.Vc * w.ld_dlt) : nullptr;
  w.dx = ce_grad_plan(d.T < w.Tc ? d.T : w.Tc, d.D, d.V < w.Vc ? d.V : w.Vc, s.triple, w.Vc < d.V);
  w.dw = ce_grad_plan(d.V < w.Vc ? d.V : w.Vc, d.D, d.T < w.Tc ? d.T : w.Tc, s.triple, w.Tc < d.T);
  w.pdx = need_dx && w.dx.part ? c.take<float>((i64)w.dx.splits * w.Tc * d.D) : nullptr;
  // (dW's sum over several row pieces is kept for every class piece)
  w.pdw_piece = (i64)w.dw.splits * w.Vc * d.D;
  w.pdw = need_dw && w.dw.part ? c.take<float>(w.pdw_piece * (w.Tc < d.T ? (d.V + w.Vc - 1) / w.Vc : 1)) : nullptr;
  w.bytes = c.at;
  return w;
}


template <class Core, typename T>
int ce_launch_grad(const CeGrad& a, hipStream_t st) {
  static NtLdsDevices allowed;
  if (!nt_allow_lds((const void*)ce_grad_kernel<Core, T>, allowed)) return FI_ERR_UNSUPPORTED;
  const i64 n = (i64)((a.M + Core::BM - 1) / Core::BM) * ((a.N + Core::BN - 1) / Core::BN) * a.splits;
  hipLaunchKernelGGL((ce_grad_kernel<Core, T>), dim3((unsigned)ce_up(n, 8)), dim3(Core::THREADS), Core::LDS, st, a);
  FI_CHECK_LAUNCH();
  return 0;
}
int ce_grad(const CeGrad& a, bool triple, int tile, hipStream_t st) {
  if (triple)
    return tile == 0 ? ce_launch_grad<NtCore<bf16_t, 3, 128, 256, 64, 64>, bf16_t>(a, st)
           : tile == 1 ? ce_launch_grad<NtCore<bf16_t, 3, 128, 128, 64, 32, 3>, bf16_t>(a, st)
                       : ce_launch_grad<NtCore<bf16_t, 3, 64, 64, 32, 32, 3>, bf16_t>(a, st);
  return tile == 0 ? ce_launch_grad<NtCore<f16_t, 1, 256, 256, 64, 64>, f16_t>(a, st)
         : tile == 1 ? ce_launch_grad<NtCore<f16_t, 1, 128, 128, 64, 64>, f16_t>(a, st)
                     : ce_launch_grad<NtCore<f16_t, 1, 64, 64, 32, 32, 3>, f16_t>(a, st);
}
int ce_join(const CeGrad& a, hipStream_t st) {
  const int sub = a.splits >= 32 ? 16 : 1;
  const i64 n = ((i64)a.M * ((a.N + 7) / 8) * sub + 255) / 256;
  const unsigned grid = (unsigned)(n < 4096 ? n : 4096);
  if (sub == 16)
    hipLaunchKernelGGL(ce_join_kernel<16>, dim3(grid), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(ce_join_kernel<1>, dim3(grid), dim3(256), 0, st, a);
  FI_CHECK_LAUNCH();
  return 0;
}

}  // namespace

extern "C" long fi_linear_ce_saved(const FiLinearCe* d) {
  const int rc = ce_check(d);
  return rc ? rc : 64 + 4 * ce_up(4 * d->T, 64);
}
extern "C" long fi_linear_ce_fwd_workspace(const FiLinearCe* d, const void* w) {
  const int rc = ce_check(d);
  return rc ? rc : ce_fwd_ws(*d, ce_shape(*d, w, true), nullptr).bytes;
}
extern "C" int fi_linear_ce_fwd(const FiLinearCe* d, const void* x, const void* w, const float* bias, const void* labels, float* loss,
                                void* saved, void* workspace, void* stream) {
  int rc = ce_check(d);
  if (rc) return rc;
  if (!x || !w || !labels || !loss || !saved || !workspace) return FI_ERR_NULL;
  hipStream_t st = (hipStream_t)stream;
  const CeShape s = ce_shape(*d, w, true);
  const CeFwdWs ws = ce_fwd_ws(*d, s, workspace);
  const CeSaved sv = ce_saved(saved, d->T);
  float* const rows_out = d->reduction == 0 ? loss : nullptr;
  const unsigned nb = (unsigned)((d->T + CE_ROWS - 1) / CE_ROWS);
  if (nb > 1) {
    hipLaunchKernelGGL(ce_count_kernel, dim3(nb), dim3(256), 0, st, labels, d->ltype, (i64)d->T, (i64)d->ignore_index, ws.cnt);
    FI_CHECK_LAUNCH();
  }
  const int scanned = nb > CE_SCAN;
  if (scanned) {
    hipLaunchKernelGGL(ce_scan_kernel, dim3(1), dim3(1024), 0, st, ws.cnt, (int)nb);
    FI_CHECK_LAUNCH();
  }
  hipLaunchKernelGGL(ce_gather_kernel, dim3(nb), dim3(256), 0, st, labels, d->ltype, (i64)d->T, (i64)d->ignore_index, d->V, ws.cnt, scanned, sv, ws.zt, rows_out, bias, ws.bias_pad);
  FI_CHECK_LAUNCH();
  if ((rc = ce_pack(ce_pack_x(*d, s, x, sv, nullptr, nullptr, ws.xc), s.w_direct ? CePack{} : ce_pack_w(*d, s, w, nullptr, nullptr, ws.wc), st))) return rc;
  const void* const wop = s.w_direct ? w : (const void*)ws.wc;
  if (s.fused) {
    CeFused a = {};
    a.out.M = (int)d->T, a.out.N = d->D, a.out.splits = ws.nparts, a.s = sv, a.own = ws.xc, a.ld_own = s.ldx, a.tile = wop, a.ld_tile = s.ldw;
    a.bias = ws.bias_pad, a.V = d->V, a.part = ws.part, a.zt = ws.zt;
    if ((rc = ce_fused<CE_FWD>(a, *d, s.kp, st))) return rc;
  } else {
    CeLogits a = {};
    a.x = ws.xc, a.ldx = s.ldx, a.w = wop, a.ldw = s.ldw, a.stages = s.kp / s.ku, a.V = d->V, a.bias = bias;
    a.s = sv, a.part = ws.part, a.zt = ws.zt, a.ntj = ws.nparts;
    if ((rc = ce_logits_any(a, *d, s, true, st))) return rc;
  }
  const int lanes = ws.nparts > 32 ? 64 : ws.nparts > 4 ? 8 : 1;
  i64 g = (d->T * lanes + 255) / 256;
  if (g > CE_LOSS_WGS) g = CE_LOSS_WGS;
  if (g <= (lanes == 1 ? 16 : 2)) g = 1;                                // (short: one workgroup also writes the loss)
  float* const alone = g == 1 && d->reduction != 0 ? loss : nullptr;
  const int mean = d->reduction == 1;
  if (lanes == 64)
    hipLaunchKernelGGL(ce_rows_kernel<64>, dim3((unsigned)g), dim3(256), 0, st, ws.part, ws.nparts, ws.zt, sv, rows_out, ws.sums, mean, alone);
  else if (lanes == 8)
    hipLaunchKernelGGL(ce_rows_kernel<8>, dim3((unsigned)g), dim3(256), 0, st, ws.part, ws.nparts, ws.zt, sv, rows_out, ws.sums, mean, alone);
  else
    hipLaunchKernelGGL(ce_rows_kernel<1>, dim3((unsigned)g), dim3(256), 0, st, ws.part, ws.nparts, ws.zt, sv, rows_out, ws.sums, mean, alone);
  FI_CHECK_LAUNCH();
  if (d->reduction != 0 && !alone) {
    hipLaunchKernelGGL(ce_loss_kernel, dim3(1), dim3(256), 0, st, ws.sums, (int)g, sv.count, mean, loss);
    FI_CHECK_LAUNCH();
  }
  return 0;
}

extern "C" long fi_linear_ce_bwd_workspace(const FiLinearCe* d, const void* w, int need_dx, int need_dw, int need_db) {
  const int rc = ce_check(d);
  return rc ? rc : ce_bwd_ws(*d, ce_shape(*d, w, false), need_dx != 0, need_dw != 0, need_db != 0, nullptr).bytes;
}
extern "C" int fi_linear_ce_bwd(const FiLinearCe* d, const void* x, const void* w, const float* bias, const void* labels, const void* saved,
                                const float* gloss, void* dx, void* dw, int dw_accumulate, float* db, int db_accumulate, void* workspace,
                                void* stream) {
  int rc = ce_check(d);
  if (rc) return rc;
  if (!x || !w || !labels || !saved || !gloss || !workspace) return FI_ERR_NULL;
  if (dw_accumulate && d->wdtype != FI_F32) return FI_ERR_DTYPE;
  if (!dx && !dw && !db) return 0;
  hipStream_t st = (hipStream_t)stream;
  const CeShape s = ce_shape(*d, w, false);
  const CeBwdWs ws = ce_bwd_ws(*d, s, dx != nullptr, dw != nullptr, db != nullptr, workspace);
  const CeSaved sv = ce_saved((void*)saved, d->T);
  float* const scal = s.scaled ? ws.scal : nullptr;
  if (scal && (rc = ce_amax(*d, x, w, sv, ws.parts, st))) return rc;
  CePack px = ce_pack_x(*d, s, x, sv, ws.parts, scal, ws.xc), pw = ce_pack_w(*d, s, w, ws.parts, scal, ws.wc);
  const bool rows_pieces = ws.Tc < d->T;
  if (!rows_pieces) px.turned = ws.xt, px.ld_turned = ws.ld_xt, px.turned_triple = s.triple;
  pw.turned = ws.wt, pw.ld_turned = ws.ld_wt, pw.turned_triple = s.triple;
  if (s.w_direct && !ws.wt) pw.src = nullptr;                           // (its scale is dx's alone)
  if (d->reduction == 0 && !s.triple) {
    hipLaunchKernelGGL(ce_gmax_kernel, dim3(CE_PARTS), dim3(256), 0, st, gloss, sv.idx, sv.count, ws.parts + 2 * CE_PARTS);
    FI_CHECK_LAUNCH();
  }
  const CeFactors fac = {gloss, d->reduction, ws.parts + 2 * CE_PARTS, sv, (int)s.triple, ws.scal, ws.g, ws.meta, bias, ws.bias_pad, labels,
                         d->ltype, d->V, d->T, d->ignore_index, (char*)dx, (i64)d->D * (d->dtype == FI_F32 ? 4 : 2)};
  const bool few = d->T <= 4096;                                        // (a launch less; its workgroups cover every row: 64 of them to a workgroup's 256)
  if ((rc = ce_pack(px, pw, st, few ? fac : CeFactors{}))) return rc;
  if (!few) {
    hipLaunchKernelGGL(ce_factors_kernel, dim3((unsigned)((d->T + 255) / 256)), dim3(256), 0, st, fac);
    FI_CHECK_LAUNCH();
  }
  const int f = s.triple ? 3 : 1;
  CeGrad gx = {}, gw = {};
  gx.a = ws.dl, gx.lda = ws.ld_dl, gx.ldb = ws.ld_wt, gx.N = d->D, gx.count = sv.count, gx.rows_are_tokens = 1;
  gx.splits = ws.dx.splits, gx.out = dx, gx.out_dtype = d->dtype, gx.ldo = d->D, gx.idx = sv.idx, gx.scal = ws.scal, gx.rscale = s.scaled ? SC_RW : -1;
  gw.a = ws.dlt, gw.lda = ws.ld_dlt, gw.ldb = ws.ld_xt, gw.N = d->D, gw.count = sv.count;
  gw.splits = ws.dw.splits, gw.out_dtype = d->wdtype, gw.accumulate = dw_accumulate, gw.ldo = d->D, gw.scal = ws.scal, gw.rscale = s.scaled ? SC_RX : -1;
  if (s.fused) {
    const void* const wop = s.w_direct ? w : (const void*)ws.wc;
    CeFused a = {};
    a.s = sv, a.meta = ws.meta, a.bias = ws.bias_pad, a.V = d->V;
    if (dx) {
      gx.vec = d->D % 4 == 0 && ((uintptr_t)dx & 15) == 0, gx.splits = ws.sdx, gx.part = ws.pdx, gx.M = (int)d->T, gx.Tc = d->T;
      a.out = gx, a.own = ws.xc, a.ld_own = s.ldx, a.tile = wop, a.ld_tile = s.ldw, a.turned = ws.wt, a.ld_turned = ws.ld_wt;
      if ((rc = ce_fused<CE_DX>(a, *d, s.kp, st))) return rc;
      gx.vec = d->D % 8 == 0 && ((uintptr_t)dx & 15) == 0;              // (the join stores 8 at a time)
      if (gx.part && (rc = ce_join(gx, st))) return rc;
    }
    if (dw || db) {
      gw.vec = d->D % 4 == 0 && ((uintptr_t)dw & 15) == 0, gw.splits = ws.sdw, gw.part = ws.pdw, gw.M = d->V, gw.Tc = d->T, gw.out = dw;
      a.out = gw, a.own = wop, a.ld_own = s.ldw, a.tile = ws.xc, a.ld_tile = s.ldx, a.turned = ws.xt, a.ld_turned = ws.ld_xt, a.db = ws.db;
      if ((rc = ce_fused<CE_DW>(a, *d, s.kp, st))) return rc;
      gw.vec = d->D % 8 == 0 && ((uintptr_t)dw & 15) == 0;
      if (gw.part && (rc = ce_join(gw, st))) return rc;
    }
    if (db) {
      hipLaunchKernelGGL(ce_dbias_kernel, dim3((unsigned)((d->V + 15) / 16)), dim3(1024), 0, st, ws.db, 1, ws.sdw, d->V, sv.count, ws.scal, db, db_accumulate);
      FI_CHECK_LAUNCH();
    }
    return 0;
  }
  gx.rowf = ws.g;
  gx.vec = d->D % 8 == 0 && ((uintptr_t)dx & 15) == 0, gw.vec = d->D % 8 == 0 && ((uintptr_t)dw & 15) == 0;
  CeLogits a = {};
  a.x = ws.xc, a.ldx = s.ldx, a.w = s.w_direct ? w : ws.wc, a.ldw = s.ldw, a.stages = s.kp / s.ku, a.V = d->V, a.bias = bias;
  a.s = sv, a.g = ws.g, a.dl = ws.dl, a.dlt = ws.dlt, a.ld_dl = ws.ld_dl, a.ld_dlt = ws.ld_dlt, a.db = ws.db;
  if (db && d->T <= CE_BM[s.tile]) a.db = nullptr, a.db_out = db, a.db_add = db_accumulate, a.rg = ws.scal + SC_RG;
  const int wsize = d->wdtype == FI_F32 ? 4 : 2;
  // the classes innermost: dx of a row piece is complete with its last class piece, dW's parts are joined behind the last row piece
  const i64 nt = (d->T + ws.Tc - 1) / ws.Tc, nv = (d->V + ws.Vc - 1) / ws.Vc;
  for (i64 o = 0; o < nt * nv; ++o) {
    const i64 it = o / nv, iv = o % nv;
    a.t0 = it * ws.Tc, a.Tc = ws.Tc < d->T - a.t0 ? ws.Tc : d->T - a.t0;
    a.v0 = (int)(iv * ws.Vc), a.Vc = ws.Vc < d->V - a.v0 ? ws.Vc : d->V - a.v0;
    if (rows_pieces && dw && iv == 0) {
      CePack pt = ce_pack_x(*d, s, x, sv, nullptr, scal, nullptr);
      pt.begin = a.t0, pt.rows = a.Tc, pt.turned = ws.xt, pt.ld_turned = ws.ld_xt, pt.turned_triple = s.triple;
      if ((rc = ce_pack(pt, CePack{}, st))) return rc;
    }
    if ((rc = ce_logits_any(a, *d, s, false, st))) return rc;
    if (dx) {
      gx.b = ws.wt + (i64)f * a.v0, gx.M = (int)a.Tc, gx.K = a.Vc, gx.t0 = a.t0, gx.Tc = a.Tc, gx.first = iv == 0;
      gx.part = ws.pdx;
      if ((rc = ce_grad(gx, s.triple, ws.dx.tile, st))) return rc;
      if (gx.part && iv == nv - 1 && (rc = ce_join(gx, st))) return rc;
    }
    if (dw) {
      gw.b = ws.xt, gw.M = a.Vc, gw.K = a.Tc, gw.t0 = a.t0, gw.Tc = a.Tc, gw.first = it == 0;
      gw.out = (char*)dw + (i64)a.v0 * d->D * wsize;
      gw.part = ws.pdw ? ws.pdw + (rows_pieces ? iv * ws.pdw_piece : 0) : nullptr;
      if ((rc = ce_grad(gw, s.triple, ws.dw.tile, st))) return rc;
      if (gw.part && it == nt - 1 && (rc = ce_join(gw, st))) return rc;
    }
  }
  if (db && !a.db_out) {
    hipLaunchKernelGGL(ce_dbias_kernel, dim3((unsigned)((d->V + 15) / 16)), dim3(1024), 0, st, ws.db, CE_BM[s.tile], 0, d->V, sv.count, ws.scal, db, db_accumulate);
    FI_CHECK_LAUNCH();
  }
  return 0;
}
