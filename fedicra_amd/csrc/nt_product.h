// The matrix-pipe product core behind newton_schulz.hip and linear_ce.hip:  C[i][j] = sum_k A[i][k] * B[j][k], both operands with
// their contraction index contiguous ("NT"), 16-bit storage, fp32 accumulation (v_mfma_f32_16x16x32).
//
// Operands come in one of three forms, by the number of 16-bit PARTS of a value:
//   1  rows of 16-bit values, a multiple of 64 per row (the tail is zero);
//   2  (pairs) every value as the sum of two fp16 (22 significant bits): per 32 values of a row 64 bytes of high parts, then 64 bytes of
//      low parts.  Three products hi*hi + hi*lo + lo*hi give what an fp32 product gives up to 2^-22 per term, at a third of the
//      16-bit matrix rate -- three times what fp32 products reach (1430 / 3 against 154 TFLOP/s at 8192 cubed) -- and one LDS fragment serves two products.
//      For values of one size: fp16 has no exponents below 2^-24, so what is 2^-17 of the largest has lost bits;
//   3  (triples) every fp32 value exactly, as the sum of three bf16, which have fp32's exponents: 64 bytes each of first, second and third parts.  Six products
//      leave out what is below 2^-23 of a term, at a sixth of the 16-bit matrix rate.  (The matrix pipe takes a part below 2^-126 as zero: values below 2^-110, 8e-34, lose
//      their last bits.)
// 128 bytes of a row are one STAGE of the contraction, of triples 192 (64 values, 32, 32).
//
// A workgroup owns a BM x BN tile, a wave WM x WN of it.  Stages are brought into an LDS ring of SLOTS by LDS-DMA (16 bytes per lane, 8 rows
// of 128 bytes per instruction); 16-byte piece c of row r lies at piece c ^ (r & 7), the swizzle being applied to the source address
// because the LDS side of the instruction is linear: the eight lanes a ds_read_b128 serves per clock then touch all 32 banks once.  Triples' third parts
// lie behind, 16 rows of 64 bytes per instruction, piece c of row r at c ^ (r / 2 & 3).
#pragma once
#include <atomic>

#include "common.h"

typedef int nt_v4i __attribute__((ext_vector_type(4)));

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// lane L's 16 bytes at resource offset voff + soff go to LDS[lds_addr + 16 L]; zeros beyond the resource.  (s_nop: M0 is read by the
// load, and an LDS-DMA needs a wait state behind a scalar write of M0.)
__device__ __forceinline__ void nt_dma16(nt_v4i rsrc, unsigned lds_addr, unsigned voff, unsigned soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds_addr), "v"(voff), "s"(rsrc), "s"(soff)
               : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ nt_v4i nt_rsrc(const void* ptr, unsigned long long bytes) {
  const unsigned long long p = (unsigned long long)ptr;
  const unsigned n = bytes > 0xffffffffull ? 0xffffffffu : (unsigned)bytes;
  return nt_v4i{__builtin_amdgcn_readfirstlane((int)(unsigned)p), __builtin_amdgcn_readfirstlane((int)((unsigned)(p >> 32) & 0xffffu)),
                __builtin_amdgcn_readfirstlane((int)n), 0x00020000};
}
// more than 64 KB of dynamic LDS per workgroup has to be allowed per kernel and device (a CU has 160 KB); `done`: a bit per device, one object per kernel
typedef std::atomic<unsigned long long> NtLdsDevices;
static inline bool nt_allow_lds(const void* kernel, NtLdsDevices& done) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return false;
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return true;
  if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess) return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}
// orders this wave's LDS traffic: what other lanes of the wave wrote before is there after
__device__ __forceinline__ void nt_wave_lds_fence() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// SLOTS: two where two stages fill the LDS or several workgroups share a CU; more where a lone workgroup would wait for each stage's latency.
// APART (pairs): they also take lo * lo, and what has a low part is summed in accumulators of its own: the matrix pipe rounds an accumulator at every
// instruction, and small matrices are held to an fp32 sum's few roundings (orthogonalised matrices of 17 .. 31 rows are 1.1e-6 of the result off without,
// 8.5e-7 with, 1.2e-6 by fp32 products).  A third more matrix instructions; long sums have no need of it.  Triples always keep theirs apart, for no more
// instructions: a loss's fp32 gradients are 2e-7 off on average, 3.5e-7 in one accumulator, 6e-7 by fp32 products (4001 x 8003 x 384: 156 us, 144 in one).
template <typename T, int PARTS_, int BM_, int BN_, int WM_, int WN_, int SLOTS_ = 2, bool APART_ = false>
struct NtCore {
  static constexpr int PARTS = PARTS_, BM = BM_, BN = BN_, WM = WM_, WN = WN_, SLOTS = SLOTS_;
  static constexpr int NWN = BN / WN, NW = (BM / WM) * NWN, THREADS = NW * 64;
  static constexpr int TI = WM / 16, TJ = WN / 16;
  static constexpr int ROW = PARTS == 3 ? 192 : 128;              // bytes of a row per stage
  static constexpr int STAGE = (BM + BN) * ROW, LDS = SLOTS * STAGE;
  static_assert(LDS <= 160 * 1024, "LDS");
  // side of the blocks a wave stores its results by (NtBlock): its scratch lies in the ring
  static constexpr int BLOCK = WM >= 64 && WN >= 64 && NW * 64 * 64 * 4 <= LDS ? 64 : 32;
  static_assert(WM % BLOCK == 0 && WN % BLOCK == 0 && NW * BLOCK * BLOCK * 4 <= LDS, "scratch");
  static constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW;       // DMA instructions of a wave per stage: 8 rows of A, of B
  static_assert(PA * NW * 8 == BM && PB * NW * 8 == BN, "whole DMA instructions for every wave");
  static constexpr int P3 = PARTS == 3 ? ((BM + BN) / 16 + NW - 1) / NW : 0;     // and for 16 rows' third parts, A's before B's
  static_assert(SLOTS == 2 || P3 * NW * 16 == (PARTS == 3 ? BM + BN : 0), "the waits count the same loads in every wave");
  static constexpr bool APART = PARTS == 3 || PARTS == 2 && APART_;
  typedef typename DT<T>::frag_t frag_t;

  f32x4 acc[TI][TJ];

  // lane's coordinates inside the tile: row of acc[ti][..] is row0() + ti * 16 + lane % 16, columns of acc[..][tj][r] are
  // col0() + tj * 16 + 4 * (lane / 16) + r  (the fragments are handed to the matrix instruction in the order that puts four consecutive columns
  // of one row into a lane: row statistics stay mostly inside a lane, stores go out in vectors)
  static __device__ __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }
  static __device__ __forceinline__ int lane() { return (int)(threadIdx.x & 63); }
  static __device__ __forceinline__ int row0(int w) { return (w / NWN) * WM; }
  static __device__ __forceinline__ int col0(int w) { return (w % NWN) * WN; }
  static __device__ __forceinline__ int row0() { return row0(wave()); }
  static __device__ __forceinline__ int col0() { return col0(wave()); }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Adds the product to acc.  a, b: first row of the tile (ld in elements, rowsA / rowsB >= 1 valid rows from there: the rest of the tile repeats the last one and
  // its results mean nothing); stages [s0, s1) of the contraction.  BM * ld * sizeof(T) < 2^32 (the callers check).
  __device__ __forceinline__ void run(const T* a, long lda, int rowsA, const T* b, long ldb, int rowsB, int s0, int s1, char* smem) {
    typedef __attribute__((address_space(3))) char* lds_ptr_t;
    const unsigned lds0 = (unsigned)(uintptr_t)(lds_ptr_t)smem;
    const int w = wave(), l = lane();
    // (the resources end with the operands' last byte in use: nothing behind them is ever fetched)
    const nt_v4i ra = nt_rsrc(a, (unsigned long long)(rowsA - 1) * lda * 2 + (unsigned long long)s1 * ROW);
    const nt_v4i rb = nt_rsrc(b, (unsigned long long)(rowsB - 1) * ldb * 2 + (unsigned long long)s1 * ROW);
    const unsigned piece = (unsigned)(((l & 7) ^ (l >> 3)) * 16);
    unsigned va[PA], vb[PB];
#pragma unroll
    for (int q = 0; q < PA; ++q) {
      int r = (w * PA + q) * 8 + (l >> 3);
      va[q] = (unsigned)(r < rowsA ? r : rowsA - 1) * (unsigned)(lda * 2) + piece;
    }
#pragma unroll
    for (int q = 0; q < PB; ++q) {
      int r = (w * PB + q) * 8 + (l >> 3);
      vb[q] = (unsigned)(r < rowsB ? r : rowsB - 1) * (unsigned)(ldb * 2) + piece;
    }
    const unsigned la = lds0 + (unsigned)(w * PA * 1024), lb = lds0 + (unsigned)(BM * 128 + w * PB * 1024);
    unsigned vc[P3 ? P3 : 1];
#pragma unroll
    for (int q = 0; q < P3; ++q) {
      const int r = (w * P3 + q) * 16 + (l >> 2), piece3 = 128 + ((l & 3) ^ ((r >> 1) & 3)) * 16;
      vc[q] = r < BM ? (unsigned)(r < rowsA ? r : rowsA - 1) * (unsigned)(lda * 2) + piece3 : (unsigned)(r - BM < rowsB ? r - BM : rowsB - 1) * (unsigned)(ldb * 2) + piece3;
    }
    // (a stage behind the last one is asked for through an empty resource: zeros, no traffic, and every step counts the same loads)
    const int endA = ra[2], endB = rb[2];
    auto fetch = [&](int s, int slot) {
      nt_v4i xa = ra, xb = rb;
      xa[2] = s < s1 ? endA : 0;
      xb[2] = s < s1 ? endB : 0;
#pragma unroll
      for (int q = 0; q < PA; ++q) nt_dma16(xa, la + (unsigned)(slot * STAGE + q * 1024), va[q], (unsigned)s * ROW);
#pragma unroll
      for (int q = 0; q < PB; ++q) nt_dma16(xb, lb + (unsigned)(slot * STAGE + q * 1024), vb[q], (unsigned)s * ROW);
#pragma unroll
      for (int q = 0; q < P3; ++q) {
        const int r = (w * P3 + q) * 16;                                // (the same in all lanes)
        if (r < BM)
          nt_dma16(xa, lds0 + (unsigned)(slot * STAGE + (BM + BN) * 128 + r * 64), vc[q], (unsigned)s * ROW);
        else if (r < BM + BN)
          nt_dma16(xb, lds0 + (unsigned)(slot * STAGE + (BM + BN) * 128 + r * 64), vc[q], (unsigned)s * ROW);
      }
    };
    const int sw = l & 7, g = l >> 4, lr = l & 15;
    const int oa = (row0() + lr) * 128, ob = BM * 128 + (col0() + lr) * 128;
    const int p0 = ((g) ^ sw) * 16, p1 = ((4 + g) ^ sw) * 16;
    // (from oa / ob to the third parts of the same row: 64 bytes a row there)
    const int p2 = (g ^ ((l >> 1) & 3)) * 16, oa3 = (BM + BN) * 128 + (row0() + lr) * 64 + p2, ob3 = (BM + BN) * 128 + (BM + col0() + lr) * 64 + p2;

    if (s0 < s1) {
#pragma unroll
      for (int k = 0; k < SLOTS - 1; ++k) fetch(s0 + k, k);
    }
    constexpr int LI = APART ? TI : 1, LJ = APART ? TJ : 1;
    f32x4 low[LI][LJ];
#pragma unroll
    for (int i = 0; i < LI; ++i)
#pragma unroll
      for (int j = 0; j < LJ; ++j) low[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    int cur = 0, free = SLOTS - 1;                                      // slots of stage s and of the one before it
    for (int s = s0; s < s1; ++s) {
      // stage s is there for every wave, and every wave has read the one before it
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((SLOTS - 2) * (PA + PB + P3)) : "memory");
      fetch(s + SLOTS - 1, free);
      const char* sa = smem + cur * STAGE + oa;
      const char* sb = smem + cur * STAGE + ob;
      if constexpr (PARTS == 3) {
        const char* sa3 = smem + cur * STAGE + oa3;
        const char* sb3 = smem + cur * STAGE + ob3;
        frag_t b0[TJ], b1[TJ], b2[TJ];
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
          b0[j] = *(const frag_t*)(sb + j * 2048 + p0);
          b1[j] = *(const frag_t*)(sb + j * 2048 + p1);
          b2[j] = *(const frag_t*)(sb3 + j * 1024);
        }
        frag_t a0[2], a1[2], a2[2];
        a0[0] = *(const frag_t*)(sa + p0);
        a1[0] = *(const frag_t*)(sa + p1);
        a2[0] = *(const frag_t*)sa3;
#pragma unroll
        for (int i = 0; i < TI; ++i) {
          const int u = i & 1;
          if (i + 1 < TI) {
            a0[u ^ 1] = *(const frag_t*)(sa + (i + 1) * 2048 + p0);
            a1[u ^ 1] = *(const frag_t*)(sa + (i + 1) * 2048 + p1);
            a2[u ^ 1] = *(const frag_t*)(sa3 + (i + 1) * 1024);
          }
          __builtin_amdgcn_sched_barrier(0);
          // (the smallest first)
#pragma unroll
          for (int j = 0; j < TJ; ++j) low[i % LI][j % LJ] = mfma16(b0[j], a2[u], low[i % LI][j % LJ]);
#pragma unroll
          for (int j = 0; j < TJ; ++j) low[i % LI][j % LJ] = mfma16(b2[j], a0[u], low[i % LI][j % LJ]);
#pragma unroll
          for (int j = 0; j < TJ; ++j) low[i % LI][j % LJ] = mfma16(b1[j], a1[u], low[i % LI][j % LJ]);
#pragma unroll
          for (int j = 0; j < TJ; ++j) low[i % LI][j % LJ] = mfma16(b0[j], a1[u], low[i % LI][j % LJ]);
#pragma unroll
          for (int j = 0; j < TJ; ++j) low[i % LI][j % LJ] = mfma16(b1[j], a0[u], low[i % LI][j % LJ]);
#pragma unroll
          for (int j = 0; j < TJ; ++j) acc[i][j] = mfma16(b0[j], a0[u], acc[i][j]);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else if constexpr (PARTS == 2) {
        frag_t bh[TJ], bl[TJ];
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
          bh[j] = *(const frag_t*)(sb + j * 2048 + p0);
          bl[j] = *(const frag_t*)(sb + j * 2048 + p1);
        }
        // (the next 16 rows' fragments are under way while these are multiplied)
        frag_t ah[2], al[2];
        ah[0] = *(const frag_t*)(sa + p0);
        al[0] = *(const frag_t*)(sa + p1);
#pragma unroll
        for (int i = 0; i < TI; ++i) {
          const int u = i & 1;
          if (i + 1 < TI) {
            ah[u ^ 1] = *(const frag_t*)(sa + (i + 1) * 2048 + p0);
            al[u ^ 1] = *(const frag_t*)(sa + (i + 1) * 2048 + p1);
          }
          __builtin_amdgcn_sched_barrier(0);
          if constexpr (APART) {
#pragma unroll
            for (int j = 0; j < TJ; ++j) low[i][j] = mfma16(bl[j], al[u], low[i][j]);
          }
#pragma unroll
          for (int j = 0; j < TJ; ++j) (APART ? low[i % LI][j % LJ] : acc[i][j]) = mfma16(bh[j], al[u], APART ? low[i % LI][j % LJ] : acc[i][j]);
#pragma unroll
          for (int j = 0; j < TJ; ++j) (APART ? low[i % LI][j % LJ] : acc[i][j]) = mfma16(bl[j], ah[u], APART ? low[i % LI][j % LJ] : acc[i][j]);
#pragma unroll
          for (int j = 0; j < TJ; ++j) acc[i][j] = mfma16(bh[j], ah[u], acc[i][j]);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          const int p = kk ? p1 : p0;
          frag_t bf[TJ];
#pragma unroll
          for (int j = 0; j < TJ; ++j) bf[j] = *(const frag_t*)(sb + j * 2048 + p);
#pragma unroll
          for (int i = 0; i < TI; ++i) {
            const frag_t af = *(const frag_t*)(sa + i * 2048 + p);
#pragma unroll
            for (int j = 0; j < TJ; ++j) acc[i][j] = mfma16(bf[j], af, acc[i][j]);
          }
        }
      }
      free = cur;
      cur = cur + 1 < SLOTS ? cur + 1 : 0;
    }
    if constexpr (APART) {
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] += low[i][j];
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");      // the ring is free: epilogues use it as scratch
  }
};

// ---- storing a tile in both orientations ------------------------------------------------------------------------------------------
// A wave takes a block of its fp32 results through its own LDS scratch (no workgroup barrier) and stores it as rows of 8-value vectors,
// row-major and / or transposed.  Scratch word of (i, j): the 8-column group is swizzled by the row inside its 8-row group and by that group, so
// that the accumulators' writes (ds_write_b128, lanes over 16 rows), row reads (2 x ds_read_b128) and column reads (8 x ds_read_b32, lanes over
// 8 columns x 8 row groups) all spread over the banks.
template <int SI, int SJ>
struct NtBlock {
  static constexpr int BYTES = SI * SJ * 4;
  float* s;
  __device__ __forceinline__ float* at(int i, int j) const { return s + i * SJ + (j ^ ((((i >> 3) ^ i) << 3) & (SJ - 1))); }
  // the wave's accumulators of block (bi, bj), times `by`
  template <class Core>
  __device__ __forceinline__ void put(const Core& c, int bi, int bj, float by) const {
    const int l = threadIdx.x & 63;
    nt_wave_lds_fence();
#pragma unroll
    for (int i = 0; i < SI / 16; ++i)
#pragma unroll
      for (int j = 0; j < SJ / 16; ++j) {
        const f32x4 v = c.acc[bi * (SI / 16) + i][bj * (SJ / 16) + j];
        *(float4*)at(i * 16 + (l & 15), j * 16 + 4 * (l >> 4)) = make_float4(v[0] * by, v[1] * by, v[2] * by, v[3] * by);
      }
    nt_wave_lds_fence();
  }
  // f(i, j0, v): 8 values of row i from column j0 on; what it leaves in v is written back if KEEP
  template <bool KEEP, class F>
  __device__ __forceinline__ void rows(F f) const {
    constexpr int PL = SJ / 8, RP = 64 / PL;
    const int l = threadIdx.x & 63, j0 = (l % PL) * 8;
#pragma unroll
    for (int i0 = 0; i0 < SI; i0 += RP) {
      const int i = i0 + l / PL;
      float v[8];
      float4* p = (float4*)at(i, j0);
      const float4 x = p[0], y = p[1];
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
      f(i, j0, v);
      if constexpr (KEEP) {
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    }
  }
  // f(i, j, v): a value per lane, along the rows: for rows that vectors do not fit
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    const int l = threadIdx.x & 63;
#pragma unroll 8
    for (int e = l; e < SI * SJ; e += 64) f(e / SJ, e % SJ, *at(e / SJ, e % SJ));
  }
  // f(j, i0, v): 8 values of column j from row i0 on
  template <class F>
  __device__ __forceinline__ void cols(F f) const {
    constexpr int PL = SI / 8, CP = 64 / PL;
    const int l = threadIdx.x & 63, i0 = (l % PL) * 8;
#pragma unroll
    for (int jb = 0; jb < SJ; jb += CP) {
      const int j = jb + l / PL;
      float v[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) v[t] = *at(i0 + t, j);
      f(j, i0, v);
    }
  }
};

// the value as it is: where it is a product, its parts must all come of one rounded number.  (The compiler otherwise takes a high part from the rounded
// product to be stored and from the exact one, by v_fma_mixlo_f16, to be subtracted: at a tie these differ by a step of fp16, and the low part is lost.)
__device__ __forceinline__ float nt_fixed(float v) {
  asm("" : "+v"(v));
  return v;
}
// 8 values -> high and low fp16 parts (value = hi + lo up to 2^-22 of it)
__device__ __forceinline__ void nt_split8(const float (&v)[8], uint4& hi, uint4& lo) {
  unsigned h[4], q[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const float x = nt_fixed(v[2 * t]), y = nt_fixed(v[2 * t + 1]);
    f16x2_t a, b;
    a[0] = (f16_t)x, a[1] = (f16_t)y;
    b[0] = (f16_t)(x - (float)a[0]), b[1] = (f16_t)(y - (float)a[1]);
    h[t] = __builtin_bit_cast(unsigned, a), q[t] = __builtin_bit_cast(unsigned, b);
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(q[0], q[1], q[2], q[3]);
}
// element offset of value k (a multiple of 8) inside a pair row; its low part lies 32 elements further
__device__ __forceinline__ long nt_pair_at(long k) { return ((k >> 5) << 6) + (k & 31); }
__device__ __forceinline__ void nt_store_pair(f16_t* row, long k, const float (&v)[8]) {
  uint4 hi, lo;
  nt_split8(v, hi, lo);
  f16_t* p = row + nt_pair_at(k);
  *(uint4*)p = hi;
  *(uint4*)(p + 32) = lo;
}
__device__ __forceinline__ void nt_load_pair(const f16_t* row, long k, float (&v)[8]) {
  const f16_t* p = row + nt_pair_at(k);
  const uint4 hi = *(const uint4*)p, lo = *(const uint4*)(p + 32);
  float a[8], b[8];
  VecWords<f16_t>::unpack(hi, a);
  VecWords<f16_t>::unpack(lo, b);
#pragma unroll
  for (int t = 0; t < 8; ++t) v[t] = a[t] + b[t];
}

// 8 fp32 values -> three bf16 parts, exactly: the first within half its step of 2^-8, so that 16 bits are left for the others.  (Next to fp32's largest
// bf16 would round up to infinity: the first part ends at its own largest.  NaN and infinities come out as NaN.)
__device__ __forceinline__ void nt_store_triple(bf16_t* row, long k, const float (&v)[8]) {           // k: a multiple of 8
  float a[8], b[8], c[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const float x = nt_fixed(v[t]);
    a[t] = (float)(bf16_t)__builtin_amdgcn_fmed3f(x, -0x1.fep127f, 0x1.fep127f);
    const float r = x - a[t];
    b[t] = (float)(bf16_t)r;
    c[t] = r - b[t];
  }
  bf16_t* p = row + (k >> 5) * 96 + (k & 31);
  *(uint4*)p = VecWords<bf16_t>::pack(a);
  *(uint4*)(p + 32) = VecWords<bf16_t>::pack(b);
  *(uint4*)(p + 64) = VecWords<bf16_t>::pack(c);
}

// Workgroups are handed to the eight XCDs in turn (id % 8): this maps a launch of `n` work items (grid rounded up to a multiple of 8) so that each
// XCD's L2 sees one contiguous run of items.  Returns an item, or -1 for the rounding's surplus.
__device__ __forceinline__ int nt_xcd_item(int bid, int grid, int n) {
  const int per = grid >> 3, t = (bid & 7) * per + (bid >> 3);
  return t < n ? t : -1;
}
