// tileops.hip.h -- element types, matrix-instruction fragments and the swizzled LDS tile shared by the training operators' kernels.
//
// One wave-level product is D[32][32] += A[32][KS] B[KS][32]; the accumulator register q*4 + i of a lane holds row 8q + 4*(lane >> 5) + i of
// column lane & 31.  A fragment is 16 bytes per lane for every element type:
//   fp32      KS = 8   four v_mfma_f32_32x32x2_f32, contraction index 4*(lane >> 5) + j
//   bf16/fp16 KS = 16  one v_mfma_f32_32x32x16, contraction index 8*(lane >> 5) + j
// The contraction order is free as long as both operands agree.  "Row" fragments take 16 consecutive bytes of a tile row (index above);
// "column" fragments and accumulators turned into operands use the order 4*(lane >> 5) + j (j < 4), then KS/2 + 4*(lane >> 5) + j: exactly the
// rows a lane's accumulator registers hold, so a softmax tile becomes the next product's operand without leaving its lane.
#pragma once
#include "common.hip.h"

namespace fdx {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Elem;
template <> struct Elem<float> {
  typedef f32x4 frag;
  static constexpr int KS = 8, VEC = 4;
  static __device__ inline f32x16 mma(frag a, frag b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};
template <> struct Elem<bf16_t> {
  typedef bf16_t frag __attribute__((ext_vector_type(8)));
  static constexpr int KS = 16, VEC = 8;
  static __device__ inline f32x16 mma(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Elem<f16_t> {
  typedef f16_t frag __attribute__((ext_vector_type(8)));
  static constexpr int KS = 16, VEC = 8;
  static __device__ inline f32x16 mma(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// A tile of rows of DH elements in LDS, in chunks of 16 bytes; chunk c of row r sits at chunk c ^ x(r).  x() spreads over the 64 banks
//   * the 16 rows of a row-fragment read (same chunk, consecutive rows), and
//   * for 16-bit elements the 4 rows x 64 bytes of a transposing read, for fp32 the two half-waves' rows r, r + 4 of a column read.
template <typename T, int DH> struct Tile {
  typedef typename Elem<T>::frag frag;
  static constexpr int CPR = DH * (int)sizeof(T) / 16;   // chunks per row: 4 ... 32
  static constexpr int KS = Elem<T>::KS;
  static __device__ inline int swz(int r) {
    if constexpr (sizeof(T) == 2) {
      if constexpr (CPR == 4) return (r >> 2) & 3;
      else if constexpr (CPR == 8) return ((r & 2) << 1) | ((r >> 2) & 3);
      else return ((r & 3) << 2) | ((r >> 2) & 3);
    } else {
      if constexpr (CPR == 8) return (r >> 1) & 7;
      else return ((r & 4) << 1) | ((r & 8) >> 1) | (r & 3);
    }
  }
  static __device__ inline int at(int r, int c) { return r * CPR + (c ^ swz(r)); }   // in chunks

  // LDS byte addresses.  x() takes row bits 0 ... 3 only and a row is a power of two of bytes, so a lane's address is ONE number xored with constants
  // (which chunk) plus constants (which rows): two registers per lane address every fragment of a tile.
  template <typename V> static __device__ inline V lds(unsigned at) { return *reinterpret_cast<__attribute__((address_space(3))) const V*>((size_t)at); }
  // row fragments: rows r0 + (lane & 31), r0 a multiple of 16; chunk 2 * i + (lane >> 5)
  static __device__ inline unsigned row_base(int lane) { return (unsigned)at(lane & 31, lane >> 5) * 16; }
  static __device__ inline frag row(unsigned base, int r0, int i) { return __builtin_bit_cast(frag, lds<u32x4>((base ^ (32 * i)) + r0 * CPR * 16)); }
  // column fragments: rows r0 + (column order above) of columns 32 * m + (lane & 31); r0 a multiple of KS
  static __device__ inline unsigned col_base(int lane) {
    if constexpr (sizeof(T) == 4) return (unsigned)at(4 * (lane >> 5), (lane & 31) >> 2) * 16 + (lane & 3) * 4;
    else return (unsigned)at(4 * (lane >> 5) + ((lane & 15) >> 2), 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) * 16 + (lane & 1) * 8;
  }
  static __device__ inline frag col(unsigned base, int r0, int m) {
    if constexpr (sizeof(T) == 4) {
      frag f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int x = (CPR == 8 ? j >> 1 : j) ^ (r0 & 8 ? 4 : 0);   // x(r0 + 4 * (lane >> 5) + j) ^ x(4 * (lane >> 5))
        f[j] = lds<float>((base ^ (128 * m) ^ (16 * x)) + (r0 + j) * CPR * 16);
      }
      return f;
    } else {
      // ds_read_b64_tr_b16: the 16 lanes of a group read 4 rows x 16 columns (lane i: row i >> 2, columns 4 * (i & 3) ...), lane i receives column i
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(size_t)((base ^ (64 * m)) + r0 * CPR * 16));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(size_t)((base ^ (64 * m) ^ 32) + (r0 + 8) * CPR * 16));   // x(r + 8) = x(r) ^ 2
      return __builtin_bit_cast(frag, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

__device__ inline unsigned lds_of(const void* p) { return (unsigned)(size_t)(__attribute__((address_space(3))) const char*)p; }
// a value the compiler must not precompute from: keeps what is derived from it inside the loop instead of in registers across it
__device__ inline unsigned opaque(unsigned x) {
  asm volatile("" : "+v"(x));
  return x;
}

static __device__ __attribute__((aligned(16))) unsigned g_zero[4];   // where rows that do not exist are read

// TK rows of DH elements from memory straight to LDS (global_load_lds_dwordx4: a wave-instruction lands 64 chunks in a row at a wave-uniform address, so
// the tile's swizzle is applied to the SOURCE address).  No staging registers: that is what lets two workgroups share a CU.  The loads are counted by
// the wait in front of the barrier that publishes the tile (landed()); written as asm because with the builtin in flight the compiler waits for every
// LDS read.  A load has no register output, so nothing can overwrite what is in flight.
template <typename T, int DH, int TK> struct Fill {
  typedef Tile<T, DH> Tl;
  static constexpr int N = TK * Tl::CPR / 256, RPI = 64 / Tl::CPR;   // wave-instructions per wave, rows each covers
  static_assert(N * 256 == TK * Tl::CPR && 64 % Tl::CPR == 0, "whole rows per instruction");
  // rows t0 ... t0 + TK - 1 of `pitch` elements apart; `all`: every one of them exists and a row is DH elements (uniform), else has(row) says so, and chunks
  // from D on are zeros; `part`: which of the four waves that share the tile this one is
  template <typename F> static __device__ inline void issue(uint4* lds, const T* t0, long pitch, int D, bool all, F&& has, int part = (int)threadIdx.x >> 6) {
    const int wave = __builtin_amdgcn_readfirstlane(part), lane = threadIdx.x & 63;
    const unsigned base = (unsigned)(size_t)(__attribute__((address_space(3))) uint4*)lds;
    if (all && pitch * TK * (long)sizeof(T) < (1L << 31)) {
      // one 32-bit lane offset (two where the swizzle alternates from instruction to instruction) on a scalar address: no vector arithmetic per step
      constexpr int V = 4 * RPI % 16 ? 2 : 1;
      const unsigned step = 4 * RPI * (unsigned)pitch * (unsigned)sizeof(T);
      unsigned off[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int row = wave * RPI + lane / Tl::CPR, c = (lane % Tl::CPR) ^ Tl::swz(row + v * 4 * RPI);
        off[v] = (unsigned)row * (unsigned)pitch * (unsigned)sizeof(T) + (unsigned)c * 16u;
      }
      const char* from = reinterpret_cast<const char*>(t0);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const unsigned to = base + (unsigned)(i * 4 + wave) * 1024u;
        unsigned keep;
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\ts_mov_b32 m0, %0"
                     : "=&s"(keep) : "v"(off[i % V]), "s"(to), "s"(from) : "memory");
        from += step;
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = (i * 4 + wave) * RPI + lane / Tl::CPR, c = (lane % Tl::CPR) ^ Tl::swz(row);
      const void* from = has(row) && c * Elem<T>::VEC < D ? static_cast<const void*>(t0 + row * pitch + c * Elem<T>::VEC) : g_zero;
      const unsigned to = base + (unsigned)(i * 4 + wave) * 1024u;
      unsigned keep;
      asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                   : "=&s"(keep) : "v"(from), "s"(to) : "memory");
    }
  }
};
// every wave's loads into LDS have landed, and every wave is done with the tile before
__device__ inline void landed() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// accumulator rows of k-step s (KS rows) as an operand; one rounding to T (half a step of T relative) where T is 16 bits
template <typename T> __device__ inline typename Elem<T>::frag acc_frag(const f32x16& v, int s) {
  typename Elem<T>::frag f;
  constexpr int N = Elem<T>::VEC;
#pragma unroll
  for (int j = 0; j < N; ++j) f[j] = (T)v[s * N + j];
  return f;
}

// ---- scalar loads / stores of a runtime element type (parameters, tails)
enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };
template <typename T> struct DtOf;
template <> struct DtOf<float> { static constexpr int v = DT_F32; };
template <> struct DtOf<bf16_t> { static constexpr int v = DT_BF16; };
template <> struct DtOf<f16_t> { static constexpr int v = DT_F16; };

// makes the handle's device current for an entry point and puts the caller's back
struct DeviceScope {
  int prev = -1;
  hipError_t err;
  explicit DeviceScope(int dev) {
    err = hipGetDevice(&prev);
    if (err != hipSuccess || prev == dev) prev = -1;   // nothing to put back
    else err = hipSetDevice(dev);
  }
  ~DeviceScope() { if (prev >= 0) (void)hipSetDevice(prev); }
};

template <typename Args> inline hipError_t launch(void (*k)(Args), unsigned grid, unsigned block, const Args& a, hipStream_t s) {
  Args copy = a;
  void* argv[] = {&copy};
  return hipLaunchKernel(reinterpret_cast<const void*>(k), dim3(grid), dim3(block), argv, 0, s);
}

}  // namespace fdx
