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
  static __device__ inline frag row(const uint4* t, int r, int c) {
    return __builtin_bit_cast(frag, t[at(r, c)]);
  }
  // rows r0 + (column order above) of columns 32 * m + (lane & 31); r0 a multiple of KS
  static __device__ inline frag col(const uint4* t, int r0, int m, int lane) {
    const int hi = lane >> 5;
    if constexpr (sizeof(T) == 4) {
      frag f;
      const int c = lane & 31;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = r0 + 4 * hi + j;
        f[j] = reinterpret_cast<const float*>(t)[at(r, 8 * m + (c >> 2)) * 4 + (c & 3)];
      }
      return f;
    } else {
      // ds_read_b64_tr_b16: the 16 lanes of a group read 4 rows x 16 columns (lane i: row i >> 2, columns 4 * (i & 3) ...), lane i receives column i
      const int c = 4 * m + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      const int ra = r0 + 4 * hi + ((lane & 15) >> 2), rb = ra + 8;
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const char* p = reinterpret_cast<const char*>(t);
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + at(ra, c) * 16 + (lane & 1) * 8));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + at(rb, c) * 16 + (lane & 1) * 8));
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      const s16x8 v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(frag, v);
    }
  }
};

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
