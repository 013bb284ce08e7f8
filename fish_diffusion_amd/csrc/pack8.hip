// pack8.hip -- activations kept in 8 bits for the backward pass, and the gradients taken straight from them (fdx_pack8 ... fdx_gelu8_*).
//
// Format: groups of 32 channels of a row share one power of two, 2^(e - 127), e the smallest integer >= 1 with max|x| <= 127 * 2^(e - 127);
// code = x / 2^(e - 127) rounded to nearest even, -127 ... 127.  The step is at most 2/127 of the group's largest value, the error half of it.
// At the largest exponent, 249, codes end at 63 (64 * 2^122 would read back as infinity).  A group that holds an infinity or a NaN has e = 255 and
// reads back as NaN.
//
// Why a power of two: code * 2^k has 7 significant bits, so it IS a bf16 number.  The weight gradient dW[o][i] = sum_n dy[n][o] x8[n][i] therefore runs
// on the bf16 matrix instruction without rounding its second operand; its first one is split into bf16 numbers that sum to it exactly (bf16: one,
// fp16: two, fp32: three), so every product is exact and sums are fp32, at 1, 1/2 and 1/3 of the bf16 rate (the fp32 instruction: 1/16).
#include "tileops.hip.h"

#include <algorithm>
#include <climits>

using namespace fdx;

namespace {

typedef unsigned char u8x8 __attribute__((ext_vector_type(8)));
__device__ inline float pow2_of(int e) { return __builtin_bit_cast(float, (unsigned)e << 23); }   // 255: inf, and 0 * inf = NaN

// ---------------------------------------------------------------------------------------------------------------- GELU
// Phi(u) = 1 - erfc(|u| / sqrt 2) / 2 (mirrored for u < 0) with erfc(z) = t P(t) exp(-z^2), t = 1 / (1 + 0.45 z): P is a least-squares fit of degree 9
// (weighted towards equal relative error), 3.3e-8 relative over z >= 0.  One exponential and one reciprocal, shared with u phi(u).
__device__ inline void gelu_parts(float u, float& cdf, float& upd) {   // Phi(u), u phi(u)
  const float z = fabsf(u) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.45f, z, 1.f));
  const float g = __builtin_amdgcn_exp2f(u * u * -0.72134752044448170f);   // exp(-u^2 / 2)
  float p = -0.04140259751416385f;
  p = __builtin_fmaf(p, t, 0.19073786368796514f);
  p = __builtin_fmaf(p, t, -0.3006732548065257f);
  p = __builtin_fmaf(p, t, 0.1424903150892374f);
  p = __builtin_fmaf(p, t, -0.022409666527826486f);
  p = __builtin_fmaf(p, t, 0.11996832229019475f);
  p = __builtin_fmaf(p, t, 0.17524854027735134f);
  p = __builtin_fmaf(p, t, 0.2282720257804334f);
  p = __builtin_fmaf(p, t, 0.2538831444508843f);
  p = __builtin_fmaf(p, t, 0.2538853210040617f);
  const float half = 0.5f * p * t * g;
  cdf = u < 0.f ? half : 1.f - half;
  upd = u * g * 0.39894228040143268f;
}

// ---------------------------------------------------------------------------------------------------------------- elementwise passes
// A thread takes 8 channels (a quarter of a group: four neighbouring lanes), so a row of C channels has 4 * ceil(C / 32) threads.
struct EltArgs {
  const void *x, *dy;
  void *y;
  int8_t* codes;
  uint8_t* exps;
  long N;
  int C, G, vec;
};
// thread i of a pass: its first element, how many of its 8 exist, its group.  Whole groups in a row follow each other without gaps; otherwise the row is
// found by a division (64 bits: as many instructions as a GELU of 4 elements).
struct Eighth { long o, group; int n; };
__device__ inline Eighth eighth(const EltArgs& a, long i) {
  if (a.C % 32 == 0) return {8 * i, i >> 2, 8};
  const long per = 4L * a.G, row = i / per;
  const int q = (int)(i - row * per);
  return {row * a.C + 8 * q, row * a.G + (q >> 2), a.C - 8 * q};
}

template <typename T> __device__ inline void load8(const T* p, int n, bool vec, float* v) {   // n of 8 valid
  if (vec && n >= 8) {
    typedef T vt __attribute__((ext_vector_type(8)));
    const vt r = *reinterpret_cast<const vt*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)r[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? (float)p[j] : 0.f;
  }
}
template <typename T> __device__ inline void store8(T* p, int n, bool vec, const float* v) {
  if (vec && n >= 8) {
    typedef T vt __attribute__((ext_vector_type(8)));
    vt r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (T)v[j];
    *reinterpret_cast<vt*>(p) = r;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = (T)v[j];
  }
}
__device__ inline void load_codes(const int8_t* p, int n, bool vec, float scale, float* v) {
  if (vec && n >= 8) {
    typedef signed char i8x8 __attribute__((ext_vector_type(8)));
    const i8x8 r = *reinterpret_cast<const i8x8*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)r[j] * scale;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (j < n ? (float)p[j] : 0.f) * scale;
  }
}

// codes of x; GELU: y = gelu(x) beside them
template <typename T, bool GELU> __global__ __launch_bounds__(256) void k_pack8(EltArgs a) {
  const long total = a.N * 4L * a.G;
  const long first = (long)blockIdx.x * 256 + threadIdx.x, stride = (long)gridDim.x * 256;
  for (long i = first; i < total; i += stride) {   // (the four lanes of a group leave together: total and stride are multiples of 4)
    const auto [o, group, n] = eighth(a, i);
    float v[8];
    load8<T>(static_cast<const T*>(a.x) + o, n, a.vec, v);
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __builtin_bit_cast(unsigned, v[j]) & 0x7fffffffu);
    top = max(top, (unsigned)__shfl_xor((int)top, 1, 64));
    top = max(top, (unsigned)__shfl_xor((int)top, 2, 64));
    // top = 1.f * 2^(E - 127): 127 * 2^(E - 133) >= top unless the fraction is above 63/64
    int e = (int)(top >> 23) - 6 + ((top & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    e = max(e, 1);
    const bool bad = top >= 0x7f800000u;
    if (bad) e = 255;
    const float s = bad ? 0.f : pow2_of(254 - e);   // 2^(127 - e)
    const float end = e == 249 ? 63.f : 127.f;
    u8x8 code;
#pragma unroll
    for (int j = 0; j < 8; ++j) code[j] = (unsigned char)(bad ? 0 : (int)fminf(fmaxf(__builtin_rintf(v[j] * s), -end), end));
    if (n > 0) {
      if (a.vec && n >= 8) *reinterpret_cast<u8x8*>(a.codes + o) = code;
      else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < n) a.codes[o + j] = (int8_t)code[j];
      }
      if ((i & 3) == 0) a.exps[group] = (uint8_t)e;
      if constexpr (GELU) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float cdf, upd;
          gelu_parts(v[j], cdf, upd);
          v[j] *= cdf;
        }
        store8<T>(static_cast<T*>(a.y) + o, n, a.vec, v);
      }
    }
  }
}

// y = what the codes stand for; GRAD: y = dy * gelu'(that)
template <typename T, bool GRAD> __global__ __launch_bounds__(256) void k_unpack8(EltArgs a) {
  const long total = a.N * 4L * a.G;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    const auto [o, group, n] = eighth(a, i);
    if (n <= 0) continue;
    float v[8];
    load_codes(a.codes + o, n, a.vec, pow2_of(a.exps[group]), v);
    if constexpr (GRAD) {
      float d[8];
      load8<T>(static_cast<const T*>(a.dy) + o, n, a.vec, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float cdf, upd;
        gelu_parts(v[j], cdf, upd);
        v[j] = d[j] * (cdf + upd);
      }
    } else if constexpr (DtOf<T>::v == DT_F16) {   // 65504 may have been rounded up to 65536: the largest fp16 number, not infinity
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = fabsf(v[j]) > 65504.f ? __builtin_copysignf(65504.f, v[j]) : v[j];
    }
    store8<T>(static_cast<T*>(a.y) + o, n, a.vec, v);
  }
}

// ---------------------------------------------------------------------------------------------------------------- weight gradient
// A workgroup computes a tile of dW over its share of the rows n: 256 x 128 channels, (32 MO) x (32 NI) a wave.  fp32 and fp16: in two halves of four waves, each
// with all of the tile over every other step of rows.  The halves' sums meet in LDS at the end, so a CU full of accumulators leaves one partial tile instead of
// two, and one half splits dy while the other one multiplies (fp32, 6888 rows, 2048 x 512, with the join: 73 us in independent workgroups of four waves, 63 so).
// bf16: independent workgroups of four waves, two on a CU; there is little to convert, and halves wait for each other (27552 rows, 512 x 2048, with pack and
// join: 136 us, 144 in halves).
// KT rows of dy (in bf16 planes) and of x8 (decoded) stand in LDS, two stages per half, both read as column fragments by transposing reads: MO + NI fragments
// feed MO * NI matrix instructions.  bf16 dy goes straight to LDS, and the 256 are its channels: decoding x is all the arithmetic (per product least so).
// The wider types pass registers to be split, the 256 are x's: splitting is the arithmetic then.
// 128 x 128 tiles take what is odd.  Bound by the matrix instructions with the conversions between them (fp32: 770 TFLOP/s of bf16 products at 6888 rows) and,
// for bf16 dy, the LDS (per 16 rows 24 KB of reads and 12 of writes for 256 cycles of matrix instructions).
// Rows are shared out over `splits` workgroups (an XCD takes whole shares: dy and x8 stay in its L2 for all tiles) whose fp32 partial tiles a second
// launch joins in order.  db is summed from what is staged, each tile column taking every ti-th step.
struct WgradArgs {
  const void* dy;
  const int8_t* codes;
  const uint8_t* exps;
  float *part, *part_b;   // [splits][O][I], [splits][ti][O]
  long N, rows;           // rows per split: a multiple of 32
  int O, I, G, to, ti, splits, bias;
};

template <typename T> struct Planes { static constexpr int n = 3; };
template <> struct Planes<bf16_t> { static constexpr int n = 1; };
template <> struct Planes<f16_t> { static constexpr int n = 2; };

__device__ inline unsigned hi_bits(float x) { return __builtin_bit_cast(unsigned, x) & 0xffff0000u; }
__device__ inline unsigned pair(unsigned lo, unsigned up) { return __builtin_amdgcn_perm(up, lo, 0x07060302); }   // the upper halves of two words

// 8 codes as 8 bf16 numbers (exact)
__device__ inline uint4 decode8(uint2 c, float scale) {
  uint4 w;
  unsigned* const wp = &w.x;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const unsigned v = q < 2 ? c.x : c.y;
    const float f0 = (float)(signed char)(v >> (16 * (q & 1))) * scale, f1 = (float)(signed char)(v >> (16 * (q & 1) + 8)) * scale;
    wp[q] = pair(__builtin_bit_cast(unsigned, f0), __builtin_bit_cast(unsigned, f1));
  }
  return w;
}

template <typename T> constexpr int halves() { return Planes<T>::n == 1 ? 1 : 2; }
template <typename T, int MO, int NI, bool VEC>
__global__ __launch_bounds__(256 * halves<T>(), 2) void k_linear8_wgrad(WgradArgs a) {
  typedef Tile<bf16_t, 128> Tl;
  typedef Elem<bf16_t>::frag frag;
  constexpr int P = Planes<T>::n, HV = halves<T>(), KT = P == 1 ? 32 : 16, NO = MO / 2, NX = NI / 2;   // NO, NX: 128-channel tiles of dy and x
  constexpr int kY = KT * 16, kStage = (P * NO + NX) * kY;   // in 16-byte units; kY: one tile
  constexpr int kSum = HV > 1 ? 256 * MO * NI * 4 : 0;   // one half's accumulators
  __shared__ __attribute__((aligned(1024))) uint4 smem[2 * HV * kStage > kSum ? 2 * HV * kStage : kSum];
  const int per = a.to * a.ti;
  int split, j;
  if (a.splits % 8 == 0) { split = (blockIdx.x & 7) + 8 * ((blockIdx.x >> 3) / per); j = (blockIdx.x >> 3) % per; }
  else { split = blockIdx.x / per; j = blockIdx.x % per; }
  const int jo = j / a.ti, ji = j % a.ti, o0 = jo * 128 * NO, i0 = ji * 128 * NX;
  const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) & 3, wo = wave >> 1, wi = wave & 1, tid = threadIdx.x & 255;
  const int half = HV > 1 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 8) : 0;
  uint4* const own = smem + half * 2 * kStage;
  // staging of x: 8 columns of XR rows; of dy (through registers): 8 columns of YR rows
  constexpr int XC = 16 * NX, XR = KT * XC / 256, YC = 16 * NO, YR = KT * YC / 256;
  const int xc = tid % XC, xr = tid / XC, yc = tid % YC, yr = tid / YC;
  const int ic = i0 + 8 * xc, in = a.I - ic, oc = o0 + 8 * yc, on = a.O - oc;
  float db[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  f32x16 acc[MO][NI];
#pragma unroll
  for (int m = 0; m < MO; ++m)
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[m][n] = f32x16{0};
  const long nb = (long)split * a.rows, ne = min(a.N, nb + a.rows);
  // wave wo's channels: MO == 4: its own 128-channel tile, MO == 2: half of the one (wi, NI: the same for x)
  const unsigned coly = lds_of(own) + (Tl::col_base(lane) ^ (MO == 2 ? 128 * wo : 0)) + (MO == 4 ? wo * P * kY * 16 : 0);
  const unsigned colx = lds_of(own) + P * NO * kY * 16 + (Tl::col_base(lane) ^ (NI == 2 ? 128 * wi : 0)) + (NI == 4 ? wi * kY * 16 : 0);

  // Registers of two steps ahead.  They hold what was loaded as it was loaded: any instruction on it here -- a conversion, the masking of a byte --
  // would wait for the load in front of the products instead of behind them.  Rows past the last one are read as the last one and made zeros when they
  // are used; columns past the last one are never stored.
  typedef T t8 __attribute__((ext_vector_type(8)));
  uint2 xcode[2][XR];
  int xexp[2][XR];
  t8 y[2][YR];
  const int icv = in > 0 ? ic : 0, ocv = on > 0 ? oc : 0;
  auto load_x = [&](long n0, int set) {
    const int last = (int)min((long)KT, ne - n0) - 1;
    const int8_t* const p = a.codes + n0 * a.I + icv;
    const uint8_t* const pe = a.exps + n0 * a.G + (icv >> 5);
#pragma unroll
    for (int h = 0; h < XR; ++h) xexp[set][h] = pe[(long)min(xr + (256 / XC) * h, last) * a.G];
#pragma unroll
    for (int h = 0; h < XR; ++h) {
      const int8_t* const q = p + (long)min(xr + (256 / XC) * h, last) * a.I;
      if constexpr (VEC) xcode[set][h] = *reinterpret_cast<const uint2*>(q);
      else {
        uint2 w = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (icv + j < a.I) (j < 4 ? w.x : w.y) |= (unsigned)(uint8_t)q[j] << (8 * (j & 3));
        xcode[set][h] = w;
      }
    }
  };
  auto load_y = [&](long n0, int set) {
    const int last = (int)min((long)KT, ne - n0) - 1;
    const T* const p = static_cast<const T*>(a.dy) + n0 * a.O + ocv;
#pragma unroll
    for (int h = 0; h < YR; ++h) {
      const T* const q = p + (long)min(yr + (256 / YC) * h, last) * a.O;
      if constexpr (VEC) y[set][h] = *reinterpret_cast<const t8*>(q);
      else {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[set][h][j] = ocv + j < a.O ? q[j] : (T)0.f;
      }
    }
  };
  // bring a step's dy and x into a stage
  auto fill_y = [&](long n0, int stage, bool count, int set) {
    uint4* const to = own + stage * kStage;
    const int rows = (int)min((long)KT, ne - n0);
    if constexpr (P == 1) {
      if constexpr (VEC) {
#pragma unroll
        for (int h = 0; h < NO; ++h)
          Fill<bf16_t, 128, KT>::issue(to + h * kY, static_cast<const bf16_t*>(a.dy) + n0 * a.O + o0 + 128 * h, a.O, a.O - o0 - 128 * h,
                                       n0 + KT <= ne && o0 + 128 * h + 128 <= a.O, [&](int row) { return n0 + row < ne; }, wave);
      } else {
#pragma unroll
        for (int h = 0; h < YR; ++h) {
          const int row = yr + (256 / YC) * h;
          to[(yc >> 4) * kY + Tl::at(row, yc & 15)] = row < rows ? __builtin_bit_cast(uint4, y[set][h]) : uint4{0, 0, 0, 0};
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < YR; ++h) {
        const int row = yr + (256 / YC) * h;
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = (float)y[set][h][q];
        if (rows < KT) {
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] = row < rows ? v[q] : 0.f;
        }
        if (count) {
#pragma unroll
          for (int q = 0; q < 8; ++q) db[q] += v[q];
        }
        const int at = (yc >> 4) * P * kY + Tl::at(row, yc & 15);
#pragma unroll
        for (int p = 0; p < P; ++p) {
          uint4 w;
          unsigned* const wp = &w.x;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float &lo = v[2 * q], &up = v[2 * q + 1];
            wp[q] = pair(__builtin_bit_cast(unsigned, lo), __builtin_bit_cast(unsigned, up));
            if (p + 1 < P) {   // exact: the bits below
              lo -= __builtin_bit_cast(float, hi_bits(lo));
              up -= __builtin_bit_cast(float, hi_bits(up));
            }
          }
          to[at + p * kY] = w;
        }
      }
    }
  };
  auto fill_x = [&](long n0, int stage, int set) {
    uint4* const to = own + stage * kStage + P * NO * kY;
    const int rows = (int)min((long)KT, ne - n0);
#pragma unroll
    for (int h = 0; h < XR; ++h) {
      const int row = xr + (256 / XC) * h;
      to[(xc >> 4) * kY + Tl::at(row, xc & 15)] = decode8(xcode[set][h], pow2_of(row < rows ? xexp[set][h] : 0));
    }
  };
  auto mine = [&](long n0) { return a.bias && (n0 - nb) / KT % a.ti == ji; };
  int stage = 0;
  constexpr int STEP = HV * KT;
  constexpr bool kDirect = P == 1 && VEC;   // dy goes straight to LDS
  auto load = [&](long n0, int set) {   // (behind the last step the last row again: no branch)
    n0 = min(n0, ne - 1);
    if constexpr (!kDirect) load_y(n0, set);
    load_x(n0, set);
  };
  const long first = nb + half * KT;
  if (first < ne) {
    load(first, 0);
    fill_y(first, 0, mine(first), 0);
    fill_x(first, 0, 0);
    load(first + STEP, 0);
    if constexpr (!kDirect) load(first + 2 * STEP, 1);
  }
  auto products = [&](long n0) {
    const unsigned cy = opaque(coly + stage * kStage * 16), cx = opaque(colx + stage * kStage * 16);
    if constexpr (P == 1) {
      if (mine(n0)) {
        const uint4* const t = own + stage * kStage + (yc >> 4) * kY;
#pragma unroll
        for (int h = 0; h < YR; ++h) {
          const frag v = __builtin_bit_cast(frag, t[Tl::at(yr + (256 / YC) * h, yc & 15)]);
#pragma unroll
          for (int q = 0; q < 8; ++q) db[q] += (float)v[q];
        }
      }
    }
#pragma unroll
    for (int ks = 0; ks < KT / 16; ++ks) {
      frag b[NI];
#pragma unroll
      for (int n = 0; n < NI; ++n) b[n] = Tl::col(cx, 16 * ks, n);
#pragma unroll
      for (int p = P - 1; p >= 0; --p)   // small parts first
#pragma unroll
        for (int m = 0; m < MO; ++m) {
          const frag f = Tl::col(cy, p * KT + 16 * ks, m);
#pragma unroll
          for (int n = 0; n < NI; ++n) acc[m][n] = Elem<bf16_t>::mma(f, b[n], acc[m][n]);
        }
    }
  };
  // The two halves share the SIMDs: where dy has to be split, one converts while the other one multiplies
  auto step = [&](long n0, int set) {
    if constexpr (kDirect) landed();
    else __syncthreads();
    const long now = n0 + half * KT, then = now + STEP;
    const bool more = then < ne;
    if constexpr (kDirect) {
      if (more) {
        fill_y(then, stage ^ 1, false, 0);
        load(then + STEP, set ^ 1);
        fill_x(then, stage ^ 1, set);
      }
      if (now < ne) products(now);
    } else {
      auto fill = [&] {
        if (!more) return;
        fill_y(then, stage ^ 1, mine(then), set);
        fill_x(then, stage ^ 1, set);
        load(then + 2 * STEP, set);
      };
      if (half == 0) fill();
      if (now < ne) products(now);
      if (half == 1) fill();
    }
    stage ^= 1;
  };
  for (long n0 = nb; n0 < ne; n0 += 2 * STEP) {
    step(n0, 0);
    if (n0 + STEP < ne) step(n0 + STEP, 1);
  }
  // each half gives the other one half of its accumulators and stores the sums of the rest
  landed();
  f32x4* const sums = reinterpret_cast<f32x4*>(smem) + wave * MO * NI * 4 * 64 + lane;
  constexpr int MH = MO / 2;
  auto give = [&](int m0) {
#pragma unroll
    for (int m = 0; m < MH; ++m)
#pragma unroll
      for (int n = 0; n < NI; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x16& v = acc[m0 + m][n];
          sums[(((m0 + m) * NI + n) * 4 + q) * 64] = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        }
  };
  float* const out = a.part + (long)split * a.O * a.I;
  auto store = [&](int m0) {
#pragma unroll
    for (int m = m0; m < m0 + MO / HV; ++m)
#pragma unroll
      for (int n = 0; n < NI; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f32x4 other = {0, 0, 0, 0};
          if constexpr (HV > 1) other = sums[((m * NI + n) * 4 + q) * 64];
          const int o = o0 + wo * 32 * MO + m * 32 + 8 * q + 4 * (lane >> 5), i = i0 + wi * 32 * NI + n * 32 + (lane & 31);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (o + e < a.O && i < a.I) out[(long)(o + e) * a.I + i] = acc[m][n][4 * q + e] + other[e];
        }
  };
  if constexpr (HV > 1) {
    if (half == 0) give(MH);
    else give(0);
    __syncthreads();
    if (half == 0) store(0);
    else store(MH);
  } else store(0);
  if (a.bias) {
    constexpr int NR = 256 * HV / YC;
    float* const lb = reinterpret_cast<float*>(smem);   // [NR][8 * YC]
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 8; ++q) lb[(half * (256 / YC) + yr) * 8 * YC + 8 * yc + q] = db[q];
    __syncthreads();
    if ((int)threadIdx.x < 8 * YC && o0 + (int)threadIdx.x < a.O) {
      float s = 0.f;
      for (int r = 0; r < NR; ++r) s += lb[r * 8 * YC + threadIdx.x];
      a.part_b[((long)split * a.ti + ji) * a.O + o0 + threadIdx.x] = s;
    }
  }
}

// The partial tiles joined in their order, four elements a thread with eight loads in flight; behind them db: 32 channels a workgroup, every thread sums an
// eighth of the rows.
struct Join8Args { const float *part, *part_b; void *dw, *db; long n; int splits, O, rows_b, main, vec; };
template <typename T> __global__ __launch_bounds__(256) void k_join8(Join8Args a) {
  __shared__ float red[8][32];
  if ((int)blockIdx.x < a.main) {
    const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= a.n) return;
    if (a.vec) {
      f32x4 v = {0, 0, 0, 0};
      const float* p = a.part + i;
      int s = 0;
      for (; s + 8 <= a.splits; s += 8) {
        f32x4 t[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) t[q] = *reinterpret_cast<const f32x4*>(p + (s + q) * a.n);
#pragma unroll
        for (int q = 0; q < 8; ++q) v += t[q];
      }
      for (; s < a.splits; ++s) v += *reinterpret_cast<const f32x4*>(p + s * a.n);
      typedef T vt __attribute__((ext_vector_type(4)));
      *reinterpret_cast<vt*>(static_cast<T*>(a.dw) + i) = vt{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    } else {
      for (long j = i; j < min(i + 4, a.n); ++j) {
        float v = 0.f;
        for (int s = 0; s < a.splits; ++s) v += a.part[s * a.n + j];
        static_cast<T*>(a.dw)[j] = (T)v;
      }
    }
    return;
  }
  const int c = ((int)blockIdx.x - a.main) * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
  float v = 0.f;
  if (c < a.O) {
    int r = g;
    for (; r + 7 * 8 < a.rows_b; r += 8 * 8) {
      float t[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) t[q] = a.part_b[(long)(r + 8 * q) * a.O + c];
#pragma unroll
      for (int q = 0; q < 8; ++q) v += t[q];
    }
    for (; r < a.rows_b; r += 8) v += a.part_b[(long)r * a.O + c];
  }
  red[g][threadIdx.x & 31] = v;
  __syncthreads();
  if (g == 0 && c < a.O) {
#pragma unroll
    for (int q = 1; q < 8; ++q) v += red[q][threadIdx.x & 31];
    static_cast<T*>(a.db)[c] = (T)v;
  }
}

// ---------------------------------------------------------------------------------------------------------------- launches
const char* check(int dtype, long long rows, int channels) {
  if (dtype < 0 || dtype > 2) return "dtype must be FDX_F32, FDX_BF16 or FDX_F16";
  if (rows < 0 || rows > (1LL << 40) || channels < 1 || channels > (1 << 24)) return "rows or channels out of range";
  return nullptr;
}
bool aligned(std::initializer_list<const void*> ps, int channels, int bytes) {
  if (channels % 8) return false;
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
  return true;
}
EltArgs elt(long long rows, int channels) {
  EltArgs a{};
  a.N = rows; a.C = channels; a.G = (channels + 31) / 32;
  return a;
}
unsigned elt_grid(const EltArgs& a) { return (unsigned)std::min<long>((a.N * 4 * a.G + 255) / 256, 1L << 22); }
template <template <typename> class K> hipError_t go(int dt, const EltArgs& a, hipStream_t s) {
  return dt == DT_F32 ? launch(K<float>::get(), elt_grid(a), 256, a, s) : dt == DT_BF16 ? launch(K<bf16_t>::get(), elt_grid(a), 256, a, s)
                                                                                       : launch(K<f16_t>::get(), elt_grid(a), 256, a, s);
}
template <typename T> struct KPack { static auto get() { return k_pack8<T, false>; } };
template <typename T> struct KGelu { static auto get() { return k_pack8<T, true>; } };
template <typename T> struct KUnpack { static auto get() { return k_unpack8<T, false>; } };
template <typename T> struct KGeluGrad { static auto get() { return k_unpack8<T, true>; } };

// 256 channels where they fit as well as 128 do (bf16, 27552 rows, 512 x 2048: 284 us in 128 x 128 tiles, 102 in 256 x 128).  Rows are split until eight
// waves stand on every CU, each workgroup with 256 rows at least: a shorter share costs more in partial tiles (8 bytes per element of dW and share) than it gains.
struct Cut8 { int wide, to, ti, splits; };
Cut8 wgrad_cut(int dtype, long N, int O, int I, bool vec) {
  Cut8 c;
  c.to = (O + 127) / 128;
  c.ti = (I + 127) / 128;
  int& w = dtype == DT_BF16 ? c.to : c.ti;
  c.wide = vec && w % 2 == 0;
  if (c.wide) w /= 2;
  const long tiles = (long)c.to * c.ti;
  const long want = dtype == DT_BF16 ? 512 : 256;
  long s = std::min<long>((want + tiles - 1) / tiles, N / 256);
  if (s > 8) s = s / 8 * 8;
  c.splits = (int)std::max<long>(1, std::min<long>(s, 64));
  return c;
}
size_t wgrad_floats(const Cut8& c, int O, int I) { return (size_t)c.splits * ((size_t)O * I + (size_t)c.ti * O); }
size_t wgrad_bytes(int dtype, long N, int O, int I) {   // whatever the pointers turn out to be aligned to
  return std::max(wgrad_floats(wgrad_cut(dtype, N, O, I, false), O, I), wgrad_floats(wgrad_cut(dtype, N, O, I, true), O, I)) * sizeof(float);
}

}  // namespace

extern "C" int fdx_pack8(fdx_handle h, int dtype, const void* x, long long rows, int channels, int8_t* codes, uint8_t* exps, fdx_stream st) {
  if (!h) return fail(nullptr, FDX_E_ARG, "fdx_pack8: null handle");
  if (const char* why = check(dtype, rows, channels)) return fail(h, FDX_E_ARG, "fdx_pack8: %s", why);
  if (rows == 0) return FDX_OK;
  if (!x || !codes || !exps) return fail(h, FDX_E_ARG, "fdx_pack8: null tensor");
  EltArgs a = elt(rows, channels);
  a.x = x; a.codes = codes; a.exps = exps; a.vec = aligned({x}, channels, 16) && aligned({codes}, channels, 8);
  DeviceScope dev(h->device);
  FDX_HIP(h, dev.err);
  FDX_HIP(h, go<KPack>(dtype, a, as_stream(st)));
  return FDX_OK;
}

extern "C" int fdx_unpack8(fdx_handle h, int dtype, const int8_t* codes, const uint8_t* exps, long long rows, int channels, void* x, fdx_stream st) {
  if (!h) return fail(nullptr, FDX_E_ARG, "fdx_unpack8: null handle");
  if (const char* why = check(dtype, rows, channels)) return fail(h, FDX_E_ARG, "fdx_unpack8: %s", why);
  if (rows == 0) return FDX_OK;
  if (!x || !codes || !exps) return fail(h, FDX_E_ARG, "fdx_unpack8: null tensor");
  EltArgs a = elt(rows, channels);
  a.y = x; a.codes = const_cast<int8_t*>(codes); a.exps = const_cast<uint8_t*>(exps); a.vec = aligned({x}, channels, 16) && aligned({codes}, channels, 8);
  DeviceScope dev(h->device);
  FDX_HIP(h, dev.err);
  FDX_HIP(h, go<KUnpack>(dtype, a, as_stream(st)));
  return FDX_OK;
}

extern "C" int fdx_gelu8_forward(fdx_handle h, int dtype, const void* x, long long rows, int channels, void* y, int8_t* codes, uint8_t* exps,
                                 fdx_stream st) {
  if (!h) return fail(nullptr, FDX_E_ARG, "fdx_gelu8_forward: null handle");
  if (const char* why = check(dtype, rows, channels)) return fail(h, FDX_E_ARG, "fdx_gelu8_forward: %s", why);
  if (rows == 0) return FDX_OK;
  if (!x || !y || !codes || !exps) return fail(h, FDX_E_ARG, "fdx_gelu8_forward: null tensor");
  EltArgs a = elt(rows, channels);
  a.x = x; a.y = y; a.codes = codes; a.exps = exps; a.vec = aligned({x, y}, channels, 16) && aligned({codes}, channels, 8);
  DeviceScope dev(h->device);
  FDX_HIP(h, dev.err);
  FDX_HIP(h, go<KGelu>(dtype, a, as_stream(st)));
  return FDX_OK;
}

extern "C" int fdx_gelu8_backward(fdx_handle h, int dtype, const void* dy, const int8_t* codes, const uint8_t* exps, long long rows, int channels,
                                  void* dx, fdx_stream st) {
  if (!h) return fail(nullptr, FDX_E_ARG, "fdx_gelu8_backward: null handle");
  if (const char* why = check(dtype, rows, channels)) return fail(h, FDX_E_ARG, "fdx_gelu8_backward: %s", why);
  if (rows == 0) return FDX_OK;
  if (!dy || !dx || !codes || !exps) return fail(h, FDX_E_ARG, "fdx_gelu8_backward: null tensor");
  EltArgs a = elt(rows, channels);
  a.dy = dy; a.y = dx; a.codes = const_cast<int8_t*>(codes); a.exps = const_cast<uint8_t*>(exps);
  a.vec = aligned({dy, dx}, channels, 16) && aligned({codes}, channels, 8);
  DeviceScope dev(h->device);
  FDX_HIP(h, dev.err);
  FDX_HIP(h, go<KGeluGrad>(dtype, a, as_stream(st)));
  return FDX_OK;
}

extern "C" int fdx_linear8_weight_grad_workspace(int dtype, long long rows, int out_features, int in_features, size_t* bytes) {
  const char* why = check(dtype, rows, out_features);
  if (!why) why = check(dtype, rows, in_features);
  if (!why && !bytes) why = "null size pointer";
  if (why) return fail(nullptr, FDX_E_ARG, "fdx_linear8_weight_grad_workspace: %s", why);
  *bytes = wgrad_bytes(dtype, rows, out_features, in_features);
  return FDX_OK;
}

extern "C" int fdx_linear8_weight_grad(fdx_handle h, int dtype, const void* dy, const int8_t* codes, const uint8_t* exps, long long rows,
                                       int out_features, int in_features, int grad_dtype, void* dw, void* db, void* workspace, size_t bytes,
                                       fdx_stream st) {
  if (!h) return fail(nullptr, FDX_E_ARG, "fdx_linear8_weight_grad: null handle");
  const char* why = check(dtype, rows, out_features);
  if (!why) why = check(grad_dtype, rows, in_features);
  const long tiles = (long)((out_features + 127) / 128) * ((in_features + 127) / 128);
  constexpr long most = (1L << 24) - 1;   // workgroups of 256 threads in one launch
  if (!why && (tiles > most / 64 || (long)out_features * in_features / 1024 + out_features / 32 + 2 > most)) why = "too many tiles for one launch";
  if (!why && (!dw || (rows > 0 && (!dy || !codes || !exps)))) why = "null tensor";
  if (why) return fail(h, FDX_E_ARG, "fdx_linear8_weight_grad: %s", why);
  const bool vec = aligned({dy}, out_features, 16) && aligned({codes}, in_features, 8);
  const Cut8 c = wgrad_cut(dtype, rows, out_features, in_features, vec);
  const size_t need = wgrad_bytes(dtype, rows, out_features, in_features);
  if (bytes < need || !workspace) return fail(h, FDX_E_ARG, "fdx_linear8_weight_grad: workspace of %zu bytes, %zu needed", bytes, need);
  WgradArgs a{};
  a.dy = dy; a.codes = codes; a.exps = exps; a.N = rows; a.O = out_features; a.I = in_features; a.G = (in_features + 31) / 32;
  a.to = c.to; a.ti = c.ti; a.splits = c.splits; a.bias = db != nullptr;
  a.rows = ((rows + a.splits - 1) / a.splits + 31) / 32 * 32;
  a.part = static_cast<float*>(workspace);
  a.part_b = a.part + (size_t)a.splits * a.O * a.I;
  DeviceScope dev(h->device);
  FDX_HIP(h, dev.err);
  hipStream_t s = as_stream(st);
  const auto go = [&](auto any, auto narrow, auto wide) { return launch(c.wide ? wide : vec ? narrow : any, (unsigned)((long)c.to * c.ti * c.splits), dtype == DT_BF16 ? 256 : 512, a, s); };
  FDX_HIP(h, dtype == DT_F32    ? go(k_linear8_wgrad<float, 2, 2, false>, k_linear8_wgrad<float, 2, 2, true>, k_linear8_wgrad<float, 2, 4, true>)
             : dtype == DT_BF16 ? go(k_linear8_wgrad<bf16_t, 2, 2, false>, k_linear8_wgrad<bf16_t, 2, 2, true>, k_linear8_wgrad<bf16_t, 4, 2, true>)
                                : go(k_linear8_wgrad<f16_t, 2, 2, false>, k_linear8_wgrad<f16_t, 2, 2, true>, k_linear8_wgrad<f16_t, 2, 4, true>));
  Join8Args j{a.part, a.part_b, dw, db, (long)a.O * a.I, a.splits, a.O, a.splits * a.ti, 0, 0};
  j.vec = j.n % 4 == 0 && (reinterpret_cast<uintptr_t>(dw) & 15) == 0 && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0;
  j.main = (int)((j.n + 1023) / 1024);
  const unsigned grid = (unsigned)j.main + (db ? (a.O + 31) / 32 : 0);
  FDX_HIP(h, grad_dtype == DT_F32 ? launch(k_join8<float>, grid, 256, j, s) : grad_dtype == DT_BF16 ? launch(k_join8<bf16_t>, grid, 256, j, s)
                                                                                                    : launch(k_join8<f16_t>, grid, 256, j, s));
  return FDX_OK;
}
