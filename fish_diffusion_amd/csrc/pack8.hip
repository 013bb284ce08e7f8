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
  int C, G, vec, out_dt;
};

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
  const long per = 4L * a.G, total = a.N * per;
  const long first = (long)blockIdx.x * 256 + threadIdx.x, stride = (long)gridDim.x * 256;
  for (long i = first; i < total; i += stride) {   // (the four lanes of a group leave together: total and stride are multiples of 4)
    const long row = i / per;
    const int q = (int)(i - row * per), c = q * 8, n = a.C - c;
    const long o = row * a.C + c;
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
      if ((q & 3) == 0) a.exps[row * a.G + (q >> 2)] = (uint8_t)e;
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
  const long per = 4L * a.G, total = a.N * per;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    const long row = i / per;
    const int q = (int)(i - row * per), c = q * 8, n = a.C - c;
    if (n <= 0) continue;
    const long o = row * a.C + c;
    float v[8];
    load_codes(a.codes + o, n, a.vec, pow2_of(a.exps[row * a.G + (q >> 2)]), v);
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
// A workgroup computes a 128 x 128 tile of dW over its share of the rows n: 32 rows of dy (in bf16 planes) and of x8 (decoded) at a time in LDS, both
// read as column fragments by transposing reads, 4 waves of 64 x 64.  Rows are shared out over `splits` workgroups whose fp32 partial tiles a second
// launch joins in order.  db is added up by the threads that stage dy in the first column of tiles.
struct WgradArgs {
  const void* dy;
  const int8_t* codes;
  const uint8_t* exps;
  float *part, *part_b;   // [splits][O][I], [splits][O]
  long N, rows;           // rows per split: a multiple of 32
  int O, I, G, to, ti, splits, bias, vec_dy, vec_x;
};

template <typename T> struct Planes { static constexpr int n = 3; };
template <> struct Planes<bf16_t> { static constexpr int n = 1; };
template <> struct Planes<f16_t> { static constexpr int n = 2; };

__device__ inline unsigned hi_bits(float x) { return __builtin_bit_cast(unsigned, x) & 0xffff0000u; }

template <typename T>
__global__ __launch_bounds__(256) void k_linear8_wgrad(WgradArgs a) {
  typedef Tile<bf16_t, 128> Tl;
  typedef Elem<bf16_t>::frag frag;
  constexpr int P = Planes<T>::n, KT = 32;
  __shared__ __attribute__((aligned(1024))) uint4 ly[P][KT * 16], lx[KT * 16];
  __shared__ float lb[16][128];
  const int per = a.to * a.ti, split = blockIdx.x / per, j = blockIdx.x % per, o0 = j / a.ti * 128, i0 = j % a.ti * 128;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wo = wave >> 1, wi = wave & 1;
  const int chunk = threadIdx.x & 15, srow = threadIdx.x >> 4;   // staging: 8 columns of rows srow, srow + 16
  const int oc = o0 + 8 * chunk, on = a.O - oc, ic = i0 + 8 * chunk, in = a.I - ic;
  const bool want_b = a.bias && i0 == 0;
  float db[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  f32x16 acc[2][2];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n) acc[m][n] = f32x16{0};
  const unsigned coly = lds_of(ly) + (Tl::col_base(lane) ^ (128 * wo)), colx = lds_of(lx) + (Tl::col_base(lane) ^ (128 * wi));
  const long nb = (long)split * a.rows, ne = min(a.N, nb + a.rows);
  float y[2][8], x[2][8];
  auto fetch = [&](long n0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long n = n0 + srow + 16 * h;
      const bool ok = n < ne;
      load8<T>(static_cast<const T*>(a.dy) + n * a.O + oc, ok ? on : 0, a.vec_dy, y[h]);
      if (ok && in > 0) load_codes(a.codes + n * a.I + ic, in, a.vec_x, pow2_of(a.exps[n * a.G + (ic >> 5)]), x[h]);
      else {
#pragma unroll
        for (int q = 0; q < 8; ++q) x[h][q] = 0.f;
      }
    }
  };
  if (nb < ne) fetch(nb);
  for (long n0 = nb; n0 < ne; n0 += KT) {
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = Tl::at(srow + 16 * h, chunk);
      if (want_b) {
#pragma unroll
        for (int q = 0; q < 8; ++q) db[q] += y[h][q];
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        uint4 w;
        unsigned* const wp = &w.x;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const unsigned lo = hi_bits(y[h][2 * q]), up = hi_bits(y[h][2 * q + 1]);
          wp[q] = (lo >> 16) | up;
          y[h][2 * q] -= __builtin_bit_cast(float, lo);   // exact: the remaining low bits
          y[h][2 * q + 1] -= __builtin_bit_cast(float, up);
        }
        ly[p][at] = w;
      }
      uint4 w;
      unsigned* const wp = &w.x;
#pragma unroll
      for (int q = 0; q < 4; ++q) wp[q] = (hi_bits(x[h][2 * q]) >> 16) | hi_bits(x[h][2 * q + 1]);
      lx[at] = w;
    }
    __syncthreads();
    if (n0 + KT < ne) fetch(n0 + KT);
#pragma unroll
    for (int ks = 0; ks < KT / 16; ++ks) {
      frag b[2];
#pragma unroll
      for (int n = 0; n < 2; ++n) b[n] = Tl::col(colx, 16 * ks, n);
#pragma unroll
      for (int p = P - 1; p >= 0; --p)   // small parts first
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const frag f = Tl::col(coly, p * KT + 16 * ks, m);
#pragma unroll
          for (int n = 0; n < 2; ++n) acc[m][n] = Elem<bf16_t>::mma(f, b[n], acc[m][n]);
        }
    }
  }
  float* const out = a.part + (long)split * a.O * a.I;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int o = o0 + wo * 64 + m * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3), i = i0 + wi * 64 + n * 32 + (lane & 31);
        if (o < a.O && i < a.I) out[(long)o * a.I + i] = acc[m][n][e];
      }
  if (want_b) {   // (uniform over the workgroup)
#pragma unroll
    for (int q = 0; q < 8; ++q) lb[srow][8 * chunk + q] = db[q];
    __syncthreads();
    if (threadIdx.x < 128 && o0 + (int)threadIdx.x < a.O) {
      float s = 0.f;
      for (int r = 0; r < 16; ++r) s += lb[r][threadIdx.x];
      a.part_b[(long)split * a.O + o0 + threadIdx.x] = s;
    }
  }
}

struct Join8Args { const float* part; void* out; long n; int splits; };
template <typename T> __global__ __launch_bounds__(256) void k_join8(Join8Args a) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < a.n; i += (long)gridDim.x * 256) {
    float v = 0.f;
    for (int s = 0; s < a.splits; ++s) v += a.part[s * a.n + i];
    static_cast<T*>(a.out)[i] = (T)v;
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

// Rows are split until two workgroups stand on every CU, each of them with 256 rows at least: a shorter share costs more in partial tiles
// (8 bytes per element of dW and share) than it gains.
int wgrad_splits(long N, int O, int I) {
  const long tiles = (long)((O + 127) / 128) * ((I + 127) / 128);
  const long s = std::min<long>((512 + tiles - 1) / tiles, N / 256);
  return (int)std::max<long>(1, std::min<long>(s, 64));
}
size_t wgrad_floats(long N, int O, int I) { return (size_t)wgrad_splits(N, O, I) * ((size_t)O * I + O); }

template <typename T> hipError_t join8(const float* part, void* out, long n, int splits, hipStream_t s) {
  Join8Args j{part, out, n, splits};
  return launch(k_join8<T>, (unsigned)std::min<long>((n + 255) / 256, 4096), 256, j, s);
}
hipError_t join8(int dt, const float* part, void* out, long n, int splits, hipStream_t s) {
  return dt == DT_F32 ? join8<float>(part, out, n, splits, s) : dt == DT_BF16 ? join8<bf16_t>(part, out, n, splits, s) : join8<f16_t>(part, out, n, splits, s);
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
  *bytes = wgrad_floats(rows, out_features, in_features) * sizeof(float);
  return FDX_OK;
}

extern "C" int fdx_linear8_weight_grad(fdx_handle h, int dtype, const void* dy, const int8_t* codes, const uint8_t* exps, long long rows,
                                       int out_features, int in_features, int grad_dtype, void* dw, void* db, void* workspace, size_t bytes,
                                       fdx_stream st) {
  if (!h) return fail(nullptr, FDX_E_ARG, "fdx_linear8_weight_grad: null handle");
  const char* why = check(dtype, rows, out_features);
  if (!why) why = check(grad_dtype, rows, in_features);
  const long tiles = (long)((out_features + 127) / 128) * ((in_features + 127) / 128);
  if (!why && tiles > INT_MAX / 64) why = "too many tiles for one launch";
  if (!why && (!dw || (rows > 0 && (!dy || !codes || !exps)))) why = "null tensor";
  if (why) return fail(h, FDX_E_ARG, "fdx_linear8_weight_grad: %s", why);
  const size_t need = wgrad_floats(rows, out_features, in_features) * sizeof(float);
  if (bytes < need || !workspace) return fail(h, FDX_E_ARG, "fdx_linear8_weight_grad: workspace of %zu bytes, %zu needed", bytes, need);
  WgradArgs a{};
  a.dy = dy; a.codes = codes; a.exps = exps; a.N = rows; a.O = out_features; a.I = in_features; a.G = (in_features + 31) / 32;
  a.to = (a.O + 127) / 128; a.ti = (a.I + 127) / 128; a.splits = wgrad_splits(rows, a.O, a.I); a.bias = db != nullptr;
  a.rows = ((rows + a.splits - 1) / a.splits + 31) / 32 * 32;
  a.vec_dy = aligned({dy}, a.O, 16); a.vec_x = aligned({codes}, a.I, 8);
  a.part = static_cast<float*>(workspace);
  a.part_b = a.part + (size_t)a.splits * a.O * a.I;
  DeviceScope dev(h->device);
  FDX_HIP(h, dev.err);
  const unsigned grid = (unsigned)(tiles * a.splits);
  hipStream_t s = as_stream(st);
  FDX_HIP(h, dtype == DT_F32 ? launch(k_linear8_wgrad<float>, grid, 256, a, s) : dtype == DT_BF16 ? launch(k_linear8_wgrad<bf16_t>, grid, 256, a, s)
                                                                                              : launch(k_linear8_wgrad<f16_t>, grid, 256, a, s));
  FDX_HIP(h, join8(grad_dtype, a.part, dw, (long)a.O * a.I, a.splits, s));
  if (db) FDX_HIP(h, join8(grad_dtype, a.part_b, db, a.O, a.splits, s));
  return FDX_OK;
}
