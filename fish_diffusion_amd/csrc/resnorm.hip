// resnorm.hip -- the step between two blocks of a network in one launch each way (fdx_resnorm_*):
//
//   n = post(block)      h = a x + g n      y = pre(h)          post, pre: LayerNorm, RMSNorm or nothing; g: nothing or a gate
//
//   dh = grad_h + pre'(grad_y)   dx = a dh   dn = g dh   dblock = post'(dn)   dg = sum dh n
//   norm'(gy): w = gy weight, r (w - mean(w) - hat mean(w hat))   (RMSNorm: without mean(w));   dweight = sum gy hat, dbias = sum gy
//
// Bound by memory: forward reads x, block, writes h, y; backward reads x, block, grad_h, grad_y and writes dx, dblock.  n, h and both normalised
// tensors are computed again from x and block in fp32 (reading h, y instead of x would cost the same bytes and add their rounding); the forward
// leaves mean and 1 / deviation of both norms (16 bytes a row).  One wave holds a row in registers up to 2048 channels (backward 1024), 4 or 8
// waves above; means are taken before the squares are summed (two passes over registers).  The sums over rows run per thread in row order,
// then over the waves of a workgroup in LDS, then over the workgroups in a second launch, always in the same order.
#include "tileops.hip.h"

#include <algorithm>
#include <climits>

using namespace fdx;

namespace {

struct NormArgs {
  const void *x, *block, *gate, *post_w, *post_b, *pre_w, *pre_b, *gh, *gy;
  void *h, *y, *dx, *dblock, *dgate;
  float *stats, *part;
  long N, gate_rows;       // rows that share one gate row (0: no gate)
  int C, pdt, gdt, rms;    // types of the norms' parameters / of the gate
  int has_post, has_pre, same_dx;   // same_dx: dblock is dx
  float a, eps, inv_c;
  // backward: `groups` runs of rows_per_group rows (one gate row each, or everything), cut into `cuts` workgroups each; or, where gate rows are short
  // (flush), every unit of waves takes whole groups and writes their dgate itself
  long groups, rows_per_group;
  int cuts, flush, slots;
};

// -------------------------------------------------------------------------------------------------------------- pieces of a row
// A thread's IT pieces of VEC channels: channel (i * threads + t) * VEC + j.
template <typename T, int VEC> __device__ inline void ld(const T* p, float* v) {
  if constexpr (VEC == 1) v[0] = (float)*p;
  else {
    typedef T vt __attribute__((ext_vector_type(VEC)));
    const vt r = *reinterpret_cast<const vt*>(p);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = (float)r[j];
  }
}
template <typename T, int VEC> __device__ inline void st(T* p, const float* v) {
  if constexpr (VEC == 1) *p = (T)v[0];
  else {
    typedef T vt __attribute__((ext_vector_type(VEC)));
    vt r;
#pragma unroll
    for (int j = 0; j < VEC; ++j) r[j] = (T)v[j];
    *reinterpret_cast<vt*>(p) = r;
  }
}
template <typename T, int VEC> __device__ inline void ldp(const void* p, int dt, long i, float* v) {   // parameter: T or fp32
  if (DtOf<T>::v == DT_F32 || dt != DT_F32) ld<T, VEC>(static_cast<const T*>(p) + i, v);
  else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = static_cast<const float*>(p)[i + j];
  }
}

template <int CTRL, int ROWS> __device__ inline float dpp_add(float x) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
}
// sum over the 64 lanes, in every lane: row_shr 1, 2, 4, 8, row_bcast 15, 31 leave it in lane 63
__device__ inline float wave_sum(float x) {
  x = dpp_add<0x111, 0xf>(x);
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);
  x = dpp_add<0x143, 0xc>(x);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
// over the NW waves of a unit (NW > 1: the whole workgroup); `buf` alternates between two blocks of 2 * NW floats
template <int NW> __device__ inline void unit_sum(float& a, float& b, float* buf, int& turn) {
  a = wave_sum(a);
  b = wave_sum(b);
  if constexpr (NW > 1) {
    float* p = buf + turn * 2 * NW;
    turn ^= 1;
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) { p[w] = a; p[NW + w] = b; }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) { a += p[i]; b += p[NW + i]; }
  }
}

template <typename T, int VEC, int IT, int NW> struct Row {
  static constexpr int NT = 64 * NW, E = VEC * IT;
  static constexpr int kThreads = NW > 4 ? 64 * NW : 256, kUnits = kThreads / NT;
  static __device__ inline int col(int i) { return (i * NT + (int)threadIdx.x % NT) * VEC; }
  template <typename F> static __device__ inline void each(int C, F&& f) {
#pragma unroll
    for (int i = 0; i < IT; ++i)
      if (col(i) < C) f(col(i), i * VEC);
  }
};

// mean (RMSNorm: 0) and 1 / sqrt(variance + eps) of a row
template <typename R, int VEC, int NW> __device__ inline void stats_of(const float* v, const NormArgs& a, float* buf, int& turn, float& mean, float& rstd) {
  float s = 0.f, none = 0.f;
  mean = 0.f;
  if (!a.rms) {
    R::each(a.C, [&](int, int e) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) s += v[e + j];
    });
    unit_sum<NW>(s, none, buf, turn);
    mean = s * a.inv_c;
  }
  float q = 0.f;
  R::each(a.C, [&](int, int e) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) { const float d = v[e + j] - mean; q = __builtin_fmaf(d, d, q); }
  });
  none = 0.f;
  unit_sum<NW>(q, none, buf, turn);
  rstd = 1.f / sqrtf(q * a.inv_c + a.eps);
}

// h (holding x) <- a x + g n
template <typename R, int VEC> __device__ inline void gate_and_add(const NormArgs& a, const float (&g)[R::E], const float (&n)[R::E], float (&h)[R::E]) {
  R::each(a.C, [&](int, int e) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) h[e + j] = __builtin_fmaf(a.a, h[e + j], a.gate ? g[e + j] * n[e + j] : n[e + j]);
  });
}
template <typename T, typename R, int VEC>
__device__ inline void affine(const NormArgs& a, const void* w, const void* b, float mean, float rstd, float* v) {
  R::each(a.C, [&](int c, int e) {
    float wv[VEC], bv[VEC];
    ldp<T, VEC>(w, a.pdt, c, wv);
    if (b) ldp<T, VEC>(b, a.pdt, c, bv);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[e + j] = __builtin_fmaf((v[e + j] - mean) * rstd, wv[j], b ? bv[j] : 0.f);
  });
}

template <typename T, int VEC, int IT, int NW>
__global__ __launch_bounds__((Row<T, VEC, IT, NW>::kThreads)) void k_resnorm_fwd(NormArgs a) {
  typedef Row<T, VEC, IT, NW> R;
  __shared__ float buf[NW > 1 ? 4 * NW : 1];
  int turn = 0;
  const int unit = threadIdx.x / R::NT;
  for (long row = (long)blockIdx.x * R::kUnits + unit; row < a.N; row += (long)gridDim.x * R::kUnits) {
    const long o = row * a.C;
    float x[R::E], n[R::E], g[R::E];
    R::each(a.C, [&](int c, int e) {
      ld<T, VEC>(static_cast<const T*>(a.x) + o + c, x + e);
      ld<T, VEC>(static_cast<const T*>(a.block) + o + c, n + e);
      if (a.gate) ldp<T, VEC>(a.gate, a.gdt, row / a.gate_rows * a.C + c, g + e);
    });
    float m0 = 0.f, r0 = 0.f, m1 = 0.f, r1 = 0.f;
    if (a.has_post) {
      stats_of<R, VEC, NW>(n, a, buf, turn, m0, r0);
      affine<T, R, VEC>(a, a.post_w, a.post_b, m0, r0, n);
    }
    gate_and_add<R, VEC>(a, g, n, x);
    R::each(a.C, [&](int c, int e) { st<T, VEC>(static_cast<T*>(a.h) + o + c, x + e); });
    if (a.has_pre) {
      stats_of<R, VEC, NW>(x, a, buf, turn, m1, r1);
      affine<T, R, VEC>(a, a.pre_w, a.pre_b, m1, r1, x);
      R::each(a.C, [&](int c, int e) { st<T, VEC>(static_cast<T*>(a.y) + o + c, x + e); });
    }
    if (a.stats && threadIdx.x % R::NT == 0) *reinterpret_cast<f32x4*>(a.stats + 4 * row) = f32x4{m0, r0, m1, r1};
  }
}

// sums over rows that a workgroup leaves: slot 0 dgate, 1 dpre_w, 2 dpre_b, 3 dpost_w, 4 dpost_b (those in `slots`)
template <typename T, int VEC, int IT, int NW>
__global__ __launch_bounds__((Row<T, VEC, IT, NW>::kThreads)) void k_resnorm_bwd(NormArgs a) {
  typedef Row<T, VEC, IT, NW> R;
  constexpr int E = R::E;
  __shared__ float buf[NW > 1 ? 4 * NW : 1];
  __shared__ float red[R::kUnits > 1 ? R::NT * VEC : 1];
  int turn = 0;
  const int unit = threadIdx.x / R::NT;
  // this unit's rows: r, r + step, ... < end
  long r, end, step;
  if (a.flush) {
    const long units = (long)gridDim.x * R::kUnits, per = (a.groups + units - 1) / units, u = (long)blockIdx.x * R::kUnits + unit;
    r = min(u * per, a.groups) * a.rows_per_group;
    end = min((u + 1) * per, a.groups) * a.rows_per_group;
    step = 1;
  } else {
    const long grp = blockIdx.x / a.cuts, cut = blockIdx.x % a.cuts, per = (a.rows_per_group + a.cuts - 1) / a.cuts;
    r = grp * a.rows_per_group + min(cut * per, a.rows_per_group) + unit;
    end = grp * a.rows_per_group + min((cut + 1) * per, a.rows_per_group);
    step = R::kUnits;
  }
  float sum[5][E];
#pragma unroll
  for (int s = 0; s < 5; ++s)
#pragma unroll
    for (int e = 0; e < E; ++e) sum[s][e] = 0.f;

  // units of one wave may run out of rows at different times: none of them waits for another one in the loop (NW > 1: one unit per workgroup)
  for (; r < end; r += step) {
    const long o = r * a.C;
    float h[E], n[E], g[E], gh[E], gy[E];
    R::each(a.C, [&](int c, int e) {
      if (a.has_pre) ld<T, VEC>(static_cast<const T*>(a.x) + o + c, h + e);
      ld<T, VEC>(static_cast<const T*>(a.block) + o + c, n + e);
      if (a.gate) ldp<T, VEC>(a.gate, a.gdt, r / a.gate_rows * a.C + c, g + e);
      if (a.gh) ld<T, VEC>(static_cast<const T*>(a.gh) + o + c, gh + e);
      if (a.gy) ld<T, VEC>(static_cast<const T*>(a.gy) + o + c, gy + e);
    });
    const f32x4 ms = *reinterpret_cast<const f32x4*>(a.stats + 4 * r);
    const float m0 = ms[0], r0 = ms[1], m1 = ms[2], r1 = ms[3];
    if (a.has_post) affine<T, R, VEC>(a, a.post_w, a.post_b, m0, r0, n);
    float dh[E];
    if (a.gy) {
      gate_and_add<R, VEC>(a, g, n, h);
      float s1 = 0.f, s2 = 0.f;
      R::each(a.C, [&](int c, int e) {
        float w[VEC];
        ldp<T, VEC>(a.pre_w, a.pdt, c, w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float hat = (h[e + j] - m1) * r1;
          sum[1][e + j] = __builtin_fmaf(gy[e + j], hat, sum[1][e + j]);
          sum[2][e + j] += gy[e + j];
          gy[e + j] *= w[j];
          h[e + j] = hat;
          s1 += gy[e + j];
          s2 = __builtin_fmaf(gy[e + j], hat, s2);
        }
      });
      unit_sum<NW>(s1, s2, buf, turn);
      s1 = a.rms ? 0.f : s1 * a.inv_c;
      s2 *= a.inv_c;
      R::each(a.C, [&](int, int e) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) dh[e + j] = __builtin_fmaf(r1, gy[e + j] - s1 - h[e + j] * s2, a.gh ? gh[e + j] : 0.f);
      });
    } else {
      R::each(a.C, [&](int, int e) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) dh[e + j] = a.gh ? gh[e + j] : 0.f;
      });
    }
    R::each(a.C, [&](int c, int e) {
      float v[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = a.a * dh[e + j];
      st<T, VEC>(static_cast<T*>(a.dx) + o + c, v);
    });
    if (a.gate) {
      R::each(a.C, [&](int c, int e) {
        float v[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          v[j] = dh[e + j] * n[e + j];
          sum[0][e + j] += v[j];
          dh[e + j] *= g[e + j];   // dn
        }
        if (a.gate_rows == 1) {
          if (a.gdt == DT_F32) st<float, VEC>(static_cast<float*>(a.dgate) + o + c, v);
          else st<T, VEC>(static_cast<T*>(a.dgate) + o + c, v);
        }
      });
      if (a.flush && (r + 1) % a.rows_per_group == 0) {
        R::each(a.C, [&](int c, int e) {
          const long at = r / a.rows_per_group * a.C + c;
          if (a.gdt == DT_F32) st<float, VEC>(static_cast<float*>(a.dgate) + at, sum[0] + e);
          else st<T, VEC>(static_cast<T*>(a.dgate) + at, sum[0] + e);
#pragma unroll
          for (int j = 0; j < VEC; ++j) sum[0][e + j] = 0.f;
        });
      }
    }
    if (a.has_post) {
      // block again (its registers became n)
      float s1 = 0.f, s2 = 0.f;
      R::each(a.C, [&](int c, int e) {
        float w[VEC], b[VEC];
        ldp<T, VEC>(a.post_w, a.pdt, c, w);
        ld<T, VEC>(static_cast<const T*>(a.block) + o + c, b);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float hat = (b[j] - m0) * r0;
          sum[3][e + j] = __builtin_fmaf(dh[e + j], hat, sum[3][e + j]);
          sum[4][e + j] += dh[e + j];
          dh[e + j] *= w[j];
          n[e + j] = hat;
          s1 += dh[e + j];
          s2 = __builtin_fmaf(dh[e + j], hat, s2);
        }
      });
      unit_sum<NW>(s1, s2, buf, turn);
      s1 = a.rms ? 0.f : s1 * a.inv_c;
      s2 *= a.inv_c;
      R::each(a.C, [&](int, int e) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) dh[e + j] = r0 * (dh[e + j] - s1 - n[e + j] * s2);
      });
    }
    if (!a.same_dx) R::each(a.C, [&](int c, int e) { st<T, VEC>(static_cast<T*>(a.dblock) + o + c, dh + e); });
  }

  // the workgroup's sums, unit by unit
#pragma unroll
  for (int s = 0; s < 5; ++s) {
    if (!((a.slots >> s) & 1)) continue;
    float* const out = a.part + ((long)blockIdx.x * 5 + s) * a.C;
    if constexpr (R::kUnits == 1) {
      R::each(a.C, [&](int c, int e) { st<float, VEC>(out + c, sum[s] + e); });
    } else {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int t = (int)threadIdx.x % R::NT;
        for (int u = 0; u < R::kUnits; ++u) {
          if (unit == u) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) red[t * VEC + j] = (u ? red[t * VEC + j] : 0.f) + sum[s][i * VEC + j];
          }
          __syncthreads();
        }
        if (unit == 0 && R::col(i) < a.C) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) out[R::col(i) + j] = red[t * VEC + j];
        }
        __syncthreads();
      }
    }
  }
}

// the workgroups' sums joined in their order.  y: which output (sum over everything) or, behind those, which gate row
struct NormJoin {
  const float* part;
  void* out[5];
  int dt[5], C, wgs, gate_cuts;   // gate_cuts: workgroups per gate row (slot 0 with more than one row), 0: as the others
  int n_out, slot[5];
};
template <typename T> __global__ __launch_bounds__(256) void k_resnorm_join(NormJoin a) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  int s, first = 0, last = a.wgs, k;
  long row = 0;
  if ((int)blockIdx.y < a.n_out) { k = blockIdx.y; s = a.slot[k]; }
  else { s = 0; k = a.n_out; row = (int)blockIdx.y - a.n_out; first = (int)row * a.gate_cuts; last = first + a.gate_cuts; }
  float v = 0.f;
  if (c < a.C)
    for (int i = first + w; i < last; i += 4) v += a.part[((long)i * 5 + s) * a.C + c];
  red[w][lane] = v;
  __syncthreads();
  if (w == 0 && c < a.C) {
    v = red[0][lane] + red[1][lane] + red[2][lane] + red[3][lane];
    if (a.dt[k] == DT_F32) static_cast<float*>(a.out[k])[row * a.C + c] = v;
    else static_cast<T*>(a.out[k])[row * a.C + c] = (T)v;
  }
}

// ---------------------------------------------------------------------------------------------------------------- launches
const char* check(const fdx_resnorm_desc* d) {
  if (!d) return "null descriptor";
  if (d->dtype < 0 || d->dtype > 2 || (d->param_dtype != DT_F32 && d->param_dtype != d->dtype) || (d->gate_dtype != DT_F32 && d->gate_dtype != d->dtype))
    return "dtype must be FDX_F32, FDX_BF16 or FDX_F16, the parameters' and the gate's the same or FDX_F32";
  if (d->rows < 0 || d->channels < 1 || d->channels > 8192) return "channels must be 1 ... 8192";
  if (d->gate_rows < 0 || (d->gate_rows > 0 && d->rows % d->gate_rows)) return "gate_rows must divide rows";
  if (d->rows > (1LL << 40)) return "too many rows";
  return nullptr;
}

// Cut of the backward pass.  About a thousand workgroups fill the chip four times over; a gate row is never shared by two cuts of another one.
// Gate rows shorter than 8 rows per unit are summed and written where they are read.
struct Cut { int wgs, cuts, flush; long groups, per; };
Cut cut_of(const fdx_resnorm_desc* d, int units) {
  Cut c{};
  const long N = d->rows, want = std::max<long>(1, std::min<long>(1024, (N + 4 * units - 1) / (4 * units)));
  const bool many = d->gate_rows > 1 && d->gate_rows < N;
  c.groups = many ? N / d->gate_rows : 1;
  c.per = many ? d->gate_rows : N;
  c.flush = many && c.groups >= want;
  if (c.flush) { c.wgs = (int)std::max<long>(1, std::min<long>(want, (c.groups + units - 1) / units)); c.cuts = 1; }
  else {
    c.cuts = (int)std::max<long>(1, std::min<long>(want / c.groups, (c.per + units - 1) / units));
    c.wgs = (int)c.groups * c.cuts;
  }
  return c;
}

struct Shape { int vec, it, nw; };   // pieces of a row per thread and waves per row
Shape shape_of(const fdx_resnorm_desc* d, bool vec, bool bwd) {
  const int v = !vec ? 1 : d->dtype == DT_F32 ? 4 : 8, C = d->channels;
  const int per1 = bwd ? 16 : 32;   // channels a thread may hold with one wave per row
  if (C <= 64 * 8) return {v, 8 / v, 1};
  if (C <= 64 * 16) return {v, 16 / v, 1};
  if (C <= 64 * per1) return {v, 32 / v, 1};
  if (C <= 256 * 16) return {v, 16 / v, 4};
  return {v, 16 / v, 8};
}

template <typename T, int VEC, bool BWD, int IT, int NW> hipError_t run(const NormArgs& a, unsigned grid, hipStream_t s) {
  if constexpr (BWD) return launch(k_resnorm_bwd<T, VEC, IT, NW>, grid, Row<T, VEC, IT, NW>::kThreads, a, s);
  else return launch(k_resnorm_fwd<T, VEC, IT, NW>, grid, Row<T, VEC, IT, NW>::kThreads, a, s);
}
template <typename T, int VEC, bool BWD> hipError_t run(const NormArgs& a, Shape sh, unsigned grid, hipStream_t s) {
  constexpr int A = 8 / VEC, B = 16 / VEC, D = 32 / VEC;
  if (sh.nw == 1 && sh.it == A) return run<T, VEC, BWD, A, 1>(a, grid, s);
  if (sh.nw == 1 && sh.it == B) return run<T, VEC, BWD, B, 1>(a, grid, s);
  if constexpr (!BWD)
    if (sh.nw == 1) return run<T, VEC, BWD, D, 1>(a, grid, s);
  if (sh.nw == 4) return run<T, VEC, BWD, B, 4>(a, grid, s);
  return run<T, VEC, BWD, B, 8>(a, grid, s);
}
template <bool BWD> hipError_t by_type(const fdx_resnorm_desc* d, const NormArgs& a, Shape sh, unsigned grid, hipStream_t s) {
  const bool one = sh.vec == 1;
  if (d->dtype == DT_F32) return one ? run<float, 1, BWD>(a, sh, grid, s) : run<float, 4, BWD>(a, sh, grid, s);
  if (d->dtype == DT_BF16) return one ? run<bf16_t, 1, BWD>(a, sh, grid, s) : run<bf16_t, 8, BWD>(a, sh, grid, s);
  return one ? run<f16_t, 1, BWD>(a, sh, grid, s) : run<f16_t, 8, BWD>(a, sh, grid, s);
}
int units_of(Shape sh) { return sh.nw == 1 ? 4 : 1; }

NormArgs args_of(const fdx_resnorm_desc* d) {
  NormArgs a{};
  a.N = d->rows; a.C = d->channels; a.gate_rows = d->gate_rows; a.pdt = d->param_dtype; a.gdt = d->gate_dtype; a.rms = d->rms != 0;
  a.a = d->residual_scale; a.eps = d->eps; a.inv_c = 1.f / (float)d->channels;
  return a;
}
bool vec_ok(const fdx_resnorm_desc* d, std::initializer_list<const void*> ps) {
  if (d->channels % 8) return false;
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & 15) return false;
  return true;
}

}  // namespace

extern "C" int fdx_resnorm_forward(fdx_handle h, const fdx_resnorm_desc* d, const void* x, const void* block, const void* gate, const void* post_w,
                                   const void* post_b, const void* pre_w, const void* pre_b, void* out_h, void* out_y, float* stats, fdx_stream st) {
  if (!h) return fail(nullptr, FDX_E_ARG, "fdx_resnorm_forward: null handle");
  if (const char* why = check(d)) return fail(h, FDX_E_ARG, "fdx_resnorm_forward: %s", why);
  if (d->rows == 0) return FDX_OK;
  if (!x || !block || !out_h || (pre_w && !out_y) || (d->gate_rows > 0) != (gate != nullptr) || (post_b && !post_w) || (pre_b && !pre_w) ||
      (reinterpret_cast<uintptr_t>(stats) & 15))
    return fail(h, FDX_E_ARG, "fdx_resnorm_forward: null tensor, or gate_rows / weights that do not fit the tensors given");
  NormArgs a = args_of(d);
  a.x = x; a.block = block; a.gate = gate; a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.pre_b = pre_b;
  a.h = out_h; a.y = out_y; a.stats = stats; a.has_post = post_w != nullptr; a.has_pre = pre_w != nullptr;
  const Shape sh = shape_of(d, vec_ok(d, {x, block, gate, post_w, post_b, pre_w, pre_b, out_h, out_y}), false);
  const long units = units_of(sh), grid = std::min<long>((d->rows + units - 1) / units, 1L << 20);
  DeviceScope dev(h->device);
  FDX_HIP(h, dev.err);
  FDX_HIP(h, by_type<false>(d, a, sh, (unsigned)grid, as_stream(st)));
  return FDX_OK;
}

// (the larger of the two shapes the launch may take: the workspace does not depend on the tensors' alignment)
extern "C" int fdx_resnorm_backward_workspace(const fdx_resnorm_desc* d, size_t* bytes) {
  if (const char* why = check(d)) return fail(nullptr, FDX_E_ARG, "fdx_resnorm_backward_workspace: %s", why);
  if (!bytes) return fail(nullptr, FDX_E_ARG, "fdx_resnorm_backward_workspace: null size pointer");
  size_t n = 0;
  for (bool vec : {false, true}) n = std::max<size_t>(n, cut_of(d, units_of(shape_of(d, vec, true))).wgs);
  *bytes = n * 5 * d->channels * sizeof(float);
  return FDX_OK;
}

extern "C" int fdx_resnorm_backward(fdx_handle h, const fdx_resnorm_desc* d, const void* grad_h, const void* grad_y, const void* x, const void* block,
                                    const void* gate, const void* post_w, const void* post_b, const void* pre_w, const void* pre_b, const float* stats,
                                    void* dx, void* dblock, void* dgate, void* dpost_w, void* dpost_b, void* dpre_w, void* dpre_b, void* workspace,
                                    size_t bytes, fdx_stream st) {
  if (!h) return fail(nullptr, FDX_E_ARG, "fdx_resnorm_backward: null handle");
  if (const char* why = check(d)) return fail(h, FDX_E_ARG, "fdx_resnorm_backward: %s", why);
  if ((grad_y && !pre_w) || (d->gate_rows > 0) != (dgate != nullptr) || (post_w != nullptr) != (dpost_w != nullptr) || (dpre_w && !pre_w) ||
      (dpost_b && !post_b) || (dpre_b && !pre_b) || (post_b && !post_w) || (pre_b && !pre_w))
    return fail(h, FDX_E_ARG, "fdx_resnorm_backward: gradients that do not fit the tensors given");
  if (d->rows > 0 && (!x || !block || !stats || (reinterpret_cast<uintptr_t>(stats) & 15) || !dx || !dblock || (d->gate_rows > 0 && !gate)))
    return fail(h, FDX_E_ARG, "fdx_resnorm_backward: null tensor (or stats not 16-byte aligned)");
  NormArgs a = args_of(d);
  a.x = x; a.block = block; a.gate = gate; a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.pre_b = pre_b;
  a.gh = grad_h; a.gy = grad_y; a.stats = const_cast<float*>(stats); a.dx = dx; a.dblock = dblock; a.dgate = dgate;
  a.has_post = post_w != nullptr; a.has_pre = grad_y != nullptr;
  a.same_dx = dblock == dx;
  if (a.same_dx && (post_w || gate || d->residual_scale != 1.f))
    return fail(h, FDX_E_ARG, "fdx_resnorm_backward: dblock may be dx only where they are equal (no gate, no post norm, residual_scale 1)");
  const Shape sh = shape_of(d, vec_ok(d, {x, block, gate, post_w, post_b, pre_w, pre_b, grad_h, grad_y, dx, dblock, dgate}), true);
  const Cut c = cut_of(d, units_of(sh));
  const size_t need = (size_t)c.wgs * 5 * d->channels * sizeof(float);
  if (bytes < need || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return fail(h, FDX_E_ARG, "fdx_resnorm_backward: workspace of %zu bytes, %zu needed (16-byte aligned)", bytes, need);
  a.part = static_cast<float*>(workspace);
  a.groups = c.groups; a.rows_per_group = c.per; a.cuts = c.cuts; a.flush = c.flush;
  NormJoin j{};
  j.part = a.part; j.C = d->channels; j.wgs = c.wgs;
  auto add = [&](int slot, void* out, int dt) {
    if (!out) return;
    a.slots |= 1 << slot;
    j.slot[j.n_out] = slot; j.out[j.n_out] = out; j.dt[j.n_out++] = dt;
  };
  add(1, dpre_w, d->param_dtype); add(2, dpre_b, d->param_dtype); add(3, dpost_w, d->param_dtype); add(4, dpost_b, d->param_dtype);
  int gate_out = 0;   // gate rows the second launch writes
  if (dgate && d->gate_rows != 1 && !c.flush) {
    a.slots |= 1;
    if (c.groups == 1) { j.slot[j.n_out] = 0; j.out[j.n_out] = dgate; j.dt[j.n_out++] = d->gate_dtype; }
    else { gate_out = (int)c.groups; j.gate_cuts = c.cuts; j.out[j.n_out] = dgate; j.dt[j.n_out] = d->gate_dtype; }
  }
  DeviceScope dev(h->device);
  FDX_HIP(h, dev.err);
  FDX_HIP(h, by_type<true>(d, a, sh, (unsigned)c.wgs, as_stream(st)));
  if (j.n_out + gate_out > 0) {
    const dim3 grid((d->channels + 63) / 64, j.n_out + gate_out);
    void* argv[] = {&j};
    const void* k = d->dtype == DT_BF16 ? reinterpret_cast<const void*>(k_resnorm_join<bf16_t>)
                    : d->dtype == DT_F16 ? reinterpret_cast<const void*>(k_resnorm_join<f16_t>) : reinterpret_cast<const void*>(k_resnorm_join<float>);
    FDX_HIP(h, hipLaunchKernel(k, grid, dim3(256), argv, 0, as_stream(st)));
  }
  return FDX_OK;
}
