// resnorm.hip -- the step between two blocks of a network in one launch each way (fdx_resnorm_*):
//
//   n = post(block)      h = a x + g n      y = pre(h)          post, pre: LayerNorm, RMSNorm or nothing; g: nothing or a gate
//
//   dh = grad_h + pre'(grad_y)   dx = a dh   dn = g dh   dblock = post'(dn)   dg = sum dh n
//   norm'(gy): w = gy weight, r (w - mean(w) - hat mean(w hat))   (RMSNorm: without mean(w));   dweight = sum gy hat, dbias = sum gy
//
// Bound by memory: forward reads x, block, writes h, y; backward reads x, block, grad_h, grad_y and writes dx, dblock.  n, h and both normalised
// tensors are computed again from x and block in fp32 (reading h, y instead of x would cost the same bytes and add their rounding); the forward
// leaves mean and 1 / deviation of both norms (16 bytes a row).  One wave holds a row of up to 512 channels in registers, 2, 4 or 8 waves
// a longer one; means are taken before the squares are summed (two passes over registers).  The sums over rows run per thread in row order,
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
template <typename T, int VEC> struct Piece {   // as loaded
  typedef T vt __attribute__((ext_vector_type(VEC)));
  vt v;
  __device__ inline void load(const T* p) { v = *reinterpret_cast<const vt*>(p); }
  __device__ inline float at(int j) const { return (float)v[j]; }
};
template <typename T> struct Piece<T, 1> {
  T v;
  __device__ inline void load(const T* p) { v = *p; }
  __device__ inline float at(int) const { return (float)v; }
};
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
  if (DtOf<T>::v == DT_F32 || dt != DT_F32) {
    Piece<T, VEC> r;
    r.load(static_cast<const T*>(p) + i);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = r.at(j);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = static_cast<const float*>(p)[i + j];
  }
}
template <typename T, int VEC> __device__ inline void stp(void* p, int dt, long i, const float* v) {
  if (DtOf<T>::v == DT_F32 || dt != DT_F32) st<T, VEC>(static_cast<T*>(p) + i, v);
  else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) static_cast<float*>(p)[i + j] = v[j];
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

template <typename T, int VEC_, int IT_, int NW_> struct Row {
  static constexpr int VEC = VEC_, IT = IT_, NW = NW_, NT = 64 * NW, E = VEC * IT;
  static constexpr int kThreads = NW > 1 ? NT : 256, kUnits = kThreads / NT;   // NW > 1: one row at a time per workgroup
  typedef Piece<T, VEC> Raw[IT];
  static __device__ inline int col(int i) { return (i * NT + (int)threadIdx.x % NT) * VEC; }
  template <typename F> static __device__ inline void each(int C, F&& f) {
#pragma unroll
    for (int i = 0; i < IT; ++i)
      if (col(i) < C) f(col(i), i * VEC);
  }
  static __device__ inline void load(Raw& r, const void* p, long o, int C) {
#pragma unroll
    for (int i = 0; i < IT; ++i)
      if (col(i) < C) r[i].load(static_cast<const T*>(p) + o + col(i));
  }
  static __device__ inline void widen(const Raw& r, float (&v)[E]) {
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i * VEC + j] = r[i].at(j);
  }
  static __device__ inline void param(const void* p, int dt, int C, float other, float (&v)[E]) {   // `other` where there is none
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = other;
    if (p) each(C, [&](int c, int e) { ldp<T, VEC>(p, dt, c, v + e); });
  }
  // sums over the row's waves; `buf` alternates between two blocks of 2 * NW floats
  static __device__ inline void sum(float& a, float& b, float* buf, int& turn) {
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
  // mean (RMSNorm: 0) and 1 / sqrt(variance + eps)
  static __device__ inline void stats(const float (&v)[E], const NormArgs& a, float* buf, int& turn, float& mean, float& rstd) {
    float s = 0.f, none = 0.f;
    mean = 0.f;
    if (!a.rms) {
      each(a.C, [&](int, int e) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += v[e + j];
      });
      sum(s, none, buf, turn);
      mean = s * a.inv_c;
    }
    float q = 0.f;
    each(a.C, [&](int, int e) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) { const float d = v[e + j] - mean; q = __builtin_fmaf(d, d, q); }
    });
    none = 0.f;
    sum(q, none, buf, turn);
    rstd = 1.f / sqrtf(q * a.inv_c + a.eps);
  }
};

// Rows are taken in turn by a fixed number of units, the next row's loads issued before this one's sums: with two workgroups on a CU and a barrier per
// sum the loads' latency is what costs otherwise.  The norms' parameters stay in registers.
template <typename T, int VEC, int IT, int NW>
__global__ __launch_bounds__((Row<T, VEC, IT, NW>::kThreads)) void k_resnorm_fwd(NormArgs a) {
  typedef Row<T, VEC, IT, NW> R;
  constexpr int E = R::E;
  __shared__ float buf[NW > 1 ? 4 * NW : 1];
  int turn = 0;
  float pw[E], pb[E], nw[E], nb[E];
  R::param(a.post_w, a.pdt, a.C, 1.f, pw);
  R::param(a.post_b, a.pdt, a.C, 0.f, pb);
  R::param(a.pre_w, a.pdt, a.C, 1.f, nw);
  R::param(a.pre_b, a.pdt, a.C, 0.f, nb);
  const long step = (long)gridDim.x * R::kUnits;
  long row = (long)blockIdx.x * R::kUnits + threadIdx.x / R::NT;
  typename R::Raw rx, rb;
  if (row < a.N) {
    R::load(rx, a.x, row * a.C, a.C);
    R::load(rb, a.block, row * a.C, a.C);
  }
  for (; row < a.N; row += step) {
    const long o = row * a.C;
    float x[E], n[E];
    R::widen(rx, x);
    R::widen(rb, n);
    float g[E];
    if (a.gate) {
      const long at = a.gate_rows == 1 ? o : a.gate_rows == a.N ? 0 : row / a.gate_rows * a.C;
      R::each(a.C, [&](int c, int e) { ldp<T, VEC>(a.gate, a.gdt, at + c, g + e); });
    }
    if (row + step < a.N) {
      R::load(rx, a.x, (row + step) * a.C, a.C);
      R::load(rb, a.block, (row + step) * a.C, a.C);
    }
    float m0 = 0.f, r0 = 0.f, m1 = 0.f, r1 = 0.f;
    if (a.has_post) {
      R::stats(n, a, buf, turn, m0, r0);
#pragma unroll
      for (int e = 0; e < E; ++e) n[e] = __builtin_fmaf((n[e] - m0) * r0, pw[e], pb[e]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = __builtin_fmaf(a.a, x[e], a.gate ? g[e] * n[e] : n[e]);
    if (a.h) R::each(a.C, [&](int c, int e) { st<T, VEC>(static_cast<T*>(a.h) + o + c, x + e); });
    if (a.has_pre) {
      R::stats(x, a, buf, turn, m1, r1);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = __builtin_fmaf((x[e] - m1) * r1, nw[e], nb[e]);
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
  float sum[5][E], pw[E], pb[E], nw[E];
#pragma unroll
  for (int s = 0; s < 5; ++s)
#pragma unroll
    for (int e = 0; e < E; ++e) sum[s][e] = 0.f;
  R::param(a.post_w, a.pdt, a.C, 1.f, pw);
  R::param(a.post_b, a.pdt, a.C, 0.f, pb);
  R::param(a.pre_w, a.pdt, a.C, 1.f, nw);
  typename R::Raw rx, rb, rh, ry;
  f32x4 ms = {0, 0, 0, 0};
  auto fetch = [&](long row) {
    const long o = row * a.C;
    if (a.gy) { R::load(rx, a.x, o, a.C); R::load(ry, a.gy, o, a.C); }
    R::load(rb, a.block, o, a.C);
    if (a.gh) R::load(rh, a.gh, o, a.C);
    ms = *reinterpret_cast<const f32x4*>(a.stats + 4 * row);
  };
  if (r < end) fetch(r);
  // units of one wave may run out of rows at different times: none of them waits for another one in the loop (NW > 1: one unit per workgroup)
  for (; r < end; r += step) {
    const long o = r * a.C;
    const float m0 = ms[0], r0 = ms[1], m1 = ms[2], r1 = ms[3];
    float h[E], bhat[E], gy[E], dh[E], g[E];
    R::widen(rb, bhat);
#pragma unroll
    for (int e = 0; e < E; ++e) dh[e] = 0.f;
    if (a.gh) R::widen(rh, dh);
    if (a.gy) { R::widen(rx, h); R::widen(ry, gy); }
    if (a.gate) {
      const long at = a.gate_rows == 1 ? o : a.gate_rows == a.N ? 0 : r / a.gate_rows * a.C;
      R::each(a.C, [&](int c, int e) { ldp<T, VEC>(a.gate, a.gdt, at + c, g + e); });
    }
    if (r + step < end) fetch(r + step);
    if (a.has_post) {
#pragma unroll
      for (int e = 0; e < E; ++e) bhat[e] = (bhat[e] - m0) * r0;
    }
    auto n = [&](int e) { return a.has_post ? __builtin_fmaf(bhat[e], pw[e], pb[e]) : bhat[e]; };
    if (a.gy) {
      float s1 = 0.f, s2 = 0.f;
      R::each(a.C, [&](int, int e0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int e = e0 + j;
          h[e] = (__builtin_fmaf(a.a, h[e], a.gate ? g[e] * n(e) : n(e)) - m1) * r1;   // normalised h
          sum[1][e] = __builtin_fmaf(gy[e], h[e], sum[1][e]);
          sum[2][e] += gy[e];
          gy[e] *= nw[e];
          s1 += gy[e];
          s2 = __builtin_fmaf(gy[e], h[e], s2);
        }
      });
      R::sum(s1, s2, buf, turn);
      s1 = a.rms ? 0.f : s1 * a.inv_c;
      s2 *= a.inv_c;
#pragma unroll
      for (int e = 0; e < E; ++e) dh[e] = __builtin_fmaf(r1, gy[e] - s1 - h[e] * s2, dh[e]);
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
          v[j] = dh[e + j] * n(e + j);
          sum[0][e + j] += v[j];
          dh[e + j] *= g[e + j];   // dn
        }
        if (a.gate_rows == 1) stp<T, VEC>(a.dgate, a.gdt, o + c, v);
      });
      if (a.flush && (r + 1) % a.rows_per_group == 0) {
        R::each(a.C, [&](int c, int e) {
          stp<T, VEC>(a.dgate, a.gdt, r / a.rows_per_group * a.C + c, sum[0] + e);
#pragma unroll
          for (int j = 0; j < VEC; ++j) sum[0][e + j] = 0.f;
        });
      }
    }
    if (a.has_post) {
      float s1 = 0.f, s2 = 0.f;
      R::each(a.C, [&](int, int e0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int e = e0 + j;
          sum[3][e] = __builtin_fmaf(dh[e], bhat[e], sum[3][e]);
          sum[4][e] += dh[e];
          dh[e] *= pw[e];
          s1 += dh[e];
          s2 = __builtin_fmaf(dh[e], bhat[e], s2);
        }
      });
      R::sum(s1, s2, buf, turn);
      s1 = a.rms ? 0.f : s1 * a.inv_c;
      s2 *= a.inv_c;
#pragma unroll
      for (int e = 0; e < E; ++e) dh[e] = r0 * (dh[e] - s1 - bhat[e] * s2);
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
// A workgroup: 32 channels, 32 threads each; a thread sums every 32nd partial row, eight loads in flight.
template <typename T> __global__ __launch_bounds__(1024) void k_resnorm_join(NormJoin a) {
  __shared__ float red[32][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  int s, first = 0, last = a.wgs, k;
  long row = 0;
  if ((int)blockIdx.y < a.n_out) { k = blockIdx.y; s = a.slot[k]; }
  else { s = 0; k = a.n_out; row = (int)blockIdx.y - a.n_out; first = (int)row * a.gate_cuts; last = first + a.gate_cuts; }
  float v = 0.f;
  if (c < a.C) {
    const float* p = a.part + (long)s * a.C + c;
    const long pitch = 5L * a.C;
    int i = first + w;
    for (; i + 7 * 32 < last; i += 8 * 32) {
      float t[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) t[q] = p[(i + q * 32) * pitch];
#pragma unroll
      for (int q = 0; q < 8; ++q) v += t[q];
    }
    for (; i < last; i += 32) v += p[i * pitch];
  }
  red[w][lane] = v;
  __syncthreads();
  if (w == 0 && c < a.C) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v += red[i][lane];
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

// 8 channels a thread (16 above 4096 channels) and as many waves as that takes: the backward pass holds five sums and five values per channel, and with 8 of
// them two waves fit on a SIMD.  (8 / 16 channels, backward, us: 16 x 861 x 512 fp32 30 / 55, 8 x 2048 x 2048 bf16 96 / 118.)
// Above 4096 channels the backward pass spills (1024 x 8192: fp32 134 us, bf16 53; reading the parameters again for every row and loading no row ahead does not
// save enough registers: 155, 56).
struct Shape { int vec, it, nw; };
Shape shape_of(const fdx_resnorm_desc* d, bool vec) {
  const int v = !vec ? 1 : d->dtype == DT_F32 ? 4 : 8, C = d->channels;
  return C <= 4096 ? Shape{v, 8 / v, C <= 512 ? 1 : C <= 1024 ? 2 : C <= 2048 ? 4 : 8} : Shape{v, 16 / v, 8};
}
int units_of(Shape sh) { return sh.nw == 1 ? 4 : 1; }   // rows a workgroup works on at a time

// Cut of the backward pass: as many workgroups as the chip holds (two waves on a SIMD), one round of them; a unit has four rows at least.  More or fewer leave
// places empty in the last round (256 / 384 / 512 / 768 / 1024 workgroups of four waves, us: 16 x 861 x 512 fp32 31.3 / 30.3 / 29.8 / 34.3 / 33.2,
// 8 x 2048 x 2048 bf16 129 / 120 / 96 / 118 / 100).  A gate row is never shared by two cuts of another one.
// Gate rows of which there are more than workgroups are summed and written where they are read.
struct Cut { int wgs, cuts, flush; long groups, per; };
Cut cut_of(const fdx_resnorm_desc* d, Shape sh) {
  Cut c{};
  const int units = units_of(sh);
  const long N = d->rows, room = 2048 / std::max(units, sh.nw), want = std::max<long>(1, std::min<long>(room, (N + 4 * units - 1) / (4 * units)));
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

template <typename T, int VEC, bool BWD, int IT, int NW> hipError_t run(const NormArgs& a, unsigned grid, hipStream_t s) {
  if constexpr (BWD) return launch(k_resnorm_bwd<T, VEC, IT, NW>, grid, Row<T, VEC, IT, NW>::kThreads, a, s);
  else return launch(k_resnorm_fwd<T, VEC, IT, NW>, grid, Row<T, VEC, IT, NW>::kThreads, a, s);
}
template <typename T, int VEC, bool BWD> hipError_t run(const NormArgs& a, Shape sh, unsigned grid, hipStream_t s) {
  constexpr int A = 8 / VEC, B = 16 / VEC;
  if (sh.it == B) return run<T, VEC, BWD, B, 8>(a, grid, s);
  if (sh.nw == 1) return run<T, VEC, BWD, A, 1>(a, grid, s);
  if (sh.nw == 2) return run<T, VEC, BWD, A, 2>(a, grid, s);
  if (sh.nw == 4) return run<T, VEC, BWD, A, 4>(a, grid, s);
  return run<T, VEC, BWD, A, 8>(a, grid, s);
}
template <bool BWD> hipError_t by_type(const fdx_resnorm_desc* d, const NormArgs& a, Shape sh, unsigned grid, hipStream_t s) {
  const bool one = sh.vec == 1;
  if (d->dtype == DT_F32) return one ? run<float, 1, BWD>(a, sh, grid, s) : run<float, 4, BWD>(a, sh, grid, s);
  if (d->dtype == DT_BF16) return one ? run<bf16_t, 1, BWD>(a, sh, grid, s) : run<bf16_t, 8, BWD>(a, sh, grid, s);
  return one ? run<f16_t, 1, BWD>(a, sh, grid, s) : run<f16_t, 8, BWD>(a, sh, grid, s);
}

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
  if (!x || !block || (!out_h && !pre_w) || (pre_w && !out_y) || (d->gate_rows > 0) != (gate != nullptr) || (post_b && !post_w) || (pre_b && !pre_w) ||
      (reinterpret_cast<uintptr_t>(stats) & 15))
    return fail(h, FDX_E_ARG, "fdx_resnorm_forward: null tensor, or gate_rows / weights that do not fit the tensors given");
  NormArgs a = args_of(d);
  a.x = x; a.block = block; a.gate = gate; a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.pre_b = pre_b;
  a.h = out_h; a.y = out_y; a.stats = stats; a.has_post = post_w != nullptr; a.has_pre = pre_w != nullptr;
  const Shape sh = shape_of(d, vec_ok(d, {x, block, gate, post_w, post_b, pre_w, pre_b, out_h, out_y}));
  const long units = units_of(sh), grid = std::min<long>((d->rows + units - 1) / units, 1024 * 4 / std::max(4, sh.nw));
  DeviceScope dev(h->device);
  FDX_HIP(h, dev.err);
  FDX_HIP(h, by_type<false>(d, a, sh, (unsigned)grid, as_stream(st)));
  return FDX_OK;
}

extern "C" int fdx_resnorm_backward_workspace(const fdx_resnorm_desc* d, size_t* bytes) {
  if (const char* why = check(d)) return fail(nullptr, FDX_E_ARG, "fdx_resnorm_backward_workspace: %s", why);
  if (!bytes) return fail(nullptr, FDX_E_ARG, "fdx_resnorm_backward_workspace: null size pointer");
  *bytes = (size_t)cut_of(d, shape_of(d, true)).wgs * 5 * d->channels * sizeof(float);
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
  const Shape sh = shape_of(d, vec_ok(d, {x, block, gate, post_w, post_b, pre_w, pre_b, grad_h, grad_y, dx, dblock, dgate}));
  const Cut c = cut_of(d, sh);
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
    const dim3 grid((d->channels + 31) / 32, j.n_out + gate_out);
    void* argv[] = {&j};
    const void* k = d->dtype == DT_BF16 ? reinterpret_cast<const void*>(k_resnorm_join<bf16_t>)
                    : d->dtype == DT_F16 ? reinterpret_cast<const void*>(k_resnorm_join<f16_t>) : reinterpret_cast<const void*>(k_resnorm_join<float>);
    FDX_HIP(h, hipLaunchKernel(k, grid, dim3(1024), argv, 0, as_stream(st)));
  }
  return FDX_OK;
}
