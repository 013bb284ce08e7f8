// attention.hip -- attention with its backward pass, as callable operators (fdx_attn_*).
//
//   s_ij = scale q_i.k_j (-inf where key j is masked, or causal and j > i + Tk - Tq)    P = exp(s - lse)    o = P v
//   delta_i = do_i.o_i    dS = P (do v^T - delta)    dq = scale dS k    dk = scale dS^T q    dv = P^T do
//
// The G query heads that share a key / value head are one list of R = G * Tq rows: a tile of rows may cross heads, K / V are staged once for
// all of them, and the sum of dk / dv over the shared heads is the ordinary sum over rows (no atomics: the same bits on every run).
//
// Every kernel holds its 32 rows (keys, for dk / dv) per wave as the COLUMN operand, so that a lane owns one row of the softmax (half of it:
// lanes l and l + 32 hold 16 of 32 keys each).  Forward and dq compute S^T = K Q^T and then O^T += V^T P^T, dQ^T += K^T dS^T: the accumulator
// of the first product is the operand of the second one without leaving its lane (tileops.hip.h), statistics need one exchange with the other half.
// dk / dv mirror it with S = Q K^T and dK^T += Q^T dS, dV^T += dO^T P.  Scores and statistics are fp32; P and dS are rounded once to the
// operand type (fp32: not at all) to enter the matrix instruction, as the inputs were.
// dq and dk / dv are two passes that each recompute S and P (7 products instead of 5): sharing one would need atomics on dq or 1/64 of the
// score matrix' traffic in partial sums, 4 bytes per (query, key) at head size 64 against 256 flops.
#include "tileops.hip.h"

#include <algorithm>
#include <climits>
#include <cmath>

using namespace fdx;

namespace {

struct Str { long b, h, t; };
struct AttnArgs {
  const void *q, *k, *v, *go;
  void *o, *dq, *dk, *dv;
  Str sq, sk, sv, sgo, so, sdq, sdk, sdv;
  const uint8_t* mask;   // [B][Tk], 1 = masked
  float *lse, *delta, *part;
  int B, H, Hkv, G, Tq, Tk, D, R, off, causal, splits, tiles;
  float c, scale;        // c = scale * log2(e)
};

// Two waves on a SIMD (256 registers each): the exponentials of one run under the matrix instructions of the other.  fp32 at head size 128 holds 128
// accumulators and as many operands and stays at one.  (bf16, head size 128, 2 x 16 / 4 x 4096 causal: dq 540 us where one is asked for, 268 so; dk / dv 511, 352.)
template <typename T, int DH> constexpr int waves_of() { return sizeof(T) == 4 && DH == 128 ? 1 : 2; }

constexpr float kLn2 = 0.69314718055994530942f, kLog2e = 1.44269504088896340736f;
__device__ inline float inf() { return __builtin_inff(); }
__device__ inline float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// of lane l and lane l ^ 32, in both: the swap exchanges the upper half of its first register with the lower half of its second one, so it needs two
__device__ inline float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), opaque(__builtin_bit_cast(unsigned, x)), false, false);
  const unsigned lo = r[0], up = r[1];   // (bit_cast of a vector element as it stands reads element 0)
  return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, up));
}
__device__ inline float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), opaque(__builtin_bit_cast(unsigned, x)), false, false);
  const unsigned lo = r[0], up = r[1];
  return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, up);
}

// workgroup -> (batch and kv head, tile, split).  Workgroups go to the 8 XCDs in turn: where the heads divide, all tiles of a head run on one
// XCD and find its K / V in that XCD's L2.  Causal tiles start in the order of their length, the G heads' longest first: the grid then has G times
// ceil(tiles / G) places and those past the last tile end at once (2 x 16 / 4 heads x 4096 x 128: forward 212 -> 169 us, dq 346 -> 280 us against head after head).
__device__ inline void decode(const AttnArgs& a, int G, int& bh, int& tile, int& split) {
  const int nb = a.B * a.Hkv, per = a.tiles * a.splits, i = blockIdx.x;
  int j;
  if (nb % 8 == 0) { bh = (i & 7) + 8 * ((i >> 3) / per); j = (i >> 3) % per; }
  else { bh = i / per; j = i % per; }
  split = j % a.splits;
  j /= a.splits;
  tile = a.causal ? j % G * (a.tiles / G) + a.tiles / G - 1 - j / G : j;
}

// one past the last key any row of [r0, r1] sees
__device__ inline int key_end(const AttnArgs& a, int r0, int r1) {
  if (!a.causal) return a.Tk;
  const int t = r0 / a.Tq == r1 / a.Tq ? r1 % a.Tq : a.Tq - 1;
  return max(0, min(a.Tk, t + a.off + 1));
}

// stages of a tile pair of `bytes`: two (a step's loads fly while the one before is computed) where two workgroups still fit on a CU, else one (the
// other workgroup's products cover the loads)
constexpr int stages_of(int bytes) { return 2 * bytes <= 80 * 1024 ? 2 : 1; }

// which of a step's TK rows exist and are not masked, in every wave: loaded one step before it is needed.  (Picked by comparison: an array indexed by
// a lane's value goes to LDS, addressed through the dispatch packet in host memory -- 12 us per launch.)
__device__ inline bool bit_of(const unsigned long long* bits, int n, int row) { return ((n > 1 && row >= 64 ? bits[n > 1 ? 1 : 0] : bits[0]) >> (row & 63)) & 1; }
template <int TK> struct RowBits {
  static constexpr int N = (TK + 63) / 64;
  static_assert(N <= 2, "two words");
  unsigned char m[N];
  unsigned long long bits[N];
  __device__ inline void load(const uint8_t* mask, int first, int end, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = first + 64 * i + lane;
      m[i] = k >= end || (TK < 64 && lane >= TK) ? 1 : mask ? mask[k] : 0;
    }
  }
  __device__ inline void vote() {
#pragma unroll
    for (int i = 0; i < N; ++i) bits[i] = __ballot(m[i] == 0);
  }
  __device__ inline bool has(int row) const { return bit_of(bits, N, row); }
  // KT rows from wk * KT on
  template <int KT> __device__ inline unsigned long long part(int wk) const {
    if constexpr (N == 1 && KT >= 64) return bits[0];
    else return ((N > 1 && wk * KT >= 64 ? bits[N - 1] : bits[0]) >> (wk * KT % 64)) & (~0ull >> (64 - KT));
  }
  __device__ inline bool all() const {
    unsigned long long o = ~0ull;
#pragma unroll
    for (int i = 0; i < N; ++i) o &= bits[i];
    return o == (TK < 64 ? ~0ull >> (64 - TK) : ~0ull);
  }
  __device__ inline bool any() const {
    unsigned long long o = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) o |= bits[i];
    return o != 0;
  }
};

// a wave's 32 rows of DH elements as column operands (lane: row lane & 31), zeros beyond D and where p is null
template <typename T, int DH> __device__ inline void load_rows(typename Elem<T>::frag* f, const T* p, int D, int lane) {
#pragma unroll
  for (int s = 0; s < DH / Elem<T>::KS; ++s) {
    const int e = (2 * s + (lane >> 5)) * Elem<T>::VEC;
    f[s] = __builtin_bit_cast(typename Elem<T>::frag, p && e < D ? *reinterpret_cast<const uint4*>(p + e) : uint4{0, 0, 0, 0});
  }
}

// The wave's own column operands either in registers or, where accumulators and two of them would not leave room for two waves per SIMD (16-bit types,
// head size 128), parked in LDS in lane order and read back at every use.
template <typename T, int DH, bool PARK> struct Own {
  typedef typename Elem<T>::frag frag;
  static constexpr int NS = DH / Elem<T>::KS;
  frag f[PARK ? 1 : NS];
  uint4* at;
  // waves that share rows share their place: one of them writes it, before a barrier
  __device__ inline void set(const frag* v, uint4* lds, int place, bool write, int lane) {
    at = lds + place * NS * 64 + lane;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      if constexpr (PARK) {
        if (write) at[s * 64] = __builtin_bit_cast(uint4, v[s]);
      } else f[s] = v[s];
    }
  }
  __device__ inline frag get(int s) const {
    if constexpr (PARK) return __builtin_bit_cast(frag, at[s * 64]);
    else return f[s];
  }
};
template <typename T, int DH> constexpr bool parked() { return sizeof(T) == 2 && DH == 128; }

template <typename T> __device__ inline void store4(T* p, float a, float b, float c, float d) {
  typedef T v4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<v4*>(p) = v4{(T)a, (T)b, (T)c, (T)d};
}

// transposed accumulators acc[m] (row d, column = this lane's row) times f to a row of D elements
template <typename T, int MT> __device__ inline void store_cols(T* p, const f32x16* acc, float f, int D, int lane) {
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int d = 32 * m + 8 * b + 4 * (lane >> 5);
      if (d < D) store4<T>(p + d, acc[m][4 * b] * f, acc[m][4 * b + 1] * f, acc[m][4 * b + 2] * f, acc[m][4 * b + 3] * f);
    }
}

// the same to LDS as [32][DH] fp32 (chunks of 4 swizzled by the row), one such block per wave, and one element of the blocks' sum
__device__ inline int red_at(int row, int d, int DH) { return row * DH + (((d >> 2) ^ (row & 7)) << 2); }
template <int DH> __device__ inline void put_rows(float* red, const f32x16* acc, float f, int lane) {
#pragma unroll
  for (int m = 0; m < DH / 32; ++m)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<f32x4*>(red + red_at(lane & 31, 32 * m + 8 * q + 4 * (lane >> 5), DH)) =
          f32x4{acc[m][4 * q] * f, acc[m][4 * q + 1] * f, acc[m][4 * q + 2] * f, acc[m][4 * q + 3] * f};
}
template <int DH> __device__ inline f32x4 sum_rows(const float* red, int row, int d) {
  f32x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < 4; ++w) v += *reinterpret_cast<const f32x4*>(red + w * 32 * DH + red_at(row, d, DH));
  return v;
}

// fp16: probabilities are carried times 2^11 (at most 2^15, with the slack of the forward's reference), which keeps those down to 2^-25 normal numbers;
// every sum has the same factor.
template <typename T> struct PShift { static constexpr float log2 = 0.f, back = 1.f; };
template <> struct PShift<f16_t> { static constexpr float log2 = 11.f, back = 0x1p-11f; };

// ---------------------------------------------------------------------------------------------------------------- forward
// WQ waves take 32 rows each, the other factor of the 4 waves (WK) shares those rows and takes KT keys each of every step; their
// (reference, sum, O) meet in LDS at the end.  Online softmax: P = exp2(c s - m) with m a reference that follows the row's maximum (below).
template <typename T, int DH, int WQ, int KT>
__global__ __launch_bounds__(256, (waves_of<T, DH>())) void k_attn_fwd(AttnArgs a) {
  typedef Tile<T, DH> Tl;
  typedef typename Elem<T>::frag frag;
  constexpr int KS = Elem<T>::KS, WK = 4 / WQ, TK = KT * WK, NS = DH / KS, MT = DH / 32, NU = KT / 32, NP = 32 / KS;
  constexpr int kTile = TK * Tl::CPR, kMerge = WK > 1 ? WK * 32 * DH / 4 : 0;   // in 16-byte units
  constexpr int S = stages_of(32 * kTile);
  __shared__ __attribute__((aligned(1024))) uint4 smem[2 * S * kTile > kMerge ? 2 * S * kTile : kMerge];       // S stages of K and V
  __shared__ float ml[2][4][32];
  int bh, tile, split;
  decode(a, a.G, bh, tile, split);
  if (tile * 32 * WQ >= a.R) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wq = wave / WK, wk = wave % WK, hi = lane >> 5;
  const int b = bh / a.Hkv, hk = bh % a.Hkv;
  const int r0 = tile * 32 * WQ, r = r0 + wq * 32 + (lane & 31), rc = min(r, a.R - 1), g = rc / a.Tq, t = rc - g * a.Tq;
  const int kmax = key_end(a, r0, min(r0 + 32 * WQ, a.R) - 1), steps = (kmax + TK - 1) / TK;
  const int lim = a.causal ? t + a.off : INT_MAX;
  const T* const K = static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h;
  const T* const V = static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h;
  const uint8_t* const mask = a.mask ? a.mask + (long)b * a.Tk : nullptr;
  frag qf[NS];
  load_rows<T, DH>(qf, static_cast<const T*>(a.q) + b * a.sq.b + (hk * a.G + g) * a.sq.h + t * a.sq.t, a.D, lane);
  f32x16 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = f32x16{0};
  float mc = -inf(), l = 0.f;   // the row's reference, times c; its sum
  constexpr float kSlack = DtOf<T>::v == DT_F16 ? 4.f : 8.f;

  RowBits<TK> rb;
  int stage = 0;
  const unsigned row0 = lds_of(smem) + Tl::row_base(lane) + wk * KT * Tl::CPR * 16, col0 = lds_of(smem) + Tl::col_base(lane) + wk * KT * Tl::CPR * 16;
  auto fetch = [&](int st) {   // (masked rows enter as zeros: 0 * NaN never happens)
    const long k0 = (long)st * TK;
    uint4* const to = smem + stage * 2 * kTile;
    const bool all = a.D == DH && rb.all();
    const auto has = [&](int row) { return rb.has(row); };
    Fill<T, DH, TK>::issue(to, K + k0 * a.sk.t, a.sk.t, a.D, all, has);
    Fill<T, DH, TK>::issue(to + kTile, V + k0 * a.sv.t, a.sv.t, a.D, all, has);
  };
  if (split < steps) {
    rb.load(mask, split * TK, a.Tk, lane);
    rb.vote();
    if (S == 2) {
      if (rb.any()) fetch(split);
      rb.load(mask, (split + a.splits) * TK, a.Tk, lane);
    }
  }
  for (int st = split; st < steps; st += a.splits) {
    if constexpr (S == 1) {
      __syncthreads();
      if (rb.any()) fetch(st);
      rb.load(mask, (st + a.splits) * TK, a.Tk, lane);
    }
    landed();
    const unsigned row = opaque(row0 + stage * 2 * kTile * 16), col = opaque(col0 + stage * 2 * kTile * 16);   // K; V: TK rows behind
    constexpr int V0 = TK;
    const unsigned long long bits = rb.template part<KT>(wk);
    if constexpr (S == 2) stage ^= 1;
    if (st + a.splits < steps) {
      rb.vote();
      if constexpr (S == 2) {
        if (rb.any()) fetch(st + a.splits);
        rb.load(mask, (st + 2 * a.splits) * TK, a.Tk, lane);
      }
    }
    if (bits == 0) continue;   // (the wave's keys are all masked; the barriers are outside)
    f32x16 s[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      s[u] = f32x16{0};
#pragma unroll
      for (int i = 0; i < NS; ++i) s[u] = Elem<T>::mma(Tl::row(row, 32 * u, i), qf[i], s[u]);
    }
    const int rel = lim - (st * TK + wk * KT);   // last visible key of this lane's row, relative
    constexpr unsigned long long full = ~0ull >> (64 - KT);
    if (!__all(bits == full && rel >= KT - 1)) {
      unsigned long long ok = bits & (rel >= 63 ? ~0ull : rel < 0 ? 0ull : (2ull << rel) - 1);
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const unsigned w = (unsigned)(ok >> (32 * u)) >> (4 * hi);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[u][e] = (w >> (8 * (e >> 2) + (e & 3))) & 1 ? s[u][e] : -inf();
      }
    }
    float mt = -inf();
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) mt = fmaxf(mt, s[u][e]);
    mt = half_max(mt) * a.c;
    // The reference of a row moves only when a score passes it by kSlack (powers of two): nearly never behind the first tiles
    const bool move = mt > mc + kSlack || (mc == -inf() && mt > -inf());
    if (__any(move)) {
      const float to = move ? mt : mc;
      const float alpha = to == -inf() ? 1.f : exp2_(mc - to);
      mc = to;
      l *= alpha;
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m] *= alpha;
    }
    const float ref = PShift<T>::log2 - (mc == -inf() ? 0.f : mc);
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        // fp32: the score is rounded as the reference was, so that the only key of a row has P = 1 exactly (16-bit results do not see the difference)
        s[u][e] = exp2_(sizeof(T) == 4 ? s[u][e] * a.c + ref : __builtin_fmaf(s[u][e], a.c, ref));
        sum += s[u][e];
      }
    l += sum;
    __builtin_amdgcn_s_setprio(1);   // this wave's products before the other one's exponentials, which then run under them: 172 -> 168 us
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const frag pf = acc_frag<T>(s[u], p);
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m] = Elem<T>::mma(Tl::col(col, V0 + 32 * u + KS * p, m), pf, acc[m]);
      }
    __builtin_amdgcn_s_setprio(0);
  }
  l = half_sum(l);

  const long row_out = (long)bh * a.R + r;
  T* const O = static_cast<T*>(a.o) + b * a.so.b + (hk * a.G + g) * a.so.h + t * a.so.t;
  const long prow = ((long)bh * a.splits + split) * a.R;
  float2* const part_ml = reinterpret_cast<float2*>(a.part + (long)a.B * a.Hkv * a.splits * a.R * a.D);
  if constexpr (WK == 1) {
    if (r >= a.R) return;
    if (a.splits > 1) {
      store_cols<float, MT>(a.part + (prow + r) * a.D, acc, 1.f, a.D, lane);
      if (hi == 0) part_ml[prow + r] = float2{mc, l};
    } else {
      store_cols<T, MT>(O, acc, l == 0.f ? 0.f : 1.f / l, a.D, lane);
      if (hi == 0) a.lse[row_out] = l == 0.f ? -inf() : (mc + __builtin_amdgcn_logf(l) - PShift<T>::log2) * kLn2;
    }
  } else {
    static_assert(WQ == 1, "the waves that share rows are all four");
    if (hi == 0) { ml[0][wk][lane] = mc; ml[1][wk][lane] = l; }
    landed();   // also: the last tile has been read (and nothing is on its way)
    float M = -inf(), L = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w) M = fmaxf(M, ml[0][w][lane & 31]);
    const float Mz = M == -inf() ? 0.f : M;
#pragma unroll
    for (int w = 0; w < WK; ++w) L += ml[1][w][lane & 31] * exp2_(ml[0][w][lane & 31] - Mz);
    const float f = exp2_(mc - Mz) * (a.splits > 1 ? 1.f : L == 0.f ? 0.f : 1.f / L);
    float* const red = reinterpret_cast<float*>(smem);
    put_rows<DH>(red + wk * 32 * DH, acc, f, lane);
    __syncthreads();
    if (wave == 0 && hi == 0 && r < a.R) {
      if (a.splits > 1) part_ml[prow + r] = float2{M, L};
      else a.lse[row_out] = L == 0.f ? -inf() : (M + __builtin_amdgcn_logf(L) - PShift<T>::log2) * kLn2;
    }
    for (int i = threadIdx.x; i < 32 * (DH / 4); i += 256) {
      const int row = i / (DH / 4), d = i % (DH / 4) * 4, rr = r0 + row;
      if (rr >= a.R || d >= a.D) continue;
      const f32x4 v = sum_rows<DH>(red, row, d);
      if (a.splits > 1) *reinterpret_cast<f32x4*>(a.part + (prow + rr) * a.D + d) = v;
      else {
        const int gg = rr / a.Tq, tt = rr - gg * a.Tq;
        store4<T>(static_cast<T*>(a.o) + b * a.so.b + (hk * a.G + gg) * a.so.h + tt * a.so.t + d, v[0], v[1], v[2], v[3]);
      }
    }
  }
}

// splits of the keys joined: one wave per row, two channels a lane.  Every lane takes one split's (reference, sum) -- at most 64 -- and the weights travel by
// lane reads, so the rows of O are the only chain: eight loads in flight.
template <typename T> __global__ __launch_bounds__(256) void k_attn_join(AttnArgs a) {
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (long)a.B * a.Hkv * a.R) return;
  const long bh = row / a.R, r = row - bh * a.R;
  const float2* ml = reinterpret_cast<const float2*>(a.part + (long)a.B * a.Hkv * a.splits * a.R * a.D) + bh * a.splits * a.R + r;
  const float2 mine = lane < a.splits ? ml[(long)lane * a.R] : float2{-inf(), 0.f};
  const float* const p = a.part + (bh * a.splits * a.R + r) * a.D + 2 * lane;
  const long pitch = (long)a.R * a.D;
  const bool in = 2 * lane < a.D;
  float M = mine.x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) M = fmaxf(M, __shfl_xor(M, d, 64));
  const float w = exp2_(mine.x - (M == -inf() ? 0.f : M));
  float L = mine.y * w;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) L += __shfl_xor(L, d, 64);
  float o0 = 0.f, o1 = 0.f;
  for (int s = 0; s < a.splits; s += 8) {
    float2 o[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) o[q] = in && s + q < a.splits ? *reinterpret_cast<const float2*>(p + (s + q) * pitch) : float2{0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float ws = __shfl(w, (s + q) & 63, 64);
      o0 = __builtin_fmaf(o[q].x, ws, o0);
      o1 = __builtin_fmaf(o[q].y, ws, o1);
    }
  }
  const float f = L == 0.f ? 0.f : 1.f / L;
  const int b = (int)(bh / a.Hkv), hk = (int)(bh % a.Hkv), g = (int)r / a.Tq, t = (int)r - g * a.Tq;
  if (in) {
    T* out = static_cast<T*>(a.o) + b * a.so.b + (hk * a.G + g) * a.so.h + t * a.so.t + 2 * lane;
    out[0] = (T)(o0 * f);
    out[1] = (T)(o1 * f);
  }
  if (lane == 0) a.lse[row] = L == 0.f ? -inf() : (M + __builtin_amdgcn_logf(L) - PShift<T>::log2) * kLn2;
}

// ---------------------------------------------------------------------------------------------------------------- backward
// fp16 only: dS can lie far below fp16's smallest normal number (6e-5) although do and the result do not.  Each lane's column of dS carries a
// power of two that puts its largest element so far near 2^14; the accumulators carry the same factor and are moved along when it shrinks.
struct RunScale {
  float s = 0x1p100f;
  template <int MT> __device__ inline void fit(f32x16& ds, f32x16* acc) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(ds[e]));
    top = half_max(top);
    const bool move = top * s > 0x1p15f;
    if (__any(move)) {
      const float n = move ? __builtin_ldexpf(1.f, 14 - (int)((__builtin_bit_cast(unsigned, top) >> 23) & 255) + 127) : s, f = n / s;
      s = n;
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m] *= f;
    }
    ds *= s;
  }
};

// dq, and delta for the dk / dv pass (which runs behind this one).  Same split of rows and keys over the waves as the forward.
// 16-bit types: delta = do.o sees o as it was rounded, off by d.  P(dP - delta) sums to 0 over a row, so the sum r of what was computed IS d, up to
// fp32: dq = scale (sum dS k - r sum P k), at the price of one more product whose operand is in place, and the dk / dv pass gets delta + r.
template <typename T, int DH, int WQ, int KT>
__global__ __launch_bounds__(256, (waves_of<T, DH>())) void k_attn_dq(AttnArgs a) {
  typedef Tile<T, DH> Tl;
  typedef typename Elem<T>::frag frag;
  constexpr bool kScaled = DtOf<T>::v == DT_F16, kMend = sizeof(T) == 2;
  constexpr int KS = Elem<T>::KS, WK = 4 / WQ, TK = KT * WK, NS = DH / KS, MT = DH / 32, NU = KT / 32, NP = 32 / KS;
  constexpr int kTile = TK * Tl::CPR, kMerge = WK > 1 ? WK * 32 * DH / 4 : 0;
  constexpr int S = stages_of(32 * kTile);
  __shared__ __attribute__((aligned(1024))) uint4 smem[2 * S * kTile > kMerge ? 2 * S * kTile : kMerge];
  __shared__ float rest[4][32];
  constexpr bool PARK = parked<T, DH>();
  __shared__ uint4 own[PARK ? WQ * NS * 64 : 1];
  int bh, tile, split;
  decode(a, a.G, bh, tile, split);
  if (tile * 32 * WQ >= a.R) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wq = wave / WK, wk = wave % WK, hi = lane >> 5;
  const int b = bh / a.Hkv, hk = bh % a.Hkv;
  const int r0 = tile * 32 * WQ, r = r0 + wq * 32 + (lane & 31), rc = min(r, a.R - 1), g = rc / a.Tq, t = rc - g * a.Tq;
  const int h = hk * a.G + g;
  const int kmax = key_end(a, r0, min(r0 + 32 * WQ, a.R) - 1), steps = (kmax + TK - 1) / TK;
  const int lim = a.causal ? t + a.off : INT_MAX;
  const T* const K = static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h;
  const T* const V = static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h;
  const uint8_t* const mask = a.mask ? a.mask + (long)b * a.Tk : nullptr;
  RowBits<TK> rb;
  int stage = 0;
  const unsigned row0 = lds_of(smem) + Tl::row_base(lane) + wk * KT * Tl::CPR * 16, col0 = lds_of(smem) + Tl::col_base(lane) + wk * KT * Tl::CPR * 16;
  auto fetch = [&](int st) {
    const long k0 = (long)st * TK;
    uint4* const to = smem + stage * 2 * kTile;
    const bool all = a.D == DH && rb.all();
    const auto has = [&](int row) { return rb.has(row); };
    Fill<T, DH, TK>::issue(to, K + k0 * a.sk.t, a.sk.t, a.D, all, has);
    Fill<T, DH, TK>::issue(to + kTile, V + k0 * a.sv.t, a.sv.t, a.D, all, has);
  };
  if (split < steps) {
    rb.load(mask, split * TK, a.Tk, lane);
    rb.vote();
    if (S == 2) {
      if (rb.any()) fetch(split);
      rb.load(mask, (split + a.splits) * TK, a.Tk, lane);
    }
  }
  frag qf[NS];
  Own<T, DH, PARK> gf;
  load_rows<T, DH>(qf, static_cast<const T*>(a.q) + b * a.sq.b + h * a.sq.h + t * a.sq.t, a.D, lane);
  const float lse = a.lse[(long)bh * a.R + rc];
  const bool empty = lse == -inf();
  float delta = 0.f;
  {
    frag of[NS], go[NS];
    load_rows<T, DH>(go, static_cast<const T*>(a.go) + b * a.sgo.b + h * a.sgo.h + t * a.sgo.t, a.D, lane);
    load_rows<T, DH>(of, static_cast<const T*>(a.o) + b * a.so.b + h * a.so.h + t * a.so.t, a.D, lane);
    // the diagonal of do o^T, by the instruction and in the order that dP is summed: a row of one key has o = v, dP - delta = 0 and gradients of exactly 0
    f32x16 d = {0};
#pragma unroll
    for (int s = 0; s < NS; ++s) d = Elem<T>::mma(of[s], go[s], d);
#pragma unroll
    for (int e = 0; e < 16; ++e) delta += 8 * (e >> 2) + 4 * hi + (e & 3) == (lane & 31) ? d[e] : 0.f;
    delta = half_sum(delta);
    if (empty) delta = 0.f;   // (whatever stands in do there)
    gf.set(go, own, wq, wk == 0, lane);
  }
  const float L = empty ? inf() : lse * kLog2e;   // exp2(x - inf) = 0
  f32x16 acc[MT], pk[kMend ? MT : 1];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = f32x16{0};
  if constexpr (kMend) {
#pragma unroll
    for (int m = 0; m < MT; ++m) pk[m] = f32x16{0};
  }
  float left = 0.f;   // sum of dS over the row
  RunScale rs;

  for (int st = split; st < steps; st += a.splits) {
    if constexpr (S == 1) {
      __syncthreads();
      if (rb.any()) fetch(st);
      rb.load(mask, (st + a.splits) * TK, a.Tk, lane);
    }
    landed();
    const unsigned row = opaque(row0 + stage * 2 * kTile * 16), col = opaque(col0 + stage * 2 * kTile * 16);   // K; V: TK rows behind
    constexpr int V0 = TK;
    const unsigned long long bits = rb.template part<KT>(wk);
    if constexpr (S == 2) stage ^= 1;
    if (st + a.splits < steps) {
      rb.vote();
      if constexpr (S == 2) {
        if (rb.any()) fetch(st + a.splits);
        rb.load(mask, (st + 2 * a.splits) * TK, a.Tk, lane);
      }
    }
    if (bits == 0) continue;
    const int rel = lim - (st * TK + wk * KT);
    constexpr unsigned long long full = ~0ull >> (64 - KT);
    const bool whole = __all(bits == full && rel >= KT - 1 && !empty);
    const unsigned long long ok = empty ? 0ull : bits & (rel >= 63 ? ~0ull : rel < 0 ? 0ull : (2ull << rel) - 1);
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      f32x16 s = {0}, dp = {0};
      __builtin_amdgcn_s_setprio(1);   // as in the forward, around the products with the longer chains: 292 -> 268 us
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        s = Elem<T>::mma(Tl::row(row, 32 * u, i), qf[i], s);
        dp = Elem<T>::mma(Tl::row(row, V0 + 32 * u, i), gf.get(i), dp);
      }
      __builtin_amdgcn_s_setprio(0);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = exp2_(__builtin_fmaf(s[e], a.c, PShift<T>::log2 - L));
      if (!whole) {
        const unsigned w = (unsigned)(ok >> (32 * u)) >> (4 * hi);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const bool in = (w >> (8 * (e >> 2) + (e & 3))) & 1;
          s[e] = in ? s[e] : 0.f;
          dp[e] = in ? dp[e] : delta;
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) dp[e] = s[e] * PShift<T>::back * (dp[e] - delta);
      if constexpr (kMend) {
#pragma unroll
        for (int e = 0; e < 16; ++e) left += dp[e];
      }
      if constexpr (kScaled) rs.fit<MT>(dp, acc);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const frag df = acc_frag<T>(dp, p);
        frag pf;
        if constexpr (kMend) pf = acc_frag<T>(s, p);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const frag kf = Tl::col(col, 32 * u + KS * p, m);
          acc[m] = Elem<T>::mma(kf, df, acc[m]);
          if constexpr (kMend) pk[m] = Elem<T>::mma(kf, pf, pk[m]);
        }
      }
    }
  }
  float f = a.scale;
  if constexpr (kScaled) f /= rs.s;
  if constexpr (kMend) left = half_sum(left);
  const float fp = a.scale * PShift<T>::back;   // of pk
  const long prow = ((long)bh * a.splits + split) * a.R;
  float* const part_pk = a.part + (long)a.B * a.Hkv * a.splits * a.R * a.D;
  float* const part_r = part_pk + (kMend ? (long)a.B * a.Hkv * a.splits * a.R * a.D : 0);
  if constexpr (WK > 1) {
    if constexpr (kMend) {   // the row's sum over the waves
      if (hi == 0) rest[wk][lane] = left;
      __syncthreads();
      left = rest[0][lane & 31] + rest[1][lane & 31] + rest[2][lane & 31] + rest[3][lane & 31];
    }
  }
  if (wk == 0 && hi == 0 && r < a.R) {
    if (a.splits == 1) a.delta[(long)bh * a.R + r] = delta + left;
    else {
      if (split == 0) a.delta[(long)bh * a.R + r] = delta;   // k_attn_join_dq adds the rest
      if constexpr (kMend) part_r[prow + r] = left;
    }
  }
  const bool whole_row = a.splits == 1;
  if constexpr (kMend) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      acc[m] *= f;
      if (whole_row) acc[m] -= pk[m] * (fp * left);
    }
    f = 1.f;
  }
  if constexpr (WK == 1) {
    if (r >= a.R) return;
    if (whole_row) store_cols<T, MT>(static_cast<T*>(a.dq) + b * a.sdq.b + h * a.sdq.h + t * a.sdq.t, acc, f, a.D, lane);
    else {
      store_cols<float, MT>(a.part + (prow + r) * a.D, acc, f, a.D, lane);
      if constexpr (kMend) store_cols<float, MT>(part_pk + (prow + r) * a.D, pk, fp, a.D, lane);
    }
  } else {
    float* const red = reinterpret_cast<float*>(smem);
    auto out = [&](float* part) {   // the waves' blocks in LDS, summed, to the partial rows or to dq
      for (int i = threadIdx.x; i < 32 * (DH / 4); i += 256) {
        const int row = i / (DH / 4), d = i % (DH / 4) * 4, rr = r0 + row;
        if (rr >= a.R || d >= a.D) continue;
        const f32x4 v = sum_rows<DH>(red, row, d);
        if (!whole_row) *reinterpret_cast<f32x4*>(part + (prow + rr) * a.D + d) = v;
        else {
          const int gg = rr / a.Tq, tt = rr - gg * a.Tq;
          store4<T>(static_cast<T*>(a.dq) + b * a.sdq.b + (hk * a.G + gg) * a.sdq.h + tt * a.sdq.t + d, v[0], v[1], v[2], v[3]);
        }
      }
    };
    landed();
    put_rows<DH>(red + wk * 32 * DH, acc, f, lane);
    __syncthreads();
    out(a.part);
    if constexpr (kMend) {
      if (!whole_row) {
        __syncthreads();
        put_rows<DH>(red + wk * 32 * DH, pk, fp, lane);
        __syncthreads();
        out(part_pk);
      }
    }
  }
}

// splits of the keys joined for dq (and delta): one wave per row, two channels a lane
template <typename T> __global__ __launch_bounds__(256) void k_attn_join_dq(AttnArgs a) {
  constexpr bool kMend = sizeof(T) == 2;
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6), rows = (long)a.B * a.Hkv * a.R;
  if (row >= rows) return;
  const long bh = row / a.R, r = row - bh * a.R;
  const float* const part_pk = a.part + rows * a.splits * a.D;
  const float* const part_r = part_pk + (kMend ? rows * a.splits * a.D : 0);
  float left = 0.f, o0 = 0.f, o1 = 0.f, p0 = 0.f, p1 = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const long at = (bh * a.splits + s) * a.R + r;
    if constexpr (kMend) left += part_r[at];
    if (2 * lane < a.D) {
      const float2 o = *reinterpret_cast<const float2*>(a.part + at * a.D + 2 * lane);
      o0 += o.x;
      o1 += o.y;
      if constexpr (kMend) {
        const float2 p = *reinterpret_cast<const float2*>(part_pk + at * a.D + 2 * lane);
        p0 += p.x;
        p1 += p.y;
      }
    }
  }
  const int b = (int)(bh / a.Hkv), hk = (int)(bh % a.Hkv), g = (int)r / a.Tq, t = (int)r - g * a.Tq;
  if (2 * lane < a.D) {
    T* p = static_cast<T*>(a.dq) + b * a.sdq.b + (hk * a.G + g) * a.sdq.h + t * a.sdq.t + 2 * lane;
    p[0] = (T)(o0 - left * p0);
    p[1] = (T)(o1 - left * p1);
  }
  if (kMend && lane == 0) a.delta[row] += left;
}

// partial sums [B * Hkv][splits][Tk][D] of dk and, behind them, dv joined in split order: four channels a thread, eight loads in flight
template <typename T> __global__ __launch_bounds__(256) void k_attn_join_dkv(AttnArgs a) {
  const int d4 = a.D / 4;
  const long n = (long)a.B * a.Hkv * a.Tk * d4;
  long i = (long)blockIdx.x * 256 + threadIdx.x;
  const bool second = i >= n;
  if (second) i -= n;
  if (i >= n) return;
  const int d = (int)(i % d4) * 4;
  const long row = i / d4, bh = row / a.Tk, key = row - bh * a.Tk, pitch = (long)a.Tk * a.D;
  const float* const p = a.part + (second ? n * 4 * a.splits : 0) + (bh * a.splits * a.Tk + key) * a.D + d;
  f32x4 v = {0, 0, 0, 0};
  for (int s = 0; s < a.splits; s += 8) {
    f32x4 t[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) t[q] = s + q < a.splits ? *reinterpret_cast<const f32x4*>(p + (s + q) * pitch) : f32x4{0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < 8; ++q) v += t[q];
  }
  const Str& st = second ? a.sdv : a.sdk;
  store4<T>(static_cast<T*>(second ? a.dv : a.dk) + (bh / a.Hkv) * st.b + (bh % a.Hkv) * st.h + key * st.t + d, v[0], v[1], v[2], v[3]);
}

// dk, dv: WN waves own 32 keys each, the other factor (WR) shares those keys and takes RT rows each of every step
template <typename T, int DH, int WN, int RT>
__global__ __launch_bounds__(256, (waves_of<T, DH>())) void k_attn_dkv(AttnArgs a) {
  typedef Tile<T, DH> Tl;
  typedef typename Elem<T>::frag frag;
  constexpr bool kScaled = DtOf<T>::v == DT_F16;
  constexpr int KS = Elem<T>::KS, WR = 4 / WN, TR = RT * WR, NS = DH / KS, MT = DH / 32, NU = RT / 32, NP = 32 / KS;
  constexpr int kTile = TR * Tl::CPR, kMerge = WR > 1 ? WR * 32 * DH / 4 : 0;
  static_assert(TR % 64 == 0 || TR == 32, "rows voted on 64 at a time");
  constexpr bool PARK = parked<T, DH>();
  // (64 rows in one stage beat 32 in two where v is parked: 368 against 399 us, bf16, head size 128, 2 x 16 / 4 x 4096 causal)
  constexpr int S = stages_of(32 * kTile + (PARK ? WN * NS * 1024 : 0));
  __shared__ __attribute__((aligned(1024))) uint4 smem[2 * S * kTile > kMerge ? 2 * S * kTile : kMerge];   // S stages of q and do
  __shared__ __attribute__((aligned(16))) float rowL[2][TR], rowD[2][TR];
  __shared__ uint4 own[PARK ? WN * NS * 64 : 1];
  int bh, tile, split;
  decode(a, 1, bh, tile, split);
  if (a.causal) tile = a.tiles - 1 - tile;   // early keys are the long ones here
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wn = wave / WR, wr = wave % WR, hi = lane >> 5;
  const int b = bh / a.Hkv, hk = bh % a.Hkv;
  const int k0 = tile * 32 * WN, key = k0 + wn * 32 + (lane & 31);
  const bool kok = key < a.Tk && !(a.mask && a.mask[(long)b * a.Tk + min(key, a.Tk - 1)]);
  frag kf[NS];
  Own<T, DH, PARK> vf;
  load_rows<T, DH>(kf, kok ? static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h + (long)key * a.sk.t : nullptr, a.D, lane);
  {
    frag v[NS];
    load_rows<T, DH>(v, kok ? static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h + (long)key * a.sv.t : nullptr, a.D, lane);
    vf.set(v, own, wn, wr == 0, lane);
  }
  f32x16 dk[MT], dv[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) dk[m] = dv[m] = f32x16{0};
  RunScale rs;

  const T* const Q = static_cast<const T*>(a.q) + b * a.sq.b + (long)hk * a.G * a.sq.h;
  const T* const Go = static_cast<const T*>(a.go) + b * a.sgo.b + (long)hk * a.G * a.sgo.h;
  // a step: TR rows of one query head (none crosses heads); causal: heads' first rows that see key k0
  const int per = (a.Tq + TR - 1) / TR;
  const int steps = __syncthreads_or(kok) ? a.G * per : 0;   // all keys masked: zeros
  auto needed = [&](int st) { return !a.causal || min((st % per + 1) * TR, a.Tq) - 1 + a.off >= k0; };
  auto after = [&](int st) {
    do st += a.splits; while (st < steps && !needed(st));
    return st;
  };
  // a step's lse and delta, one step ahead of its rows: lane l holds those of rows l, l + 64; a row that sees nothing (or does not exist) enters as zeros,
  // whatever stands in it
  constexpr int NB = (TR + 63) / 64;
  float nL[NB], nD[NB];
  unsigned long long live[NB];
  auto stats = [&](int st) {
    const int g = st / per, t0 = (st - g * per) * TR;
    const long at = (long)bh * a.R + (long)g * a.Tq;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int row = 64 * i + lane, t = t0 + row;
      const bool in = row < TR && t < a.Tq;
      nL[i] = in ? a.lse[at + t] : -inf();
      nD[i] = in ? a.delta[at + t] : 0.f;
    }
  };
  int stage = 0;
  const unsigned row0 = lds_of(smem) + Tl::row_base(lane) + wr * RT * Tl::CPR * 16, col0 = lds_of(smem) + Tl::col_base(lane) + wr * RT * Tl::CPR * 16;
  auto fetch = [&](int st) {
    const int g = st / per, t0 = (st - g * per) * TR;
    const T* const q = Q + g * a.sq.h + (long)t0 * a.sq.t;
    const T* const go = Go + g * a.sgo.h + (long)t0 * a.sgo.t;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      live[i] = __ballot(nL[i] != -inf());
      if (wave == i && (TR >= 64 || lane < TR)) {
        rowL[stage][64 * i + lane] = nL[i] == -inf() ? inf() : nL[i] * kLog2e;
        rowD[stage][64 * i + lane] = nL[i] == -inf() ? 0.f : nD[i];
      }
    }
    auto has = [&](int row) { return bit_of(live, NB, row); };
    uint4* const to = smem + stage * 2 * kTile;
    bool all = a.D == DH;
#pragma unroll
    for (int i = 0; i < NB; ++i) all = all && live[i] == (TR < 64 ? ~0ull >> (64 - TR) : ~0ull);
    Fill<T, DH, TR>::issue(to, q, a.sq.t, a.D, all, has);
    Fill<T, DH, TR>::issue(to + kTile, go, a.sgo.t, a.D, all, has);
  };
  int st = split;
  if (st < steps && !needed(st)) st = after(st);
  int nx = st < steps ? after(st) : steps;
  if (st < steps) {
    stats(st);
    if (S == 2) {
      fetch(st);
      if (nx < steps) stats(nx);
    }
  }
  while (st < steps) {
    if constexpr (S == 1) {
      __syncthreads();
      fetch(st);
      if (nx < steps) stats(nx);
    }
    landed();
    const unsigned row = opaque(row0 + stage * 2 * kTile * 16), col = opaque(col0 + stage * 2 * kTile * 16);   // q; do: TR rows behind
    const float *const rL = rowL[stage], *const rD = rowD[stage];
    const int here = (st % per) * TR;
    if constexpr (S == 2) stage ^= 1;
    st = nx;
    if (st < steps) {
      nx = after(st);
      if constexpr (S == 2) {
        fetch(st);
        if (nx < steps) stats(nx);
      }
    }
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      f32x16 s = {0}, dp = {0};
      const int rr = wr * RT + 32 * u;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        s = Elem<T>::mma(Tl::row(row, 32 * u, i), kf[i], s);
        dp = Elem<T>::mma(Tl::row(row, TR + 32 * u, i), vf.get(i), dp);
      }
      f32x16 p;
      const bool edge = a.causal && here + a.off + rr < k0 + 32 * WN - 1;   // some of these rows do not see some of the workgroup's keys
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int rq = rr + 8 * q + 4 * hi;
        const f32x4 L = *reinterpret_cast<const f32x4*>(rL + rq), dl = *reinterpret_cast<const f32x4*>(rD + rq);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = 4 * q + i;
          float x = exp2_(__builtin_fmaf(s[e], a.c, PShift<T>::log2 - L[i]));
          if (edge) x = key <= here + a.off + rq + i ? x : 0.f;
          p[e] = x;
          s[e] = x * PShift<T>::back * (dp[e] - dl[i]);
        }
      }
      if constexpr (kScaled) rs.fit<MT>(s, dk);
      // as in the forward; here it also keeps the compiler from moving the next rows' products in between, whose operands then spill (742 -> 933 us both ways)
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const frag pf = acc_frag<T>(p, i), df = acc_frag<T>(s, i);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          dv[m] = Elem<T>::mma(Tl::col(col, TR + 32 * u + KS * i, m), pf, dv[m]);
          dk[m] = Elem<T>::mma(Tl::col(col, 32 * u + KS * i, m), df, dk[m]);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    }
  }
  float f = a.scale, fv = PShift<T>::back;
  if constexpr (kScaled) f /= rs.s;
  if (!kok) {   // a masked key: its column saw the row sums of the others
    f = fv = 0.f;
#pragma unroll
    for (int m = 0; m < MT; ++m) dk[m] = dv[m] = f32x16{0};
  }
  const long prow = ((long)bh * a.splits + split) * a.Tk, pv = (long)a.B * a.Hkv * a.splits * a.Tk * a.D;
  if constexpr (WR == 1) {
    if (key >= a.Tk) return;
    if (a.splits > 1) {
      store_cols<float, MT>(a.part + (prow + key) * a.D, dk, f, a.D, lane);
      store_cols<float, MT>(a.part + pv + (prow + key) * a.D, dv, fv, a.D, lane);
    } else {
      store_cols<T, MT>(static_cast<T*>(a.dk) + b * a.sdk.b + hk * a.sdk.h + (long)key * a.sdk.t, dk, f, a.D, lane);
      store_cols<T, MT>(static_cast<T*>(a.dv) + b * a.sdv.b + hk * a.sdv.h + (long)key * a.sdv.t, dv, fv, a.D, lane);
    }
  } else {
    float* const red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      landed();
      put_rows<DH>(red + wr * 32 * DH, which ? dv : dk, which ? fv : f, lane);
      __syncthreads();
      for (int i = threadIdx.x; i < 32 * (DH / 4); i += 256) {
        const int row = i / (DH / 4), d = i % (DH / 4) * 4, kk = k0 + row;
        if (kk >= a.Tk || d >= a.D) continue;
        const f32x4 v = sum_rows<DH>(red, row, d);
        if (a.splits > 1) *reinterpret_cast<f32x4*>(a.part + which * pv + (prow + kk) * a.D + d) = v;
        else if (which) store4<T>(static_cast<T*>(a.dv) + b * a.sdv.b + hk * a.sdv.h + (long)kk * a.sdv.t + d, v[0], v[1], v[2], v[3]);
        else store4<T>(static_cast<T*>(a.dk) + b * a.sdk.b + hk * a.sdk.h + (long)kk * a.sdk.t + d, v[0], v[1], v[2], v[3]);
      }
    }
  }
}
}  // namespace

// ---------------------------------------------------------------------------------------------------------------- launches
namespace {

// How a pass is cut.  Four waves x 32 rows share every staged tile where that gives more than one workgroup per CU (1024 tiles of 32 rows); below, 32-row
// workgroups whose waves share the keys.  Forward, 128-row / 32-row form, us: fp32 head size 64, 86 rows x 8 heads 13.1 / 7.7; bf16 64: 256 tiles of 32 rows
// 13.3 / 6.0, 864: 35.2 / 24.2, 1024: 48.1 / 42.6, 1728: 26.9 / 45.5.
// Causal tiles stop there at half as many: a 32-row workgroup's waves have few keys each in the short ones (1024: forward 56.6 / 55.5, dk and dv 389 / 434).
// While even those leave CUs empty the other axis is split over workgroups and joined.  512 workgroups are resident; causal tiles differ in length by up to
// all of it, and twice as many workgroups as are resident, long ones first, even that out (dk / dv, 2 x 4 heads x 4096 x 128: 1094 us in 256 workgroups, 408 in 1024).
struct Plan { int narrow, tiles, splits; };   // narrow: 32 rows per workgroup
Plan plan_of(int nb, int rows, int across, bool causal, int G) {   // G: heads in the rows
  Plan p;
  const long n32 = (long)nb * ((rows + 31) / 32);
  p.narrow = n32 <= (causal ? 512 : 1024);
  p.tiles = p.narrow ? (rows + 31) / 32 : (rows + 127) / 128;
  const long base = std::max<long>(1, (long)nb * p.tiles), want = causal ? 1024 : 512;
  const int steps = p.narrow ? (across + 127) / 128 : (across + 63) / 64;
  if (causal) p.tiles = (p.tiles + G - 1) / G * G;
  long s = base > want * 3 / 4 ? 1 : (want + base / 2) / base;
  s = std::min<long>(s, steps / 2);
  p.splits = (int)std::max<long>(1, std::min<long>(s, 64));
  return p;
}

const char* check(const fdx_attn_desc* d) {
  if (!d) return "null descriptor";
  if (d->dtype < 0 || d->dtype > 2) return "dtype must be FDX_F32, FDX_BF16 or FDX_F16";
  if (d->batch < 0 || d->heads <= 0 || d->kv_heads <= 0 || d->q_len < 0 || d->k_len < 0) return "negative size or no heads";
  if (d->heads % d->kv_heads) return "heads must be a multiple of kv_heads";
  if (d->head_dim <= 0 || d->head_dim > 128 || d->head_dim % 8) return "head_dim must be a multiple of 8 up to 128";
  if (!(d->scale > 0.f) || !std::isfinite(d->scale)) return "scale must be positive and finite";
  const long R = (long)(d->heads / d->kv_heads) * d->q_len, nb = (long)d->batch * d->kv_heads;
  if (R > INT_MAX / 2 || d->k_len > INT_MAX / 2) return "too many rows for one key / value head";
  constexpr long most = (1L << 24) - 1;   // workgroups of 256 threads in one launch
  if (nb * ((R + 31) / 32 + d->heads) > most || nb * (((long)d->k_len + 31) / 32) > most) return "too many tiles for one launch";
  return nullptr;
}

struct Checked { const fdx_bht* t; bool need; int heads, rows; };   // heads, rows: of a tensor that is written, else 0
const char* check(const fdx_attn_desc* d, const Checked& x) {
  const fdx_bht* const t = x.t;
  if (!t || !t->data) return x.need ? "null tensor" : nullptr;
  if (t->b < 0 || t->h < 0 || t->t < 0) return "strides must not be negative";
  if (x.heads && ((d->batch > 1 && !t->b) || (x.heads > 1 && !t->h) || (x.rows > 1 && !t->t))) return "results must not overlap themselves (stride 0)";
  const int vec = d->dtype == DT_F32 ? 4 : 8;
  if ((reinterpret_cast<uintptr_t>(t->data) & 15) || t->b % vec || t->h % vec || t->t % vec) return "tensors must be 16-byte aligned, strides whole 16 bytes";
  return nullptr;
}

AttnArgs args_of(const fdx_attn_desc* d) {
  AttnArgs a{};
  a.B = d->batch; a.H = d->heads; a.Hkv = d->kv_heads; a.G = d->heads / d->kv_heads;
  a.Tq = d->q_len; a.Tk = d->k_len; a.D = d->head_dim; a.R = a.G * a.Tq;
  a.off = a.Tk - a.Tq; a.causal = d->causal != 0;
  a.scale = d->scale; a.c = d->scale * kLog2e;
  return a;
}
Str str_of(const fdx_bht* t) { return t ? Str{(long)t->b, (long)t->h, (long)t->t} : Str{0, 0, 0}; }

size_t fwd_floats(const fdx_attn_desc* d, Plan p) {
  return p.splits > 1 ? (size_t)d->batch * d->heads * d->q_len * p.splits * (d->head_dim + 2) : 0;
}
size_t dq_floats(const fdx_attn_desc* d, Plan p) {
  const size_t row = d->dtype == DT_F32 ? d->head_dim : 2 * d->head_dim + 1;
  return p.splits > 1 ? (size_t)d->batch * d->heads * d->q_len * p.splits * row : 0;
}
size_t dkv_floats(const fdx_attn_desc* d, Plan p) { return p.splits > 1 ? (size_t)2 * d->batch * d->kv_heads * d->k_len * p.splits * d->head_dim : 0; }
size_t delta_floats(const fdx_attn_desc* d) { return ((size_t)d->batch * d->heads * d->q_len + 3) / 4 * 4; }

template <template <typename, int> class Run, typename... A> hipError_t by_type(const fdx_attn_desc* d, A&&... x) {
  const int w = d->head_dim <= 32 ? 0 : d->head_dim <= 64 ? 1 : 2;
  switch (d->dtype * 3 + w) {
    case 0: return Run<float, 32>::go(x...);
    case 1: return Run<float, 64>::go(x...);
    case 2: return Run<float, 128>::go(x...);
    case 3: return Run<bf16_t, 32>::go(x...);
    case 4: return Run<bf16_t, 64>::go(x...);
    case 5: return Run<bf16_t, 128>::go(x...);
    case 6: return Run<f16_t, 32>::go(x...);
    case 7: return Run<f16_t, 64>::go(x...);
    default: return Run<f16_t, 128>::go(x...);
  }
}

template <typename T, int DH> struct RunFwd {
  static hipError_t go(AttnArgs& a, const Plan& p, hipStream_t s) {
    a.tiles = p.tiles; a.splits = p.splits;
    const unsigned grid = (unsigned)((long)a.B * a.Hkv * p.tiles * p.splits);
    hipError_t e = p.narrow ? launch(k_attn_fwd<T, DH, 1, 32>, grid, 256, a, s) : launch(k_attn_fwd<T, DH, 4, 64>, grid, 256, a, s);
    if (e == hipSuccess && p.splits > 1) e = launch(k_attn_join<T>, (unsigned)(((long)a.B * a.Hkv * a.R + 3) / 4), 256, a, s);
    return e;
  }
};

template <typename T, int DH> struct RunBwd {
  static hipError_t go(AttnArgs& a, const Plan& pq, const Plan& pk, float* part, hipStream_t s) {
    hipError_t e = hipSuccess;
    a.part = part;
    if (a.R > 0) {
      a.tiles = pq.tiles; a.splits = pq.splits;
      const unsigned grid = (unsigned)((long)a.B * a.Hkv * pq.tiles * pq.splits);
      e = pq.narrow ? launch(k_attn_dq<T, DH, 1, 32>, grid, 256, a, s) : launch(k_attn_dq<T, DH, 4, (DH * sizeof(T) >= 256 ? 32 : 64)>, grid, 256, a, s);
      if (e == hipSuccess && pq.splits > 1) e = launch(k_attn_join_dq<T>, (unsigned)(((long)a.B * a.Hkv * a.R + 3) / 4), 256, a, s);
    }
    if (e == hipSuccess && a.Tk > 0) {   // (reuses the partial sums' memory: ordered by the stream)
      a.tiles = pk.tiles; a.splits = pk.splits;
      const unsigned grid = (unsigned)((long)a.B * a.Hkv * pk.tiles * pk.splits);
      e = pk.narrow ? launch(k_attn_dkv<T, DH, 1, 32>, grid, 256, a, s) : launch(k_attn_dkv<T, DH, 4, (sizeof(T) == 4 && DH > 32 ? 32 : 64)>, grid, 256, a, s);
      if (e == hipSuccess && pk.splits > 1)
        e = launch(k_attn_join_dkv<T>, (unsigned)(((long)a.B * a.Hkv * a.Tk * (a.D / 4) * 2 + 255) / 256), 256, a, s);
    }
    return e;
  }
};

}  // namespace

extern "C" int fdx_attn_forward_workspace(const fdx_attn_desc* d, size_t* bytes) {
  if (const char* why = check(d)) return fail(nullptr, FDX_E_ARG, "fdx_attn_forward_workspace: %s", why);
  if (!bytes) return fail(nullptr, FDX_E_ARG, "fdx_attn_forward_workspace: null size pointer");
  const int rows = d->heads / d->kv_heads * d->q_len;
  *bytes = fwd_floats(d, plan_of(d->batch * d->kv_heads, rows, d->k_len, d->causal, d->heads / d->kv_heads)) * sizeof(float);
  return FDX_OK;
}

extern "C" int fdx_attn_backward_workspace(const fdx_attn_desc* d, size_t* bytes) {
  if (const char* why = check(d)) return fail(nullptr, FDX_E_ARG, "fdx_attn_backward_workspace: %s", why);
  if (!bytes) return fail(nullptr, FDX_E_ARG, "fdx_attn_backward_workspace: null size pointer");
  const int rows = d->heads / d->kv_heads * d->q_len, nb = d->batch * d->kv_heads;
  *bytes = (delta_floats(d) + std::max(dq_floats(d, plan_of(nb, rows, d->k_len, d->causal, d->heads / d->kv_heads)), dkv_floats(d, plan_of(nb, d->k_len, rows, d->causal, 1)))) * sizeof(float);
  return FDX_OK;
}

extern "C" int fdx_attn_forward(fdx_handle h, const fdx_attn_desc* d, const fdx_bht* q, const fdx_bht* k, const fdx_bht* v, const uint8_t* key_mask,
                                const fdx_bht* out, float* lse, void* workspace, size_t bytes, fdx_stream st) {
  if (!h) return fail(nullptr, FDX_E_ARG, "fdx_attn_forward: null handle");
  if (const char* why = check(d)) return fail(h, FDX_E_ARG, "fdx_attn_forward: %s", why);
  if (d->batch == 0 || d->q_len == 0) return FDX_OK;
  const bool keys = d->k_len > 0;
  for (const Checked& x : {Checked{q, true, 0, 0}, {k, keys, 0, 0}, {v, keys, 0, 0}, {out, true, d->heads, d->q_len}})
    if (const char* why = check(d, x)) return fail(h, FDX_E_ARG, "fdx_attn_forward: %s", why);
  if (!lse) return fail(h, FDX_E_ARG, "fdx_attn_forward: null lse");
  AttnArgs a = args_of(d);
  const Plan p = plan_of(a.B * a.Hkv, a.R, a.Tk, a.causal, a.G);
  if (bytes < fwd_floats(d, p) * sizeof(float) || (p.splits > 1 && !workspace) || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return fail(h, FDX_E_ARG, "fdx_attn_forward: workspace of %zu bytes, %zu needed (16-byte aligned)", bytes, fwd_floats(d, p) * sizeof(float));
  a.q = q->data; a.k = k ? k->data : nullptr; a.v = v ? v->data : nullptr; a.o = out->data;
  a.sq = str_of(q); a.sk = str_of(k); a.sv = str_of(v); a.so = str_of(out);
  a.mask = key_mask; a.lse = lse; a.part = static_cast<float*>(workspace);
  DeviceScope dev(h->device);
  FDX_HIP(h, dev.err);
  FDX_HIP(h, by_type<RunFwd>(d, a, p, as_stream(st)));
  return FDX_OK;
}

extern "C" int fdx_attn_backward(fdx_handle h, const fdx_attn_desc* d, const fdx_bht* grad_out, const fdx_bht* q, const fdx_bht* k, const fdx_bht* v,
                                 const fdx_bht* out, const float* lse, const uint8_t* key_mask, const fdx_bht* dq, const fdx_bht* dk,
                                 const fdx_bht* dv, void* workspace, size_t bytes, fdx_stream st) {
  if (!h) return fail(nullptr, FDX_E_ARG, "fdx_attn_backward: null handle");
  if (const char* why = check(d)) return fail(h, FDX_E_ARG, "fdx_attn_backward: %s", why);
  if (d->batch == 0 || (d->q_len == 0 && d->k_len == 0)) return FDX_OK;
  const bool rows = d->q_len > 0, keys = d->k_len > 0;
  for (const Checked& x : {Checked{grad_out, rows, 0, 0}, {q, rows, 0, 0}, {out, rows, 0, 0}, {dq, rows, d->heads, d->q_len}, {k, keys, 0, 0}, {v, keys, 0, 0},
                           {dk, keys, d->kv_heads, d->k_len}, {dv, keys, d->kv_heads, d->k_len}})
    if (const char* why = check(d, x)) return fail(h, FDX_E_ARG, "fdx_attn_backward: %s", why);
  if (rows && !lse) return fail(h, FDX_E_ARG, "fdx_attn_backward: null lse");
  AttnArgs a = args_of(d);
  const Plan pq = plan_of(a.B * a.Hkv, a.R, a.Tk, a.causal, a.G), pk = plan_of(a.B * a.Hkv, a.Tk, a.R, a.causal, 1);
  const size_t need = (delta_floats(d) + std::max(dq_floats(d, pq), dkv_floats(d, pk))) * sizeof(float);
  if (bytes < need || (need && !workspace) || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return fail(h, FDX_E_ARG, "fdx_attn_backward: workspace of %zu bytes, %zu needed (16-byte aligned)", bytes, need);
  const auto data = [](const fdx_bht* t) { return t ? t->data : nullptr; };
  a.q = data(q); a.k = data(k); a.v = data(v); a.go = data(grad_out); a.o = data(out);
  a.dq = data(dq); a.dk = data(dk); a.dv = data(dv);
  a.sq = str_of(q); a.sk = str_of(k); a.sv = str_of(v); a.sgo = str_of(grad_out); a.so = str_of(out);
  a.sdq = str_of(dq); a.sdk = str_of(dk); a.sdv = str_of(dv);
  a.mask = key_mask; a.lse = const_cast<float*>(lse); a.delta = static_cast<float*>(workspace);
  DeviceScope dev(h->device);
  FDX_HIP(h, dev.err);
  FDX_HIP(h, by_type<RunBwd>(d, a, pq, pk, static_cast<float*>(workspace) + delta_floats(d), as_stream(st)));
  return FDX_OK;
}
