// Norm of every q / k head followed by the rotation of rotary positions with several axes: the
// kernels.  Instantiated per element type in fln_rotary_{f32,bf16,f16}.cu; entry points in
// fln_rotary.cu.
//
// A row is one head of one token.  It is owned by L lanes of a warp (a power of two), each of
// which holds U units; a unit is two vectors of V elements that belong to each other:
//   half layout         columns [uV, uV + V) and [pairs + uV, pairs + uV + V): pair j is
//                       element j of both
//   interleaved layout  columns [2uV, 2uV + 2V): pair j is elements 2j, 2j + 1
//   behind the rotated part, two neighbouring vectors (the second may lie behind the row)
// so both members of every pair are in one lane's registers, a rotation needs no exchange, and
// the row sums take log2(L) shuffles and no barrier.
//
// Angles.  position * turns modulo 2^64 is the fraction of a turn as a signed 64-bit number, so
// the range reduction is the wrap of an integer product: no table of cosines to read, nothing
// lost at far positions.  sincospi of twice that fraction gives cosine and sine.  A lane makes
// them once per token and keeps them in registers for all the heads that its warp takes of that
// token.
#pragma once

#include "fln_common.cuh"

namespace fln {

struct RotTensor {
  const void* in;
  void* out;
  int64_t in_batch, in_seq, in_head;
  int64_t out_batch, out_seq, out_head;
  const void* weight;
  const void* bias;
  void* dx;          // backward only
  float* partials;   // backward only: [CTAs of this tensor][2][head_dim], or NULL
  int heads;
};
struct RotParams {
  RotTensor t[2];
  const void* positions;
  int64_t pos_axis, pos_batch, pos_seq;
  const unsigned long long* turns;
  const unsigned char* axis;
  int tokens, seq;
  int dim, pairs;
  int rot_units, units;  // units of the rotated part, of the whole row
  int log2_l;            // lanes per row
  int pos64, kind;
  float woff, eps, mag;
  // forward: items = tokens * splits, each a run of `per_split` heads of the q heads followed by
  // the k heads.  backward: the first nb0 CTAs take q, the others k; items of `per_split` heads.
  int splits[2], per_split[2];
  int nb0;
};

constexpr int kRotThreads = 256;

// first columns of a unit's two vectors; hi < 0: the second vector does not exist
template <int V, bool HALF>
__device__ __forceinline__ void unit_columns(const RotParams& p, int u, int& lo, int& hi) {
  if (u < p.rot_units) {
    lo = HALF ? u * V : 2 * u * V;
    hi = HALF ? p.pairs + u * V : lo + V;
  } else {
    lo = 2 * p.pairs + 2 * (u - p.rot_units) * V;
    hi = lo + V < p.dim ? lo + V : -1;
  }
}

// cosine and sine (times the magnitude) of the V pairs of a unit
template <int V>
__device__ __forceinline__ void unit_angles(const RotParams& p, int u, int b, int s, float (&c)[V], float (&sn)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    c[j] = 1.f;
    sn[j] = 0.f;
  }
  if (u >= p.rot_units) return;
  const int64_t at0 = (int64_t)b * p.pos_batch + (int64_t)s * p.pos_seq;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = u * V + j;
    const int64_t at = at0 + (int64_t)__ldg(p.axis + i) * p.pos_axis;
    const long long pos = p.pos64 ? reinterpret_cast<const long long*>(p.positions)[at]
                                  : (long long)reinterpret_cast<const int*>(p.positions)[at];
    const long long frac = (long long)((unsigned long long)pos * __ldg(p.turns + i));
    // frac / 2^64 turns = frac / 2^63 half turns, in [-1, 1]
    float sv, cv;
    sincospif(__ll2float_rn(frac) * 1.0842021724855044e-19f, &sv, &cv);
    c[j] = cv * p.mag;
    sn[j] = sv * p.mag;
  }
}

// the two vectors of a unit of one row as floats e[0, V) and e[V, 2V); zeros where absent
template <typename T, int V>
__device__ __forceinline__ void unit_load(const T* row, int lo, int hi, bool ok, Pack<T, V>& a, Pack<T, V>& b) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    a.e[j] = Cvt<T>::from_f(0.f);
    b.e[j] = Cvt<T>::from_f(0.f);
  }
  if (ok) {
    a = ld_stream<T, V>(row + lo);
    if (hi >= 0) b = ld_stream<T, V>(row + hi);
  }
}
template <typename T, int V>
__device__ __forceinline__ void unit_param(const T* w, int lo, int hi, bool ok, float fill, float (&f)[2 * V]) {
#pragma unroll
  for (int j = 0; j < 2 * V; ++j) f[j] = fill;
  if (w == nullptr || !ok) return;
  float t[V];
  unpack<T, V>(ld_param<T, V>(w + lo), t);
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = t[j];
  if (hi >= 0) {
    unpack<T, V>(ld_param<T, V>(w + hi), t);
#pragma unroll
    for (int j = 0; j < V; ++j) f[V + j] = t[j];
  }
}
template <typename T, int V>
__device__ __forceinline__ void unit_store(T* row, int lo, int hi, const float (&f)[2 * V]) {
  float t[V];
  Pack<T, V> o;
#pragma unroll
  for (int j = 0; j < V; ++j) t[j] = f[j];
  pack<T, V>(t, o);
  st_plain<T, V>(row + lo, o);
  if (hi >= 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) t[j] = f[V + j];
    pack<T, V>(t, o);
    st_plain<T, V>(row + hi, o);
  }
}
template <typename T, int V>
__device__ __forceinline__ void unit_unpack(const Pack<T, V>& a, const Pack<T, V>& b, float (&f)[2 * V]) {
  float t[V];
  unpack<T, V>(a, t);
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = t[j];
  unpack<T, V>(b, t);
#pragma unroll
  for (int j = 0; j < V; ++j) f[V + j] = t[j];
}

// rotation by the angle (sign = 1) or back (sign = -1) of the V pairs of a unit
template <int V, bool HALF, bool BACK>
__device__ __forceinline__ void unit_rotate(float (&f)[2 * V], const float (&c)[V], const float (&s)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int ia = HALF ? j : 2 * j, ib = HALF ? V + j : 2 * j + 1;
    const float a = f[ia], b = f[ib];
    f[ia] = BACK ? fmaf(b, s[j], a * c[j]) : fmaf(-b, s[j], a * c[j]);
    f[ib] = BACK ? fmaf(-a, s[j], b * c[j]) : fmaf(a, s[j], b * c[j]);
  }
}

template <int N>
__device__ __forceinline__ void lane_sum(float (&v)[N], int log2_l) {
  for (int off = (1 << log2_l) >> 1; off > 0; off >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], off);
  }
}

// Statistics of NB rows at once: x becomes xh = (x - mean) * rstd in place (untouched without a
// norm).  Elements behind the row count as zeros of the centred row.
template <int NB, int U, int V>
__device__ __forceinline__ void rows_normalize(const RotParams& p, float (&x)[NB][U][2 * V], const bool (&lo_ok)[U],
                                               const bool (&hi_ok)[U], float (&rstd)[NB]) {
#pragma unroll
  for (int n = 0; n < NB; ++n) rstd[n] = 1.f;
  if (p.kind == FLN_NO_NORM) return;
  const float inv_d = 1.0f / (float)p.dim;
  float v[NB];
  if (p.kind == FLN_LAYERNORM) {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      v[n] = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) v[n] += x[n][u][j];
    }
    lane_sum<NB>(v, p.log2_l);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const float mean = v[n] * inv_d;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 2 * V; ++j)
          if (j < V ? lo_ok[u] : hi_ok[u]) x[n][u][j] -= mean;
    }
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    v[n] = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) v[n] = fmaf(x[n][u][j], x[n][u][j], v[n]);
  }
  lane_sum<NB>(v, p.log2_l);
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    rstd[n] = rsqrtf(fmaf(v[n], inv_d, p.eps));
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) x[n][u][j] *= rstd[n];
  }
}

// ----------------------------------------------------------------------------------------
// forward: a warp takes items (token, run of heads); each of its 32 / L row groups takes every
// (32 / L)-th head of the run, NB of them at a time so that NB rows are on their way from memory
// together.  All lanes of a warp make the same number of turns, so the shuffles are whole.
// ----------------------------------------------------------------------------------------
template <typename T, int V, int U, bool HALF, int NB>
__global__ void __launch_bounds__(kRotThreads) rotary_fwd_kernel(const RotParams p) {
  const int lane = threadIdx.x & 31;
  const int L = 1 << p.log2_l;
  const int groups = 32 >> p.log2_l;
  const int grp = lane >> p.log2_l, ul = lane & (L - 1);
  int lo[U], hi[U];
  bool lo_ok[U], hi_ok[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int u = ul + k * L;
    lo_ok[k] = u < p.units;
    lo[k] = hi[k] = 0;
    if (lo_ok[k]) unit_columns<V, HALF>(p, u, lo[k], hi[k]);
    hi_ok[k] = lo_ok[k] && hi[k] >= 0;
  }
  const int64_t items = (int64_t)p.tokens * p.splits[0];
  const int64_t step = (int64_t)gridDim.x * (kRotThreads / 32);
  const int heads_all = p.t[0].heads + p.t[1].heads;
  for (int64_t it = (int64_t)blockIdx.x * (kRotThreads / 32) + (threadIdx.x >> 5); it < items; it += step) {
    const int token = (int)(it / p.splits[0]);
    const int part = (int)(it - (int64_t)token * p.splits[0]);
    const int h0 = part * p.per_split[0];
    const int h1 = h0 + p.per_split[0] < heads_all ? h0 + p.per_split[0] : heads_all;
    const int b = token / p.seq, s = token - b * p.seq;
    float cs[U][V], sn[U][V];
#pragma unroll
    for (int k = 0; k < U; ++k) unit_angles<V>(p, ul + k * L, b, s, cs[k], sn[k]);
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
      const RotTensor& t = p.t[which];
      const int first = which == 0 ? h0 : (h0 > p.t[0].heads ? h0 - p.t[0].heads : 0);
      const int end = which == 0 ? (h1 < p.t[0].heads ? h1 : p.t[0].heads) : h1 - p.t[0].heads;
      if (first >= end) continue;
      float w[U][2 * V], bi[U][2 * V];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        unit_param<T, V>(reinterpret_cast<const T*>(t.weight), lo[k], hi[k], lo_ok[k], t.weight != nullptr ? 0.f : 1.f, w[k]);
        unit_param<T, V>(reinterpret_cast<const T*>(t.bias), lo[k], hi[k], lo_ok[k], 0.f, bi[k]);
        if (t.weight != nullptr) {
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) w[k][j] += p.woff;
        }
      }
      const T* in = reinterpret_cast<const T*>(t.in) + (int64_t)b * t.in_batch + (int64_t)s * t.in_seq;
      T* out = reinterpret_cast<T*>(t.out) + (int64_t)b * t.out_batch + (int64_t)s * t.out_seq;
#pragma unroll 1
      for (int h = first; h < end; h += groups * NB) {
        Pack<T, V> pa[NB][U], pb[NB][U];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const int hh = h + n * groups + grp;
#pragma unroll
          for (int k = 0; k < U; ++k)
            unit_load<T, V>(in + (int64_t)hh * t.in_head, lo[k], hi[k], hh < end && lo_ok[k], pa[n][k], pb[n][k]);
        }
        float x[NB][U][2 * V], rstd[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int k = 0; k < U; ++k) unit_unpack<T, V>(pa[n][k], pb[n][k], x[n][k]);
        rows_normalize<NB, U, V>(p, x, lo_ok, hi_ok, rstd);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const int hh = h + n * groups + grp;
          if (hh < end) {
#pragma unroll
            for (int k = 0; k < U; ++k) {
              if (lo_ok[k]) {
                float f[2 * V];
#pragma unroll
                for (int j = 0; j < 2 * V; ++j) f[j] = fmaf(x[n][k][j], w[k][j], bi[k][j]);
                unit_rotate<V, HALF, false>(f, cs[k], sn[k]);
                unit_store<T, V>(out + (int64_t)hh * t.out_head, lo[k], hi[k], f);
              }
            }
          }
        }
      }
    }
  }
}

// ----------------------------------------------------------------------------------------
// backward: the rows are normalized again from the inputs (nothing but them is kept), the
// gradient is rotated back, and the norm is differentiated.  The sums for weight and bias stay
// in the lanes' registers over all rows of a CTA and are added in a fixed order at its end, so a
// CTA works for one tensor only.
// ----------------------------------------------------------------------------------------
template <typename T, int V, int U, bool HALF, int NB>
__global__ void __launch_bounds__(kRotThreads) rotary_bwd_kernel(const RotParams p) {
  extern __shared__ float sacc[];  // [warps][2][dim]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int L = 1 << p.log2_l;
  const int groups = 32 >> p.log2_l;
  const int grp = lane >> p.log2_l, ul = lane & (L - 1);
  const int which = (int)blockIdx.x < p.nb0 ? 0 : 1;
  const RotTensor& t = p.t[which];
  const int cta = which == 0 ? (int)blockIdx.x : (int)blockIdx.x - p.nb0;
  const int ctas = which == 0 ? p.nb0 : (int)gridDim.x - p.nb0;
  int lo[U], hi[U];
  bool lo_ok[U], hi_ok[U];
  float w[U][2 * V], dw[U][2 * V], db[U][2 * V];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int u = ul + k * L;
    lo_ok[k] = u < p.units;
    lo[k] = hi[k] = 0;
    if (lo_ok[k]) unit_columns<V, HALF>(p, u, lo[k], hi[k]);
    hi_ok[k] = lo_ok[k] && hi[k] >= 0;
    unit_param<T, V>(reinterpret_cast<const T*>(t.weight), lo[k], hi[k], lo_ok[k], t.weight != nullptr ? 0.f : 1.f, w[k]);
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) {
      if (t.weight != nullptr) w[k][j] += p.woff;
      dw[k][j] = 0.f;
      db[k][j] = 0.f;
    }
  }
  const float inv_d = 1.0f / (float)p.dim;
  const int splits = p.splits[which], per_split = p.per_split[which];
  const int64_t items = (int64_t)p.tokens * splits;
  const int64_t step = (int64_t)ctas * (kRotThreads / 32);
  for (int64_t it = (int64_t)cta * (kRotThreads / 32) + warp; it < items; it += step) {
    const int token = (int)(it / splits);
    const int h0 = (int)(it - (int64_t)token * splits) * per_split;
    const int end = h0 + per_split < t.heads ? h0 + per_split : t.heads;
    const int b = token / p.seq, s = token - b * p.seq;
    float cs[U][V], sn[U][V];
#pragma unroll
    for (int k = 0; k < U; ++k) unit_angles<V>(p, ul + k * L, b, s, cs[k], sn[k]);
    const T* in = reinterpret_cast<const T*>(t.in) + (int64_t)b * t.in_batch + (int64_t)s * t.in_seq;
    const T* go = reinterpret_cast<const T*>(t.out) + (int64_t)b * t.out_batch + (int64_t)s * t.out_seq;
    T* dx = reinterpret_cast<T*>(t.dx) + (int64_t)token * t.heads * p.dim;
#pragma unroll 1
    for (int h = h0; h < end; h += groups * NB) {
      Pack<T, V> pa[NB][U], pb[NB][U], ga[NB][U], gb[NB][U];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int hh = h + n * groups + grp;
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const bool ok = hh < end && lo_ok[k];
          unit_load<T, V>(in + (int64_t)hh * t.in_head, lo[k], hi[k], ok, pa[n][k], pb[n][k]);
          unit_load<T, V>(go + (int64_t)hh * t.out_head, lo[k], hi[k], ok, ga[n][k], gb[n][k]);
        }
      }
      float x[NB][U][2 * V], rstd[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int k = 0; k < U; ++k) unit_unpack<T, V>(pa[n][k], pb[n][k], x[n][k]);
      rows_normalize<NB, U, V>(p, x, lo_ok, hi_ok, rstd);
      float g[NB][U][2 * V], red[2 * NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float r0 = 0.f, r1 = 0.f;
#pragma unroll
        for (int k = 0; k < U; ++k) {
          unit_unpack<T, V>(ga[n][k], gb[n][k], g[n][k]);
          unit_rotate<V, HALF, true>(g[n][k], cs[k], sn[k]);
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) {
            dw[k][j] = fmaf(g[n][k][j], x[n][k][j], dw[k][j]);
            db[k][j] += g[n][k][j];
            g[n][k][j] *= w[k][j];
            r0 = fmaf(g[n][k][j], x[n][k][j], r0);
            r1 += g[n][k][j];
          }
        }
        red[2 * n] = r0;
        red[2 * n + 1] = r1;
      }
      if (p.kind != FLN_NO_NORM) lane_sum<2 * NB>(red, p.log2_l);
      if (t.dx == nullptr) continue;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int hh = h + n * groups + grp;
        if (hh < end) {
          const float c1 = red[2 * n] * inv_d;
          const float c2 = p.kind == FLN_LAYERNORM ? red[2 * n + 1] * inv_d : 0.f;
#pragma unroll
          for (int k = 0; k < U; ++k) {
            if (lo_ok[k]) {
              if (p.kind != FLN_NO_NORM) {
#pragma unroll
                for (int j = 0; j < 2 * V; ++j) g[n][k][j] = rstd[n] * fmaf(-x[n][k][j], c1, g[n][k][j] - c2);
              }
              unit_store<T, V>(dx + (int64_t)hh * p.dim, lo[k], hi[k], g[n][k]);
            }
          }
        }
      }
    }
  }
  if (t.partials == nullptr) return;
  // row groups of the warp, then the warps of the CTA
#pragma unroll
  for (int k = 0; k < U; ++k) {
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) {
      for (int off = 16; off >= L; off >>= 1) {
        dw[k][j] += __shfl_xor_sync(0xffffffffu, dw[k][j], off);
        db[k][j] += __shfl_xor_sync(0xffffffffu, db[k][j], off);
      }
      const bool ok = j < V ? lo_ok[k] : hi_ok[k];
      const int c = (j < V ? lo[k] + j : hi[k] + j - V);
      if (grp == 0 && ok) {
        sacc[(warp * 2) * p.dim + c] = dw[k][j];
        sacc[(warp * 2 + 1) * p.dim + c] = db[k][j];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.dim; i += kRotThreads) {
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < kRotThreads / 32; ++q) v += sacc[q * 2 * p.dim + i];
    t.partials[(int64_t)cta * 2 * p.dim + i] = v;
  }
}

// plan of a problem (host), and the launches of one element type
struct RotPlan {
  int V, U;
  bool half;
};
template <typename T>
int rotary_launch(const RotParams& p, const RotPlan& plan, bool backward, unsigned grid, cudaStream_t st);

template <typename T, int V, int U>
static int rotary_launch_vu(const RotParams& p, bool half, bool backward, unsigned grid, cudaStream_t st) {
  // rows in flight per row group: 64 bytes of each tensor per lane where the registers allow it
  constexpr int W = V * U * (int)sizeof(T);
  constexpr int NBF = W <= 16 ? 4 : (W <= 32 ? 2 : 1);
  constexpr int NBB = W <= 16 ? 2 : 1;
  if (!backward) {
    if (half) rotary_fwd_kernel<T, V, U, true, NBF><<<grid, kRotThreads, 0, st>>>(p);
    else rotary_fwd_kernel<T, V, U, false, NBF><<<grid, kRotThreads, 0, st>>>(p);
  } else {
    const size_t smem = (size_t)(kRotThreads / 32) * 2 * p.dim * sizeof(float);
    if (half) rotary_bwd_kernel<T, V, U, true, NBB><<<grid, kRotThreads, smem, st>>>(p);
    else rotary_bwd_kernel<T, V, U, false, NBB><<<grid, kRotThreads, smem, st>>>(p);
  }
  FLN_CHECK_LAUNCH();
  return FLN_OK;
}

template <typename T, int V>
static int rotary_launch_v(const RotParams& p, const RotPlan& plan, bool backward, unsigned grid, cudaStream_t st) {
  switch (plan.U) {
    case 1:
      return rotary_launch_vu<T, V, 1>(p, plan.half, backward, grid, st);
    case 3:
      return rotary_launch_vu<T, V, 3>(p, plan.half, backward, grid, st);
    case 8:
      if constexpr (V <= 2) return rotary_launch_vu<T, V, 8>(p, plan.half, backward, grid, st);
      return FLN_ERR_UNSUPPORTED;
    default:
      return FLN_ERR_UNSUPPORTED;
  }
}

#define FLN_ROTARY_INSTANTIATE(T)                                                                                  \
  template <>                                                                                                      \
  int rotary_launch<T>(const RotParams& p, const RotPlan& plan, bool backward, unsigned grid, cudaStream_t st) {   \
    switch (plan.V) {                                                                                              \
      case 8:                                                                                                      \
        if constexpr (sizeof(T) == 2) return rotary_launch_v<T, 8>(p, plan, backward, grid, st);                   \
        return FLN_ERR_UNSUPPORTED;                                                                                \
      case 4:                                                                                                      \
        return rotary_launch_v<T, 4>(p, plan, backward, grid, st);                                                 \
      case 2:                                                                                                      \
        return rotary_launch_v<T, 2>(p, plan, backward, grid, st);                                                 \
      default:                                                                                                     \
        return rotary_launch_v<T, 1>(p, plan, backward, grid, st);                                                 \
    }                                                                                                              \
  }

}  // namespace fln
