// The norms around a block fused with its gate and residual scale: what the kernels of
// fln_nga.cu share.
//
//     s = ra * residual + ba * act(gate) * N1(x)         y = N2(s)
//     N(z) = xh * w + b,  xh = (z - mean) * rstd          w = weight_offset + weight
//
// The sum s stays in 32 bits for N2 and is rounded once, when it is stored; so is y.
// Backward, from dy and dsum, with n1 = N1(x) and sh = (s - mean2) * rstd2, where s is made again
// from x and residual: as many bytes as reading the stored sum, without its rounding (which would
// put 2^-9 |s| rstd2 on every sh at 16 bits), and none at all where there is no residual:
//     g2 = dy * w2;  c1 = mean(g2 * sh);  c2 = mean(g2) (LayerNorm, else 0)
//     ds = dsum + rstd2 * ((g2 - c2) - sh * c1)                dresidual = ra * ds
//     e  = ba * ds;  f = e * act(gate)                         dgate = e * n1 * act'(gate)
//     g1 = f * w1;  d1 = mean(g1 * xh);  d2 = mean(g1) (LayerNorm, else 0)
//     dx = rstd1 * ((g1 - d2) - xh * d1)
// The sums over rows that the parameters need are four at most, whatever is asked for:
//     U = sum dy * sh, V = sum dy                 dweight = U, dbias = V
//     P = sum h * xh,  Q = sum h                  h = f for a gate per element, else h = e
// With a gate shared by the rows of a group, act(gate) is constant under the sum, so
//     dpost_weight = sum_groups act(gate) * P,  dpost_bias = sum_groups act(gate) * Q,
//     dgate = act'(gate) * (w1 * P + b1 * Q)
// and no third pair of column sums is carried.
//
// Rows are cut into slots of at most `chunk` consecutive rows that never cross a group; every
// slot leaves its own partial sums in the workspace (fp32), and a last kernel adds the partial
// sums of a group, or of all groups, in slot order.  So the results do not depend on which CTA
// took which slot.
#pragma once

#include "fln_common.cuh"

namespace fln {

struct NgaParams {
  const void* x;
  const void* res;
  const void* gate;
  const void* w1;
  const void* b1;
  const void* w2;
  const void* b2;
  int64_t rows;
  int64_t group_rows;
  int cols;
  int post_kind, kind, gate_mode, act;
  int affine_grouped;
  float ba, ra, woff, eps1, eps2;
  // forward
  void* y;
  void* sum;
  float* mean1;
  float* rstd1;
  float* mean2;
  float* rstd2;
  // backward (the statistics are inputs there)
  const void* dy;
  const void* ds;
  void* dx;
  void* dres;
  void* dgate;
  float* row_c;     // [rows][2]: c1, c2 of every row, for the column kernel
  float* partials;  // [partial rows][nacc][cols]
  int acc;          // which sums: 1 P, 2 Q, 4 U, 8 V
  int nacc;
  int64_t chunk;           // rows per slot
  int64_t slots_per_group;
  int64_t slots;
  int64_t groups;  // set for the last kernel
  // Rows that are not whole 16-byte vectors start at one of `period` places of a vector in turn.  A
  // slot then holds rows of one such class (every period-th row of the group), `classes` of them per
  // group, cut into `pieces` slots each.  period 1: whole vectors, slots of `chunk` rows.
  int period, classes;
  int64_t pieces;
};
constexpr int kAccP = 1, kAccQ = 2, kAccU = 4, kAccV = 8;

// act(v) and act'(v).  32-bit types: the full-precision exponential and tanh; the reciprocal is the
// hardware's, good to one unit in the last place, where a correctly rounded one costs some eight
// instructions.  16-bit types: the hardware exponential too.  Its argument v log2(e) is rounded to 24
// bits, so a sigmoid is good to 2^-22 + |v| 2^-24 of itself: 2^-18 at v = -40, below the half step of
// 2^-12 that fp16 has and the 2^-9 of bf16.
template <bool EXACT>
__device__ __forceinline__ float sigmoid_of(float v) {
  if (EXACT) return rcp_approx(1.0f + expf(-v));  // (the reciprocal is good to one unit in the last place)
  return rcp_approx(1.0f + ex2_approx(-1.4426950408889634f * v));
}
template <bool EXACT>
__device__ __forceinline__ float gate_act(float v, int act) {
  if (act == FLN_GATE_ACT_SIGMOID) return sigmoid_of<EXACT>(v);
  // v * (the reciprocal of an overflowed 1 + exp(-v), which is 0) is -0 for large negative v
  if (act == FLN_GATE_ACT_SILU) return v * sigmoid_of<EXACT>(v);
  if (act == FLN_GATE_ACT_TANH) return tanhf(v);
  return v;
}
template <bool EXACT>
__device__ __forceinline__ void gate_act_grad(float v, int act, float* a, float* da) {
  if (act == FLN_GATE_ACT_SIGMOID) {
    const float q = sigmoid_of<EXACT>(v);
    *a = q;
    *da = q * (1.0f - q);
  } else if (act == FLN_GATE_ACT_SILU) {
    const float q = sigmoid_of<EXACT>(v);
    *a = v * q;
    *da = q * fmaf(v, 1.0f - q, 1.0f);
  } else if (act == FLN_GATE_ACT_TANH) {
    const float t = tanhf(v);
    *a = t;
    *da = fmaf(-t, t, 1.0f);
  } else {
    *a = v;
    *da = 1.0f;
  }
}
template <int V>
struct Known {
  static constexpr int value = V;
};
// the same of N pairs: which function is asked once for all of them, so that their special-function
// instructions follow each other instead of each waiting behind a branch (262144 x 128 bf16: forward
// 42.8 -> 38.5 us, backward 58.7 -> 54.3).  The general backward has no registers left for it and takes
// one pair after the other (2047 x 5120 fp32: 67 us, 78 all at once).
template <bool EXACT, int N>
__device__ __forceinline__ void gate_act_all(float2 (&v)[N], int act) {
  auto all = [&](auto known) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = make_float2(gate_act<EXACT>(v[e].x, known.value), gate_act<EXACT>(v[e].y, known.value));
  };
  if (act == FLN_GATE_ACT_SIGMOID) all(Known<FLN_GATE_ACT_SIGMOID>());
  else if (act == FLN_GATE_ACT_SILU) all(Known<FLN_GATE_ACT_SILU>());
  else if (act == FLN_GATE_ACT_TANH) all(Known<FLN_GATE_ACT_TANH>());
}
template <bool EXACT, int N>
__device__ __forceinline__ void gate_act_grad_all(float2 (&v)[N], float2 (&d)[N], int act) {  // v becomes act(v)
  auto all = [&](auto known) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      float2 a;
      gate_act_grad<EXACT>(v[e].x, known.value, &a.x, &d[e].x);
      gate_act_grad<EXACT>(v[e].y, known.value, &a.y, &d[e].y);
      v[e] = a;
    }
  };
  if (act == FLN_GATE_ACT_SIGMOID) all(Known<FLN_GATE_ACT_SIGMOID>());
  else if (act == FLN_GATE_ACT_SILU) all(Known<FLN_GATE_ACT_SILU>());
  else if (act == FLN_GATE_ACT_TANH) all(Known<FLN_GATE_ACT_TANH>());
  else all(Known<FLN_GATE_ACT_NONE>());
}

// sum of NV values over the CTA, result in every thread, the same order everywhere; red holds
// 2 x NV x 32 floats, `flip` alternates so that one barrier per call is enough
template <int NV>
__device__ __forceinline__ void cta_sum(float (&v)[NV], float* red, int& flip) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], off);
  }
  float* r = red + flip * (NV * 32);
  flip ^= 1;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) r[i * 32 + (threadIdx.x >> 5)] = v[i];
  }
  __syncthreads();
  const int nw = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float t = 0.f;
    for (int w = 0; w < nw; ++w) t += r[i * 32 + w];
    v[i] = t;
  }
}

// the rows of slot `slot`
struct SlotRows {
  int64_t group, first, last;  // rows first, first + p.period, ... below last; last - 1 is one of them
};
__device__ __forceinline__ SlotRows slot_rows(const NgaParams& p, int64_t slot) {
  SlotRows s;
  s.group = slot / p.slots_per_group;
  const int64_t j = slot - s.group * p.slots_per_group;
  const int64_t g0 = s.group * p.group_rows;
  if (p.period > 1) {
    const int64_t c = j % p.classes, piece = j / p.classes;
    const int64_t n = (p.group_rows - c + p.period - 1) / p.period;  // rows of the class, at least `pieces`
    s.first = g0 + c + piece * n / p.pieces * p.period;
    s.last = g0 + c + ((piece + 1) * n / p.pieces - 1) * p.period + 1;
    return s;
  }
  s.first = g0 + j * p.chunk;
  s.last = s.first + p.chunk < g0 + p.group_rows ? s.first + p.chunk : g0 + p.group_rows;
  return s;
}

struct NgaGrads {
  void* dgate;  // of a shared gate
  void* dw1;
  void* db1;
  void* dw2;
  void* db2;
};

}  // namespace fln
