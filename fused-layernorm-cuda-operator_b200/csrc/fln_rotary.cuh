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
// Angles.  position * turns modulo 2^64 is the fraction of a turn as a 64-bit integer, so the range
// reduction is the wrap of an integer product: no table of cosines to read, nothing lost at far
// positions.  sincospi of what is left behind whole quarter turns gives cosine and sine.  A warp
// makes them once per token, in shared memory, for all the heads that it takes of that token.
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
  int nb0;      // backward: the first nb0 CTAs take q, the others k
  int want_db;  // a bias gradient is asked for
};

constexpr int kRotThreads = 256;
// CTAs per SM that the registers are cut for, by the pairs a lane holds of a row
__host__ __device__ constexpr int rot_blocks(int pairs, bool backward) {
  return pairs <= 8 ? (backward ? 2 : 3) : (pairs <= 12 ? 2 : 1);
}

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

// Tables in shared memory, in 32 bits.  Every warp keeps the cosines and sines of its token, one
// entry per pair: the lanes make the angles between them, P / 32 each, and all row groups of the
// warp read them.  The CTA keeps
// weight_offset + weight and bias of both tensors.  (With the angles made by every lane for its own
// unit and held in registers beside the weights, the bf16 forward at 8192 x 48 x 128 ran with 80
// registers, 16.7 instructions per element, 55 us.)
struct RotTables {
  float *c, *s;  // of this warp: [rot_units * V] each
  float *w, *b;  // of q; those of k lie `step` behind them
  int step;
};
__host__ __device__ constexpr size_t rot_tables_floats(int rot_units, int V, int dim, bool gen) {
  return (size_t)(kRotThreads / 32) * 2 * rot_units * V + (size_t)(gen ? 4 : 2) * ((dim + 3) & ~3);
}
template <typename T, int V, bool GEN>
__device__ __forceinline__ RotTables rot_tables(const RotParams& p, float* mem) {
  RotTables t;
  const int n = p.rot_units * V, warp = threadIdx.x >> 5, dim4 = (p.dim + 3) & ~3;
  t.c = mem + warp * 2 * n;
  t.s = t.c + n;
  t.w = mem + (kRotThreads / 32) * 2 * n;
  t.b = t.w + dim4;
  t.step = GEN ? 2 * dim4 : dim4;
  for (int i = threadIdx.x; i < 2 * p.dim; i += kRotThreads) {
    const int which = i >= p.dim ? 1 : 0, c = i - which * p.dim;
    const T* w = reinterpret_cast<const T*>(p.t[which].weight);
    t.w[which * t.step + c] = w != nullptr ? p.woff + Cvt<T>::to_f(w[c]) : 1.f;
    if (GEN) {
      const T* b = reinterpret_cast<const T*>(p.t[which].bias);
      t.b[which * t.step + c] = b != nullptr ? Cvt<T>::to_f(b[c]) : 0.f;
    }
  }
  __syncthreads();
  return t;
}
// the angles of a token into its warp's table
__device__ __forceinline__ void token_angles(const RotParams& p, const RotTables& t, int batch, int seq) {
  const int64_t at0 = (int64_t)batch * p.pos_batch + (int64_t)seq * p.pos_seq;
  __syncwarp();  // nobody reads the last token's any more
  for (int i = threadIdx.x & 31; i < p.pairs; i += 32) {
    const int64_t at = at0 + (int64_t)__ldg(p.axis + i) * p.pos_axis;
    const long long pos = p.pos64 ? __ldg(reinterpret_cast<const long long*>(p.positions) + at)
                                  : (long long)__ldg(reinterpret_cast<const int*>(p.positions) + at);
    // The fraction of a turn in 2^64ths.  Whole quarter turns are taken off while it is an integer:
    // what goes into 32 bits is an eighth of a turn at most, so a cosine or sine keeps its own relative
    // precision next to its zeros too (the whole fraction rounded: 1.1e-7 at most, so 5e-8).
    const unsigned long long frac = (unsigned long long)pos * __ldg(p.turns + i);
    const unsigned quarters = (unsigned)((frac + (1ull << 61)) >> 62);
    float sv, cv;  // rest / 2^63 half turns, in [-1/4, 1/4]
    sincospif(__ll2float_rn((long long)(frac - ((unsigned long long)quarters << 62))) * 1.0842021724855044e-19f, &sv, &cv);
    const float c = quarters & 1 ? sv : cv, s = quarters & 1 ? cv : sv;
    t.c[i] = ((quarters + 1) & 2 ? -c : c) * p.mag;
    t.s[i] = (quarters & 2 ? -s : s) * p.mag;
  }
  __syncwarp();
}
// V floats of a table
template <int V>
__device__ __forceinline__ void table_take(const float* t, float (&f)[V]) {
  if constexpr (V >= 4) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const float4 q = *reinterpret_cast<const float4*>(t + j);
      f[j] = q.x;
      f[j + 1] = q.y;
      f[j + 2] = q.z;
      f[j + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = t[j];
  }
}
// a unit's share of a row table, as register pairs
template <int V>
__device__ __forceinline__ void table_unit(const float* t, int lo, int hi, float2 (&f)[V]) {
  float a[V], b[V];
  table_take<V>(t + lo, a);
  table_take<V>(t + hi, b);
  if constexpr (V == 1) {
    f[0] = make_float2(a[0], b[0]);
  } else {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      f[j] = make_float2(a[2 * j], a[2 * j + 1]);
      f[V / 2 + j] = make_float2(b[2 * j], b[2 * j + 1]);
    }
  }
}

// A unit as V register pairs: f[0, V / 2) its first vector and f[V / 2, V) its second one; with
// V == 1 both elements in one pair.
template <typename T, int V>
struct UnitPack {
  Pack<T, V> a, b;
};
// (absent vectors read as zeros)
template <typename T, int V, bool WHOLE>
__device__ __forceinline__ UnitPack<T, V> unit_load(const T* row, int lo, int hi, bool lo_ok, bool hi_ok) {
  UnitPack<T, V> u;
  if (!WHOLE) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      u.a.e[j] = Cvt<T>::from_f(0.f);
      u.b.e[j] = Cvt<T>::from_f(0.f);
    }
  }
  if (WHOLE || lo_ok) u.a = ld_stream<T, V>(row + lo);
  if (WHOLE || hi_ok) u.b = ld_stream<T, V>(row + hi);
  return u;
}
template <typename T, int V>
__device__ __forceinline__ void unit_unpack(const UnitPack<T, V>& u, float2 (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = make_float2(Cvt<T>::to_f(u.a.e[0]), Cvt<T>::to_f(u.b.e[0]));
  } else {
    float2 t[V / 2];
    unpack2<T, V>(u.a, t);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) f[j] = t[j];
    unpack2<T, V>(u.b, t);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) f[V / 2 + j] = t[j];
  }
}
template <typename T, int V>
__device__ __forceinline__ void unit_store(T* row, int lo, int hi, bool hi_ok, const float2 (&f)[V]) {
  if constexpr (V == 1) {
    row[lo] = Cvt<T>::from_f(f[0].x);
    if (hi_ok) row[hi] = Cvt<T>::from_f(f[0].y);
  } else {
    float2 t[V / 2];
    Pack<T, V> o;
#pragma unroll
    for (int j = 0; j < V / 2; ++j) t[j] = f[j];
    pack2<T, V>(t, o);
    st_plain<T, V>(row + lo, o);
    if (hi_ok) {
#pragma unroll
      for (int j = 0; j < V / 2; ++j) t[j] = f[V / 2 + j];
      pack2<T, V>(t, o);
      st_plain<T, V>(row + hi, o);
    }
  }
}
// rotation of the V pairs of a unit by the angle, or back
template <int V, bool HALF, bool BACK>
__device__ __forceinline__ void unit_rotate(float2 (&f)[V], const float (&c)[V], const float (&s)[V]) {
  if constexpr (HALF && V > 1) {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const float2 cc = make_float2(c[2 * j], c[2 * j + 1]);
      const float2 ss = make_float2(s[2 * j], s[2 * j + 1]), ns = make_float2(-s[2 * j], -s[2 * j + 1]);
      const float2 a = f[j], b = f[V / 2 + j];
      f[j] = f2fma(b, BACK ? ss : ns, f2mul(a, cc));
      f[V / 2 + j] = f2fma(a, BACK ? ns : ss, f2mul(b, cc));
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float a = f[j].x, b = f[j].y;
      f[j].x = BACK ? fmaf(b, s[j], a * c[j]) : fmaf(-b, s[j], a * c[j]);
      f[j].y = BACK ? fmaf(-a, s[j], b * c[j]) : fmaf(a, s[j], b * c[j]);
    }
  }
}

// ... by its angles in the table; a unit of the part that is not rotated stays as it is (a rotation
// by nothing would multiply by zero, and take an infinity to its neighbour as NaN)
template <int V, bool HALF, bool BACK>
__device__ __forceinline__ void unit_turn(float2 (&f)[V], const RotTables& tab, int at, bool turn) {
  if (!turn) return;
  float c[V], s[V];
  table_take<V>(tab.c + at, c);
  table_take<V>(tab.s + at, s);
  unit_rotate<V, HALF, BACK>(f, c, s);
}

template <int N, int LL>
__device__ __forceinline__ void lane_sum(float (&v)[N], int log2_l) {
  if constexpr (LL >= 0) {
#pragma unroll
    for (int off = (1 << LL) >> 1; off > 0; off >>= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], off);
    }
  } else {
    for (int off = (1 << log2_l) >> 1; off > 0; off >>= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], off);
    }
  }
}

// v where the element exists, else 0: elements behind the row must not count as -mean
template <int V>
__device__ __forceinline__ float2 in_row(float2 v, int j, bool lo_ok, bool hi_ok) {
  if constexpr (V == 1) return make_float2(lo_ok ? v.x : 0.f, hi_ok ? v.y : 0.f);
  const bool ok = j < V / 2 ? lo_ok : hi_ok;
  return make_float2(ok ? v.x : 0.f, ok ? v.y : 0.f);
}

// what every lane of both kernels holds of its place in the row
template <int V, int U, bool HALF>
struct RotLane {
  int L, groups, grp, ul;
  int lo[U], hi[U];          // first columns of the unit's vectors (of another vector where there is none)
  int at[U];                 // its first entry in the table of angles
  bool rot[U];               // it is rotated
  bool lo_ok[U], hi_ok[U];
  template <int LL>
  __device__ __forceinline__ void init(const RotParams& p) {
    const int lane = threadIdx.x & 31;
    const int ll = LL >= 0 ? LL : p.log2_l;
    L = 1 << ll;
    groups = 32 >> ll;
    grp = lane >> ll;
    ul = lane & (L - 1);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int u = ul + k * L;
      lo_ok[k] = u < p.units;
      unit_columns<V, HALF>(p, lo_ok[k] ? u : 0, lo[k], hi[k]);
      hi_ok[k] = lo_ok[k] && hi[k] >= 0;
      if (hi[k] < 0) hi[k] = lo[k];
      rot[k] = u < p.rot_units;
      at[k] = (rot[k] ? u : 0) * V;
      if (LL >= 0) lo_ok[k] = hi_ok[k] = true;  // whole units on every lane
    }
  }
};

// ----------------------------------------------------------------------------------------
// forward: the work is one sequence of steps, token after token; a step is NB heads of q or of k for
// each of a warp's 32 / L row groups, so that NB rows per group are on their way from memory
// together.  The warps of as many CTAs as are resident at once take equal runs of it (with a token
// per warp and its CTA's tables made for eight tokens, 8192 x 48 x 128 bf16 took 44 us, 40 so); a run
// that starts inside a token makes that token's angles again.  All lanes of a warp take part in
// every step, so the shuffles are whole.  The rows stay packed as they came; they are unpacked once
// for the sums and once more for the result, which costs an instruction per element and saves the
// registers that let more warps (and so more loads) be in flight.
// GEN: layer norm or bias.  LL >= 0: log2 of the lanes per row, known at compile time.  PART: there are
// units that are not rotated (asked for each unit where every one is: 8192 x 48 x 128 bf16, backward
// 70.8 -> 74.9 us with its sums).
// ----------------------------------------------------------------------------------------
template <typename T, int V, int U, bool HALF, int NB, bool GEN, int LL, bool PART>
__global__ void __launch_bounds__(kRotThreads, rot_blocks(V * U, false)) rotary_fwd_kernel(const RotParams p) {
  RotLane<V, U, HALF> r;
  r.template init<LL>(p);
  extern __shared__ __align__(16) float tables[];
  const RotTables tab = rot_tables<T, V, GEN>(p, tables);
  constexpr bool WHOLE = LL >= 0;
  const float inv_d = 1.0f / (float)p.dim;
  const int q_heads = p.t[0].heads, turn = r.groups * NB;
  const int q_steps = (q_heads + turn - 1) / turn, steps = q_steps + (p.t[1].heads + turn - 1) / turn;
  const int64_t total = (int64_t)p.tokens * steps, warps = (int64_t)gridDim.x * (kRotThreads / 32);
  const int64_t me = (int64_t)blockIdx.x * (kRotThreads / 32) + (threadIdx.x >> 5);
  const int64_t lo = total * me / warps, hi = total * (me + 1) / warps;
  int token = (int)(lo / steps), step = (int)(lo - (int64_t)token * steps);
  int b = 0, s = 0;
  bool fresh = true;
#pragma unroll 1
  for (int64_t i = lo; i < hi; ++i) {
    if (fresh) {
      b = p.tokens == p.seq ? 0 : token / p.seq;
      s = token - b * p.seq;
    }
    const int which = step >= q_steps ? 1 : 0;
    const RotTensor& t = p.t[which];
    const int h = (step - (which == 0 ? 0 : q_steps)) * turn, end = t.heads;
    const T* in = reinterpret_cast<const T*>(t.in) + (int64_t)b * t.in_batch + (int64_t)s * t.in_seq;
    T* out = reinterpret_cast<T*>(t.out) + (int64_t)b * t.out_batch + (int64_t)s * t.out_seq;
    UnitPack<T, V> x[NB][U];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      // (row groups behind the last head take it once more and store nothing)
      const int hh = min(h + n * r.groups + r.grp, end - 1);
      const T* row = in + (int64_t)hh * t.in_head;
#pragma unroll
      for (int k = 0; k < U; ++k) x[n][k] = unit_load<T, V, WHOLE>(row, r.lo[k], r.hi[k], r.lo_ok[k], r.hi_ok[k]);
    }
    if (fresh) {  // behind the loads, so that both wait for memory together
      fresh = false;
      token_angles(p, tab, b, s);
    }
    float mean[NB], rstd[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      mean[n] = 0.f;
      rstd[n] = 1.f;
    }
    if (p.kind != FLN_NO_NORM) {
      float v[NB];
      if (GEN && p.kind == FLN_LAYERNORM) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          float2 a = f2(0.f);
#pragma unroll
          for (int k = 0; k < U; ++k) {
            float2 f[V];
            unit_unpack<T, V>(x[n][k], f);
#pragma unroll
            for (int j = 0; j < V; ++j) a = f2add(a, f[j]);
          }
          v[n] = a.x + a.y;
        }
        lane_sum<NB, LL>(v, p.log2_l);
#pragma unroll
        for (int n = 0; n < NB; ++n) mean[n] = v[n] * inv_d;
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float2 a = f2(0.f);
#pragma unroll
        for (int k = 0; k < U; ++k) {
          float2 f[V];
          unit_unpack<T, V>(x[n][k], f);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            if (GEN) {
              f[j] = f2add(f[j], f2(-mean[n]));
              if (!WHOLE) f[j] = in_row<V>(f[j], j, r.lo_ok[k], r.hi_ok[k]);
            }
            a = f2fma(f[j], f[j], a);
          }
        }
        v[n] = a.x + a.y;
      }
      lane_sum<NB, LL>(v, p.log2_l);
#pragma unroll
      for (int n = 0; n < NB; ++n) rstd[n] = rsqrtf(fmaf(v[n], inv_d, p.eps));
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int hh = h + n * r.groups + r.grp;
      T* row = out + (int64_t)hh * t.out_head;
#pragma unroll
      for (int k = 0; k < U; ++k) {
        float2 f[V], w[V], bi[V];
        unit_unpack<T, V>(x[n][k], f);
        table_unit<V>(tab.w + which * tab.step, r.lo[k], r.hi[k], w);
        if (GEN) table_unit<V>(tab.b + which * tab.step, r.lo[k], r.hi[k], bi);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (GEN) f[j] = f2add(f[j], f2(-mean[n]));
          f[j] = f2mul(f[j], f2(rstd[n]));
          f[j] = GEN ? f2fma(f[j], w[j], bi[j]) : f2mul(f[j], w[j]);
        }
        unit_turn<V, HALF, false>(f, tab, r.at[k], !PART || r.rot[k]);
        if (hh < end && r.lo_ok[k]) unit_store<T, V>(row, r.lo[k], r.hi[k], r.hi_ok[k], f);
      }
    }
    if (++step == steps) {
      step = 0;
      ++token;
      fresh = true;
    }
  }
}

// ----------------------------------------------------------------------------------------
// backward: the rows are normalized again from the inputs (nothing but them is kept), the
// gradient is rotated back, and the norm is differentiated:
//     dn = rotated back,  g = dn * w,  c1 = mean(g * xh), c2 = mean(g) (LayerNorm),
//     dx = rstd * ((g - c2) - xh * c1),  dw = sum dn * xh,  db = sum dn
// RMSNorm needs one exchange between the lanes: mean(g * xh) = rstd * mean(g * x).  The sums for
// weight and bias stay in the lanes' registers over all rows of a CTA and are added in a fixed
// order at its end, so a CTA works for one tensor only.
// ----------------------------------------------------------------------------------------
template <typename T, int V, int U, bool HALF, int NB, bool GEN, int LL, bool PART>
__global__ void __launch_bounds__(kRotThreads, rot_blocks(V * U, true)) rotary_bwd_kernel(const RotParams p) {
  extern __shared__ __align__(16) float sacc[];  // the tables; at the end [warps][2][dim]
  const RotTables tab = rot_tables<T, V, GEN>(p, sacc);
  constexpr bool WHOLE = LL >= 0;
  const int warp = threadIdx.x >> 5;
  RotLane<V, U, HALF> r;
  r.template init<LL>(p);
  const int which = (int)blockIdx.x < p.nb0 ? 0 : 1;
  const RotTensor& t = p.t[which];
  const int cta = which == 0 ? (int)blockIdx.x : (int)blockIdx.x - p.nb0;
  const int ctas = which == 0 ? p.nb0 : (int)gridDim.x - p.nb0;
  float2 dw[U][V], db[GEN ? U : 1][V];
#pragma unroll
  for (int k = 0; k < U; ++k) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      dw[k][j] = f2(0.f);
      if (GEN) db[GEN ? k : 0][j] = f2(0.f);
    }
  }
  const float inv_d = 1.0f / (float)p.dim;
  const int turn = r.groups * NB, steps = (t.heads + turn - 1) / turn;
  const int64_t total = (int64_t)p.tokens * steps, warps = (int64_t)ctas * (kRotThreads / 32);
  const int64_t me = (int64_t)cta * (kRotThreads / 32) + warp;
  const int64_t lo = total * me / warps, hi = total * (me + 1) / warps;
  int token = (int)(lo / steps), step = (int)(lo - (int64_t)token * steps);
  int b = 0, s = 0;
  bool fresh = true;
#pragma unroll 1
  for (int64_t i = lo; i < hi; ++i) {
    if (fresh) {
      b = p.tokens == p.seq ? 0 : token / p.seq;
      s = token - b * p.seq;
    }
    const int h = step * turn, end = t.heads;
    const T* in = reinterpret_cast<const T*>(t.in) + (int64_t)b * t.in_batch + (int64_t)s * t.in_seq;
    const T* go = reinterpret_cast<const T*>(t.out) + (int64_t)b * t.out_batch + (int64_t)s * t.out_seq;
    T* dx = reinterpret_cast<T*>(t.dx) + (int64_t)token * t.heads * p.dim;
    UnitPack<T, V> px[NB][U], pg[NB][U];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      // (row groups behind the last head read it once more; their gradient is zero)
      const int hh = min(h + n * r.groups + r.grp, end - 1);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        px[n][k] = unit_load<T, V, WHOLE>(in + (int64_t)hh * t.in_head, r.lo[k], r.hi[k], r.lo_ok[k], r.hi_ok[k]);
        pg[n][k] = unit_load<T, V, WHOLE>(go + (int64_t)hh * t.out_head, r.lo[k], r.hi[k], r.lo_ok[k], r.hi_ok[k]);
      }
    }
    if (fresh) {
      fresh = false;
      token_angles(p, tab, b, s);
    }
    float mean[NB], rstd[NB], c1[NB], c2[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      mean[n] = 0.f;
      rstd[n] = 1.f;
      c1[n] = c2[n] = 0.f;
    }
    if (p.kind != FLN_NO_NORM) {
      if (GEN && p.kind == FLN_LAYERNORM) {
        float v[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          float2 a = f2(0.f);
#pragma unroll
          for (int k = 0; k < U; ++k) {
            float2 f[V];
            unit_unpack<T, V>(px[n][k], f);
#pragma unroll
            for (int j = 0; j < V; ++j) a = f2add(a, f[j]);
          }
          v[n] = a.x + a.y;
        }
        lane_sum<NB, LL>(v, p.log2_l);
#pragma unroll
        for (int n = 0; n < NB; ++n) mean[n] = v[n] * inv_d;
      }
      constexpr int NS = GEN ? 3 : 2;
      float v[NS * NB];  // the squares, g times the centred row, g
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float2 a = f2(0.f), gx = f2(0.f), gs = f2(0.f);
#pragma unroll
        for (int k = 0; k < U; ++k) {
          float2 x[V], g[V], w[V];
          unit_unpack<T, V>(px[n][k], x);
          unit_unpack<T, V>(pg[n][k], g);
          unit_turn<V, HALF, true>(g, tab, r.at[k], !PART || r.rot[k]);
          table_unit<V>(tab.w + which * tab.step, r.lo[k], r.hi[k], w);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            if (GEN) {
              x[j] = f2add(x[j], f2(-mean[n]));
              if (!WHOLE) x[j] = in_row<V>(x[j], j, r.lo_ok[k], r.hi_ok[k]);
            }
            const float2 q = f2mul(g[j], w[j]);
            a = f2fma(x[j], x[j], a);
            gx = f2fma(q, x[j], gx);
            if (GEN) gs = f2add(gs, q);
          }
        }
        v[NS * n] = a.x + a.y;
        v[NS * n + 1] = gx.x + gx.y;
        if (GEN) v[NS * n + NS - 1] = gs.x + gs.y;
      }
      lane_sum<NS * NB, LL>(v, p.log2_l);
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        rstd[n] = rsqrtf(fmaf(v[NS * n], inv_d, p.eps));
        c1[n] = rstd[n] * v[NS * n + 1] * inv_d;
        if (GEN && p.kind == FLN_LAYERNORM) c2[n] = v[NS * n + NS - 1] * inv_d;
      }
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int hh = h + n * r.groups + r.grp;
      const bool live = hh < end;
#pragma unroll
      for (int k = 0; k < U; ++k) {
        float2 x[V], g[V], w[V];
        unit_unpack<T, V>(px[n][k], x);
        unit_unpack<T, V>(pg[n][k], g);
        unit_turn<V, HALF, true>(g, tab, r.at[k], !PART || r.rot[k]);
        table_unit<V>(tab.w + which * tab.step, r.lo[k], r.hi[k], w);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (GEN) x[j] = f2add(x[j], f2(-mean[n]));
          x[j] = f2mul(x[j], f2(rstd[n]));
          if (live) {
            dw[k][j] = f2fma(g[j], x[j], dw[k][j]);
            if (GEN) db[GEN ? k : 0][j] = f2add(db[GEN ? k : 0][j], g[j]);
          }
          g[j] = f2mul(g[j], w[j]);
          if (p.kind != FLN_NO_NORM) {
            if (GEN) g[j] = f2add(g[j], f2(-c2[n]));
            g[j] = f2mul(f2fma(x[j], f2(-c1[n]), g[j]), f2(rstd[n]));
          }
        }
        if (t.dx != nullptr && live && r.lo_ok[k])
          unit_store<T, V>(dx + (int64_t)hh * p.dim, r.lo[k], r.hi[k], r.hi_ok[k], g);
      }
    }
    if (++step == steps) {
      step = 0;
      ++token;
      fresh = true;
    }
  }
  if (t.partials == nullptr) return;
  __syncthreads();  // the tables are done with
  // row groups of the warp, then the warps of the CTA
#pragma unroll
  for (int k = 0; k < U; ++k) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      for (int off = 16; off >= r.L; off >>= 1) {
        dw[k][j].x += __shfl_xor_sync(0xffffffffu, dw[k][j].x, off);
        dw[k][j].y += __shfl_xor_sync(0xffffffffu, dw[k][j].y, off);
        if (GEN) {
          db[GEN ? k : 0][j].x += __shfl_xor_sync(0xffffffffu, db[GEN ? k : 0][j].x, off);
          db[GEN ? k : 0][j].y += __shfl_xor_sync(0xffffffffu, db[GEN ? k : 0][j].y, off);
        }
      }
      if (r.grp == 0) {
        const int i = 2 * j;  // elements i and i + 1 of the unit, of the first vector and then the second
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const bool second = i + e >= V;
          if (second ? !r.hi_ok[k] : !r.lo_ok[k]) continue;
          const int c = second ? r.hi[k] + i + e - V : r.lo[k] + i + e;
          sacc[(warp * 2) * p.dim + c] = e == 0 ? dw[k][j].x : dw[k][j].y;
          sacc[(warp * 2 + 1) * p.dim + c] = GEN ? (e == 0 ? db[GEN ? k : 0][j].x : db[GEN ? k : 0][j].y) : 0.f;
        }
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
int rotary_launch(const RotParams& p, const RotPlan& plan, bool backward, unsigned grid, cudaStream_t st);  // grid: of a backward

template <typename T, int V, int U, bool HALF, bool GEN, int LL, bool PART>
static int rotary_launch_one(const RotParams& p, bool backward, unsigned grid, cudaStream_t st) {
  // rows in flight per row group: 128 bytes of each tensor per lane where the registers allow it
  constexpr int W = 2 * V * U * (int)sizeof(T);
  constexpr int NBF = W <= 64 ? 2 : 1;
  constexpr int NBB = W <= 32 ? 2 : 1;
  size_t smem = rot_tables_floats(p.rot_units, V, p.dim, GEN) * sizeof(float);
  if (!backward) {
    // CTAs: those that are resident at once, fewer where there are not steps for all of their warps
    const int turn = (32 >> p.log2_l) * NBF;
    const int64_t total = (int64_t)p.tokens * ((p.t[0].heads + turn - 1) / turn + (p.t[1].heads + turn - 1) / turn);
    const int64_t all = (int64_t)sm_count() * rot_blocks(V * U, false), most = (total + kRotThreads / 32 - 1) / (kRotThreads / 32);
    grid = (unsigned)(most < all ? most : all);
    rotary_fwd_kernel<T, V, U, HALF, NBF, GEN, LL, PART><<<grid, kRotThreads, smem, st>>>(p);
  } else {
    const size_t sums = (size_t)(kRotThreads / 32) * 2 * p.dim * sizeof(float);
    if (sums > smem) smem = sums;
    rotary_bwd_kernel<T, V, U, HALF, NBB, GEN, LL, PART><<<grid, kRotThreads, smem, st>>>(p);
  }
  FLN_CHECK_LAUNCH();
  return FLN_OK;
}
template <typename T, int V, int U, bool HALF, bool GEN>
static int rotary_launch_ll(const RotParams& p, bool backward, unsigned grid, cudaStream_t st) {
  // heads that fill the lanes with whole 16-byte vectors (64, 128 and 256 elements of 16 bits) have
  // their own kernels
  if constexpr (U == 1 && V * (int)sizeof(T) == 16) {
    if (2 * p.units * V == p.dim && p.units == 1 << p.log2_l) {
#define FLN_ROT_LL(LL)                                                                                            \
  if (p.log2_l == LL)                                                                                             \
    return p.rot_units < p.units ? rotary_launch_one<T, V, U, HALF, GEN, LL, true>(p, backward, grid, st)         \
                                 : rotary_launch_one<T, V, U, HALF, GEN, LL, false>(p, backward, grid, st);
      FLN_ROT_LL(2)
      FLN_ROT_LL(3)
      FLN_ROT_LL(4)
#undef FLN_ROT_LL
    }
  }
  return rotary_launch_one<T, V, U, HALF, GEN, -1, true>(p, backward, grid, st);
}
template <typename T, int V, int U>
static int rotary_launch_vu(const RotParams& p, bool half, bool backward, unsigned grid, cudaStream_t st) {
  const bool gen = p.kind == FLN_LAYERNORM || p.t[0].bias != nullptr || p.t[1].bias != nullptr || p.want_db;
  if (half)
    return gen ? rotary_launch_ll<T, V, U, true, true>(p, backward, grid, st)
               : rotary_launch_ll<T, V, U, true, false>(p, backward, grid, st);
  return gen ? rotary_launch_ll<T, V, U, false, true>(p, backward, grid, st)
             : rotary_launch_ll<T, V, U, false, false>(p, backward, grid, st);
}

template <typename T, int V>
static int rotary_launch_v(const RotParams& p, const RotPlan& plan, bool backward, unsigned grid, cudaStream_t st) {
  switch (plan.U) {
    case 1:
      return rotary_launch_vu<T, V, 1>(p, plan.half, backward, grid, st);
    case 3:
      if constexpr (V <= 4) return rotary_launch_vu<T, V, 3>(p, plan.half, backward, grid, st);
      return FLN_ERR_UNSUPPORTED;
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
