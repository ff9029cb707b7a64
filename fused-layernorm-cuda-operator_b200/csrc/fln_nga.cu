// fln_norm_gate_add_norm: entry points and launch plans; the kernels that serve every row length
// and alignment (element loads, the row read once per pass), and the sum of the partial rows.
// Rows that start on 16-byte boundaries and fit a CTA's registers, or those of two in the backward, go
// to fln_nga_rows.cuh.  The formulas stand in fln_nga.cuh.
#include <initializer_list>

#include "fln_nga_rows.cuh"

namespace fln {

// explicit instantiations live in fln_nga_{f32,bf16,f16}.cu
#define FLN_NGA_DECLARE(T)                                                              \
  template <>                                                                           \
  int nga_fwd_rows<T>(const NgaParams&, const NgaGeom&, int, cudaStream_t);             \
  template <>                                                                           \
  int nga_bwd_rows<T>(const NgaParams&, const NgaGeom&, int, cudaStream_t);
FLN_NGA_DECLARE(float)
FLN_NGA_DECLARE(__nv_bfloat16)
FLN_NGA_DECLARE(__half)
#undef FLN_NGA_DECLARE

constexpr int kLoopThreads = 256;

// ----------------------------------------------------------------------------------------
// forward, any shape: one CTA per row, which is read up to five times (mean and spread of N1, mean and
// spread of the sum, y), mostly out of L1 / L2 after the first, element by element: 2048 x 16384 fp32 in
// 352 us, 4.3 times its bytes.
// ----------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float nga_sum(const NgaParams& p, float v, int c, const T* w1, const T* b1, const T* gate,
                                         const T* res) {
  if (w1 != nullptr) v *= p.woff + Cvt<T>::to_f(w1[c]);
  if (b1 != nullptr) v += Cvt<T>::to_f(b1[c]);
  if (p.gate_mode != FLN_GATE_NONE) v *= gate_act<sizeof(T) == 4>(Cvt<T>::to_f(gate[c]), p.act);
  v *= p.ba;
  if (res != nullptr) v = fmaf(p.ra, Cvt<T>::to_f(res[c]), v);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kLoopThreads) nga_fwd_loop_kernel(const NgaParams p) {
  __shared__ float red[2 * 32];
  int flip = 0;
  const int cols = p.cols;
  const float inv_n = 1.0f / (float)cols;
  const T* w1 = reinterpret_cast<const T*>(p.w1);
  const T* b1 = reinterpret_cast<const T*>(p.b1);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const int64_t base = row * (int64_t)cols;
    const int64_t group = row / p.group_rows;
    const T* x = reinterpret_cast<const T*>(p.x) + base;
    const T* res = p.res != nullptr ? reinterpret_cast<const T*>(p.res) + base : nullptr;
    const T* gate = reinterpret_cast<const T*>(p.gate);
    if (p.gate_mode == FLN_GATE_GROUP) gate += group * (int64_t)cols;
    if (p.gate_mode == FLN_GATE_ELEMENT) gate += base;
    const T* w2 = reinterpret_cast<const T*>(p.w2);
    const T* b2 = reinterpret_cast<const T*>(p.b2);
    if (p.affine_grouped) {
      if (w2 != nullptr) w2 += group * (int64_t)cols;
      if (b2 != nullptr) b2 += group * (int64_t)cols;
    }
    float mean1 = 0.f, rstd1 = 1.f;
    if (p.post_kind != FLN_NO_NORM) {
      float v[1] = {0.f};
      if (p.post_kind == FLN_LAYERNORM) {
        for (int c = threadIdx.x; c < cols; c += kLoopThreads) v[0] += Cvt<T>::to_f(x[c]);
        cta_sum<1>(v, red, flip);
        mean1 = v[0] * inv_n;
        v[0] = 0.f;
      }
      for (int c = threadIdx.x; c < cols; c += kLoopThreads) {
        const float d = Cvt<T>::to_f(x[c]) - mean1;
        v[0] = fmaf(d, d, v[0]);
      }
      cta_sum<1>(v, red, flip);
      rstd1 = rsqrtf(fmaf(v[0], inv_n, p.eps1));
    }
    auto s_of = [&](int c) { return nga_sum<T>(p, (Cvt<T>::to_f(x[c]) - mean1) * rstd1, c, w1, b1, gate, res); };
    float mean2 = 0.f, rstd2 = 1.f;
    if (p.kind != FLN_NO_NORM) {
      float v[1] = {0.f};
      if (p.kind == FLN_LAYERNORM) {
        for (int c = threadIdx.x; c < cols; c += kLoopThreads) v[0] += s_of(c);
        cta_sum<1>(v, red, flip);
        mean2 = v[0] * inv_n;
        v[0] = 0.f;
      }
      for (int c = threadIdx.x; c < cols; c += kLoopThreads) {
        const float d = s_of(c) - mean2;
        v[0] = fmaf(d, d, v[0]);
      }
      cta_sum<1>(v, red, flip);
      rstd2 = rsqrtf(fmaf(v[0], inv_n, p.eps2));
    }
    for (int c = threadIdx.x; c < cols; c += kLoopThreads) {
      const float s = s_of(c);
      reinterpret_cast<T*>(p.sum)[base + c] = Cvt<T>::from_f(s);
      if (p.kind != FLN_NO_NORM) {
        float v = (s - mean2) * rstd2;
        if (w2 != nullptr) v *= p.woff + Cvt<T>::to_f(w2[c]);
        if (b2 != nullptr) v += Cvt<T>::to_f(b2[c]);
        reinterpret_cast<T*>(p.y)[base + c] = Cvt<T>::from_f(v);
      }
    }
    if (threadIdx.x == 0) {
      if (p.mean1 != nullptr && p.post_kind == FLN_LAYERNORM) p.mean1[row] = mean1;
      if (p.rstd1 != nullptr && p.post_kind != FLN_NO_NORM) p.rstd1[row] = rstd1;
      if (p.mean2 != nullptr && p.kind == FLN_LAYERNORM) p.mean2[row] = mean2;
      if (p.rstd2 != nullptr && p.kind != FLN_NO_NORM) p.rstd2[row] = rstd2;
    }
  }
}

// ----------------------------------------------------------------------------------------
// backward, any shape
// ----------------------------------------------------------------------------------------
// what one element of one row needs, given the row's scalars
template <typename T>
struct NgaBwdRow {
  const T *x, *res, *dy, *dsum, *gate, *w1, *b1, *w2;
  float mean1, rstd1, mean2, rstd2, c1, c2;
  __device__ __forceinline__ void open(const NgaParams& p, int64_t row) {
    const int64_t base = row * (int64_t)p.cols;
    const int64_t group = row / p.group_rows;
    x = reinterpret_cast<const T*>(p.x) + base;
    res = p.res != nullptr ? reinterpret_cast<const T*>(p.res) + base : nullptr;
    dy = p.dy != nullptr ? reinterpret_cast<const T*>(p.dy) + base : nullptr;
    dsum = p.ds != nullptr ? reinterpret_cast<const T*>(p.ds) + base : nullptr;
    gate = reinterpret_cast<const T*>(p.gate);
    if (p.gate_mode == FLN_GATE_GROUP) gate += group * (int64_t)p.cols;
    if (p.gate_mode == FLN_GATE_ELEMENT) gate += base;
    w1 = reinterpret_cast<const T*>(p.w1);
    b1 = reinterpret_cast<const T*>(p.b1);
    w2 = reinterpret_cast<const T*>(p.w2);
    if (p.affine_grouped && w2 != nullptr) w2 += group * (int64_t)p.cols;
    mean1 = p.post_kind == FLN_LAYERNORM ? p.mean1[row] : 0.f;
    rstd1 = p.post_kind != FLN_NO_NORM ? p.rstd1[row] : 1.f;
    mean2 = p.kind == FLN_LAYERNORM && dy != nullptr ? p.mean2[row] : 0.f;
    rstd2 = p.kind != FLN_NO_NORM && dy != nullptr ? p.rstd2[row] : 1.f;
    c1 = c2 = 0.f;
  }
  __device__ __forceinline__ float g2(const NgaParams& p, int c) const {
    float v = Cvt<T>::to_f(dy[c]);
    if (w2 != nullptr) v *= p.woff + Cvt<T>::to_f(w2[c]);
    return v;
  }
  __device__ __forceinline__ float xh(int c) const { return (Cvt<T>::to_f(x[c]) - mean1) * rstd1; }
  // the forward's 32-bit sum, made again, normalized
  __device__ __forceinline__ float sh(const NgaParams& p, int c) const {
    return (nga_sum<T>(p, xh(c), c, w1, b1, gate, res) - mean2) * rstd2;
  }
  __device__ __forceinline__ float dsv(const NgaParams& p, int c) const {
    float v = dsum != nullptr ? Cvt<T>::to_f(dsum[c]) : 0.f;
    if (dy != nullptr) v += rstd2 * ((g2(p, c) - c2) - sh(p, c) * c1);
    return v;
  }
};

template <typename T>
__global__ void __launch_bounds__(kLoopThreads) nga_bwd_loop_kernel(const NgaParams p) {
  constexpr bool EXACT = sizeof(T) == 4;
  __shared__ float red[2 * 2 * 32];
  int flip = 0;
  const int cols = p.cols;
  const float inv_n = 1.0f / (float)cols;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const int64_t base = row * (int64_t)cols;
    NgaBwdRow<T> r;
    r.open(p, row);
    if (r.dy != nullptr) {
      float v[2] = {0.f, 0.f};
      for (int c = threadIdx.x; c < cols; c += kLoopThreads) {
        const float g = r.g2(p, c);
        v[0] = fmaf(g, r.sh(p, c), v[0]);
        v[1] += g;
      }
      cta_sum<2>(v, red, flip);
      r.c1 = v[0] * inv_n;
      r.c2 = p.kind == FLN_LAYERNORM ? v[1] * inv_n : 0.f;
      if (p.row_c != nullptr && threadIdx.x == 0) {
        p.row_c[2 * row] = r.c1;
        p.row_c[2 * row + 1] = r.c2;
      }
    }
    auto g1_of = [&](int c, float e) {
      if (p.gate_mode != FLN_GATE_NONE) e *= gate_act<EXACT>(Cvt<T>::to_f(r.gate[c]), p.act);
      if (r.w1 != nullptr) e *= p.woff + Cvt<T>::to_f(r.w1[c]);
      return e;
    };
    float v[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < cols; c += kLoopThreads) {
      const float ds = r.dsv(p, c);
      if (p.dres != nullptr) reinterpret_cast<T*>(p.dres)[base + c] = Cvt<T>::from_f(p.ra * ds);
      const float e = p.ba * ds;
      if (p.dgate != nullptr && p.gate_mode == FLN_GATE_ELEMENT) {
        float n = r.xh(c);
        if (r.w1 != nullptr) n *= p.woff + Cvt<T>::to_f(r.w1[c]);
        if (r.b1 != nullptr) n += Cvt<T>::to_f(r.b1[c]);
        float a, da;
        gate_act_grad<EXACT>(Cvt<T>::to_f(r.gate[c]), p.act, &a, &da);
        reinterpret_cast<T*>(p.dgate)[base + c] = Cvt<T>::from_f(e * n * da);
      }
      if (p.dx != nullptr && p.post_kind != FLN_NO_NORM) {
        const float g1 = g1_of(c, e);
        v[0] = fmaf(g1, r.xh(c), v[0]);
        v[1] += g1;
      }
    }
    if (p.dx != nullptr) {
      float d1 = 0.f, d2 = 0.f;
      if (p.post_kind != FLN_NO_NORM) {
        cta_sum<2>(v, red, flip);
        d1 = v[0] * inv_n;
        d2 = p.post_kind == FLN_LAYERNORM ? v[1] * inv_n : 0.f;
      }
      for (int c = threadIdx.x; c < cols; c += kLoopThreads) {
        const float g1 = g1_of(c, p.ba * r.dsv(p, c));
        // without a norm xh * d1 would be inf * 0 where x is infinite
        const float d = p.post_kind != FLN_NO_NORM ? r.rstd1 * ((g1 - d2) - r.xh(c) * d1) : g1;
        reinterpret_cast<T*>(p.dx)[base + c] = Cvt<T>::from_f(d);
      }
    }
  }
}

// Column sums of a slot: 32 columns x 8 row lanes per CTA, every term recomputed from the row's
// scalars (c1, c2 as the row kernel left them).
template <typename T>
__global__ void __launch_bounds__(256) nga_bwd_columns_kernel(const NgaParams p) {
  constexpr bool EXACT = sizeof(T) == 4;
  __shared__ float tile[8][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31);
  const int lane = threadIdx.x >> 5;
  const bool col_ok = c < p.cols;
  for (int64_t slot = blockIdx.y; slot < p.slots; slot += gridDim.y) {
    const SlotRows sr = slot_rows(p, slot);
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    if (col_ok) {
      for (int64_t row = sr.first + lane; row < sr.last; row += 8) {
        NgaBwdRow<T> r;
        r.open(p, row);
        if (r.dy != nullptr) {
          r.c1 = p.row_c[2 * row];
          r.c2 = p.row_c[2 * row + 1];
          const float d = Cvt<T>::to_f(r.dy[c]);
          if (p.acc & kAccU) acc[2] = fmaf(d, r.sh(p, c), acc[2]);
          acc[3] += d;
        }
        if (p.acc & (kAccP | kAccQ)) {
          float h = p.ba * r.dsv(p, c);
          if (p.gate_mode == FLN_GATE_ELEMENT) h *= gate_act<EXACT>(Cvt<T>::to_f(r.gate[c]), p.act);
          if (p.acc & kAccP) acc[0] = fmaf(h, r.xh(c), acc[0]);
          acc[1] += h;
        }
      }
    }
    int k = 0;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      if (!(p.acc & (1 << a))) continue;
      __syncthreads();
      tile[lane][threadIdx.x & 31] = acc[a];
      __syncthreads();
      if (lane == 0 && col_ok) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) t += tile[i][threadIdx.x & 31];
        p.partials[(slot * p.nacc + k) * (int64_t)p.cols + c] = t;
      }
      ++k;
    }
  }
}

// ----------------------------------------------------------------------------------------
// Sums of the partial rows.  Job y < grouped: the gradients that belong to one group each (dgate of
// a gate per group, dweight / dbias per group); job y == grouped: those of the vectors shared by all
// rows.  A CTA takes LANES x (256 / LANES) columns of a job: lane l adds partial rows l, l + LANES,
// ... of all the sums that the job needs, and the lanes are added in order.  One lane where a group
// has few partial rows (32 samples x 9 slots of 2048 columns: 16 lanes with a pass per sum took
// 29 us), 16 where all of them are added for a few hundred columns. 
// ----------------------------------------------------------------------------------------
template <typename T, int LANES>
__global__ void __launch_bounds__(256) nga_finalize_kernel(const NgaParams p, const NgaGrads g, int grouped) {
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int COLS = 256 / LANES;
  __shared__ float tile[LANES > 1 ? 4 : 1][LANES][LANES > 1 ? COLS + 1 : 1];
  const int tx = threadIdx.x % COLS, lane = threadIdx.x / COLS;
  const int64_t c = (int64_t)blockIdx.x * COLS + tx;
  const bool ok = c < p.cols;
  const int64_t per_group = p.slots_per_group;
  const bool gate_grouped = p.gate_mode == FLN_GATE_GROUP, gate_vec = p.gate_mode == FLN_GATE_VECTOR;
  const int64_t pitch = (int64_t)p.nacc * p.cols;
  const T* gate = reinterpret_cast<const T*>(p.gate);
  auto dgate_of = [&](float P, float Q, int64_t at) {
    float a, da;
    gate_act_grad<EXACT>(Cvt<T>::to_f(gate[at]), p.act, &a, &da);
    float w = 1.f;
    if (p.w1 != nullptr) w = p.woff + Cvt<T>::to_f(reinterpret_cast<const T*>(p.w1)[c]);
    float n = w * P;
    if (p.b1 != nullptr) n = fmaf(Cvt<T>::to_f(reinterpret_cast<const T*>(p.b1)[c]), Q, n);
    reinterpret_cast<T*>(g.dgate)[at] = Cvt<T>::from_f(n * da);
  };
  auto put = [&](void* out, int64_t at, float v) {
    if (out != nullptr) reinterpret_cast<T*>(out)[at] = Cvt<T>::from_f(v);
  };
  const int64_t jobs = p.groups + 1;
  for (int64_t y = (int64_t)blockIdx.y + (grouped ? 0 : p.groups); y < jobs; y += gridDim.y) {
    const bool all = y == p.groups;
    // the sums this job needs (bits as in p.acc), and whether P and Q are weighted with act(gate) of
    // their group
    int want = 0;
    if (all) {
      if (g.dw1 != nullptr || (gate_vec && g.dgate != nullptr)) want |= kAccP;
      if (g.db1 != nullptr || (gate_vec && g.dgate != nullptr && p.b1 != nullptr)) want |= kAccQ;
      if (!p.affine_grouped) want |= (g.dw2 != nullptr ? kAccU : 0) | (g.db2 != nullptr ? kAccV : 0);
    } else {
      if (gate_grouped && g.dgate != nullptr) want |= kAccP | (p.b1 != nullptr ? kAccQ : 0);
      if (p.affine_grouped) want |= (g.dw2 != nullptr ? kAccU : 0) | (g.db2 != nullptr ? kAccV : 0);
    }
    if (want == 0) continue;
    const bool weighted = all && gate_grouped;
    const int64_t from = all ? 0 : y * per_group, to = all ? p.slots : from + per_group;
    float t[4] = {0.f, 0.f, 0.f, 0.f};
    if (ok) {
      const float* src[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) src[i] = p.partials + (int64_t)__popc(p.acc & ((1 << i) - 1)) * p.cols + c;
      int64_t r = from + lane;
      for (; r + 3 * LANES < to; r += 4 * LANES) {
        float v[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[j][i] = (want >> i) & 1 ? __ldcg(src[i] + (r + j * LANES) * pitch) : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (weighted) {
            const float a = gate_act<EXACT>(Cvt<T>::to_f(gate[(r + j * LANES) / per_group * p.cols + c]), p.act);
            v[j][0] *= a;
            v[j][1] *= a;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) t[i] += v[j][i];
        }
      }
      for (; r < to; r += LANES) {
        float a = 1.f;
        if (weighted) a = gate_act<EXACT>(Cvt<T>::to_f(gate[r / per_group * p.cols + c]), p.act);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if ((want >> i) & 1) t[i] = fmaf(i < 2 ? a : 1.f, __ldcg(src[i] + r * pitch), t[i]);
      }
    }
    if (LANES > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) tile[i][lane][tx] = t[i];
      __syncthreads();
      if (lane == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          t[i] = 0.f;
#pragma unroll
          for (int l = 0; l < LANES; ++l) t[i] += tile[LANES > 1 ? i : 0][l][LANES > 1 ? tx : 0];
        }
      }
    }
    if (!ok || lane != 0) continue;
    if (!all) {
      const int64_t at = y * p.cols + c;
      if (gate_grouped && g.dgate != nullptr) dgate_of(t[0], t[1], at);
      if (p.affine_grouped) {
        put(g.dw2, at, t[2]);
        put(g.db2, at, t[3]);
      }
    } else {
      const float a = gate_vec ? gate_act<EXACT>(Cvt<T>::to_f(gate[c]), p.act) : 1.f;
      put(g.dw1, c, a * t[0]);
      put(g.db1, c, a * t[1]);
      if (gate_vec && g.dgate != nullptr) dgate_of(t[0], t[1], c);
      if (!p.affine_grouped) {
        put(g.dw2, c, t[2]);
        put(g.db2, c, t[3]);
      }
    }
  }
}

// ----------------------------------------------------------------------------------------
// host side
// ----------------------------------------------------------------------------------------
static int check_args(const fln_nga_args* a) {
  if (a == nullptr) return FLN_ERR_NULL;
  auto kind_ok = [](int k) { return k == FLN_LAYERNORM || k == FLN_RMSNORM || k == FLN_NO_NORM; };
  if (!kind_ok(a->post_kind) || !kind_ok(a->kind)) return FLN_ERR_ARG;
  if (a->gate_mode < FLN_GATE_NONE || a->gate_mode > FLN_GATE_ELEMENT) return FLN_ERR_ARG;
  if (a->gate_act < FLN_GATE_ACT_NONE || a->gate_act > FLN_GATE_ACT_TANH) return FLN_ERR_ARG;
  if (a->dtype != FLN_F32 && a->dtype != FLN_BF16 && a->dtype != FLN_F16) return FLN_ERR_DTYPE;
  if (a->rows < 0 || a->cols <= 0 || a->cols > 0x7fffffff || a->rows > 0x7fffffff) return FLN_ERR_SHAPE;
  if (a->rows > 0 && (a->group_rows <= 0 || a->rows % a->group_rows != 0)) return FLN_ERR_SHAPE;
  if ((a->gate != nullptr) != (a->gate_mode != FLN_GATE_NONE) && a->rows > 0) return FLN_ERR_ARG;
  if (a->post_kind == FLN_NO_NORM && (a->post_weight != nullptr || a->post_bias != nullptr)) return FLN_ERR_ARG;
  if (a->kind == FLN_NO_NORM && (a->weight != nullptr || a->bias != nullptr)) return FLN_ERR_ARG;
  return FLN_OK;
}

static NgaParams base_params(const fln_nga_args* a) {
  NgaParams p = {};
  p.x = a->x;
  p.res = a->residual;
  p.gate = a->gate;
  p.w1 = a->post_weight;
  p.b1 = a->post_bias;
  p.w2 = a->weight;
  p.b2 = a->bias;
  p.rows = a->rows;
  p.group_rows = a->group_rows;
  p.cols = (int)a->cols;
  p.post_kind = a->post_kind;
  p.kind = a->kind;
  p.gate_mode = a->gate_mode;
  p.act = a->gate_act;
  p.affine_grouped = a->affine_grouped != 0;
  p.ba = a->branch_scale;
  p.ra = a->residual_scale;
  p.woff = a->weight_offset;
  p.eps1 = a->post_eps;
  p.eps2 = a->eps;
  // groups matter only where something is held per group
  if (p.gate_mode != FLN_GATE_GROUP && !p.affine_grouped) p.group_rows = a->rows;
  return p;
}

// Slots of the loop kernels: 64 rows, more when that would make over a thousand of them.
static void plan_slots(NgaParams* p) {
  p->period = 1;
  const int64_t groups = p->rows / p->group_rows;
  int64_t most = 1024 / groups;
  if (most < 1) most = 1;
  int64_t chunk = 64;
  if ((p->group_rows + chunk - 1) / chunk > most) chunk = (p->group_rows + most - 1) / most;
  p->chunk = chunk;
  p->slots_per_group = (p->group_rows + chunk - 1) / chunk;
  p->slots = p->slots_per_group * groups;
}

// threads that own a row when each holds K of its nv vectors
static int threads_per_row(int nv, int K) {
  const int t = (nv + K - 1) / K;
  if (t > 32) return (t + 31) & ~31;
  int w = 1;
  while (w < t) w <<= 1;
  return w;
}

// Places of a 16-byte vector that the rows start at in turn, and with them p's classes.
static bool row_vectors(NgaParams* p, int es) {
  // (the kernels count rows in 32 bits, a few steps past the last one)
  if (p->cols > (1 << 20) || p->rows > 0x7fff0000) return false;
  const int vec = 16 / es;
  p->period = vec;
  for (int c = p->cols; p->period > 1 && c % 2 == 0; c /= 2) p->period /= 2;
  p->classes = p->group_rows < p->period ? (int)p->group_rows : p->period;
  p->pieces = 1;
  return true;
}
// Cuts every class of a group into about `want` slots, none of them empty.
static void cut_classes(NgaParams* p, int64_t want) {
  const int64_t most = p->group_rows / p->period;
  p->pieces = want > most ? most : want;
  if (p->pieces < 1) p->pieces = 1;
  p->slots_per_group = p->classes * p->pieces;
  p->slots = p->slots_per_group * (p->rows / p->group_rows);
}
// vectors that cover a row, wherever it starts
static int row_vector_count(const NgaParams& p, int es) {
  const int vec = 16 / es;
  return p.period == 1 ? p.cols / vec : (p.cols + 2 * (vec - 1)) / vec;
}

// rows per CTA: rows of 128 threads and more one at a time, shorter ones until there are 256 threads
static void rows_per_cta(NgaGeom* g) {
  g->R = g->tpr >= 128 ? 1 : (g->tpr > 32 ? 2 : 256 / g->tpr);
  g->threads = g->R * g->tpr;
}

// The forward's plan.  K = 0: not for the row kernels.
static int plan_forward(NgaParams* pp, int es, NgaGeom* g) {
  if (!row_vectors(pp, es)) return 0;
  const NgaParams& p = *pp;
  const int nv = row_vector_count(p, es), vec = 16 / es;
  g->nv = nv;
  int E = 16;  // elements per thread
  int fK = 0, ftpr = 0;
  plan_override(&fK, &ftpr);
  if (fK == 1 || fK == 2 || fK == 4) E = 8 * fK;
  if (threads_per_row(nv, E / vec) > 512) E = E < 16 ? 16 : 32;
  if (threads_per_row(nv, E / vec) > 512) E = 32;
  if (threads_per_row(nv, E / vec) > 512) return 0;
  const int K = E / vec;
  g->tpr = threads_per_row(nv, K);
  if (p.period == 1 && E == 16) {
    const int fixed = fixed_tpr(g->tpr, K * g->tpr == nv, 512);
    if (fixed != 0) g->tpr = fixed;
  }
  rows_per_cta(g);
  const int tensors = 1 + (p.res != nullptr) + (p.gate_mode == FLN_GATE_ELEMENT);
  g->stages = 3;
  g->smem = 512 + (size_t)g->stages * tensors * K * g->threads * 16;
  while (g->smem > 220 * 1024) {
    if (--g->stages < 2) return 0;
    g->smem = 512 + (size_t)g->stages * tensors * K * g->threads * 16;
  }
  // Rows per CTA: about eight row steps, so that a CTA's coefficients and the start of its ring are
  // paid for, and one wave of CTAs where there are fewer rows than that.  16384 x 8192 bf16: 170 us
  // with 8 steps, 176 with 16, 182 with 32.  Resident CTAs: some 64 .. 84 registers without biases and
  // means, up to 119 with them.
  const int64_t groups = p.rows / p.group_rows;
  int64_t resident = (nga_general(p) ? 512 : 768) / g->threads;
  const int64_t by_smem = (int64_t)(227 * 1024 / (g->smem + 1024));
  if (resident > by_smem) resident = by_smem;
  if (resident < 1) resident = 1;
  const int64_t slots = (int64_t)sm_count() * resident * g->R, steps = nga_general(p) ? 12 : 8;
  const int64_t waves = (p.rows + slots * steps - 1) / (slots * steps);
  int64_t chunk = (p.rows + slots * waves - 1) / (slots * waves) * g->R;
  if (chunk > p.group_rows) chunk = p.group_rows;
  g->per_group = (p.group_rows + chunk - 1) / chunk;
  g->chunk = (p.group_rows + g->per_group - 1) / g->per_group;
  g->chunk = (g->chunk + g->R - 1) / g->R * g->R;
  g->per_group = (p.group_rows + g->chunk - 1) / g->chunk;
  if (p.period > 1) {
    cut_classes(pp, (g->per_group + p.period - 1) / p.period);
    g->per_group = p.slots_per_group;
  }
  g->grid = g->per_group * groups;
  if (g->grid > 0x7fffffff) return 0;
  return K;
}

// What a backward plan reads of the library's settings.  A call reads them once: the workspace that it asks
// for and the slots that it fills come from the same numbers, also while another thread changes them.
struct NgaSettings {
  int sms = usable_sms(), K = 0, tpr = 0;
  NgaSettings() { plan_override(&K, &tpr); }
};

// The backward's plan: threads and shared memory so that an SM holds as many threads as the
// kernels' registers allow (640 with 8 elements per thread, 512 with 16), at least two rows on
// their way per row group.  Fills p's slots.  K = 0: not for the row kernels.
static int plan_backward(NgaParams* p, int es, const NgaSettings& settings, NgaGeom* g) {
  if (!row_vectors(p, es)) return 0;
  const int vec = 16 / es;
  g->nv = row_vector_count(*p, es);
  auto most = [&](int e) { return e <= 8 ? 640 : 512; };
  // 16 elements per thread, 8 with four column sums and for fp32 (whose staged rows leave room for
  // one CTA of either: 8192 x 4096, 145 us with 512 threads, 165 with 256)
  const bool eight = nga_general(*p) || es == 4;
  int E = eight ? 8 : 16;
  if (settings.K == 1 || settings.K == 2) E = 8 * settings.K;
  if (threads_per_row(g->nv, E / vec) > most(E)) E = 16;
  const int K = E / vec;
  g->tpr = threads_per_row(g->nv, K);
  if (g->tpr > most(E)) {  // E is 16 here
    g->pair = 1;
    g->tpr = threads_per_row((g->nv + 1) / 2, K);
    if (g->tpr > 512) return 0;
  }
  const int set = p->period == 1 && !g->pair ? nga_set_of(*p) : 0;  // (0: dsum never past the ring)
  int ctas = 1;
  // Lays out a CTA for rows of `tpr` threads: as many CTAs as the registers allow if two rows each fit, else
  // fewer; then dsum past the ring, then the coefficients out of it, and a ring of one row last.
  auto lay_out = [&](int tpr) {
    g->tpr = tpr;
    rows_per_cta(g);
    g->rep = g->tpr < 32 ? g->threads / 32 : g->R;
    const size_t unit = (size_t)K * g->threads * 16;
    auto fit = [&](int ctas, int csm, int direct, int rows) {
      const size_t per = (size_t)227 * 1024 / ctas - 1024;  // the runtime keeps 1 KB of every CTA
      const NgaBwdLayout l = nga_bwd_layout(*p, es, csm != 0, nga_general(*p), direct != 0);
      const size_t joint = g->rep > 1 ? (size_t)g->rep * g->tpr * vec * 4 : 0;
      const size_t fixed = kNgaBwdHeader + (size_t)l.coefs * unit + joint, stage = (size_t)l.tensors * unit;
      if (fixed + rows * stage > per) return false;
      int s = (int)((per - fixed) / stage);
      if (s > 3) s = 3;
      g->csm = csm;
      g->direct = direct;
      g->stages = s;
      g->smem = fixed + (size_t)s * stage;
      return true;
    };
    ctas = most(E) / g->threads;
    if (ctas < 1) ctas = 1;
    for (; ctas >= 1; --ctas)
      if (fit(ctas, 1, 0, 2)) return true;
    ctas = 1;
    return (set == 1 && fit(1, 1, 1, 2)) || fit(1, 0, 0, 2) || (set == 1 && fit(1, 0, 1, 2)) || fit(1, 1, 0, 1) || fit(1, 0, 0, 1);
  };
  // A compile-time number of threads, unless only its idle ones put dsum past the ring or the coefficients
  // out of it, or dsum is past it and there is no such kernel (not the general form).
  auto grade = [&](bool fits) { return !fits ? 0 : (!g->csm ? 1 : (g->direct ? 2 : 3)); };
  const int tpr = g->tpr, fixed = set == 1 && E == (eight ? 8 : 16) ? fixed_tpr(tpr, K * tpr == g->nv, most(E)) : 0;
  bool fits = lay_out(fixed != 0 ? fixed : tpr);
  if (fixed != 0 && fixed != tpr && grade(fits) < 3) {
    const int with_fixed = grade(fits);
    fits = lay_out(tpr);
    if (grade(fits) < with_fixed || (grade(fits) == with_fixed && nga_general(*p))) fits = lay_out(fixed);
  }
  if (!fits) return 0;
  // Slots: as many per group as give every CTA the same number of row steps, nearly; a slot's own
  // cost (its partial rows) counts as one more step.
  const int64_t groups = p->rows / p->group_rows, T = p->group_rows;
  const int64_t slots_max = (T + g->R - 1) / g->R;
  const int64_t cta = g->pair ? settings.sms / 2 : (int64_t)settings.sms * ctas;  // (or pairs of them)
  if (cta < 1) return 0;
  if (p->period > 1) {
    const int64_t n = (T + p->period - 1) / p->period, per = groups * p->classes;
    int64_t best = 1, best_cost = -1;
    for (int64_t w = 1; w <= 8; ++w) {
      cut_classes(p, w * cta / per);
      const int64_t cost = (p->slots + cta - 1) / cta * (((n + p->pieces - 1) / p->pieces + g->R - 1) / g->R + 1);
      if (best_cost < 0 || cost < best_cost) {
        best = p->pieces;
        best_cost = cost;
      }
    }
    cut_classes(p, best);
    g->grid = (p->slots < cta ? p->slots : cta) * (g->pair ? 2 : 1);
    return p->slots > 0x7fffffff - g->grid ? 0 : K;
  }
  int64_t best = -1, best_cost = 0;
  auto consider = [&](int64_t spg) {
    if (spg < 1) spg = 1;
    if (spg > slots_max) spg = slots_max;
    int64_t chunk = (T + spg - 1) / spg;
    chunk = (chunk + g->R - 1) / g->R * g->R;
    const int64_t n = (T + chunk - 1) / chunk * groups;
    const int64_t cost = (n + cta - 1) / cta * ((chunk + g->R - 1) / g->R + 1);
    if (best < 0 || cost < best_cost) {
      best = spg;
      best_cost = cost;
    }
  };
  for (int64_t w = 1; w <= 8; ++w) consider(w * cta / groups);
  consider(1);
  p->chunk = ((T + best - 1) / best + g->R - 1) / g->R * g->R;
  p->slots_per_group = (T + p->chunk - 1) / p->chunk;
  p->slots = p->slots_per_group * groups;
  g->grid = (p->slots < cta ? p->slots : cta) * (g->pair ? 2 : 1);
  if (p->slots > 0x7fffffff - g->grid) return 0;
  return K;
}

static size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

template <typename T>
static int finalize(NgaParams p, const NgaGrads& g, cudaStream_t st) {
  p.groups = p.rows / p.group_rows;
  const bool grouped = (p.gate_mode == FLN_GATE_GROUP && g.dgate != nullptr) ||
                       (p.affine_grouped && (g.dw2 != nullptr || g.db2 != nullptr));
  const bool shared = g.dw1 != nullptr || g.db1 != nullptr || (p.gate_mode == FLN_GATE_VECTOR && g.dgate != nullptr) ||
                      (!p.affine_grouped && (g.dw2 != nullptr || g.db2 != nullptr));
  // 16 lanes wherever the shared vectors are among the outputs or a group has many partial rows
  const bool wide = shared || p.slots_per_group > 32;
  const int64_t jobs = grouped ? p.groups + (shared ? 1 : 0) : 1;
  const dim3 grid((unsigned)((p.cols + (wide ? 16 : 256) - 1) / (wide ? 16 : 256)), (unsigned)(jobs < 65535 ? jobs : 65535));
  if (wide) nga_finalize_kernel<T, 16><<<grid, 256, 0, st>>>(p, g, grouped ? 1 : 0);
  else nga_finalize_kernel<T, 1><<<grid, 256, 0, st>>>(p, g, grouped ? 1 : 0);
  FLN_CHECK_LAUNCH();
  return FLN_OK;
}

template <typename T>
static int run_backward(NgaParams p, const NgaGrads& g, bool aligned, const NgaSettings& settings, cudaStream_t st) {
  if (aligned) {
    NgaParams q = p;
    NgaGeom geom = {};
    const int K = plan_backward(&q, (int)sizeof(T), settings, &geom);
    if (K != 0) {
      q.partials = p.row_c;  // the whole workspace: the row scalars are not kept
      const int rc = nga_bwd_rows<T>(q, geom, K, st);
      if (rc != FLN_OK || q.acc == 0) return rc;
      return finalize<T>(q, g, st);
    }
  }
  plan_slots(&p);
  const int64_t grid = p.rows < 0x7fffffff ? p.rows : 0x7fffffff;
  nga_bwd_loop_kernel<T><<<(unsigned)grid, kLoopThreads, 0, st>>>(p);
  FLN_CHECK_LAUNCH();
  if (p.acc != 0) {
    const dim3 cg((unsigned)((p.cols + 31) / 32), (unsigned)(p.slots < 65535 ? p.slots : 65535));
    nga_bwd_columns_kernel<T><<<cg, 256, 0, st>>>(p);
    FLN_CHECK_LAUNCH();
    return finalize<T>(p, g, st);
  }
  return FLN_OK;
}

static size_t workspace_bytes_of(const fln_nga_args* a, const NgaSettings& settings) {
  // the most that any of the plans takes: which one it is depends on the gradients asked for and
  // on the alignment of all tensors
  NgaParams p = base_params(a);
  const size_t row = 4 * (size_t)p.cols * 4;
  plan_slots(&p);
  size_t most = align256((size_t)p.rows * 8) + (size_t)p.slots * row;
  for (int acc = kAccP | kAccU; acc <= 15; acc += kAccQ | kAccV) {
    for (int grads = 1; grads <= 3; ++grads) {  // dy, dsum, both
      NgaParams q = base_params(a);
      NgaGeom g = {};
      q.acc = acc;
      q.dy = (grads & 1) != 0 && a->kind != FLN_NO_NORM ? a->x : nullptr;
      q.ds = (grads & 2) != 0 ? a->x : nullptr;
      if (plan_backward(&q, a->dtype == FLN_F32 ? 4 : 2, settings, &g) == 0) continue;
      const size_t n = (size_t)q.slots * row;
      if (n > most) most = n;
    }
  }
  return most;
}

static bool all_aligned(std::initializer_list<const void*> ps) {
  for (const void* q : ps)
    if (!is_aligned16(q)) return false;
  return true;
}

// Byte ranges of a call: no output may share a byte with an input or with another output.
struct NgaRanges {
  struct Range {
    uintptr_t from, to;
  };
  Range in[12], out[8];
  int ins = 0, outs = 0;
  static Range of(const void* p, size_t n) { return {reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + n}; }
  void reads(const void* p, size_t n) {
    if (p != nullptr) in[ins++] = of(p, n);
  }
  void writes(const void* p, size_t n) {
    if (p != nullptr) out[outs++] = of(p, n);
  }
  bool apart() const {
    auto meet = [](const Range& a, const Range& b) { return a.from < b.to && b.from < a.to; };
    for (int o = 0; o < outs; ++o) {
      for (int i = 0; i < ins; ++i)
        if (meet(out[o], in[i])) return false;
      for (int i = 0; i < o; ++i)
        if (meet(out[o], out[i])) return false;
    }
    return true;
  }
};
struct NgaSizes {
  size_t all, vec, gate, affine, stat;
  explicit NgaSizes(const fln_nga_args* a) {
    const size_t es = a->dtype == FLN_F32 ? 4 : 2, groups = (size_t)(a->rows / a->group_rows);
    vec = (size_t)a->cols * es;
    all = (size_t)a->rows * vec;
    gate = a->gate_mode == FLN_GATE_ELEMENT ? all : (a->gate_mode == FLN_GATE_GROUP ? groups * vec : vec);
    affine = a->affine_grouped ? groups * vec : vec;
    stat = (size_t)a->rows * sizeof(float);
  }
};
static NgaRanges input_ranges(const fln_nga_args* a, const NgaSizes& n) {
  NgaRanges r;
  r.reads(a->x, n.all);
  r.reads(a->residual, n.all);
  r.reads(a->gate, n.gate);
  r.reads(a->post_weight, n.vec);
  r.reads(a->post_bias, n.vec);
  r.reads(a->weight, n.affine);
  return r;
}

// the column sums of parameters when there are no rows: zeros
static int zero_grads(const fln_nga_args* a, const NgaGrads& g, cudaStream_t st) {
  const size_t n = (size_t)a->cols * (a->dtype == FLN_F32 ? 4 : 2);
  void* const v[] = {g.dw1, g.db1, a->affine_grouped ? nullptr : g.dw2, a->affine_grouped ? nullptr : g.db2,
                     a->gate_mode == FLN_GATE_VECTOR ? g.dgate : nullptr};
  for (void* q : v)
    if (q != nullptr && cudaMemsetAsync(q, 0, n, st) != cudaSuccess) {
      cudaGetLastError();
      return FLN_ERR_LAUNCH;
    }
  return FLN_OK;
}

}  // namespace fln

using namespace fln;

extern "C" int fln_norm_gate_add_norm_forward(const fln_nga_args* a, void* y, void* sum, float* post_mean,
                                              float* post_rstd, float* mean, float* rstd, void* stream) {
  const int rc = check_args(a);
  if (rc != FLN_OK) return rc;
  if (a->rows == 0) return FLN_OK;
  if (a->x == nullptr || sum == nullptr) return FLN_ERR_NULL;
  if (a->kind != FLN_NO_NORM && y == nullptr) return FLN_ERR_NULL;
  // (a statistic that the call has none of is not written)
  if (a->post_kind != FLN_LAYERNORM) post_mean = nullptr;
  if (a->post_kind == FLN_NO_NORM) post_rstd = nullptr;
  if (a->kind != FLN_LAYERNORM) mean = nullptr;
  if (a->kind == FLN_NO_NORM) y = nullptr, rstd = nullptr;
  const NgaSizes n(a);
  NgaRanges ranges = input_ranges(a, n);
  ranges.reads(a->bias, n.affine);
  ranges.writes(y, n.all);
  ranges.writes(sum, n.all);
  for (const float* q : {post_mean, post_rstd, mean, rstd}) ranges.writes(q, n.stat);
  if (!ranges.apart()) return FLN_ERR_ARG;
  NgaParams p = base_params(a);
  p.y = y;
  p.sum = sum;
  p.mean1 = post_mean;
  p.rstd1 = post_rstd;
  p.mean2 = mean;
  p.rstd2 = rstd;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (all_aligned({a->x, a->residual, a->gate, a->post_weight, a->post_bias, a->weight, a->bias, y, sum})) {
    NgaGeom g = {};
    const int K = plan_forward(&p, a->dtype == FLN_F32 ? 4 : 2, &g);
    if (K != 0) {
      if (a->dtype == FLN_F32) return nga_fwd_rows<float>(p, g, K, st);
      if (a->dtype == FLN_BF16) return nga_fwd_rows<__nv_bfloat16>(p, g, K, st);
      return nga_fwd_rows<__half>(p, g, K, st);
    }
  }
  const unsigned grid = (unsigned)p.rows;
  switch (a->dtype) {
    case FLN_F32:
      nga_fwd_loop_kernel<float><<<grid, kLoopThreads, 0, st>>>(p);
      break;
    case FLN_BF16:
      nga_fwd_loop_kernel<__nv_bfloat16><<<grid, kLoopThreads, 0, st>>>(p);
      break;
    default:
      nga_fwd_loop_kernel<__half><<<grid, kLoopThreads, 0, st>>>(p);
      break;
  }
  FLN_CHECK_LAUNCH();
  return FLN_OK;
}

extern "C" size_t fln_norm_gate_add_norm_workspace_bytes(const fln_nga_args* a) {
  return check_args(a) != FLN_OK || a->rows == 0 ? 0 : workspace_bytes_of(a, NgaSettings());
}

extern "C" int fln_norm_gate_add_norm_backward(const fln_nga_args* a, const float* post_mean,
                                               const float* post_rstd, const float* mean, const float* rstd,
                                               const void* dy, const void* dsum, void* dx, void* dresidual,
                                               void* dgate, void* dpost_weight, void* dpost_bias, void* dweight,
                                               void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_args(a);
  if (rc != FLN_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dgate != nullptr && a->gate_mode == FLN_GATE_NONE) return FLN_ERR_ARG;
  if (a->post_kind == FLN_NO_NORM && (dpost_weight != nullptr || dpost_bias != nullptr)) return FLN_ERR_ARG;
  if (a->kind == FLN_NO_NORM && (dweight != nullptr || dbias != nullptr || dy != nullptr)) return FLN_ERR_ARG;
  const bool shared_gate = a->gate_mode == FLN_GATE_VECTOR || a->gate_mode == FLN_GATE_GROUP;
  NgaGrads g;
  g.dgate = shared_gate ? dgate : nullptr;
  g.dw1 = dpost_weight;
  g.db1 = dpost_bias;
  g.dw2 = dweight;
  g.db2 = dbias;
  if (a->rows == 0) return zero_grads(a, g, st);
  if (dy == nullptr && dsum == nullptr) return FLN_ERR_NULL;
  if (a->x == nullptr) return FLN_ERR_NULL;
  if (dy != nullptr && (rstd == nullptr || (a->kind == FLN_LAYERNORM && mean == nullptr)))
    return FLN_ERR_NULL;
  if (a->post_kind != FLN_NO_NORM && (post_rstd == nullptr || (a->post_kind == FLN_LAYERNORM && post_mean == nullptr)))
    return FLN_ERR_NULL;
  NgaParams p = base_params(a);
  p.mean1 = const_cast<float*>(post_mean);
  p.rstd1 = const_cast<float*>(post_rstd);
  p.mean2 = const_cast<float*>(mean);
  p.rstd2 = const_cast<float*>(rstd);
  p.dy = dy;
  p.ds = dsum;
  p.dx = dx;
  p.dres = dresidual;
  p.dgate = dgate;
  if (g.dw1 != nullptr || g.dgate != nullptr) p.acc |= kAccP;
  if (g.db1 != nullptr || (g.dgate != nullptr && p.b1 != nullptr)) p.acc |= kAccQ;
  if (g.dw2 != nullptr) p.acc |= kAccU;
  if (g.db2 != nullptr) p.acc |= kAccV;
  p.nacc = __builtin_popcount((unsigned)p.acc);
  const NgaSettings settings;
  size_t scratch = 0;
  if (p.acc != 0) {
    scratch = workspace_bytes_of(a, settings);
    if (workspace == nullptr || workspace_bytes < scratch) return FLN_ERR_WORKSPACE;
    if (!is_aligned16(workspace)) return FLN_ERR_WORKSPACE;
    p.row_c = reinterpret_cast<float*>(workspace);
    p.partials = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + align256((size_t)p.rows * 8));
  }
  const NgaSizes n(a);
  NgaRanges ranges = input_ranges(a, n);
  ranges.reads(dy, n.all);
  ranges.reads(dsum, n.all);
  if (a->post_kind == FLN_LAYERNORM) ranges.reads(post_mean, n.stat);
  if (a->post_kind != FLN_NO_NORM) ranges.reads(post_rstd, n.stat);
  if (dy != nullptr && a->kind == FLN_LAYERNORM) ranges.reads(mean, n.stat);
  if (dy != nullptr) ranges.reads(rstd, n.stat);
  ranges.writes(dx, n.all);
  ranges.writes(dresidual, n.all);
  ranges.writes(dgate, n.gate);
  ranges.writes(dpost_weight, n.vec);
  ranges.writes(dpost_bias, n.vec);
  ranges.writes(dweight, n.affine);
  ranges.writes(dbias, n.affine);
  if (p.acc != 0) ranges.writes(workspace, scratch);
  if (!ranges.apart()) return FLN_ERR_ARG;
  const bool aligned = all_aligned({a->x, a->residual, a->gate, a->post_weight, a->post_bias, a->weight, dy, dsum, dx,
                                    dresidual, dgate});
  switch (a->dtype) {
    case FLN_F32:
      return run_backward<float>(p, g, aligned, settings, st);
    case FLN_BF16:
      return run_backward<__nv_bfloat16>(p, g, aligned, settings, st);
    default:
      return run_backward<__half>(p, g, aligned, settings, st);
  }
}
