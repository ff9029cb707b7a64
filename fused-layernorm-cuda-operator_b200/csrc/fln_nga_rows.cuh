// fln_norm_gate_add_norm: the kernels that hold a row in registers, for rows of whole 16-byte
// vectors.  Instantiated per element type in fln_nga_{f32,bf16,f16}.cu; launched from fln_nga.cu.
// The formulas stand in fln_nga.cuh.
//
// A row is owned by `tpr` consecutive threads: a power of two within a warp, or whole warps.
// Thread `lane` of them holds vectors lane, lane + tpr, ... (K of them, the last ones may lie
// behind the row).
#pragma once

#include "fln_nga.cuh"

namespace fln {

struct NgaGeom {
  int tpr;      // threads per row
  int R;        // rows per CTA
  int nv;       // vectors per row
  int threads;  // per CTA: R * tpr
  int stages;   // backward: rows on their way per row group
  int rep;      // backward: partial rows a CTA leaves per slot
  int64_t grid;
  size_t smem;
};

// ----------------------------------------------------------------------------------------
// sums over the threads of a row
// ----------------------------------------------------------------------------------------
struct RowGroup {
  int width;   // lanes that share a row within a warp
  int wpr;     // warps per row, 1 where a warp or less owns it
  int warp0;   // first warp of the row in the CTA
  float cnt;   // elements of the row that warp (my lane) of the row holds
  float mine;  // elements of the row that my warp holds
  float2* red; // [2 buffers][32 warps]
  int flip;
};
__device__ __forceinline__ RowGroup row_group(const NgaGeom& g, int K, int vec, float2* red) {
  RowGroup r;
  r.width = g.tpr < 32 ? g.tpr : 32;
  r.wpr = g.tpr <= 32 ? 1 : g.tpr >> 5;
  r.warp0 = g.tpr <= 32 ? (int)(threadIdx.x >> 5) : (int)(threadIdx.x / g.tpr) * r.wpr;
  r.red = red;
  r.flip = 0;
  auto count = [&](int w) {  // elements of the row in its warp w
    int n = 0;
    for (int k = 0; k < K; ++k) {
      int left = g.nv - (k * g.tpr + w * 32);
      left = left < 0 ? 0 : (left > 32 ? 32 : left);
      n += left;
    }
    return (float)(n * vec);
  };
  const int lane = threadIdx.x & 31;
  r.cnt = lane < r.wpr ? count(lane) : 0.f;
  r.mine = r.wpr == 1 ? (float)(g.nv * vec) : count((int)(threadIdx.x >> 5) - r.warp0);
  return r;
}
template <int NV>
__device__ __forceinline__ void warp_sum(float (&v)[NV], int width) {
  if (width == 32) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], off);
    }
  } else {
    for (int off = width >> 1; off > 0; off >>= 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], off);
    }
  }
}
// one pair per warp in; every lane gets the pair of warp `lane` of its row (zeros behind them).
// One barrier; two buffers in turn, so the next exchange may start while this one is still read.
__device__ __forceinline__ float2 warp_exchange(RowGroup& g, float2 mine) {
  float2* r = g.red + g.flip * 32;
  g.flip ^= 1;
  if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = mine;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return lane < g.wpr ? r[g.warp0 + lane] : make_float2(0.f, 0.f);
}
__device__ __forceinline__ void row_sum1(RowGroup& g, float& a) {
  float v[1] = {a};
  warp_sum<1>(v, g.width);
  if (g.wpr > 1) {
    v[0] = warp_exchange(g, make_float2(v[0], 0.f)).x;
    warp_sum<1>(v, 32);
  }
  a = v[0];
}
__device__ __forceinline__ void row_sum2(RowGroup& g, float& a, float& b) {
  float v[2] = {a, b};
  warp_sum<2>(v, g.width);
  if (g.wpr > 1) {
    const float2 o = warp_exchange(g, make_float2(v[0], v[1]));
    v[0] = o.x;
    v[1] = o.y;
    warp_sum<2>(v, 32);
  }
  a = v[0];
  b = v[1];
}
// Mean and reciprocal deviation of the row held in v (zeros behind it).  LayerNorm: the spread is
// taken about the mean of the warp, and the warps' spreads are joined with that of their means
// about the row's, so one barrier is enough and nothing cancels.
template <int K, int VEC>
__device__ __forceinline__ void row_stats(RowGroup& g, int kind, const float (&v)[K][VEC], const bool (&ok)[K], float inv_n,
                                          float eps, float& mean, float& rstd) {
  float q = 0.f;
  mean = 0.f;
  if (kind == FLN_RMSNORM) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) q = fmaf(v[k][e], v[k][e], q);
    row_sum1(g, q);
  } else {
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[0] += v[k][e];
    warp_sum<1>(s, g.width);
    const float m = s[0] / fmaxf(g.mine, 1.f);
    float d2[1] = {0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (ok[k]) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float d = v[k][e] - m;
          d2[0] = fmaf(d, d, d2[0]);
        }
      }
    }
    warp_sum<1>(d2, g.width);
    mean = m;
    q = d2[0];
    if (g.wpr > 1) {
      const float2 o = warp_exchange(g, make_float2(s[0], d2[0]));
      s[0] = o.x;
      warp_sum<1>(s, 32);
      mean = s[0] * inv_n;
      const float d = o.x / fmaxf(g.cnt, 1.f) - mean;
      d2[0] = fmaf(g.cnt * d, d, o.y);
      warp_sum<1>(d2, 32);
      q = d2[0];
    }
  }
  rstd = rsqrtf(fmaf(q, inv_n, eps));
}

template <typename T, int VEC>
__device__ __forceinline__ void param_vec(const T* p, int c, float (&f)[VEC]) {
  unpack<T, VEC>(ld_param<T, VEC>(p + c), f);
}

// ----------------------------------------------------------------------------------------
// forward: R rows per CTA, one pass.  GATE 0: none, 1: shared by rows, 2: an element each.
// ----------------------------------------------------------------------------------------
template <typename T, int K, int GATE>
__global__ void __launch_bounds__(K * 16 / (int)sizeof(T) <= 16 ? 1024 : 512) nga_fwd_rows_kernel(const NgaParams p, const NgaGeom g) {
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int VEC = 16 / (int)sizeof(T);
  __shared__ float2 red[2 * 32];
  RowGroup rg = row_group(g, K, VEC, red);
  const int r_in = threadIdx.x / g.tpr, lane = threadIdx.x - r_in * g.tpr;
  const int64_t row = (int64_t)blockIdx.x * g.R + r_in;
  const bool live = row < p.rows;
  const int64_t base = row * (int64_t)p.cols;
  const float inv_n = 1.0f / (float)p.cols;
  bool ok[K];
  int col[K];
  Pack<T, VEC> px[K], pr[K], pg[GATE == 2 ? K : 1];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int v = lane + k * g.tpr;
    ok[k] = live && v < g.nv;
    col[k] = v * VEC;
    if (ok[k]) {
      px[k] = ld_stream<T, VEC>(reinterpret_cast<const T*>(p.x) + base + col[k]);
      if (p.res != nullptr) pr[k] = ld_stream<T, VEC>(reinterpret_cast<const T*>(p.res) + base + col[k]);
      if (GATE == 2) pg[k] = ld_stream<T, VEC>(reinterpret_cast<const T*>(p.gate) + base + col[k]);
    }
  }
  // (p.group_rows is the row count where nothing is held per group, so this is then 0)
  const int64_t goff =
      p.group_rows < p.rows && live ? (int64_t)((uint32_t)row / (uint32_t)p.group_rows) * p.cols : 0;
  float s[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[k][e] = 0.f;
    if (ok[k]) unpack<T, VEC>(px[k], s[k]);
  }
  float mean1 = 0.f, rstd1 = 1.f;
  if (p.post_kind != FLN_NO_NORM) row_stats<K, VEC>(rg, p.post_kind, s, ok, inv_n, p.eps1, mean1, rstd1);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (ok[k]) {
      float f[VEC];
      if (p.post_kind != FLN_NO_NORM) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[k][e] = (s[k][e] - mean1) * rstd1;
        if (p.w1 != nullptr) {
          param_vec<T, VEC>(reinterpret_cast<const T*>(p.w1), col[k], f);
#pragma unroll
          for (int e = 0; e < VEC; ++e) s[k][e] *= p.woff + f[e];
        }
        if (p.b1 != nullptr) {
          param_vec<T, VEC>(reinterpret_cast<const T*>(p.b1), col[k], f);
#pragma unroll
          for (int e = 0; e < VEC; ++e) s[k][e] += f[e];
        }
      }
      if (GATE == 1) param_vec<T, VEC>(reinterpret_cast<const T*>(p.gate) + (p.gate_mode == FLN_GATE_GROUP ? goff : 0), col[k], f);
      if (GATE == 2) unpack<T, VEC>(pg[k], f);
      if (GATE != 0) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[k][e] *= gate_act<EXACT>(f[e], p.act);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[k][e] *= p.ba;
      if (p.res != nullptr) {
        unpack<T, VEC>(pr[k], f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[k][e] = fmaf(p.ra, f[e], s[k][e]);
      }
      Pack<T, VEC> o;
      pack<T, VEC>(s[k], o);
      st_stream<T, VEC>(reinterpret_cast<T*>(p.sum) + base + col[k], o);
    }
  }
  float mean2 = 0.f, rstd2 = 1.f;
  if (p.kind != FLN_NO_NORM) {
    row_stats<K, VEC>(rg, p.kind, s, ok, inv_n, p.eps2, mean2, rstd2);
    const int64_t aoff = p.affine_grouped ? goff : 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (ok[k]) {
        float f[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[k][e] = (s[k][e] - mean2) * rstd2;
        if (p.w2 != nullptr) {
          param_vec<T, VEC>(reinterpret_cast<const T*>(p.w2) + aoff, col[k], f);
#pragma unroll
          for (int e = 0; e < VEC; ++e) s[k][e] *= p.woff + f[e];
        }
        if (p.b2 != nullptr) {
          param_vec<T, VEC>(reinterpret_cast<const T*>(p.b2) + aoff, col[k], f);
#pragma unroll
          for (int e = 0; e < VEC; ++e) s[k][e] += f[e];
        }
        Pack<T, VEC> o;
        pack<T, VEC>(s[k], o);
        st_stream<T, VEC>(reinterpret_cast<T*>(p.y) + base + col[k], o);
      }
    }
  }
  if (live && lane == 0) {
    if (p.mean1 != nullptr && p.post_kind == FLN_LAYERNORM) p.mean1[row] = mean1;
    if (p.rstd1 != nullptr && p.post_kind != FLN_NO_NORM) p.rstd1[row] = rstd1;
    if (p.mean2 != nullptr && p.kind == FLN_LAYERNORM) p.mean2[row] = mean2;
    if (p.rstd2 != nullptr && p.kind != FLN_NO_NORM) p.rstd2[row] = rstd2;
  }
}

// ----------------------------------------------------------------------------------------
// backward: persistent CTAs; CTA b takes slots b, b + grid, ...  Every thread keeps its own
// vectors of the next rows on their way into its own places in shared memory (cp.async), so
// staging needs no barrier and no flag; the barriers are those of the two row sums.  The column
// sums stay in registers over a slot.
//
// shared memory: the exchange buffers, the parameters of the current group (w1, b1, w2 as they
// are, act(gate) in 32 bits), then `stages` times the staged tensors; everything as
// [vector k][thread], each thread touching its own 16 bytes.
// ----------------------------------------------------------------------------------------
__device__ __forceinline__ void cp_async16(void* smem, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_async_wait_behind(int ahead) {  // at most `ahead` groups still on their way
  if (ahead == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else if (ahead == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 3;" ::: "memory");
}

constexpr int kNgaBwdHeader = 512;

// where a thread's pieces lie: in units of K * threads * 16 bytes behind the header
struct NgaBwdLayout {
  int w1, b1, w2, a;           // parameters, -1: absent (a takes sizeof(float) / sizeof(T) units)
  int x, res, dy, ds, gate;    // tensors inside a stage
  int params, tensors;         // units
};
inline __host__ __device__ NgaBwdLayout nga_bwd_layout(const NgaParams& p, int es) {
  NgaBwdLayout l;
  int n = 0;
  l.w1 = p.w1 != nullptr ? n++ : -1;
  l.b1 = p.b1 != nullptr ? n++ : -1;
  l.w2 = p.w2 != nullptr && p.dy != nullptr ? n++ : -1;
  l.a = -1;
  if (p.gate_mode == FLN_GATE_VECTOR || p.gate_mode == FLN_GATE_GROUP) {
    l.a = n;
    n += 4 / es;
  }
  l.params = n;
  n = 0;
  l.x = n++;
  l.res = p.res != nullptr && p.dy != nullptr ? n++ : -1;
  l.dy = p.dy != nullptr ? n++ : -1;
  l.ds = p.ds != nullptr ? n++ : -1;
  l.gate = p.gate_mode == FLN_GATE_ELEMENT ? n++ : -1;
  l.tensors = n;
  return l;
}

// FOUR: all four column sums are kept, else P and U only
template <typename T, int K, int GATE, bool FOUR>
__global__ void __launch_bounds__(K * 16 / (int)sizeof(T) <= 8 ? 768 : 512) nga_bwd_rows_kernel(const NgaParams p, const NgaGeom g) {
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int VEC = 16 / (int)sizeof(T);
  extern __shared__ __align__(128) unsigned char smem[];
  const NgaBwdLayout l = nga_bwd_layout(p, (int)sizeof(T));
  RowGroup rg = row_group(g, K, VEC, reinterpret_cast<float2*>(smem));
  const int tid = threadIdx.x;
  const int r_in = tid / g.tpr, lane = tid - r_in * g.tpr;
  const float inv_n = 1.0f / (float)p.cols;
  const uint32_t unit = (uint32_t)K * g.threads * 16u;
  unsigned char* par = smem + kNgaBwdHeader + tid * 16;
  unsigned char* stages = par + (uint32_t)l.params * unit;
  const uint32_t stage_bytes = (uint32_t)l.tensors * unit;
  bool vok[K];
  int col[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int v = lane + k * g.tpr;
    vok[k] = v < g.nv;
    col[k] = v * VEC;
  }
  auto at = [&](unsigned char* b, int piece, int k) { return b + (uint32_t)piece * unit + (uint32_t)(k * g.threads) * 16u; };

  // the row sequence of this CTA: slot after slot, R rows at a time; one walker runs ahead
  struct Walker {
    int64_t slot, row, last;
  };
  auto open = [&](Walker& w) {
    if (w.slot < p.slots) {
      const SlotRows sr = slot_rows(p, w.slot);
      w.row = sr.first;
      w.last = sr.last;
    }
  };
  auto step = [&](Walker& w) {
    w.row += g.R;
    if (w.row >= w.last) {
      w.slot += gridDim.x;
      open(w);
    }
  };
  Walker ahead{(int64_t)blockIdx.x, 0, 0};
  open(ahead);
  Walker cur = ahead;
  int in_stage = 0;  // stage the walker fills next
  auto fetch = [&]() {
    if (ahead.slot < p.slots) {
      const int64_t row = ahead.row + r_in;
      if (row < ahead.last) {
        const int64_t base = row * (int64_t)p.cols;
        unsigned char* st = stages + (uint32_t)in_stage * stage_bytes;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (vok[k]) {
            const int64_t o = base + col[k];
            cp_async16(at(st, l.x, k), reinterpret_cast<const T*>(p.x) + o);
            if (l.dy >= 0) cp_async16(at(st, l.dy, k), reinterpret_cast<const T*>(p.dy) + o);
            if (l.res >= 0) cp_async16(at(st, l.res, k), reinterpret_cast<const T*>(p.res) + o);
            if (l.ds >= 0) cp_async16(at(st, l.ds, k), reinterpret_cast<const T*>(p.ds) + o);
            if (GATE == 2) cp_async16(at(st, l.gate, k), reinterpret_cast<const T*>(p.gate) + o);
          }
        }
      }
      step(ahead);
    }
    cp_async_commit();  // a group per step, also an empty one, so that the count tells the row
    in_stage = in_stage + 1 == g.stages ? 0 : in_stage + 1;
  };
  for (int i = 0; i + 1 < g.stages; ++i) fetch();

  float acc_p[K][VEC], acc_u[K][VEC], acc_q[FOUR ? K : 1][VEC], acc_v[FOUR ? K : 1][VEC];
  auto clear = [&]() {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        acc_p[k][e] = 0.f;
        acc_u[k][e] = 0.f;
        if (FOUR) {
          acc_q[FOUR ? k : 0][e] = 0.f;
          acc_v[FOUR ? k : 0][e] = 0.f;
        }
      }
  };
  clear();
  int64_t group = -1;
  int stage = 0;
  bool opened = true;  // cur has come to a new slot
  while (cur.slot < p.slots) {
    // parameters of a new group into this thread's places
    const int64_t grp = opened ? cur.slot / p.slots_per_group : group;
    if (grp != group) {
      const bool first = group < 0;
      group = grp;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!vok[k]) continue;
        if (first) {
          if (l.w1 >= 0) *reinterpret_cast<Pack<T, VEC>*>(at(par, l.w1, k)) = ld_param<T, VEC>(reinterpret_cast<const T*>(p.w1) + col[k]);
          if (l.b1 >= 0) *reinterpret_cast<Pack<T, VEC>*>(at(par, l.b1, k)) = ld_param<T, VEC>(reinterpret_cast<const T*>(p.b1) + col[k]);
        }
        if (l.w2 >= 0 && (first || p.affine_grouped))
          *reinterpret_cast<Pack<T, VEC>*>(at(par, l.w2, k)) =
              ld_param<T, VEC>(reinterpret_cast<const T*>(p.w2) + (p.affine_grouped ? grp * p.cols : 0) + col[k]);
        if (GATE == 1 && (first || p.gate_mode == FLN_GATE_GROUP)) {
          float f[VEC];
          param_vec<T, VEC>(reinterpret_cast<const T*>(p.gate) + (p.gate_mode == FLN_GATE_GROUP ? grp * p.cols : 0), col[k], f);
#pragma unroll
          for (int e = 0; e < VEC; ++e) f[e] = gate_act<EXACT>(f[e], p.act);
#pragma unroll
          for (int q = 0; q < VEC / 4; ++q)
            *reinterpret_cast<float4*>(at(par, l.a + q, k)) = make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]);
        }
      }
    }
    fetch();
    const int64_t row = cur.row + r_in;
    const bool live = row < cur.last;
    float mean1 = 0.f, rstd1 = 1.f, mean2 = 0.f, rstd2 = 1.f;
    if (live) {
      if (p.post_kind != FLN_NO_NORM) {
        rstd1 = __ldg(p.rstd1 + row);
        if (p.post_kind == FLN_LAYERNORM) mean1 = __ldg(p.mean1 + row);
      }
      if (l.dy >= 0) {
        rstd2 = __ldg(p.rstd2 + row);
        if (p.kind == FLN_LAYERNORM) mean2 = __ldg(p.mean2 + row);
      }
    }
    cp_async_wait_behind(g.stages - 1);
    unsigned char* st = stages + (uint32_t)stage * stage_bytes;
    stage = stage + 1 == g.stages ? 0 : stage + 1;
    const int64_t base = row * (int64_t)p.cols;

    float xh[K][VEC], sh[K][VEC], g2[K][VEC];
    float r0 = 0.f, r1 = 0.f;
    auto piece = [&](int which, int k, float (&f)[VEC]) {
      unpack<T, VEC>(*reinterpret_cast<const Pack<T, VEC>*>(at(st, which, k)), f);
    };
    auto param = [&](int which, int k, float (&f)[VEC]) {
      unpack<T, VEC>(*reinterpret_cast<const Pack<T, VEC>*>(at(par, which, k)), f);
    };
    auto shared_gate = [&](int k, float (&f)[VEC]) {
#pragma unroll
      for (int q = 0; q < VEC / 4; ++q) {
        const float4 v = *reinterpret_cast<const float4*>(at(par, l.a + q, k));
        f[4 * q] = v.x;
        f[4 * q + 1] = v.y;
        f[4 * q + 2] = v.z;
        f[4 * q + 3] = v.w;
      }
    };
    // N1's value from xhat
    auto n1_of = [&](int k, float (&n)[VEC]) {
      float f[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) n[e] = xh[k][e];
      if (l.w1 >= 0) {
        param(l.w1, k, f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) n[e] *= p.woff + f[e];
      }
      if (l.b1 >= 0) {
        param(l.b1, k, f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) n[e] += f[e];
      }
    };
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool ok = live && vok[k];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        xh[k][e] = 0.f;
        sh[k][e] = 0.f;
        g2[k][e] = 0.f;
      }
      if (ok) {
        piece(l.x, k, xh[k]);
        if (p.post_kind != FLN_NO_NORM) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) xh[k][e] = (xh[k][e] - mean1) * rstd1;
        }
        if (l.dy >= 0) {
          float n[VEC], f[VEC];
          n1_of(k, n);
          if (GATE == 1) shared_gate(k, f);
          if (GATE == 2) {
            piece(l.gate, k, f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = gate_act<EXACT>(f[e], p.act);
          }
          if (GATE != 0) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) n[e] *= f[e];
          }
#pragma unroll
          for (int e = 0; e < VEC; ++e) n[e] *= p.ba;
          if (l.res >= 0) {
            piece(l.res, k, f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) n[e] = fmaf(p.ra, f[e], n[e]);
          }
          piece(l.dy, k, g2[k]);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            sh[k][e] = (n[e] - mean2) * rstd2;
            acc_u[k][e] = fmaf(g2[k][e], sh[k][e], acc_u[k][e]);
            if (FOUR) acc_v[FOUR ? k : 0][e] += g2[k][e];
          }
          if (l.w2 >= 0) {
            param(l.w2, k, f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) g2[k][e] *= p.woff + f[e];
          }
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            r0 = fmaf(g2[k][e], sh[k][e], r0);
            r1 += g2[k][e];
          }
        }
      }
    }
    float c1 = 0.f, c2 = 0.f;
    if (l.dy >= 0) {
      row_sum2(rg, r0, r1);
      c1 = r0 * inv_n;
      c2 = p.kind == FLN_LAYERNORM ? r1 * inv_n : 0.f;
    }
    r0 = 0.f;
    r1 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (live && vok[k]) {
        float d[VEC], f[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[e] = 0.f;
        if (l.ds >= 0) piece(l.ds, k, d);
        if (l.dy >= 0) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) d[e] = fmaf(rstd2, fmaf(-sh[k][e], c1, g2[k][e] - c2), d[e]);
        }
        if (p.dres != nullptr) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) f[e] = p.ra * d[e];
          Pack<T, VEC> o;
          pack<T, VEC>(f, o);
          st_stream<T, VEC>(reinterpret_cast<T*>(p.dres) + base + col[k], o);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[e] *= p.ba;  // e of the formulas
        if (GATE == 2) {
          float gv[VEC];
          piece(l.gate, k, gv);
          if (p.dgate != nullptr) {
            float n[VEC];
            n1_of(k, n);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              float a, da;
              gate_act_grad<EXACT>(gv[e], p.act, &a, &da);
              f[e] = d[e] * n[e] * da;
              d[e] *= a;
            }
            Pack<T, VEC> o;
            pack<T, VEC>(f, o);
            st_stream<T, VEC>(reinterpret_cast<T*>(p.dgate) + base + col[k], o);
          } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) d[e] *= gate_act<EXACT>(gv[e], p.act);
          }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          acc_p[k][e] = fmaf(d[e], xh[k][e], acc_p[k][e]);
          if (FOUR) acc_q[FOUR ? k : 0][e] += d[e];
        }
        if (GATE == 1) {
          shared_gate(k, f);
#pragma unroll
          for (int e = 0; e < VEC; ++e) d[e] *= f[e];
        }
        if (l.w1 >= 0) {
          param(l.w1, k, f);
#pragma unroll
          for (int e = 0; e < VEC; ++e) d[e] *= p.woff + f[e];
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          g2[k][e] = d[e];  // g1 from here on
          r0 = fmaf(d[e], xh[k][e], r0);
          r1 += d[e];
        }
      }
    }
    if (p.dx != nullptr) {
      float d1 = 0.f, d2 = 0.f;
      if (p.post_kind != FLN_NO_NORM) {
        row_sum2(rg, r0, r1);
        d1 = r0 * inv_n;
        d2 = p.post_kind == FLN_LAYERNORM ? r1 * inv_n : 0.f;
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (live && vok[k]) {
          if (p.post_kind != FLN_NO_NORM) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) g2[k][e] = rstd1 * fmaf(-xh[k][e], d1, g2[k][e] - d2);
          }
          Pack<T, VEC> o;
          pack<T, VEC>(g2[k], o);
          st_stream<T, VEC>(reinterpret_cast<T*>(p.dx) + base + col[k], o);
        }
      }
    }
    const int64_t slot = cur.slot;
    step(cur);
    opened = cur.slot != slot;
    if (opened) {
      // the slot's sums: one partial row per row group, or per warp where a warp holds several
      if (p.acc != 0) {
        const int who = g.tpr < 32 ? tid >> 5 : r_in;
        float* out = p.partials + (slot * g.rep + who) * (int64_t)p.nacc * p.cols;
        auto leave = [&](float (&acc)[VEC], int k, int which) {
          if (!(p.acc & which)) return;
          for (int off = 16; off >= g.tpr; off >>= 1) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], off);
          }
          if (!vok[k] || (g.tpr < 32 && (tid & 31) >= g.tpr)) return;
          float* q = out + (int64_t)__popc(p.acc & (which - 1)) * p.cols + col[k];
#pragma unroll
          for (int e = 0; e < VEC; e += 4) *reinterpret_cast<float4*>(q + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
        };
#pragma unroll
        for (int k = 0; k < K; ++k) {
          leave(acc_p[k], k, kAccP);
          if (FOUR) leave(acc_q[FOUR ? k : 0], k, kAccQ);
          leave(acc_u[k], k, kAccU);
          if (FOUR) leave(acc_v[FOUR ? k : 0], k, kAccV);
        }
      }
      clear();
    }
  }
}

// launches of one element type; K vectors per thread
template <typename T>
int nga_fwd_rows(const NgaParams& p, const NgaGeom& g, int K, cudaStream_t st);
template <typename T>
int nga_bwd_rows(const NgaParams& p, const NgaGeom& g, int K, cudaStream_t st);

inline int nga_gate_of(const NgaParams& p) {
  return p.gate_mode == FLN_GATE_NONE ? 0 : (p.gate_mode == FLN_GATE_ELEMENT ? 2 : 1);
}

template <typename T, int K>
static int nga_fwd_rows_k(const NgaParams& p, const NgaGeom& g, cudaStream_t st) {
  const unsigned grid = (unsigned)g.grid;
  switch (nga_gate_of(p)) {
    case 0:
      nga_fwd_rows_kernel<T, K, 0><<<grid, g.threads, 0, st>>>(p, g);
      break;
    case 1:
      nga_fwd_rows_kernel<T, K, 1><<<grid, g.threads, 0, st>>>(p, g);
      break;
    default:
      nga_fwd_rows_kernel<T, K, 2><<<grid, g.threads, 0, st>>>(p, g);
      break;
  }
  FLN_CHECK_LAUNCH();
  return FLN_OK;
}

template <typename T, int K, int GATE, bool FOUR>
static int nga_bwd_rows_one(const NgaParams& p, const NgaGeom& g, cudaStream_t st) {
  auto kern = nga_bwd_rows_kernel<T, K, GATE, FOUR>;
  if (g.smem > 48 * 1024 &&
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)g.smem) != cudaSuccess) {
    cudaGetLastError();
    return FLN_ERR_LAUNCH;
  }
  kern<<<(unsigned)g.grid, g.threads, g.smem, st>>>(p, g);
  FLN_CHECK_LAUNCH();
  return FLN_OK;
}
template <typename T, int K>
static int nga_bwd_rows_k(const NgaParams& p, const NgaGeom& g, cudaStream_t st) {
  const bool four = (p.acc & (kAccQ | kAccV)) != 0;
  switch (nga_gate_of(p)) {
    case 0:
      return four ? nga_bwd_rows_one<T, K, 0, true>(p, g, st) : nga_bwd_rows_one<T, K, 0, false>(p, g, st);
    case 1:
      return four ? nga_bwd_rows_one<T, K, 1, true>(p, g, st) : nga_bwd_rows_one<T, K, 1, false>(p, g, st);
    default:
      return four ? nga_bwd_rows_one<T, K, 2, true>(p, g, st) : nga_bwd_rows_one<T, K, 2, false>(p, g, st);
  }
}

#define FLN_NGA_INSTANTIATE(T)                                                                       \
  template <>                                                                                        \
  int nga_fwd_rows<T>(const NgaParams& p, const NgaGeom& g, int K, cudaStream_t st) {                \
    if (K == 1) return nga_fwd_rows_k<T, 1>(p, g, st);                                               \
    if (K == 2) return nga_fwd_rows_k<T, 2>(p, g, st);                                               \
    if (K == 4) return nga_fwd_rows_k<T, 4>(p, g, st);                                               \
    return FLN_ERR_UNSUPPORTED;                                                                      \
  }                                                                                                  \
  template <>                                                                                        \
  int nga_bwd_rows<T>(const NgaParams& p, const NgaGeom& g, int K, cudaStream_t st) {                \
    if (K == 1) return nga_bwd_rows_k<T, 1>(p, g, st);                                               \
    if (K == 2) return nga_bwd_rows_k<T, 2>(p, g, st);                                               \
    if constexpr (sizeof(T) == 4) {                                                                  \
      if (K == 4) return nga_bwd_rows_k<T, 4>(p, g, st);                                             \
    }                                                                                                \
    return FLN_ERR_UNSUPPORTED;                                                                      \
  }

}  // namespace fln
