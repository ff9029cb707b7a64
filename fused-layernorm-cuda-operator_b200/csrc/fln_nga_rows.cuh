// fln_norm_gate_add_norm: the kernels that hold a row in registers, for rows of whole 16-byte
// vectors.  Instantiated per element type in fln_nga_{f32,bf16,f16}.cu; launched from fln_nga.cu.
// The formulas stand in fln_nga.cuh.
//
// A row is owned by `tpr` consecutive threads: a power of two within a warp, or whole warps.
// Thread `lane` of them holds vectors lane, lane + tpr, ... (K of them, the last ones may lie
// behind the row).
//
// At 16 bits these kernels run out of issue slots before they run out of HBM, so the arithmetic is
// on register pairs (packed fp32), and what is constant over the rows of a group is folded into
// 32-bit coefficients once per group:
//     no gate or a shared one     C1 = ba * act(gate) * w1,  B1 = ba * act(gate) * b1
//                                 s  = xh * C1 + B1 + ra * residual,    g1 = ds * C1
//     a gate per element          C1 = ba * w1,  B1 = ba * b1,  a = act(gate)
//                                 s  = a * (xh * C1 + B1) + ra * residual,
//                                 dgate = ds * (xh * C1 + B1) * act'(gate),  g1 = ds * a * C1
//     C2 = w2, B2 = b2            y  = sh * C2 + B2,                    g2 = dy * C2
// The column sums P and Q are kept of ds (times a) and multiplied by ba when they are left.
// The unfolded form on single floats took 48 (forward) and 84 (backward) instructions per element
// at 16384 x 4096 bf16: 127 and 248 us.  As it is: 20 and 28, 90 and 146 us (with the sums of its partial
// rows); 16384 x 8192: 180 us (6.0 TB/s of the 8 bytes per element) and 261 us (6.2 TB/s of 12), where
// HBM is the bound.
//
// SHIFT: rows that are not whole 16-byte vectors (tensors that start on a 16-byte boundary, row length
// not a multiple of a vector).  Such a row starts at one of 2, 4 or 8 places of a vector, by its
// number; a CTA takes rows of one class at a time (fln_nga.cuh), for which a column always lies at
// the same place of the same thread's vectors.  So all that is above holds: the row is staged as
// the vectors that cover it, what belongs to the neighbouring rows in its first and last vector is
// set to zero, and only those two are stored element by element.  (Rows held element by element
// instead: 16384 x 2777 bf16 at 190 us forward and 546 us backward; this way 123 and 203.  The general
// form with a gate per element takes 246 and 498 there: its limits per vector and four column sums do
// not fit the registers.)
//
// PAIR (backward): a row is shared by the two CTAs of a cluster, half of its vectors each, where one
// CTA's registers do not hold it.  The row sums go through the shared memory of both and the
// cluster's barrier takes the place of the CTA's; both add the same values in the same order.
// 4096 x 12288 bf16, 12 bytes per element: 235 us, 1590 with the looping kernels.
//
// GEN = false: both norms RMSNorm or none and no bias, which is what most blocks have; no means, no
// Q and V.  GEN = true: everything, in more registers: 16384 x 4096 bf16, two LayerNorms with biases 135
// and 208 us, with a sigmoid gate per element too 162 and 318 (1.6 to 2 times its bytes).  Backward rows
// of 5121 to 8192 elements of 16 bits (fp32: past 5120) take 16 elements per thread, and there the
// general form spills: 16384 x 8192 in 826 us, 3.4 times its bytes.
#pragma once

#include "fln_nga.cuh"
#include "fln_pipeline.cuh"  // thread-block cluster helpers

namespace fln {

struct NgaGeom {
  int tpr;      // threads per row
  int R;        // rows per CTA
  int nv;       // vectors per row
  int threads;  // per CTA: R * tpr
  int stages;   // backward: rows on their way per row group
  int rep;      // backward: row groups (or warps of several) whose sums a CTA joins
  int64_t grid;
  size_t smem;
  int csm;      // backward: coefficients in shared memory
  int direct;   // backward: dsum past the ring
  int pair;     // backward: a row is shared by the two CTAs of a cluster
  int64_t chunk, per_group;  // forward: rows per CTA, CTAs per group
};

// Where the threads per row are known at compile time (TPR != 0) every offset in shared memory and
// between a thread's vectors is a constant, and where the row is whole as well (cols == TPR * K *
// vector, !RAG) nothing is predicated: 34 -> 22 instructions per element of the bf16 forward at
// 4096 columns, 51 -> 28 of the backward.  Rows per CTA of these:
__host__ __device__ constexpr int fixed_rows(int tpr) { return tpr >= 128 ? 1 : (tpr > 32 ? 2 : 256 / tpr); }

// Numbers of threads per row that are known at compile time: 4 to 64 for short rows that are whole (heads
// of 32 to 512 elements: 524288 x 64 bf16 with a gate per element, backward 116 us at run time, 71 so),
// and for longer ones the next of this list where that leaves few of them idle (8192 x 5064 bf16, two
// LayerNorms with biases, backward 193 us at run time, 151 so).  Whole rows of a number of their own
// keep it where the next one would idle more than an eighth of the threads (288 -> 320 threads, 8192 x
// 4608 bf16: forward 147 -> 102 us; 160 -> 192, 16384 x 2560: backward 101 -> 116).  0: everything is
// found out at run time.  All but 192, 384 and (dsum past the ring) 640 have a kernel for rows that fill
// their threads besides the one for rows that do not: there it gained nothing (16384 x 6144 bf16: 212
// and 208 us backward, 16384 x 1536 general: 91 and 95).
constexpr int kFixedTpr[] = {128, 192, 256, 320, 384, 512, 640};
inline int fixed_tpr(int tpr, bool whole, int most) {
  for (int t : kFixedTpr)
    if (t >= tpr && t <= most && (t - tpr) * (whole ? 8 : 6) <= t) return t;
  return 0;
}
// Forward: what fits once on an SM may have all of its registers; two CTAs where that leaves 96 for a
// thread and the ring of 16-bit rows leaves the shared memory (16384 x 5120 bf16 with a gate per element
// and two LayerNorms: 300 -> 207 us; up to 256 threads the bound of 128 registers does it by itself).
__host__ __device__ constexpr int fwd_threads(int tpr) { return tpr > 256 ? tpr : 512; }
__host__ __device__ constexpr int fwd_ctas(int es, int tpr) { return es == 2 && tpr > 256 && 2 * 96 * tpr <= 65536 ? 2 : 1; }

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
  int rank;    // in the cluster that shares the row, -1 where there is none
};
// (the row lies at elements [shift, shift + cols) of its nv vectors)
template <int TPR, bool FULL>
__device__ __forceinline__ RowGroup row_group(const NgaGeom& g, int K, int vec, int nv, int shift, int cols, float2* red) {
  RowGroup r;
  const int tpr = TPR ? TPR : g.tpr;
  r.width = tpr < 32 ? tpr : 32;
  r.wpr = tpr <= 32 ? 1 : tpr >> 5;
  r.warp0 = tpr <= 32 ? (int)(threadIdx.x >> 5) : (int)(threadIdx.x / tpr) * r.wpr;
  r.red = red;
  r.flip = 0;
  r.rank = -1;
  auto count = [&](int w) {  // elements of the row in its warp w
    if (FULL) return (float)(K * 32 * vec);
    int n = 0;
    for (int k = 0; k < K; ++k) {
      const int v0 = k * tpr + w * 32, v1 = v0 + 32 < nv ? v0 + 32 : nv;
      const int e0 = v0 * vec > shift ? v0 * vec : shift, e1 = v1 * vec < shift + cols ? v1 * vec : shift + cols;
      n += e1 > e0 ? e1 - e0 : 0;
    }
    return (float)n;
  };
  const int lane = threadIdx.x & 31;
  r.cnt = lane < r.wpr ? count(lane) : 0.f;
  r.mine = r.wpr == 1 ? (float)cols : count((int)(threadIdx.x >> 5) - r.warp0);
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
// the same over the two CTAs of a cluster: 16 warps at most of each
__device__ __forceinline__ float2 pair_exchange(RowGroup& g, float2 mine) {
  float2* r = g.red + g.flip * 32;
  g.flip ^= 1;
  if ((threadIdx.x & 31) == 0) {
    float2* place = r + g.rank * 16 + (threadIdx.x >> 5);
    *place = mine;
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(map_to_cta(place, (uint32_t)(g.rank ^ 1))), "f"(mine.x),
                 "f"(mine.y)
                 : "memory");
  }
  __syncwarp();
  cluster_sync_all();
  const int lane = threadIdx.x & 31;
  return (lane & 15) < g.wpr ? r[lane] : make_float2(0.f, 0.f);
}
template <bool PAIR = false>
__device__ __forceinline__ void row_sum1(RowGroup& g, float& a) {
  float v[1] = {a};
  warp_sum<1>(v, g.width);
  if (PAIR) {
    v[0] = pair_exchange(g, make_float2(v[0], 0.f)).x;
    warp_sum<1>(v, 32);
  } else if (g.wpr > 1) {
    v[0] = warp_exchange(g, make_float2(v[0], 0.f)).x;
    warp_sum<1>(v, 32);
  }
  a = v[0];
}
template <bool PAIR = false>
__device__ __forceinline__ void row_sum2(RowGroup& g, float& a, float& b) {
  float v[2] = {a, b};
  warp_sum<2>(v, g.width);
  if (PAIR || g.wpr > 1) {
    const float2 o = PAIR ? pair_exchange(g, make_float2(v[0], v[1])) : warp_exchange(g, make_float2(v[0], v[1]));
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
// only(k, e, d): d where the two elements belong to the row, else zeros.
template <int K, int V2, bool GEN, typename Only>
__device__ __forceinline__ void row_stats(RowGroup& g, int kind, const float2 (&v)[K][V2], const Only& only, float inv_n,
                                          float eps, float& mean, float& rstd) {
  float q = 0.f;
  mean = 0.f;
  if (!GEN || kind == FLN_RMSNORM) {
    float2 t = f2(0.f);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < V2; ++e) t = f2fma(v[k][e], v[k][e], t);
    q = t.x + t.y;
    row_sum1(g, q);
  } else {
    float2 t = f2(0.f);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < V2; ++e) t = f2add(v[k][e], t);
    float s[1] = {t.x + t.y};
    warp_sum<1>(s, g.width);
    const float m = s[0] / fmaxf(g.mine, 1.f);
    t = f2(0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int e = 0; e < V2; ++e) {
        const float2 d = only(k, e, f2add(v[k][e], f2(-m)));
        t = f2fma(d, d, t);
      }
    }
    float d2[1] = {t.x + t.y};
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

// vectors between global memory, a thread's own places in shared memory, and register pairs
__device__ __forceinline__ void cp_async16(void* smem, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_async_wait_behind(int ahead) {  // at most `ahead` groups (0, 1, 2) still on their way
  if (ahead == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else if (ahead == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}
__device__ __forceinline__ void cp_async16_part(void* smem, const void* src, int bytes) {  // the rest zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(src),
               "r"(bytes)
               : "memory");
}
// Where a thread's vectors lie in the row.  at[k]: column of the first element (below zero in the
// first vector of a shifted row); a vector behind the row is replaced by the row's last one and
// ok[k] is false; [lo, hi): the elements of an edge vector that belong to the row.
template <int K, int VEC, bool FULL, bool SHIFT>
struct Places {
  int at[K];
  bool ok[K], edge[SHIFT ? K : 1];
  int lo[SHIFT ? K : 1], hi[SHIFT ? K : 1];
  // (v0, v1: the vectors of this CTA where two share the row)
  __device__ __forceinline__ void set(int lane, int tpr, int nv, int cols, int shift, bool pair = false, int v0 = 0, int v1 = 0) {
    if (SHIFT) nv = (shift + cols + VEC - 1) / VEC;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int v = lane + k * tpr + (pair ? v0 : 0);
      ok[k] = FULL || (!SHIFT && !pair && K == 2 && k == 0) || (v < nv && (!pair || v < v1));  // (tpr <= nv where K is 2)
      at[k] = (ok[k] ? v : nv - 1) * VEC - (SHIFT ? shift : 0);
      if (SHIFT) {
        lo[SHIFT ? k : 0] = at[k] < 0 ? -at[k] : 0;
        hi[SHIFT ? k : 0] = cols - at[k] < VEC ? cols - at[k] : VEC;
        edge[SHIFT ? k : 0] = at[k] < 0 || at[k] + VEC > cols;
      }
    }
  }
  // a pair of the vector where it belongs to the row, else zeros (not v times zero, which would be
  // NaN where v is infinite)
  __device__ __forceinline__ float2 only(int k, int e, float2 v) const {
    if (FULL) return v;
    if (SHIFT) {
      const int l = lo[SHIFT ? k : 0], h = hi[SHIFT ? k : 0];
      return make_float2(ok[k] && 2 * e >= l && 2 * e < h ? v.x : 0.f, ok[k] && 2 * e + 1 >= l && 2 * e + 1 < h ? v.y : 0.f);
    }
    return make_float2(ok[k] ? v.x : 0.f, ok[k] ? v.y : 0.f);
  }
  // what the neighbouring rows have in an edge vector, set to zero
  __device__ __forceinline__ void trim(int k, float2 (&v)[VEC / 2]) const {
    if (SHIFT && edge[SHIFT ? k : 0]) {
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) {
        const int l = lo[SHIFT ? k : 0], h = hi[SHIFT ? k : 0];
        v[e] = make_float2(2 * e >= l && 2 * e < h ? v[e].x : 0.f, 2 * e + 1 >= l && 2 * e + 1 < h ? v[e].y : 0.f);
      }
    }
  }
};
// the first column of a row in its first vector
__device__ __forceinline__ int row_shift(int64_t row, int cols, int vec) {
  return (int)((uint32_t)(row & (vec - 1)) * (uint32_t)(cols & (vec - 1)) & (uint32_t)(vec - 1));
}
// v, or zeros (not v times zero, which would be NaN where v is infinite)
__device__ __forceinline__ float2 f2only(bool on, float2 v) { return make_float2(on ? v.x : 0.f, on ? v.y : 0.f); }
template <typename T>
__device__ __forceinline__ void take(const unsigned char* p, float2 (&f)[8 / sizeof(T)]) {
  Pack<T, 16 / sizeof(T)> v;
  *reinterpret_cast<uint4*>(&v) = *reinterpret_cast<const uint4*>(p);
  unpack2<T, 16 / sizeof(T)>(v, f);
}
template <typename T>
__device__ __forceinline__ void give(T* p, const float2 (&f)[8 / sizeof(T)]) {
  Pack<T, 16 / sizeof(T)> v;
  pack2<T, 16 / sizeof(T)>(f, v);
  st_stream<T, 16 / sizeof(T)>(p, v);
}
// a vector of a row at `row`, whole or only what belongs to the row
template <typename T, int K, bool FULL, bool SHIFT>
__device__ __forceinline__ void give_row(T* row, const Places<K, 16 / (int)sizeof(T), FULL, SHIFT>& w, int k,
                                         const float2 (&f)[8 / sizeof(T)]) {
  if (SHIFT && w.edge[SHIFT ? k : 0]) {
#pragma unroll
    for (int e = 0; e < 8 / (int)sizeof(T); ++e) {
      const int l = w.lo[SHIFT ? k : 0], h = w.hi[SHIFT ? k : 0];
      if (2 * e >= l && 2 * e < h) row[w.at[k] + 2 * e] = Cvt<T>::from_f(f[e].x);
      if (2 * e + 1 >= l && 2 * e + 1 < h) row[w.at[k] + 2 * e + 1] = Cvt<T>::from_f(f[e].y);
    }
    return;
  }
  give<T>(row + w.at[k], f);
}
// a vector of a parameter; SHIFT: element by element, the nearest there is for those beside the row
template <typename T, bool SHIFT>
__device__ __forceinline__ void param2(const void* p, int64_t off, int col, int cols, float2 (&f)[8 / sizeof(T)]) {
  const T* q = reinterpret_cast<const T*>(p) + off;
  if (!SHIFT) {
    unpack2<T, 16 / sizeof(T)>(ld_param<T, 16 / sizeof(T)>(q + col), f);
    return;
  }
  auto one = [&](int c) { return Cvt<T>::to_f(__ldg(q + (c < 0 ? 0 : (c < cols ? c : cols - 1)))); };
#pragma unroll
  for (int e = 0; e < 8 / (int)sizeof(T); ++e) f[e] = make_float2(one(col + 2 * e), one(col + 2 * e + 1));
}

// C1 and B1 of a vector of columns; `goff` is where the group's gate vector starts
template <typename T, int GATE, bool SHIFT>
__device__ __forceinline__ void coef1(const NgaParams& p, int col, int64_t goff, float2 (&c)[8 / sizeof(T)],
                                      float2 (&b)[8 / sizeof(T)]) {
  constexpr int V2 = 8 / (int)sizeof(T);
#pragma unroll
  for (int e = 0; e < V2; ++e) {
    c[e] = f2(1.f);
    b[e] = f2(0.f);
  }
  if (p.w1 != nullptr) {
    param2<T, SHIFT>(p.w1, 0, col, p.cols, c);
#pragma unroll
    for (int e = 0; e < V2; ++e) c[e] = f2add(c[e], f2(p.woff));
  }
  if (p.b1 != nullptr) param2<T, SHIFT>(p.b1, 0, col, p.cols, b);
  float2 a[V2];
#pragma unroll
  for (int e = 0; e < V2; ++e) a[e] = f2(1.f);
  if (GATE == 1) {
    param2<T, SHIFT>(p.gate, goff, col, p.cols, a);
    gate_act_all<sizeof(T) == 4>(a, p.act);
  }
#pragma unroll
  for (int e = 0; e < V2; ++e) {
    a[e] = f2mul(a[e], f2(p.ba));
    c[e] = f2mul(c[e], a[e]);
    b[e] = f2mul(b[e], a[e]);
  }
}
// (BIAS: the backward has no use for B2)
template <typename T, bool SHIFT, bool BIAS>
__device__ __forceinline__ void coef2(const NgaParams& p, int col, int64_t aoff, float2 (&c)[8 / sizeof(T)], float2 (&b)[8 / sizeof(T)]) {
  constexpr int V2 = 8 / (int)sizeof(T);
#pragma unroll
  for (int e = 0; e < V2; ++e) {
    c[e] = f2(1.f);
    b[e] = f2(0.f);
  }
  if (p.w2 != nullptr) {
    param2<T, SHIFT>(p.w2, aoff, col, p.cols, c);
#pragma unroll
    for (int e = 0; e < V2; ++e) c[e] = f2add(c[e], f2(p.woff));
  }
  if (BIAS && p.b2 != nullptr) param2<T, SHIFT>(p.b2, aoff, col, p.cols, b);
}

// ----------------------------------------------------------------------------------------
// forward: a CTA takes `chunk` consecutive rows of a group, R at a time.  Every thread keeps its
// own vectors of the next rows on their way into its own places in shared memory (cp.async), so
// staging needs no barrier and no flag; the barriers are those of the row sums.  A CTA is short
// (a few rows), so that the hardware hands the chunks out and SMs with less bandwidth get fewer.
// GATE 0: none, 1: shared by rows, 2: an element each.  HOLD: the coefficients stay in registers
// over the chunk, else they are made again for every row (rows too long for that).
// ----------------------------------------------------------------------------------------
template <typename T, int K, int GATE, bool GEN, bool HOLD, int TPR, bool RAG, bool SHIFT>
__global__ void __launch_bounds__(fwd_threads(TPR), fwd_ctas((int)sizeof(T), TPR)) nga_fwd_rows_kernel(const NgaParams p, const NgaGeom g) {
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int VEC = 16 / (int)sizeof(T), V2 = VEC / 2;
  extern __shared__ __align__(128) unsigned char smem[];
  constexpr bool FULL = TPR != 0 && !RAG;
  const int tpr = TPR ? TPR : g.tpr;
  const int R = TPR ? fixed_rows(TPR) : g.R;
  const int threads = TPR ? TPR * fixed_rows(TPR) : g.threads;
  const int cols = FULL ? TPR * K * VEC : p.cols;
  const int tid = threadIdx.x;
  const int r_in = tid / tpr, lane = tid - r_in * tpr;
  const float inv_n = 1.0f / (float)cols;
  const uint32_t unit = (uint32_t)K * threads * 16u;
  unsigned char* stages = smem + 512 + tid * 16;
  const int has_res = p.res != nullptr ? 1 : 0;
  const uint32_t stage_bytes = (uint32_t)(1 + has_res + (GATE == 2 ? 1 : 0)) * unit;
  const uint32_t gate_off = (uint32_t)(1 + has_res) * unit;
  int64_t group, first, last;
  if (SHIFT) {
    const SlotRows sr = slot_rows(p, blockIdx.x);
    group = sr.group;
    first = sr.first;
    last = sr.last;
  } else {
    group = blockIdx.x / g.per_group;
    first = group * p.group_rows + (blockIdx.x - group * g.per_group) * g.chunk;
    last = (group + 1) * p.group_rows;
    if (first + g.chunk < last) last = first + g.chunk;
  }
  const int64_t apart = SHIFT ? p.period : 1;  // from one row to the next
  const int64_t goff = p.gate_mode == FLN_GATE_GROUP ? group * cols : 0;
  const int64_t aoff = p.affine_grouped ? group * cols : 0;
  // A lane whose last vectors lie behind the row works on the row's last vector instead; what goes
  // into the sums is set to zero there and nothing is stored, so the arithmetic has no branches.
  Places<K, VEC, FULL, SHIFT> w;
  const int shift = SHIFT ? row_shift(first, cols, VEC) : 0;
  w.set(lane, tpr, g.nv, cols, shift);
  RowGroup rg = row_group<TPR, FULL>(g, K, VEC, SHIFT ? (shift + cols + VEC - 1) / VEC : g.nv, shift, cols,
                                     reinterpret_cast<float2*>(smem));
  auto only = [&](int k, int e, float2 v) { return w.only(k, e, v); };

  // row groups behind the last row work on the last row once more (and write the same values), so
  // that nothing below depends on it
  int64_t ahead = first;
  int in_stage = 0;
  auto fetch = [&]() {
    if (ahead < last) {
      const int64_t mine = ahead + r_in * apart;
      const int64_t o = (mine < last ? mine : last - 1) * (int64_t)cols;
      unsigned char* st = stages + (uint32_t)in_stage * stage_bytes;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        unsigned char* d = st + (uint32_t)(k * threads) * 16u;
        const int64_t q = o + w.at[k];
        auto bring = [&](unsigned char* to, const void* from) {
          if (SHIFT) {  // the last vector of the last row may reach behind the tensor
            const int64_t left = (p.rows * cols - q) * (int)sizeof(T);
            cp_async16_part(to, reinterpret_cast<const T*>(from) + q, left < 16 ? (int)left : 16);
          } else {
            cp_async16(to, reinterpret_cast<const T*>(from) + q);
          }
        };
        bring(d, p.x);
        if (has_res) bring(d + unit, p.res);
        if (GATE == 2) bring(d + gate_off, p.gate);
      }
      ahead += R * apart;
    }
    cp_async_commit();
    in_stage = in_stage + 1 == g.stages ? 0 : in_stage + 1;
  };
  for (int i = 0; i + 1 < g.stages; ++i) fetch();

  float2 c1[HOLD ? K : 1][V2], b1[HOLD && GEN ? K : 1][V2], c2[HOLD ? K : 1][V2], b2[HOLD && GEN ? K : 1][V2];
  if (HOLD) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      coef1<T, GATE, SHIFT>(p, w.at[k], goff, c1[HOLD ? k : 0], b1[HOLD && GEN ? k : 0]);
      coef2<T, SHIFT, true>(p, w.at[k], aoff, c2[HOLD ? k : 0], b2[HOLD && GEN ? k : 0]);
    }
  }
  const float2 ra = f2(p.ra);
  int stage = 0;
  for (int64_t row0 = first; row0 < last; row0 += R * apart) {
    fetch();
    const int64_t row = row0 + r_in * apart < last ? row0 + r_in * apart : last - 1;
    cp_async_wait_behind(g.stages - 1);
    const unsigned char* st = stages + (uint32_t)stage * stage_bytes;
    stage = stage + 1 == g.stages ? 0 : stage + 1;
    float2 s[K][V2];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      take<T>(st + (uint32_t)(k * threads) * 16u, s[k]);
      if (!FULL) {
#pragma unroll
        for (int e = 0; e < V2; ++e) s[k][e] = w.only(k, e, s[k][e]);
      }
    }
    float mean1 = 0.f, rstd1 = 1.f;
    if (p.post_kind != FLN_NO_NORM) row_stats<K, V2, GEN>(rg, p.post_kind, s, only, inv_n, p.eps1, mean1, rstd1);
    T* sum = reinterpret_cast<T*>(p.sum) + row * (int64_t)cols;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      {
        const unsigned char* d = st + (uint32_t)(k * threads) * 16u;
        float2 tc[V2], tb[V2];
        if (!HOLD) coef1<T, GATE, SHIFT>(p, w.at[k], goff, tc, tb);
#pragma unroll
        for (int e = 0; e < V2; ++e) {
          // (x - mean) * rstd: without a norm mean is 0 and rstd 1, and x passes as it is
          if (GEN) s[k][e] = f2add(s[k][e], f2(-mean1));
          s[k][e] = f2mul(s[k][e], f2(rstd1));
          const float2 c = HOLD ? c1[HOLD ? k : 0][e] : tc[e];
          const float2 b = HOLD ? b1[HOLD && GEN ? k : 0][e] : tb[e];
          s[k][e] = GEN ? f2fma(s[k][e], c, b) : f2mul(s[k][e], c);
        }
        if (GATE == 2) {
          float2 a[V2];
          take<T>(d + gate_off, a);
          gate_act_all<EXACT>(a, p.act);
#pragma unroll
          for (int e = 0; e < V2; ++e) s[k][e] = f2mul(s[k][e], a[e]);
        }
        if (has_res) {
          float2 r[V2];
          take<T>(d + unit, r);
#pragma unroll
          for (int e = 0; e < V2; ++e) s[k][e] = f2fma(r[e], ra, s[k][e]);
        }
        if (w.ok[k]) give_row<T, K, FULL, SHIFT>(sum, w, k, s[k]);
        if (!FULL) {
#pragma unroll
          for (int e = 0; e < V2; ++e) s[k][e] = w.only(k, e, s[k][e]);
        }
      }
    }
    float mean2 = 0.f, rstd2 = 1.f;
    if (p.kind != FLN_NO_NORM) {
      row_stats<K, V2, GEN>(rg, p.kind, s, only, inv_n, p.eps2, mean2, rstd2);
      T* y = reinterpret_cast<T*>(p.y) + row * (int64_t)cols;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        {
          float2 tc[V2], tb[V2];
          if (!HOLD) coef2<T, SHIFT, true>(p, w.at[k], aoff, tc, tb);
#pragma unroll
          for (int e = 0; e < V2; ++e) {
            if (GEN) s[k][e] = f2add(s[k][e], f2(-mean2));
            s[k][e] = f2mul(s[k][e], f2(rstd2));
            const float2 c = HOLD ? c2[HOLD ? k : 0][e] : tc[e];
            const float2 b = HOLD ? b2[HOLD && GEN ? k : 0][e] : tb[e];
            s[k][e] = GEN ? f2fma(s[k][e], c, b) : f2mul(s[k][e], c);
          }
          if (w.ok[k]) give_row<T, K, FULL, SHIFT>(y, w, k, s[k]);
        }
      }
    }
    if (lane == 0) {
      if (p.mean1 != nullptr && p.post_kind == FLN_LAYERNORM) p.mean1[row] = mean1;
      if (p.rstd1 != nullptr && p.post_kind != FLN_NO_NORM) p.rstd1[row] = rstd1;
      if (p.mean2 != nullptr && p.kind == FLN_LAYERNORM) p.mean2[row] = mean2;
      if (p.rstd2 != nullptr && p.kind != FLN_NO_NORM) p.rstd2[row] = rstd2;
    }
  }
}

// ----------------------------------------------------------------------------------------
// backward: persistent CTAs; CTA b takes slots b, b + grid, ...  Rows are staged as in the forward,
// the column sums stay in registers over a slot.  CSM: the coefficients lie in shared memory, in 32
// bits, each thread's own; else (no room) they are made again where they are used.
// SET: which tensors there are, 1: x, residual, dy and dsum, 2: x and dsum, 0: found out at run time;
// 3: like 1, dsum fetched into registers (rows whose ring would not fit otherwise).
// ----------------------------------------------------------------------------------------
constexpr int kNgaBwdHeader = 512;

// where a thread's pieces lie, in units of K * threads * 16 bytes behind the header; a coefficient
// takes 4 / es units
struct NgaBwdLayout {
  int c1, b1, c2;            // -1: absent
  int x, res, dy, ds, gate;  // tensors inside a stage
  int coefs, tensors;        // units
};
__host__ __device__ constexpr NgaBwdLayout nga_layout(int es, bool csm, bool bias, bool res, bool dy, bool ds, bool gate) {
  NgaBwdLayout l = {-1, -1, -1, 0, -1, -1, -1, -1, 0, 0};
  const int u = 4 / es;
  int n = 0;
  if (csm) {
    l.c1 = n;
    n += u;
    if (bias) {
      l.b1 = n;
      n += u;
    }
    if (dy) {
      l.c2 = n;
      n += u;
    }
  }
  l.coefs = n;
  n = 1;
  if (res) l.res = n++;
  if (dy) l.dy = n++;
  if (ds) l.ds = n++;
  if (gate) l.gate = n++;
  l.tensors = n;
  return l;
}
// (GEN kernels keep a place for B1 whether there is one or not)
inline NgaBwdLayout nga_bwd_layout(const NgaParams& p, int es, bool csm, bool gen, bool direct) {
  return nga_layout(es, csm, gen, p.res != nullptr && p.dy != nullptr, p.dy != nullptr, p.ds != nullptr && !direct,
                    p.gate_mode == FLN_GATE_ELEMENT);
}
inline int nga_set_of(const NgaParams& p) {
  if (p.res != nullptr && p.dy != nullptr && p.ds != nullptr) return 1;
  if (p.dy == nullptr && p.ds != nullptr) return 2;
  return 0;
}

template <typename T, int K, int GATE, bool GEN, bool CSM, int TPR, bool RAG, int SET, bool SHIFT, bool PAIR = false>
__global__ void __launch_bounds__(K * 16 / (int)sizeof(T) <= 8 ? 640 : 512) nga_bwd_rows_kernel(const NgaParams p, const NgaGeom g) {
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int VEC = 16 / (int)sizeof(T), V2 = VEC / 2;
  extern __shared__ __align__(128) unsigned char smem[];
  constexpr bool DIRECT = SET == 3;
  const bool has_dy = SET == 1 || DIRECT || (SET == 0 && p.dy != nullptr);
  const bool has_ds = SET != 0 || p.ds != nullptr;
  const bool has_res = SET == 1 || DIRECT || (SET == 0 && has_dy && p.res != nullptr);
  const NgaBwdLayout l = nga_layout((int)sizeof(T), CSM, GEN, has_res, has_dy, has_ds && !DIRECT, GATE == 2);
  constexpr bool FULL = TPR != 0 && !RAG;
  const int tpr = TPR ? TPR : g.tpr;
  const int R = TPR ? fixed_rows(TPR) : g.R;
  const int threads = TPR ? TPR * fixed_rows(TPR) : g.threads;
  const int cols = FULL ? TPR * K * VEC : p.cols;
  constexpr bool ONE = PAIR || (TPR != 0 && fixed_rows(TPR ? TPR : 1) == 1);  // one row at a time: never behind the slot
  RowGroup rg = row_group<TPR, FULL>(g, K, VEC, g.nv, 0, cols, reinterpret_cast<float2*>(smem));
  const int tid = threadIdx.x;
  const int r_in = ONE ? 0 : tid / tpr, lane = tid - r_in * tpr;
  const float inv_n = 1.0f / (float)cols;
  const uint32_t unit = (uint32_t)K * threads * 16u;
  const uint32_t kstep = (uint32_t)threads * 16u;
  unsigned char* coefs = smem + kNgaBwdHeader + tid * 16;
  unsigned char* stages = coefs + (uint32_t)l.coefs * unit;
  const uint32_t stage_bytes = (uint32_t)l.tensors * unit;
  const uint32_t ring_bytes = (uint32_t)g.stages * stage_bytes;
  // Lanes behind the row work on its last vector, row groups behind the slot on its last row; what
  // goes into the sums is set to zero there and nothing is stored, so the arithmetic has no branches.
  const int rank = PAIR ? (int)cluster_ctarank() : 0;
  const int half = (g.nv + 1) / 2, v0 = rank * half, v1 = v0 + half;
  if (PAIR) {
    rg.rank = rank;
    cluster_sync_all();  // the other CTA is there before anything is written into its shared memory
  }
  Places<K, VEC, FULL, SHIFT> w;
  if (!SHIFT) w.set(lane, tpr, g.nv, cols, 0, PAIR, v0, v1);
  const int apart = SHIFT ? p.period : 1;  // from one row to the next

  // The row sequence of this CTA: slot after slot, R rows at a time; one walker runs ahead.
  struct Walker {
    int slot, row, last;  // row: of the CTA's first row group
  };
  const int nslots = (int)p.slots, grid = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;
  auto open = [&](Walker& w) {
    if (w.slot < nslots) {
      const SlotRows sr = slot_rows(p, w.slot);
      w.row = (int)sr.first;
      w.last = (int)sr.last;
    }
  };
  auto step = [&](Walker& w) {
    w.row += R * apart;
    if (w.row >= w.last) {
      w.slot += grid;
      open(w);
    }
  };
  auto my_row = [&](const Walker& w) { return ONE ? w.row : (w.row + r_in * apart < w.last ? w.row + r_in * apart : w.last - 1); };
  Walker ahead{PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x, 0, 0};
  open(ahead);
  Walker cur = ahead;
  uint32_t fill = 0;  // byte offset of the stage the walker fills next
  auto fetch = [&]() {
    if (ahead.slot < nslots) {
      unsigned char* st = stages + fill;
      const int64_t row_at = (int64_t)my_row(ahead) * cols;
      const bool there = ONE || ahead.row + r_in * apart < ahead.last;
      Places<K, VEC, FULL, SHIFT> wa = w;
      if (SHIFT) wa.set(lane, tpr, g.nv, cols, row_shift(ahead.row, cols, VEC), PAIR, v0, v1);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        unsigned char* d = st + k * kstep;
        const int64_t o = row_at + wa.at[k];
        const int64_t left = SHIFT ? (p.rows * cols - o) * (int)sizeof(T) : 16;
        const int bytes = left < 16 ? (int)left : 16;  // (the last vector of the last row may reach behind the tensor)
        auto bring = [&](unsigned char* to, const void* from) {
          if (SHIFT) cp_async16_part(to, reinterpret_cast<const T*>(from) + o, bytes);
          else cp_async16(to, reinterpret_cast<const T*>(from) + o);
        };
        // a row group behind the slot takes x as zeros: without a norm in front of it an infinity of the last
        // row would be multiplied by that group's ds of 0
        if (ONE) bring(d, p.x);
        else cp_async16_part(d, reinterpret_cast<const T*>(p.x) + o, there ? bytes : 0);
        if (has_res) bring(d + l.res * unit, p.res);
        if (has_dy) bring(d + l.dy * unit, p.dy);
        if (has_ds && !DIRECT) bring(d + l.ds * unit, p.ds);
        if (GATE == 2) bring(d + l.gate * unit, p.gate);
      }
      step(ahead);
    }
    cp_async_commit();  // a group per step, also an empty one, so that the count tells the row
    fill += stage_bytes;
    if (fill == ring_bytes) fill = 0;
  };
  for (int i = 0; i + 1 < g.stages; ++i) fetch();

  float2 acc_p[K][V2], acc_u[K][V2], acc_q[GEN ? K : 1][V2], acc_v[GEN ? K : 1][V2];
  auto clear = [&]() {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < V2; ++e) {
        acc_p[k][e] = f2(0.f);
        acc_u[k][e] = f2(0.f);
        if (GEN) {
          acc_q[GEN ? k : 0][e] = f2(0.f);
          acc_v[GEN ? k : 0][e] = f2(0.f);
        }
      }
  };
  clear();
  // the four scalars of a row, fetched one row ahead
  struct Scalars {
    float mean1, rstd1, mean2, rstd2;
  };
  auto scalars = [&](const Walker& w) {
    Scalars s{0.f, 1.f, 0.f, 1.f};
    if (w.slot < nslots) {
      const int row = my_row(w);
      if (p.post_kind != FLN_NO_NORM) s.rstd1 = __ldg(p.rstd1 + row);
      if (GEN && p.post_kind == FLN_LAYERNORM) s.mean1 = __ldg(p.mean1 + row);
      if (has_dy) s.rstd2 = __ldg(p.rstd2 + row);
      if (GEN && has_dy && p.kind == FLN_LAYERNORM) s.mean2 = __ldg(p.mean2 + row);
    }
    return s;
  };
  Scalars sc_next = scalars(cur);
  int64_t group = -1, goff = 0, aoff = 0;
  uint32_t drain = 0;  // byte offset of the stage in hand
  bool opened = true;  // cur has come to a new slot
  const float2 ra = f2(p.ra);
  auto coef = [&](int piece, int k, float2 (&v)[V2]) {
#pragma unroll
    for (int e = 0; e < V2; e += 2) {
      const float4 q = *reinterpret_cast<const float4*>(coefs + (uint32_t)(piece + e / 2) * unit + k * kstep);
      v[e] = make_float2(q.x, q.y);
      v[e + 1] = make_float2(q.z, q.w);
    }
  };
  // C1 and (GEN) B1
  auto first_coefs = [&](int k, float2 (&c)[V2], float2 (&b)[V2]) {
    if (CSM) {
      coef(l.c1, k, c);
      if (GEN) coef(l.b1, k, b);
    } else {
      coef1<T, GATE, SHIFT>(p, w.at[k], goff, c, b);
    }
  };
  while (cur.slot < nslots) {
    if (opened) {
      const int64_t grp = cur.slot / p.slots_per_group;
      if (SHIFT) w.set(lane, tpr, g.nv, cols, row_shift(cur.row, cols, VEC), PAIR, v0, v1);
      if (SHIFT || grp != group) {  // coefficients of a new group, or for another place of the row
        const bool first = SHIFT || group < 0;
        group = grp;
        goff = p.gate_mode == FLN_GATE_GROUP ? grp * cols : 0;
        aoff = p.affine_grouped ? grp * cols : 0;
        if (CSM) {
#pragma unroll
          for (int k = 0; k < K; ++k) {
            float2 c[V2], b[V2];
            auto put = [&](int piece, const float2 (&v)[V2]) {
#pragma unroll
              for (int e = 0; e < V2; e += 2)
                *reinterpret_cast<float4*>(coefs + (uint32_t)(piece + e / 2) * unit + k * kstep) =
                    make_float4(v[e].x, v[e].y, v[e + 1].x, v[e + 1].y);
            };
            if (first || p.gate_mode == FLN_GATE_GROUP) {
              coef1<T, GATE, SHIFT>(p, w.at[k], goff, c, b);
              put(l.c1, c);
              if (GEN) put(l.b1, b);
            }
            if (has_dy && (first || p.affine_grouped)) {
              coef2<T, SHIFT, false>(p, w.at[k], aoff, c, b);
              put(l.c2, c);
            }
          }
        }
      }
    }
    fetch();
    const int slot = cur.slot;
    const int slot_shift = SHIFT ? row_shift(cur.row, cols, VEC) : 0;
    const bool live = ONE || cur.row + r_in * apart < cur.last;
    const int64_t base = (int64_t)my_row(cur) * cols;
    const Scalars sc = sc_next;
    step(cur);
    opened = cur.slot != slot;
    sc_next = scalars(cur);
    cp_async_wait_behind(g.stages - 1);
    const unsigned char* st = stages + drain;
    drain += stage_bytes;
    if (drain == ring_bytes) drain = 0;

    Pack<T, VEC> ds_now[DIRECT ? K : 1];
    if (DIRECT) {  // used behind the first row sum
#pragma unroll
      for (int k = 0; k < K; ++k) ds_now[DIRECT ? k : 0] = ld_stream<T, VEC>(reinterpret_cast<const T*>(p.ds) + base + w.at[k]);
    }
    float2 xh[K][V2], sh[K][V2], g2[K][V2];
    float2 r0 = f2(0.f), r1 = f2(0.f);
    {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const unsigned char* d = st + k * kstep;
        take<T>(d, xh[k]);
        w.trim(k, xh[k]);
#pragma unroll
        for (int e = 0; e < V2; ++e) {
          if (GEN) xh[k][e] = f2add(xh[k][e], f2(-sc.mean1));
          xh[k][e] = f2mul(xh[k][e], f2(sc.rstd1));
        }
        if (has_dy) {
          float2 c[V2], b[V2];
          first_coefs(k, c, b);
#pragma unroll
          for (int e = 0; e < V2; ++e) sh[k][e] = GEN ? f2fma(xh[k][e], c[e], b[e]) : f2mul(xh[k][e], c[e]);
          if (GATE == 2) {
            take<T>(d + l.gate * unit, c);
            if (!GEN) gate_act_all<EXACT>(c, p.act);
#pragma unroll
            for (int e = 0; e < V2; ++e) {
              if (GEN) c[e] = make_float2(gate_act<EXACT>(c[e].x, p.act), gate_act<EXACT>(c[e].y, p.act));
              sh[k][e] = f2mul(sh[k][e], c[e]);
            }
          }
          if (has_res) {
            take<T>(d + l.res * unit, c);
#pragma unroll
            for (int e = 0; e < V2; ++e) sh[k][e] = f2fma(c[e], ra, sh[k][e]);
          }
          w.trim(k, sh[k]);
          take<T>(d + l.dy * unit, g2[k]);
          w.trim(k, g2[k]);
          if (!(FULL && ONE)) {
#pragma unroll
            for (int e = 0; e < V2; ++e) g2[k][e] = f2only(live && w.ok[k], g2[k][e]);
          }
          if (CSM) coef(l.c2, k, c);
          else coef2<T, SHIFT, false>(p, w.at[k], aoff, c, b);
#pragma unroll
          for (int e = 0; e < V2; ++e) {
            if (GEN) sh[k][e] = f2add(sh[k][e], f2(-sc.mean2));
            sh[k][e] = f2mul(sh[k][e], f2(sc.rstd2));
            acc_u[k][e] = f2fma(g2[k][e], sh[k][e], acc_u[k][e]);
            if (GEN) acc_v[GEN ? k : 0][e] = f2add(acc_v[GEN ? k : 0][e], g2[k][e]);
            g2[k][e] = f2mul(g2[k][e], c[e]);
            r0 = f2fma(g2[k][e], sh[k][e], r0);
            if (GEN) r1 = f2add(r1, g2[k][e]);
          }
        }
      }
    }
    float c1 = 0.f, c2 = 0.f;
    if (has_dy) {
      float a = r0.x + r0.y, b = r1.x + r1.y;
      if (GEN) row_sum2<PAIR>(rg, a, b);
      else row_sum1<PAIR>(rg, a);
      c1 = a * inv_n;
      c2 = GEN && p.kind == FLN_LAYERNORM ? b * inv_n : 0.f;
    }
    r0 = f2(0.f);
    r1 = f2(0.f);
    {
      T* dres = reinterpret_cast<T*>(p.dres) + base;
      T* dgate = reinterpret_cast<T*>(p.dgate) + base;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const bool ok = live && w.ok[k];
        const unsigned char* st_k = st + k * kstep;
        float2 d[V2], c[V2], b[V2];
        if (DIRECT) {
          unpack2<T, VEC>(ds_now[DIRECT ? k : 0], d);
        } else if (has_ds) {
          take<T>(st_k + l.ds * unit, d);
        } else {
#pragma unroll
          for (int e = 0; e < V2; ++e) d[e] = f2(0.f);
        }
        if (has_dy) {
#pragma unroll
          for (int e = 0; e < V2; ++e) {
            const float2 q = f2fma(sh[k][e], f2(-c1), GEN ? f2add(g2[k][e], f2(-c2)) : g2[k][e]);
            d[e] = f2fma(q, f2(sc.rstd2), d[e]);
          }
        }
        if (!(FULL && ONE)) {
#pragma unroll
          for (int e = 0; e < V2; ++e) d[e] = f2only(ok, d[e]);
          w.trim(k, d);
        }
        if (p.dres != nullptr) {
#pragma unroll
          for (int e = 0; e < V2; ++e) c[e] = f2mul(d[e], ra);
          if (ok) give_row<T, K, FULL, SHIFT>(dres, w, k, c);
        }
        first_coefs(k, c, b);
        if (GATE == 2) {
          float2 gv[V2];
          take<T>(st_k + l.gate * unit, gv);
          w.trim(k, gv);
          if (p.dgate != nullptr) {
            float2 o[V2];
            if (!GEN) gate_act_grad_all<EXACT>(gv, o, p.act);
#pragma unroll
            for (int e = 0; e < V2; ++e) {
              if (GEN) {
                const float2 v = gv[e];
                gate_act_grad<EXACT>(v.x, p.act, &gv[e].x, &o[e].x);
                gate_act_grad<EXACT>(v.y, p.act, &gv[e].y, &o[e].y);
              }
              const float2 n = GEN ? f2fma(xh[k][e], c[e], b[e]) : f2mul(xh[k][e], c[e]);
              o[e] = f2mul(f2mul(d[e], n), o[e]);
              d[e] = f2mul(d[e], gv[e]);
            }
            if (ok) give_row<T, K, FULL, SHIFT>(dgate, w, k, o);
          } else {
            if (!GEN) gate_act_all<EXACT>(gv, p.act);
#pragma unroll
            for (int e = 0; e < V2; ++e) {
              if (GEN) gv[e] = make_float2(gate_act<EXACT>(gv[e].x, p.act), gate_act<EXACT>(gv[e].y, p.act));
              d[e] = f2mul(d[e], gv[e]);
            }
          }
        }
#pragma unroll
        for (int e = 0; e < V2; ++e) {
          acc_p[k][e] = f2fma(d[e], xh[k][e], acc_p[k][e]);
          if (GEN) acc_q[GEN ? k : 0][e] = f2add(acc_q[GEN ? k : 0][e], d[e]);
          g2[k][e] = f2mul(d[e], c[e]);  // g1 from here on
          r0 = f2fma(g2[k][e], xh[k][e], r0);
          if (GEN) r1 = f2add(r1, g2[k][e]);
        }
      }
    }
    if (p.dx != nullptr) {
      float d1 = 0.f, d2 = 0.f;
      if (p.post_kind != FLN_NO_NORM) {
        float a = r0.x + r0.y, b = r1.x + r1.y;
        if (GEN) row_sum2<PAIR>(rg, a, b);
        else row_sum1<PAIR>(rg, a);
        d1 = a * inv_n;
        d2 = GEN && p.post_kind == FLN_LAYERNORM ? b * inv_n : 0.f;
      }
      {
        T* dx = reinterpret_cast<T*>(p.dx) + base;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (p.post_kind != FLN_NO_NORM) {
#pragma unroll
            for (int e = 0; e < V2; ++e) {
              const float2 q = f2fma(xh[k][e], f2(-d1), GEN ? f2add(g2[k][e], f2(-d2)) : g2[k][e]);
              g2[k][e] = f2mul(q, f2(sc.rstd1));
            }
          }
          if (live && w.ok[k]) give_row<T, K, FULL, SHIFT>(dx, w, k, g2[k]);
        }
      }
    }
    if (opened) {
      // the slot's sums; several row groups are joined in the CTA first, in their order
      if (p.acc != 0) {
        const int who = tpr < 32 ? tid >> 5 : r_in;
        float* out = p.partials + (int64_t)slot * p.nacc * cols;
        float* joint = reinterpret_cast<float*>(smem + kNgaBwdHeader + (uint32_t)l.coefs * unit + ring_bytes);
        auto leave = [&](float2 (&acc)[K][V2], int which, float scale) {
          if (!(p.acc & which)) return;
          float* dst = out + (int64_t)__popc(p.acc & (which - 1)) * cols;
#pragma unroll
          for (int k = 0; k < K; ++k) {
            for (int off = 16; off >= tpr; off >>= 1) {
#pragma unroll
              for (int e = 0; e < V2; ++e) {
                acc[k][e].x += __shfl_xor_sync(0xffffffffu, acc[k][e].x, off);
                acc[k][e].y += __shfl_xor_sync(0xffffffffu, acc[k][e].y, off);
              }
            }
            const bool mine = w.ok[k] && (tpr >= 32 || (tid & 31) < tpr);
            const bool join = !ONE && g.rep > 1;
            float* q = join ? joint + (who * tpr + lane) * VEC : dst + w.at[k];
            if (SHIFT && !join) {
              if (mine) {
#pragma unroll
                for (int e = 0; e < V2; ++e) {
                  const int lo = w.lo[SHIFT ? k : 0], hi = w.hi[SHIFT ? k : 0];
                  if (2 * e >= lo && 2 * e < hi) q[2 * e] = acc[k][e].x * scale;
                  if (2 * e + 1 >= lo && 2 * e + 1 < hi) q[2 * e + 1] = acc[k][e].y * scale;
                }
              }
            } else if (mine || join) {
#pragma unroll
              for (int e = 0; e < V2; e += 2)
                *reinterpret_cast<float4*>(q + 2 * e) =
                    make_float4(acc[k][e].x * scale, acc[k][e].y * scale, acc[k][e + 1].x * scale, acc[k][e + 1].y * scale);
            }
            if (join) {
              __syncthreads();
              for (int i = tid; i < tpr * VEC; i += threads) {
                float v = 0.f;
                for (int r = 0; r < g.rep; ++r) v += joint[r * tpr * VEC + i];
                const int c = k * tpr * VEC + i - (SHIFT ? slot_shift : 0);
                if (c >= 0 && c < cols) dst[c] = v;
              }
              __syncthreads();
            }
          }
        };
        leave(acc_p, kAccP, p.ba);
        leave(acc_u, kAccU, 1.f);
        if constexpr (GEN) {
          leave(acc_q, kAccQ, p.ba);
          leave(acc_v, kAccV, 1.f);
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
inline bool nga_general(const NgaParams& p) {
  return p.post_kind == FLN_LAYERNORM || p.kind == FLN_LAYERNORM || p.b1 != nullptr || p.b2 != nullptr ||
         (p.acc & (kAccQ | kAccV)) != 0;
}

// clusters of two CTAs
template <auto KERN>
static int nga_launch_pair(const NgaParams& p, const NgaGeom& g, cudaStream_t st) {
  if (!allow_smem<KERN>(g.smem)) return FLN_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)g.grid);
  cfg.blockDim = dim3((unsigned)g.threads);
  cfg.dynamicSmemBytes = g.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, KERN, p, g) != cudaSuccess) {
    cudaGetLastError();
    return FLN_ERR_LAUNCH;
  }
  FLN_CHECK_LAUNCH();
  return FLN_OK;
}
template <auto KERN>
static int nga_launch(const NgaParams& p, const NgaGeom& g, cudaStream_t st) {
  if (!allow_smem<KERN>(g.smem)) return FLN_ERR_LAUNCH;
  KERN<<<(unsigned)g.grid, g.threads, g.smem, st>>>(p, g);
  FLN_CHECK_LAUNCH();
  return FLN_OK;
}
template <typename T, int K, int GATE, int TPR, bool RAG, bool SHIFT = false>
static int nga_fwd_rows_t(const NgaParams& p, const NgaGeom& g, cudaStream_t st) {
  constexpr bool HOLD = K * 16 / (int)sizeof(T) <= 16;
  return nga_general(p) ? nga_launch<nga_fwd_rows_kernel<T, K, GATE, true, HOLD, TPR, RAG, SHIFT>>(p, g, st)
                        : nga_launch<nga_fwd_rows_kernel<T, K, GATE, false, HOLD, TPR, RAG, SHIFT>>(p, g, st);
}
template <typename T, int K, int GATE>
static int nga_fwd_rows_k(const NgaParams& p, const NgaGeom& g, cudaStream_t st) {
  if (p.period > 1) return nga_fwd_rows_t<T, K, GATE, 0, false, true>(p, g, st);
  // compile-time rows: 16 elements per thread
  if constexpr (K * 16 / (int)sizeof(T) == 16) {
    const bool whole = g.nv == K * g.tpr;
#define FLN_NGA_SHORT(TPR) \
  case TPR:                \
    if (whole) return nga_fwd_rows_t<T, K, GATE, TPR, false>(p, g, st); \
    break;
#define FLN_NGA_RAG(TPR) \
  case TPR:              \
    return nga_fwd_rows_t<T, K, GATE, TPR, true>(p, g, st);
#define FLN_NGA_LONG(TPR) \
  case TPR:               \
    return whole ? nga_fwd_rows_t<T, K, GATE, TPR, false>(p, g, st) : nga_fwd_rows_t<T, K, GATE, TPR, true>(p, g, st);
    switch (g.tpr) {
      FLN_NGA_SHORT(4)
      FLN_NGA_SHORT(8)
      FLN_NGA_SHORT(16)
      FLN_NGA_SHORT(32)
      FLN_NGA_SHORT(64)
      FLN_NGA_LONG(128)
      FLN_NGA_RAG(192)
      FLN_NGA_LONG(256)
      FLN_NGA_LONG(320)
      FLN_NGA_RAG(384)
      FLN_NGA_LONG(512)
    }
#undef FLN_NGA_RAG
#undef FLN_NGA_SHORT
#undef FLN_NGA_LONG
  }
  return nga_fwd_rows_t<T, K, GATE, 0, false>(p, g, st);
}
template <typename T, int K, int GATE, bool GEN>
static int nga_bwd_rows_g(const NgaParams& p, const NgaGeom& g, cudaStream_t st) {
  if (g.pair) {
    if constexpr (K * 16 / (int)sizeof(T) == 16) {
      if (p.period > 1)
        return g.csm ? nga_launch_pair<nga_bwd_rows_kernel<T, K, GATE, GEN, true, 0, false, 0, true, true>>(p, g, st)
                     : nga_launch_pair<nga_bwd_rows_kernel<T, K, GATE, GEN, false, 0, false, 0, true, true>>(p, g, st);
      return g.csm ? nga_launch_pair<nga_bwd_rows_kernel<T, K, GATE, GEN, true, 0, false, 0, false, true>>(p, g, st)
                   : nga_launch_pair<nga_bwd_rows_kernel<T, K, GATE, GEN, false, 0, false, 0, false, true>>(p, g, st);
    }
    return FLN_ERR_UNSUPPORTED;
  }
  if (p.period > 1) {
    if (!g.csm) return nga_launch<nga_bwd_rows_kernel<T, K, GATE, GEN, false, 0, false, 0, true>>(p, g, st);
    return nga_set_of(p) == 1 ? nga_launch<nga_bwd_rows_kernel<T, K, GATE, GEN, true, 0, false, 1, true>>(p, g, st)
                              : nga_launch<nga_bwd_rows_kernel<T, K, GATE, GEN, true, 0, false, 0, true>>(p, g, st);
  }
  const bool whole = g.nv == K * g.tpr;
  if (g.direct) {
    // (640 threads come here in fp32 with a gate per element.  General form, 2047 rows of 4864 / 5056: 101 /
    // 103 us with the threads found out at run time, 87 / 87 so; without means and biases 4096 rows of 4864
    // take 118 us at run time, 134 so)
    if constexpr (sizeof(T) == 4 && K * 16 / (int)sizeof(T) == 8 && GATE == 2 && GEN) {
      if (g.csm && g.tpr == 640) return nga_launch<nga_bwd_rows_kernel<T, K, GATE, GEN, true, 640, true, 3, false>>(p, g, st);
    }
    return g.csm ? nga_launch<nga_bwd_rows_kernel<T, K, GATE, GEN, true, 0, false, 3, false>>(p, g, st)
                 : nga_launch<nga_bwd_rows_kernel<T, K, GATE, GEN, false, 0, false, 3, false>>(p, g, st);
  }
  if (!g.csm) return nga_launch<nga_bwd_rows_kernel<T, K, GATE, GEN, false, 0, false, 0, false>>(p, g, st);
  const int set = nga_set_of(p);
  // compile-time rows where the registers allow: 16 elements per thread, 8 of the general form and of fp32
  if constexpr (K * 16 / (int)sizeof(T) == (GEN || sizeof(T) == 4 ? 8 : 16)) {
#define FLN_NGA_SHORT(TPR, SET) \
  case TPR:                     \
    if (whole) return nga_launch<nga_bwd_rows_kernel<T, K, GATE, GEN, true, TPR, false, SET, false>>(p, g, st); \
    break;
#define FLN_NGA_RAG(TPR) \
  case TPR:              \
    return nga_launch<nga_bwd_rows_kernel<T, K, GATE, GEN, true, TPR, true, 1, false>>(p, g, st);
#define FLN_NGA_LONG(TPR)                                                                                          \
  case TPR:                                                                                                        \
    return whole ? nga_launch<nga_bwd_rows_kernel<T, K, GATE, GEN, true, TPR, false, 1, false>>(p, g, st)          \
                 : nga_launch<nga_bwd_rows_kernel<T, K, GATE, GEN, true, TPR, true, 1, false>>(p, g, st);
    if (set == 1) {
      switch (g.tpr) {
        FLN_NGA_SHORT(64, 1)
        FLN_NGA_LONG(128)
        FLN_NGA_RAG(192)
        FLN_NGA_LONG(256)
        FLN_NGA_LONG(320)
        FLN_NGA_RAG(384)
        FLN_NGA_LONG(512)
      }
      if constexpr (K * 16 / (int)sizeof(T) == 8) {  // (what 640 threads have the registers for)
        switch (g.tpr) { FLN_NGA_LONG(640) }
      }
    }
    if (set == 2) {
      switch (g.tpr) {
        FLN_NGA_SHORT(4, 2)
        FLN_NGA_SHORT(8, 2)
        FLN_NGA_SHORT(16, 2)
        FLN_NGA_SHORT(32, 2)
        FLN_NGA_SHORT(64, 2)
      }
    }
#undef FLN_NGA_RAG
#undef FLN_NGA_SHORT
#undef FLN_NGA_LONG
  }
  if (set == 1) return nga_launch<nga_bwd_rows_kernel<T, K, GATE, GEN, true, 0, false, 1, false>>(p, g, st);
  return nga_launch<nga_bwd_rows_kernel<T, K, GATE, GEN, true, 0, false, 0, false>>(p, g, st);
}
template <typename T, int K, int GATE>
static int nga_bwd_rows_k(const NgaParams& p, const NgaGeom& g, cudaStream_t st) {
  return nga_general(p) ? nga_bwd_rows_g<T, K, GATE, true>(p, g, st) : nga_bwd_rows_g<T, K, GATE, false>(p, g, st);
}

#define FLN_NGA_GATES(F, T, K)              \
  switch (nga_gate_of(p)) {                 \
    case 0:                                 \
      return F<T, K, 0>(p, g, st);          \
    case 1:                                 \
      return F<T, K, 1>(p, g, st);          \
    default:                                \
      return F<T, K, 2>(p, g, st);          \
  }
// vectors per thread: 8, 16 or (forward) 32 elements
#define FLN_NGA_INSTANTIATE(T)                                                                       \
  template <>                                                                                        \
  int nga_fwd_rows<T>(const NgaParams& p, const NgaGeom& g, int K, cudaStream_t st) {                \
    constexpr int K8 = (int)sizeof(T) / 2;                                                           \
    if (K == K8) FLN_NGA_GATES(nga_fwd_rows_k, T, K8)                                                \
    if (K == 2 * K8) FLN_NGA_GATES(nga_fwd_rows_k, T, 2 * K8)                                        \
    if (K == 4 * K8) FLN_NGA_GATES(nga_fwd_rows_k, T, 4 * K8)                                        \
    return FLN_ERR_UNSUPPORTED;                                                                      \
  }                                                                                                  \
  template <>                                                                                        \
  int nga_bwd_rows<T>(const NgaParams& p, const NgaGeom& g, int K, cudaStream_t st) {                \
    constexpr int K8 = (int)sizeof(T) / 2;                                                           \
    if (K == K8) FLN_NGA_GATES(nga_bwd_rows_k, T, K8)                                                \
    if (K == 2 * K8) FLN_NGA_GATES(nga_bwd_rows_k, T, 2 * K8)                                        \
    return FLN_ERR_UNSUPPORTED;                                                                      \
  }

}  // namespace fln
