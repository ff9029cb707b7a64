// fln_qk_norm_rotary: entry points, launch plan, and the sum of the weight gradients' partial
// rows.  The kernels stand in fln_rotary.cuh.
#include "fln_rotary.cuh"

namespace fln {

constexpr int kRotMaxDim = 512;

// explicit instantiations live in fln_rotary_{f32,bf16,f16}.cu
template <>
int rotary_launch<float>(const RotParams&, const RotPlan&, bool, unsigned, cudaStream_t);
template <>
int rotary_launch<__nv_bfloat16>(const RotParams&, const RotPlan&, bool, unsigned, cudaStream_t);
template <>
int rotary_launch<__half>(const RotParams&, const RotPlan&, bool, unsigned, cudaStream_t);

// One CTA per 32 columns of one output row; 32 lanes take the partial rows in turn, the lanes are
// added in order.
constexpr int kRotFinalLanes = 32;
template <typename T>
__global__ void __launch_bounds__(32 * kRotFinalLanes) rotary_finalize_kernel(const float* p0, int n0, const float* p1, int n1, int dim,
                                                              T* dw0, T* db0, T* dw1, T* db1) {
  __shared__ float tile[kRotFinalLanes][33];
  const int which = blockIdx.y >> 1, bias = blockIdx.y & 1;
  T* out = which == 0 ? (bias ? db0 : dw0) : (bias ? db1 : dw1);
  if (out == nullptr) return;
  const float* src = which == 0 ? p0 : p1;
  const int n = which == 0 ? n0 : n1;
  const int tx = threadIdx.x & 31, lane = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  float v = 0.f;
  if (c < dim) {
    const float* s = src + bias * dim + c;
    for (int r = lane; r < n; r += 4 * kRotFinalLanes) {
      float q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = r + j * kRotFinalLanes < n ? __ldcg(s + (int64_t)(r + j * kRotFinalLanes) * 2 * dim) : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) v += q[j];
    }
  }
  tile[lane][tx] = v;
  __syncthreads();
  if (lane == 0 && c < dim) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < kRotFinalLanes; ++i) v += tile[i][tx];
    out[c] = Cvt<T>::from_f(v);
  }
}

static int check(const fln_rotary_args* a) {
  if (a == nullptr) return FLN_ERR_NULL;
  if (a->dtype != FLN_F32 && a->dtype != FLN_BF16 && a->dtype != FLN_F16) return FLN_ERR_DTYPE;
  if (a->kind != FLN_LAYERNORM && a->kind != FLN_RMSNORM && a->kind != FLN_NO_NORM) return FLN_ERR_ARG;
  if (a->layout != FLN_ROTARY_HALF && a->layout != FLN_ROTARY_INTERLEAVED) return FLN_ERR_ARG;
  if (a->batch < 0 || a->seq < 0) return FLN_ERR_SHAPE;
  if (a->batch > 0x7fffffff || a->seq > 0x7fffffff || a->batch * a->seq > 0x7fffffff) return FLN_ERR_SHAPE;
  if (a->head_dim <= 0 || a->pairs < 0 || a->pairs > a->head_dim / 2) return FLN_ERR_SHAPE;
  if (a->head_dim > kRotMaxDim) return FLN_ERR_UNSUPPORTED;
  if (a->t[0].heads < 0 || a->t[1].heads < 0 || a->t[0].heads > (1 << 20) || a->t[1].heads > (1 << 20)) return FLN_ERR_SHAPE;
  if (a->kind == FLN_NO_NORM &&
      (a->t[0].weight != nullptr || a->t[0].bias != nullptr || a->t[1].weight != nullptr || a->t[1].bias != nullptr))
    return FLN_ERR_ARG;
  return FLN_OK;
}

static bool empty(const fln_rotary_args* a) {
  return a->batch == 0 || a->seq == 0 || (a->t[0].heads == 0 && a->t[1].heads == 0);
}

static int check_pointers(const fln_rotary_args* a) {
  for (int i = 0; i < 2; ++i)
    if (a->t[i].heads > 0 && (a->t[i].in == nullptr || a->t[i].out == nullptr)) return FLN_ERR_NULL;
  if (a->pairs > 0 && (a->positions == nullptr || a->turns == nullptr || a->axis == nullptr)) return FLN_ERR_NULL;
  return FLN_OK;
}

// The longest vector (16 bytes at most) that divides the row, its rotated half and every stride,
// and that all addresses are multiples of; then the fewest units per lane of 1, 3 and 8 that let
// 32 lanes hold the row.
static RotPlan make_rot_plan(const fln_rotary_args* a, void* const* dx, RotParams* p) {
  const int es = a->dtype == FLN_F32 ? 4 : 2;
  int V = 16 / es;
  auto fits = [&](int v) {
    if (a->head_dim % v != 0 || a->pairs % v != 0) return false;
    const int64_t bytes = (int64_t)v * es;
    for (int i = 0; i < 2; ++i) {
      const fln_rotary_tensor& t = a->t[i];
      if (t.heads == 0) continue;
      const void* ptrs[] = {t.in, t.out, t.weight, t.bias, dx != nullptr ? dx[i] : nullptr};
      for (const void* q : ptrs)
        if (reinterpret_cast<uintptr_t>(q) % bytes != 0) return false;
      // a dimension of size one may have any stride: it is never stepped along
      if ((a->batch > 1 && (t.in_batch % v != 0 || t.out_batch % v != 0)) ||
          (a->seq > 1 && (t.in_seq % v != 0 || t.out_seq % v != 0)) ||
          (t.heads > 1 && (t.in_head % v != 0 || t.out_head % v != 0)))
        return false;
    }
    return true;
  };
  while (V > 1 && !fits(V)) V >>= 1;
  RotPlan plan;
  plan.V = V;
  plan.half = a->layout == FLN_ROTARY_HALF;
  p->rot_units = a->pairs / V;
  p->units = p->rot_units + (a->head_dim - 2 * a->pairs + 2 * V - 1) / (2 * V);
  // Three units on each of a few lanes where that leaves fewer lanes idle (9 units: 3 of 4 lanes x
  // 3 units instead of 9 of 16 lanes), eight where the row needs them.
  auto lanes = [&](int u) {
    int l = 1;
    while (l * u < p->units) l <<= 1;
    return l;
  };
  plan.U = 1;
  if (lanes(1) > 32 || (V <= 4 && lanes(3) * 3 * 5 < lanes(1) * 4)) plan.U = 3;
  if (lanes(plan.U) > 32) plan.U = 8;
  int l = lanes(plan.U), lg = 0;
  while ((1 << lg) < l) ++lg;
  p->log2_l = lg;
  return plan;
}

static RotParams base_params(const fln_rotary_args* a) {
  RotParams p = {};
  for (int i = 0; i < 2; ++i) {
    const fln_rotary_tensor& s = a->t[i];
    RotTensor& t = p.t[i];
    t.in = s.in;
    t.out = s.out;
    t.in_batch = s.in_batch;
    t.in_seq = s.in_seq;
    t.in_head = s.in_head;
    t.out_batch = s.out_batch;
    t.out_seq = s.out_seq;
    t.out_head = s.out_head;
    t.weight = s.weight;
    t.bias = s.bias;
    t.heads = s.heads;
  }
  p.positions = a->positions;
  p.pos_axis = a->pos_axis;
  p.pos_batch = a->pos_batch;
  p.pos_seq = a->pos_seq;
  p.turns = reinterpret_cast<const unsigned long long*>(a->turns);
  p.axis = a->axis;
  p.tokens = (int)(a->batch * a->seq);
  p.seq = (int)a->seq;
  p.dim = a->head_dim;
  p.pairs = a->pairs;
  p.pos64 = a->pos64;
  p.kind = a->kind;
  p.woff = a->weight_offset;
  p.eps = a->eps;
  p.mag = a->magnitude;
  return p;
}

static int launch(int dtype, const RotParams& p, const RotPlan& plan, bool backward, unsigned grid, cudaStream_t st) {
  switch (dtype) {
    case FLN_F32:
      return rotary_launch<float>(p, plan, backward, grid, st);
    case FLN_BF16:
      return rotary_launch<__nv_bfloat16>(p, plan, backward, grid, st);
    default:
      return rotary_launch<__half>(p, plan, backward, grid, st);
  }
}

constexpr int kRotBwdCtasPerSm = 2;

// CTAs of the backward for q and for k: in proportion to their heads, at least one for a tensor
// that has any, and not more than one per eight rows
static void bwd_grid(const fln_rotary_args* a, int* n0, int* n1) {
  const int h0 = a->t[0].heads, h1 = a->t[1].heads;
  int64_t most = (a->batch * a->seq * (h0 + h1) + 7) / 8;
  if (most < 2) most = 2;
  int all = sm_count() * kRotBwdCtasPerSm;
  if (all > most) all = (int)most;
  int q = (int)((int64_t)all * h0 / (h0 + h1));
  if (h0 > 0 && q < 1) q = 1;
  if (h1 > 0 && q > all - 1) q = all - 1;
  if (h0 == 0) q = 0;
  *n0 = q;
  *n1 = h1 > 0 ? all - q : 0;
}

}  // namespace fln

using namespace fln;

extern "C" int fln_qk_norm_rotary_forward(const fln_rotary_args* a, void* stream) {
  int rc = check(a);
  if (rc != FLN_OK) return rc;
  if (empty(a)) return FLN_OK;
  rc = check_pointers(a);
  if (rc != FLN_OK) return rc;
  for (const fln_rotary_tensor& t : a->t) {  // in place: every row is read by the warp that writes it
    if (t.heads > 0 && t.in == t.out &&
        ((a->batch > 1 && t.in_batch != t.out_batch) || (a->seq > 1 && t.in_seq != t.out_seq) ||
         (t.heads > 1 && t.in_head != t.out_head)))
      return FLN_ERR_ARG;
  }
  RotParams p = base_params(a);
  const RotPlan plan = make_rot_plan(a, nullptr, &p);
  return launch(a->dtype, p, plan, false, 0, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t fln_qk_norm_rotary_workspace_bytes(const fln_rotary_args* a) {
  if (check(a) != FLN_OK || empty(a)) return 0;
  return (size_t)sm_count() * kRotBwdCtasPerSm * 2 * (size_t)a->head_dim * sizeof(float);
}

extern "C" int fln_qk_norm_rotary_backward(const fln_rotary_args* a, void* const dx[2], void* const dweight[2],
                                           void* const dbias[2], void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(a);
  if (rc != FLN_OK) return rc;
  if (dx == nullptr || dweight == nullptr || dbias == nullptr) return FLN_ERR_NULL;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const size_t es = a->dtype == FLN_F32 ? 4 : 2;
  bool sums = false, want_db = false;
  for (int i = 0; i < 2; ++i) {
    if (a->kind == FLN_NO_NORM && (dweight[i] != nullptr || dbias[i] != nullptr)) return FLN_ERR_ARG;
    sums = sums || dweight[i] != nullptr || dbias[i] != nullptr;
    want_db = want_db || dbias[i] != nullptr;
    // a tensor without rows: its sums are zeros
    if (empty(a) || a->t[i].heads == 0) {
      void* const z[] = {dweight[i], dbias[i]};
      for (void* q : z)
        if (q != nullptr && cudaMemsetAsync(q, 0, es * (size_t)a->head_dim, st) != cudaSuccess) {
          cudaGetLastError();
          return FLN_ERR_LAUNCH;
        }
    }
  }
  if (empty(a)) return FLN_OK;
  rc = check_pointers(a);
  if (rc != FLN_OK) return rc;
  RotParams p = base_params(a);
  const RotPlan plan = make_rot_plan(a, dx, &p);
  int n0, n1;
  bwd_grid(a, &n0, &n1);
  p.nb0 = n0;
  p.want_db = want_db ? 1 : 0;
  if (sums) {
    if (workspace == nullptr || workspace_bytes < fln_qk_norm_rotary_workspace_bytes(a) || !is_aligned16(workspace))
      return FLN_ERR_WORKSPACE;
  }
  float* ws = reinterpret_cast<float*>(workspace);
  for (int i = 0; i < 2; ++i) {
    p.t[i].dx = dx[i];
    p.t[i].partials = (dweight[i] != nullptr || dbias[i] != nullptr) && p.t[i].heads > 0
                          ? ws + (i == 0 ? 0 : (int64_t)n0 * 2 * p.dim)
                          : nullptr;
  }
  rc = launch(a->dtype, p, plan, true, (unsigned)(n0 + n1), st);
  if (rc != FLN_OK || !sums) return rc;
  const dim3 grid((unsigned)((p.dim + 31) / 32), 4);
  auto own = [&](int i, void* q) { return p.t[i].heads > 0 ? q : nullptr; };
#define FLN_FIN(T)                                                                                                     \
  rotary_finalize_kernel<T><<<grid, 32 * kRotFinalLanes, 0, st>>>(p.t[0].partials, n0, p.t[1].partials, n1, p.dim,                     \
                                                  reinterpret_cast<T*>(own(0, dweight[0])),                            \
                                                  reinterpret_cast<T*>(own(0, dbias[0])),                              \
                                                  reinterpret_cast<T*>(own(1, dweight[1])),                            \
                                                  reinterpret_cast<T*>(own(1, dbias[1])))
  if (a->dtype == FLN_F32) FLN_FIN(float);
  else if (a->dtype == FLN_BF16) FLN_FIN(__nv_bfloat16);
  else FLN_FIN(__half);
#undef FLN_FIN
  FLN_CHECK_LAUNCH();
  return FLN_OK;
}
