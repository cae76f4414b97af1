// Low-rank products chosen per route, added onto a base, and their gradients.  With B = left[e],
// A = right[e] of a route's set e:
//   p = A x,  out = base + scale B p;   q = scale B^T grad,  dx = A^T q,
//   dA = sum q x^T,  dB = scale sum grad p^T
#include "switch_plan.cuh"

namespace keepvq {
namespace dense {

constexpr int LR_MAX_RANK = 128;

// inner[r, j] = factor * sum_k m[e][j or k][k or j] v[row, k]: one warp per (route, j).
template <bool ACROSS>
__global__ void __launch_bounds__(256) inner_kernel(const void* v, int64_t ld, int x_div, const void* m, int64_t depth, int rank, int dtype, Indices indices, int sets, int64_t routes, float factor, float* inner) {
  const int64_t i = blockIdx.x * 8ll + threadIdx.x / 32;
  if (i >= routes * rank) return;
  const int64_t r = i / rank, j = i - r * rank;
  const int e = indices.set_of(r, sets), lane = threadIdx.x % 32;
  float sum = 0.0f;
  if (e >= 0)
    for (int64_t k = lane; k < depth; k += 32)
      sum += load_as_float(v, dtype, r / x_div * ld + k) * load_as_float(m, dtype, ACROSS ? (e * depth + k) * rank + j : (e * rank + j) * depth + k);
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
  if (lane == 0) inner[i] = factor * sum;
}

// out[r, n] = base[r, n] + factor * sum_j inner[r, j] left[e][n][j]
__global__ void __launch_bounds__(256) outer_kernel(keepvq_switch_low_rank_args a, Indices indices, const float* inner) {
  const int64_t i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= a.routes * a.out_dim) return;
  const int64_t r = i / a.out_dim, n = i - r * a.out_dim;
  const int e = indices.set_of(r, static_cast<int>(a.sets));
  float sum = 0.0f;
  if (e >= 0)
    for (int64_t j = 0; j < a.rank; ++j) sum += inner[r * a.rank + j] * load_as_float(a.left, a.dtype, (e * a.out_dim + n) * a.rank + j);
  const float base = a.base ? load_as_float(a.base, a.out_dtype, r * a.base_ld + n) : 0.0f;
  store_from_float(a.out, a.out_dtype, r * a.out_ld + n, e < 0 ? base : base + a.scale * sum);
}

// dx[t, k] = sum over picks, j of q[r, j] right[e][j][k]
__global__ void __launch_bounds__(256) input_grad_kernel(keepvq_switch_low_rank_args a, Indices indices, const float* q) {
  const int64_t i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= a.routes / a.x_div * a.in_dim) return;
  const int64_t t = i / a.in_dim, k = i - t * a.in_dim;
  float sum = 0.0f;
  for (int64_t r = t * a.x_div; r < (t + 1) * a.x_div; ++r) {
    const int e = indices.set_of(r, static_cast<int>(a.sets));
    if (e < 0) continue;
    for (int64_t j = 0; j < a.rank; ++j) sum += q[r * a.rank + j] * load_as_float(a.right, a.dtype, (e * a.rank + j) * a.in_dim + k);
  }
  store_from_float(a.dx, a.dtype, i, sum);
}

// grad[e][wide][j] or [e][j][wide] = factor * sum over e's routes of inner[r, j] v[row, wide]
template <bool ACROSS>
__global__ void __launch_bounds__(256) factor_grad_kernel(const void* v, int64_t ld, int x_div, int64_t wide, int rank, int dtype, Plan plan, const float* inner, float factor, void* out) {
  const int64_t e = blockIdx.y, i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= wide * rank) return;
  const int64_t n = ACROSS ? i / rank : i % wide, j = ACROSS ? i % rank : i / wide;
  float sum = 0.0f;
  for (int p = plan.offset[e]; p < plan.offset[e] + plan.count[e]; ++p) {
    const int64_t r = plan.order[p];
    sum += inner[r * rank + j] * load_as_float(v, dtype, r / x_div * ld + n);
  }
  store_from_float(out, dtype, e * wide * rank + i, factor * sum);
}

struct LowRankLayout {
  Plan plan;
  float *inner, *back;  // [routes, rank]: A x, and scale B^T grad
  int64_t bytes;
};
static LowRankLayout lay_out_low_rank(void* base, int64_t routes, int64_t sets, int64_t rank, bool grads) {
  Scratch s{static_cast<char*>(base)};
  LowRankLayout l;
  l.plan = take_plan(s, routes, sets, 64);
  l.inner = s.take<float>(routes * rank);
  l.back = grads ? s.take<float>(routes * rank) : nullptr;
  l.bytes = s.used;
  return l;
}

static int check_low_rank_sizes(int64_t routes, int64_t sets, int64_t out_dim, int64_t in_dim, int64_t rank, int32_t x_div) {
  if (routes < 0 || sets <= 0 || out_dim <= 0 || in_dim <= 0 || rank <= 0 || x_div <= 0 || in_dim % 8 != 0 || rank % 8 != 0 || routes % x_div != 0) return KEEPVQ_ERR_SHAPE;
  if (rank > LR_MAX_RANK) return KEEPVQ_ERR_UNSUPPORTED;
  if (routes > MAX_ROUTES || sets > MAX_SETS || out_dim > (1 << 24) || in_dim > (1 << 24)) return KEEPVQ_ERR_CAPACITY;
  return KEEPVQ_OK;
}

static int check_low_rank(const keepvq_switch_low_rank_args& a, bool grads) {
  if (!valid_16bit(a.dtype) || (a.index_bits != 32 && a.index_bits != 64) || (!grads && a.out_dtype != a.dtype && a.out_dtype != KEEPVQ_F32)) return KEEPVQ_ERR_DTYPE;
  if (const int rc = check_low_rank_sizes(a.routes, a.sets, a.out_dim, a.in_dim, a.rank, a.x_div)) return rc;
  if (grads ? a.grad_ld < a.out_dim || a.grad_ld % 8 != 0 : a.out_ld < a.out_dim || (a.base && a.base_ld < a.out_dim)) return KEEPVQ_ERR_SHAPE;
  if (!a.workspace || (a.routes > 0 && (!a.x || !a.left || !a.right || !a.indices || (grads ? !a.grad : !a.out)))) return KEEPVQ_ERR_NULL;
  for (const void* p : {a.x, a.left, a.right, a.grad, static_cast<const void*>(a.dx), static_cast<const void*>(a.dleft), static_cast<const void*>(a.dright)})
    if (!aligned_to(p, 16)) return KEEPVQ_ERR_ALIGN;
  if (!aligned_to(a.workspace, 256) || !aligned_to(a.indices, a.index_bits / 8) || !aligned_to(a.base, dtype_size(a.out_dtype)) || !aligned_to(a.out, dtype_size(a.out_dtype))) return KEEPVQ_ERR_ALIGN;
  return KEEPVQ_OK;
}

static unsigned blocks_of(int64_t n, int64_t per) { return static_cast<unsigned>((n + per - 1) / per); }

}  // namespace dense
}  // namespace keepvq

extern "C" {

int64_t keepvq_switch_low_rank_workspace_bytes(int64_t routes, int64_t sets, int64_t out_dim, int64_t in_dim, int64_t rank, int32_t x_div, int32_t grads) {
  using namespace keepvq::dense;
  if (const int rc = check_low_rank_sizes(routes, sets, out_dim, in_dim, rank, x_div)) return rc;
  return lay_out_low_rank(nullptr, routes, sets, rank, grads != 0).bytes;
}

int keepvq_switch_low_rank(const keepvq_switch_low_rank_args* args, void* stream) {
  using namespace keepvq::dense;
  if (!args) return KEEPVQ_ERR_NULL;
  const keepvq_switch_low_rank_args& a = *args;
  if (const int rc = check_low_rank(a, false)) return rc;
  const LowRankLayout l = lay_out_low_rank(a.workspace, a.routes, a.sets, a.rank, false);
  if (l.bytes > a.workspace_bytes) return KEEPVQ_ERR_CAPACITY;
  if (a.routes == 0) return KEEPVQ_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Indices indices{a.indices, a.index_bits};
  inner_kernel<false><<<blocks_of(a.routes * a.rank, 8), 256, 0, s>>>(a.x, a.in_dim, a.x_div, a.right, a.in_dim, static_cast<int>(a.rank), a.dtype, indices, static_cast<int>(a.sets), a.routes, 1.0f, l.inner);
  KEEPVQ_CHECK_LAUNCH();
  outer_kernel<<<blocks_of(a.routes * a.out_dim, 256), 256, 0, s>>>(a, indices, l.inner);
  KEEPVQ_CHECK_LAUNCH();
  return KEEPVQ_OK;
}

int keepvq_switch_low_rank_grads(const keepvq_switch_low_rank_args* args, void* stream) {
  using namespace keepvq::dense;
  if (!args) return KEEPVQ_ERR_NULL;
  const keepvq_switch_low_rank_args& a = *args;
  if (const int rc = check_low_rank(a, true)) return rc;
  const LowRankLayout l = lay_out_low_rank(a.workspace, a.routes, a.sets, a.rank, true);
  if (l.bytes > a.workspace_bytes) return KEEPVQ_ERR_CAPACITY;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Indices indices{a.indices, a.index_bits};
  const int rank = static_cast<int>(a.rank), sets = static_cast<int>(a.sets);
  if (const int rc = make_plan(indices, a.routes, a.sets, 64, 16, l.plan, s)) return rc;
  if (a.routes > 0) {
    inner_kernel<false><<<blocks_of(a.routes * rank, 8), 256, 0, s>>>(a.x, a.in_dim, a.x_div, a.right, a.in_dim, rank, a.dtype, indices, sets, a.routes, 1.0f, l.inner);
    inner_kernel<true><<<blocks_of(a.routes * rank, 8), 256, 0, s>>>(a.grad, a.grad_ld, 1, a.left, a.out_dim, rank, a.dtype, indices, sets, a.routes, a.scale, l.back);
    if (a.dx) input_grad_kernel<<<blocks_of(a.routes / a.x_div * a.in_dim, 256), 256, 0, s>>>(a, indices, l.back);
  }
  if (a.dleft) factor_grad_kernel<true><<<dim3(blocks_of(a.out_dim * rank, 256), sets), 256, 0, s>>>(a.grad, a.grad_ld, 1, a.out_dim, rank, a.dtype, l.plan, l.inner, a.scale, a.dleft);
  if (a.dright) factor_grad_kernel<false><<<dim3(blocks_of(a.in_dim * rank, 256), sets), 256, 0, s>>>(a.x, a.in_dim, a.x_div, a.in_dim, rank, a.dtype, l.plan, l.back, 1.0f, a.dright);
  KEEPVQ_CHECK_LAUNCH();
  return KEEPVQ_OK;
}

}  // extern "C"
