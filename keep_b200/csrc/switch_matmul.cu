// Products over 16-bit experts chosen per route, and their gradients.
//
//   forward   out[r]    = W[e_r] x[r / x_div]
//   dx        dx[r]     = W[e_r]^T grad[r], summed over a row's picks in fp32
//   dweight   dW[e]     = sum over e's routes of grad[r] x[r / x_div]^T
#include "switch_plan.cuh"

namespace keepvq {
namespace dense {

enum { FORWARD = 0, INPUT_GRAD = 1, WEIGHT_GRAD = 2 };
constexpr int TILE = 64, STEP = 16;

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

// 64 x 64 outputs per block, 4 x 4 per thread, operands widened to fp32 in shared memory.
template <typename T, int MODE>
__global__ void __launch_bounds__(256) switch_matmul_kernel(keepvq_switch_matmul_args a, Plan plan, float* route_dx) {
  __shared__ float left[STEP][TILE + 1], right[STEP][TILE + 1];  // [contraction][output column], [contraction][output row]
  const T *x = static_cast<const T*>(a.x), *w = static_cast<const T*>(a.weight), *g = static_cast<const T*>(a.grad);
  int set, start, size;
  if (MODE == WEIGHT_GRAD) {
    set = blockIdx.z;
    start = plan.offset[set];
    size = plan.offset[set + 1] - start;
  } else {
    if (static_cast<int>(blockIdx.x) >= *plan.tiles) {
      if (MODE == FORWARD)  // dead routes
        for (int64_t r = plan.offset[a.experts] + blockIdx.x - *plan.tiles; r < a.routes; r += gridDim.x - *plan.tiles)
          for (int64_t n = blockIdx.y * 256 + threadIdx.x; n < a.out_dim; n += gridDim.y * 256) store_from_float(a.out, a.dtype, plan.order[r] * a.out_dim + n, 0.0f);
      return;
    }
    const int4 t = plan.tile[blockIdx.x];
    set = t.x; start = t.y; size = t.z;
  }
  const int64_t col0 = static_cast<int64_t>(MODE == WEIGHT_GRAD ? blockIdx.x : blockIdx.y) * TILE;
  const int64_t row0 = MODE == WEIGHT_GRAD ? blockIdx.y * TILE : 0;
  const int64_t depth = MODE == FORWARD ? a.in_dim : MODE == INPUT_GRAD ? a.out_dim : size;
  const int64_t cols = MODE == FORWARD ? a.out_dim : a.in_dim, rows = MODE == WEIGHT_GRAD ? a.out_dim : size;
  const T* we = w + set * a.out_dim * a.in_dim;
  float sum[4][4] = {};
  const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
  for (int64_t k0 = 0; k0 < depth; k0 += STEP) {
    for (int i = threadIdx.x; i < STEP * TILE; i += 256) {
      const int k = i / TILE, c = i % TILE;
      const int64_t kk = k0 + k;
      float lv = 0.0f, rv = 0.0f;
      if (kk < depth) {
        if (MODE == FORWARD) {
          if (col0 + c < cols) lv = widen(we[(col0 + c) * a.in_dim + kk]);
          if (c < rows) rv = widen(x[plan.order[start + c] / a.x_div * a.in_dim + kk]);
        } else if (MODE == INPUT_GRAD) {
          if (col0 + c < cols) lv = widen(we[kk * a.in_dim + col0 + c]);
          if (c < rows) rv = widen(g[plan.order[start + c] * a.grad_ld + kk]);
        } else {
          const int64_t r = plan.order[start + kk];
          if (col0 + c < cols) lv = widen(x[r / a.x_div * a.in_dim + col0 + c]);
          if (row0 + c < rows) rv = widen(g[r * a.grad_ld + row0 + c]);
        }
      }
      left[k][c] = lv;
      right[k][c] = rv;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < STEP; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] += right[k][tr * 4 + i] * left[k][tc + 16 * j];
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t row = row0 + tr * 4 + i, col = col0 + tc + 16 * j;
      if (row >= rows || col >= cols) continue;
      if (MODE == FORWARD) store_from_float(a.out, a.dtype, plan.order[start + row] * a.out_dim + col, sum[i][j]);
      else if (MODE == WEIGHT_GRAD) store_from_float(a.dweight, a.dtype, (set * a.out_dim + row) * a.in_dim + col, sum[i][j]);
      else if (route_dx) route_dx[plan.order[start + row] * a.in_dim + col] = sum[i][j];
      else store_from_float(a.dx, a.dtype, plan.order[start + row] * a.in_dim + col, sum[i][j]);
    }
}

struct Layout {
  Plan plan;
  float* route_dx;  // [routes, in_dim], where a row has several picks
  int64_t bytes;
};
static Layout lay_out(void* base, int64_t routes, int64_t experts, int64_t in_dim, int x_div, bool grads) {
  Scratch s{static_cast<char*>(base)};
  Layout l;
  l.plan = take_plan(s, routes, experts, TILE);
  l.route_dx = grads && x_div > 1 ? s.take<float>(routes * in_dim) : nullptr;
  l.bytes = s.used;
  return l;
}

static int check_sizes(int64_t routes, int64_t experts, int64_t out_dim, int64_t in_dim, int32_t x_div) {
  if (routes < 0 || experts <= 0 || out_dim <= 0 || in_dim <= 0 || x_div <= 0 || in_dim % 8 != 0 || routes % x_div != 0) return KEEPVQ_ERR_SHAPE;
  if (routes > MAX_ROUTES || experts > MAX_SETS || out_dim > (1 << 24) || in_dim > (1 << 24)) return KEEPVQ_ERR_CAPACITY;
  return KEEPVQ_OK;
}

template <int MODE>
static int launch(const keepvq_switch_matmul_args& a, const Layout& l, cudaStream_t s) {
  auto blocks = [](int64_t n) { return static_cast<unsigned>((n + TILE - 1) / TILE); };
  const dim3 grid = MODE == WEIGHT_GRAD ? dim3(blocks(a.in_dim), blocks(a.out_dim), static_cast<unsigned>(a.experts))
                                        : dim3(static_cast<unsigned>(max_tiles(a.routes, a.experts, TILE) + 1), blocks(MODE == FORWARD ? a.out_dim : a.in_dim));
  if (a.dtype == KEEPVQ_BF16) switch_matmul_kernel<__nv_bfloat16, MODE><<<grid, 256, 0, s>>>(a, l.plan, l.route_dx);
  else switch_matmul_kernel<__half, MODE><<<grid, 256, 0, s>>>(a, l.plan, l.route_dx);
  KEEPVQ_CHECK_LAUNCH();
  return KEEPVQ_OK;
}

static int check_call(const keepvq_switch_matmul_args& a, bool grads) {
  if (!valid_16bit(a.dtype) || (a.index_bits != 32 && a.index_bits != 64)) return KEEPVQ_ERR_DTYPE;
  if (const int rc = check_sizes(a.routes, a.experts, a.out_dim, a.in_dim, a.x_div)) return rc;
  if (grads && (a.grad_ld < a.out_dim || a.grad_ld % 8 != 0)) return KEEPVQ_ERR_SHAPE;
  if (!a.workspace || (a.routes > 0 && (!a.x || !a.weight || !a.indices || (grads ? !a.grad : !a.out)))) return KEEPVQ_ERR_NULL;
  for (const void* p : {a.x, a.weight, a.grad, static_cast<const void*>(a.dx), static_cast<const void*>(a.dweight)})
    if (!aligned_to(p, 16)) return KEEPVQ_ERR_ALIGN;
  if (!aligned_to(a.workspace, 256) || !aligned_to(a.out, 16) || !aligned_to(a.indices, a.index_bits / 8)) return KEEPVQ_ERR_ALIGN;
  return KEEPVQ_OK;
}

}  // namespace dense
}  // namespace keepvq

extern "C" {

int64_t keepvq_switch_matmul_workspace_bytes(int64_t routes, int64_t experts, int64_t out_dim, int64_t in_dim, int32_t x_div, int32_t grads) {
  using namespace keepvq::dense;
  if (const int rc = check_sizes(routes, experts, out_dim, in_dim, x_div)) return rc;
  return lay_out(nullptr, routes, experts, in_dim, x_div, grads != 0).bytes;
}

int keepvq_switch_matmul(const keepvq_switch_matmul_args* args, void* stream) {
  using namespace keepvq::dense;
  if (!args) return KEEPVQ_ERR_NULL;
  const keepvq_switch_matmul_args& a = *args;
  if (const int rc = check_call(a, false)) return rc;
  const Layout l = lay_out(a.workspace, a.routes, a.experts, a.in_dim, a.x_div, false);
  if (l.bytes > a.workspace_bytes) return KEEPVQ_ERR_CAPACITY;
  if (a.routes == 0) return KEEPVQ_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (const int rc = make_plan({a.indices, a.index_bits}, a.routes, a.experts, TILE, 16, l.plan, s)) return rc;
  return launch<FORWARD>(a, l, s);
}

int keepvq_switch_matmul_grads(const keepvq_switch_matmul_args* args, void* stream) {
  using namespace keepvq::dense;
  if (!args) return KEEPVQ_ERR_NULL;
  const keepvq_switch_matmul_args& a = *args;
  if (const int rc = check_call(a, true)) return rc;
  const Layout l = lay_out(a.workspace, a.routes, a.experts, a.in_dim, a.x_div, true);
  if (l.bytes > a.workspace_bytes) return KEEPVQ_ERR_CAPACITY;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Indices indices{a.indices, a.index_bits};
  if (const int rc = make_plan(indices, a.routes, a.experts, TILE, 16, l.plan, s)) return rc;
  if (a.dx && a.routes > 0) {
    if (!l.route_dx) {  // a dead route's row
      const cudaError_t e = cudaMemsetAsync(a.dx, 0, a.routes * a.in_dim * 2, s);
      if (e != cudaSuccess) return keepvq::note_cuda_error(e);
    }
    if (const int rc = launch<INPUT_GRAD>(a, l, s)) return rc;
    if (l.route_dx)
      if (const int rc = sum_picks(l.route_dx, indices, a.experts, a.routes / a.x_div, a.x_div, a.in_dim, a.dx, a.dtype, s)) return rc;
  }
  return a.dweight ? launch<WEIGHT_GRAD>(a, l, s) : KEEPVQ_OK;
}

}  // extern "C"
