// Grouping of routes by weight set, and the pick sum of input gradients.
#include "switch_plan.cuh"

namespace keepvq {
namespace dense {

// One launch, no communication between blocks, the same order every time: every block counts all
// routes per set in shared memory and scans the counts, so it knows where each of its own sets (one
// per warp) starts; the warp then walks the routes once more and keeps its own in their order.  A
// sort would need several launches or atomics that leave an order of their own.
constexpr int PLAN_THREADS = 256, PLAN_WARPS = PLAN_THREADS / 32;

__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(Indices indices, int routes, int sets, int tile_routes, int tile_step, Plan plan) {
  grid_launch_dependents();
  grid_wait();
  extern __shared__ int32_t count[];  // [sets]
  __shared__ int warp_routes[PLAN_WARPS], warp_tiles[PLAN_WARPS];
  __shared__ int own_offset[PLAN_WARPS], own_tile[PLAN_WARPS], own_count[PLAN_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int e = tid; e < sets; e += PLAN_THREADS) count[e] = 0;
  if (tid < PLAN_WARPS) own_count[tid] = 0;
  __syncthreads();
  for (int r = tid; r < routes; r += PLAN_THREADS) {
    const int e = indices.set_of(r, sets);
    if (e >= 0) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  // exclusive scan over the sets; a thread has a contiguous run of them
  const int run = (sets + PLAN_THREADS - 1) / PLAN_THREADS, first = min(sets, tid * run), last = min(sets, first + run);
  int n = 0, t = 0;
  for (int e = first; e < last; ++e) { n += count[e]; t += (count[e] + tile_routes - 1) / tile_routes; }
  int n_scan = n, t_scan = t;
  for (int d = 1; d < 32; d <<= 1) {
    const int a = __shfl_up_sync(0xFFFFFFFFu, n_scan, d), b = __shfl_up_sync(0xFFFFFFFFu, t_scan, d);
    if (lane >= d) { n_scan += a; t_scan += b; }
  }
  if (lane == 31) { warp_routes[warp] = n_scan; warp_tiles[warp] = t_scan; }
  __syncthreads();
  int n_before = n_scan - n, t_before = t_scan - t, live = 0, tiles = 0;
  for (int w = 0; w < PLAN_WARPS; ++w) {
    if (w < warp) { n_before += warp_routes[w]; t_before += warp_tiles[w]; }
    live += warp_routes[w];
    tiles += warp_tiles[w];
  }
  const int own0 = blockIdx.x * PLAN_WARPS;
  for (int e = first; e < last; ++e) {
    if (e >= own0 && e < own0 + PLAN_WARPS) {
      own_offset[e - own0] = n_before;
      own_tile[e - own0] = t_before;
      own_count[e - own0] = count[e];
      plan.offset[e] = n_before;
    }
    n_before += count[e];
    t_before += (count[e] + tile_routes - 1) / tile_routes;
  }
  if (blockIdx.x == 0 && tid == 0) {
    *plan.status = 0;
    *plan.tiles = tiles;
    plan.offset[sets] = live;
  }
  __syncthreads();
  const int e = own0 + warp;  // e == sets: the dead routes
  if (e > sets) return;
  int at = e < sets ? own_offset[warp] : live;
  const int mine = e < sets ? own_count[warp] : routes - live;
  if (mine == 0) return;
  if (e < sets) {
    const int parts = (mine + tile_routes - 1) / tile_routes;
    const int part = (mine + parts - 1) / parts, per = (part + tile_step - 1) / tile_step * tile_step;
    for (int p = lane; p < parts; p += 32) plan.tile[own_tile[warp] + p] = make_int4(e, at + p * per, max(0, min(per, mine - p * per)), 0);
  }
  const int want = e < sets ? e : -1, end = at + mine;
  for (int base = 0; base < routes && at < end; base += 128) {
    int found[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = base + u * 32 + lane;
      found[u] = r < routes ? indices.set_of(r, sets) : -2;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const unsigned hits = __ballot_sync(0xFFFFFFFFu, found[u] == want);
      if (found[u] == want) plan.order[at + __popc(hits & ((1u << lane) - 1u))] = base + u * 32 + lane;
      at += __popc(hits);
    }
  }
}

int make_plan(const Indices& indices, int64_t routes, int64_t sets, int tile_routes, int tile_step, const Plan& plan, cudaStream_t s) {
  const size_t smem = static_cast<size_t>(sets) * sizeof(int32_t);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return note_cuda_error(e);
  }
  const unsigned blocks = static_cast<unsigned>((sets + 1 + PLAN_WARPS - 1) / PLAN_WARPS);
  const cudaError_t e = launch_after(true, plan_kernel, blocks, PLAN_THREADS, smem, s, indices, static_cast<int>(routes), static_cast<int>(sets), tile_routes, tile_step, plan);
  return e == cudaSuccess ? KEEPVQ_OK : note_cuda_error(e);
}

// HBM-bound: 4 bytes in per value and pick, 2 out; a thread has eight neighbouring values of a row.
template <typename T>
__global__ void __launch_bounds__(256) sum_picks_kernel(const float* __restrict__ in, Indices indices, int sets, int64_t rows, int picks, int64_t width, T* __restrict__ out) {
  grid_launch_dependents();
  grid_wait();
  const int64_t per_row = width / 8, total = rows * per_row;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += 256ll * gridDim.x) {
    const int64_t row = i / per_row, c = (i - row * per_row) * 8;
    float sum[8] = {};
    for (int j = 0; j < picks; ++j) {
      const int64_t r = row * picks + j;
      if (indices.set_of(r, sets) < 0) continue;
      float v[8];
      load8_as_float(in + r * width + c, v);
#pragma unroll
      for (int d = 0; d < 8; ++d) sum[d] += v[d];
    }
    store8_from_float(out + row * width + c, sum);
  }
}

int sum_picks(const float* routes, const Indices& indices, int64_t sets, int64_t rows, int picks, int64_t width, void* out, int dtype, cudaStream_t s) {
  int64_t blocks = (rows * (width / 8) + 255) / 256;
  if (blocks > 148 * 32) blocks = 148 * 32;
  const dim3 grid(static_cast<unsigned>(blocks));
  const cudaError_t e = dtype == KEEPVQ_BF16
      ? launch_after(true, sum_picks_kernel<__nv_bfloat16>, grid, 256, 0, s, routes, indices, static_cast<int>(sets), rows, picks, width, static_cast<__nv_bfloat16*>(out))
      : launch_after(true, sum_picks_kernel<__half>, grid, 256, 0, s, routes, indices, static_cast<int>(sets), rows, picks, width, static_cast<__half*>(out));
  return e == cudaSuccess ? KEEPVQ_OK : note_cuda_error(e);
}

}  // namespace dense
}  // namespace keepvq
