// Grouping of routes by weight set, and the pick sum of input gradients.
#include "switch_plan.cuh"

namespace keepvq {
namespace dense {

// One launch, no communication between blocks, the same order every time: every block counts all
// routes per set in shared memory and scans the counts, so it knows where its own sets start; a team
// of warps then walks the routes once more for each of them and keeps the set's own in their order.  A sort
// would need several launches or atomics that leave an order of their own.
//
// Latency-bound: what counts is how many loads are in flight.  Up to PLAN_FEW routes a team is one warp
// and a block has eight (4 us for a few routes); beyond that a block of 32 warps is one team, whose warps
// take a stretch of the routes each (24,576 routes of 32 sets: 15 us; one warp per set took 49).
constexpr int PLAN_FEW = 2048;
constexpr unsigned PLAN_EARLY_BLOCKS = 148;  // more of them would crowd the SMs while they wait for their predecessor

template <int WARPS, int TEAM>
__global__ void __launch_bounds__(WARPS * 32) plan_kernel(Indices indices, int routes, int sets, int tile_routes, int tile_step, Plan plan) {
  constexpr int THREADS = WARPS * 32, TEAMS = WARPS / TEAM, BATCH = 4;
  grid_launch_dependents();
  grid_wait();
  extern __shared__ int32_t count[];  // [sets]
  __shared__ int warp_sums[3][WARPS], found_before[WARPS];
  __shared__ int own_place[TEAMS], own_tile[TEAMS], own_count[TEAMS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int e = tid; e < sets; e += THREADS) count[e] = 0;
  if (tid < TEAMS) own_count[tid] = 0;
  __syncthreads();
  for (int r0 = tid; r0 < routes; r0 += BATCH * THREADS) {
    int e[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) e[u] = r0 + u * THREADS < routes ? indices.set_of(r0 + u * THREADS, sets) : -1;
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
      if (e[u] >= 0) atomicAdd(&count[e[u]], 1);
  }
  __syncthreads();
  // exclusive scans over the sets of (routes, places, tiles); a thread has a contiguous run of them
  auto places_of = [](int n) { return (n + ROW_STEP - 1) / ROW_STEP * ROW_STEP; };
  auto tiles_of = [&](int n) { return (n + tile_routes - 1) / tile_routes; };
  const int run = (sets + THREADS - 1) / THREADS, first = min(sets, tid * run), last = min(sets, first + run);
  int own[3] = {}, before[3], total[3] = {};
  for (int e = first; e < last; ++e) { own[0] += count[e]; own[1] += places_of(count[e]); own[2] += tiles_of(count[e]); }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    int scan = own[k];
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, scan, d);
      if (lane >= d) scan += v;
    }
    if (lane == 31) warp_sums[k][warp] = scan;
    before[k] = scan - own[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k)
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const int sum = warp_sums[k][w];
      if (w < warp) before[k] += sum;
      total[k] += sum;
    }
  const int own0 = blockIdx.x * TEAMS;
  for (int e = first; e < last; ++e) {
    if (e >= own0 && e < own0 + TEAMS) {
      own_place[e - own0] = plan.offset[e] = before[1];
      own_count[e - own0] = plan.count[e] = count[e];
      own_tile[e - own0] = before[2];
    }
    before[1] += places_of(count[e]);
    before[2] += tiles_of(count[e]);
  }
  const int dead = routes - total[0];
  if (blockIdx.x == 0 && tid == 0) {
    *plan.status = 0;
    *plan.tiles = total[2];
    *plan.dead_count = dead;
    plan.offset[sets] = total[1];
  }
  __syncthreads();
  const int team = warp / TEAM, member = warp % TEAM, e = own0 + team;  // e == sets: the dead routes
  if (e > sets) return;  // (a team that is a block leaves as a whole)
  const int mine = e < sets ? own_count[team] : dead;
  if (mine == 0) return;
  int32_t* to = e < sets ? plan.order + own_place[team] : plan.dead;
  if (e < sets && member == 0) {
    const int parts = tiles_of(mine), part = (mine + parts - 1) / parts, per = (part + tile_step - 1) / tile_step * tile_step;
    for (int p = lane; p < parts; p += 32) plan.tile[own_tile[team] + p] = make_int4(e, own_place[team] + p * per, min(per, mine - p * per), 0);
    if (mine + lane < places_of(mine)) to[mine + lane] = -1;
  }
  const int want = e < sets ? e : -1;
  const int stretch = (routes + TEAM * 32 * BATCH - 1) / (TEAM * 32 * BATCH) * (32 * BATCH), from = member * stretch, end = min(routes, from + stretch);
  // hits of this warp's stretch, 128 routes at a time
  auto walk = [&](auto&& each) {
    for (int base = from; base < end; base += 32 * BATCH) {
      int found[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int r = base + u * 32 + lane;
        found[u] = r < end ? indices.set_of(r, sets) : -2;
      }
#pragma unroll
      for (int u = 0; u < BATCH; ++u) each(base + u * 32 + lane, found[u] == want, __ballot_sync(0xFFFFFFFFu, found[u] == want));
    }
  };
  int at = 0;
  if (TEAM > 1) {
    int hits = 0;
    walk([&](int, bool, unsigned all) { hits += __popc(all); });
    if (lane == 0) found_before[warp] = hits;
    __syncthreads();
    for (int w = 0; w < member; ++w) at += found_before[w];
  }
  walk([&](int r, bool hit, unsigned all) {
    if (hit) to[at + __popc(all & ((1u << lane) - 1u))] = r;
    at += __popc(all);
  });
}

template <int WARPS, int TEAM>
static int launch_plan(const Indices& indices, int64_t routes, int64_t sets, int tile_routes, int tile_step, const Plan& plan, cudaStream_t s) {
  auto kernel = plan_kernel<WARPS, TEAM>;
  const size_t smem = static_cast<size_t>(sets) * sizeof(int32_t);
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return note_cuda_error(e);
  }
  const unsigned blocks = static_cast<unsigned>((sets + 1 + WARPS / TEAM - 1) / (WARPS / TEAM));
  const cudaError_t e = launch_after(blocks <= PLAN_EARLY_BLOCKS, kernel, blocks, WARPS * 32, smem, s, indices, static_cast<int>(routes), static_cast<int>(sets), tile_routes, tile_step, plan);
  return e == cudaSuccess ? KEEPVQ_OK : note_cuda_error(e);
}
int make_plan(const Indices& indices, int64_t routes, int64_t sets, int tile_routes, int tile_step, const Plan& plan, cudaStream_t s) {
  return routes <= PLAN_FEW ? launch_plan<8, 1>(indices, routes, sets, tile_routes, tile_step, plan, s) : launch_plan<32, 32>(indices, routes, sets, tile_routes, tile_step, plan, s);
}

// HBM-bound, by writing; a block per place, four loads of a thread in flight (24,576 rows of 8 KB: 42 us, 4.8 TB/s written).
__global__ void __launch_bounds__(128) copy_rows_kernel(RowCopy a, RowCopy b, Plan plan, int sets) {
  if (static_cast<int>(blockIdx.x) >= plan.offset[sets]) return;
  const RowCopy& c = blockIdx.y ? b : a;
  const int route = plan.order[blockIdx.x], n = static_cast<int>(c.width / 8);
  const uint4* in = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.in) + (route < 0 ? 0 : route / c.div) * c.ld);
  uint4* out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(c.out) + blockIdx.x * c.width);
  for (int i = threadIdx.x; i < n; i += 4 * 128) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = route >= 0 && i + u * 128 < n ? __ldg(in + i + u * 128) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * 128 < n) out[i + u * 128] = v[u];
  }
}

int copy_rows(const RowCopy* copies, int count, int64_t routes, int64_t sets, const Plan& plan, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(max_places(routes, sets)), count);
  const cudaError_t e = launch_after(false, copy_rows_kernel, grid, 128, 0, s, copies[0], copies[count - 1], plan, static_cast<int>(sets));
  return e == cudaSuccess ? KEEPVQ_OK : note_cuda_error(e);
}

// HBM-bound: 4 bytes in per value and pick, 2 out; a thread has eight neighbouring values of a row (1000 rows of six picks of
// 4096: 20 us, 5.3 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) sum_picks_kernel(const float* __restrict__ in, Indices indices, int sets, int64_t rows, int picks, int64_t width, T* __restrict__ out) {
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
      ? launch_after(false, sum_picks_kernel<__nv_bfloat16>, grid, 256, 0, s, routes, indices, static_cast<int>(sets), rows, picks, width, static_cast<__nv_bfloat16*>(out))
      : launch_after(false, sum_picks_kernel<__half>, grid, 256, 0, s, routes, indices, static_cast<int>(sets), rows, picks, width, static_cast<__half*>(out));
  return e == cudaSuccess ? KEEPVQ_OK : note_cuda_error(e);
}

}  // namespace dense
}  // namespace keepvq
