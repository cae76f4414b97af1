// Routes grouped by the weight set they name, for the products over 16-bit experts and low-rank
// adapters (switch_matmul.cu, low_rank.cu), and the sum of the routes' input gradients.
#pragma once

#include "common.cuh"

namespace keepvq {
namespace dense {

constexpr int64_t MAX_ROUTES = int64_t{1} << 24, MAX_SETS = 16384;

// What the plan kernel leaves in the workspace.  A set's routes take consecutive places, rounded up to
// ROW_STEP: places without a route hold -1, and zeros where rows are copied into that order.
constexpr int ROW_STEP = 16;
struct Plan {
  int32_t* status;  // [1] 1: a bounded wait expired, the call's outputs are invalid
  int32_t* tiles;   // [1]
  int32_t* dead_count;  // [1]
  int32_t* offset;  // [sets + 1] a set's first place; offset[sets]: the number of places
  int32_t* count;   // [sets] its routes
  int32_t* order;   // [places] the routes by set, each set's in their own order
  int32_t* dead;    // [routes] the routes without a set
  int4* tile;       // [max_tiles] (set, first place, routes, 0): a set's routes in equal parts of at most `tile_routes`
};
inline int64_t max_places(int64_t routes, int64_t sets) { return routes + (ROW_STEP - 1) * (routes < sets ? routes : sets); }

inline int64_t align_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }
inline int64_t max_tiles(int64_t routes, int64_t sets, int64_t tile_routes) { return routes / tile_routes + (routes < sets ? routes : sets); }

// A bump allocator over the workspace; with base == nullptr it only counts.
struct Scratch {
  char* base;
  int64_t used = 0;
  template <typename T>
  T* take(int64_t count) {
    T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used = align_up(used + count * static_cast<int64_t>(sizeof(T)), 256);
    return p;
  }
};
inline Plan take_plan(Scratch& s, int64_t routes, int64_t sets, int64_t tile_routes) {
  Plan p;
  p.status = s.take<int32_t>(3);
  p.tiles = p.status ? p.status + 1 : nullptr;
  p.dead_count = p.status ? p.status + 2 : nullptr;
  p.offset = s.take<int32_t>(sets + 1);
  p.count = s.take<int32_t>(sets);
  p.order = s.take<int32_t>(max_places(routes, sets));
  p.dead = s.take<int32_t>(routes);
  p.tile = s.take<int4>(max_tiles(routes, sets, tile_routes) + 1);
  return p;
}

struct Indices {
  const void* data;
  int bits;
  __device__ __forceinline__ int64_t at(int64_t r) const {
    return bits == 64 ? static_cast<const int64_t*>(data)[r] : static_cast<const int32_t*>(data)[r];
  }
  // the set of a route, or -1
  __device__ __forceinline__ int set_of(int64_t r, int sets) const {
    const int64_t e = at(r);
    return e >= 0 && e < sets ? static_cast<int>(e) : -1;
  }
};

// Sums and tiles in a launch of their own; `tile_routes` a multiple of `tile_step`, to which the parts are rounded up.
int make_plan(const Indices& indices, int64_t routes, int64_t sets, int tile_routes, int tile_step, const Plan& plan, cudaStream_t s);

// Rows of 16-bit values copied into the plan's places: out[p] = in[order[p] / div], zeros where order[p] is -1.
struct RowCopy {
  const void* in;
  void* out;
  int64_t ld, width;  // of a row in `in`, and of one in `out`: multiples of 8
  int div;
};
int copy_rows(const RowCopy* copies, int count, int64_t routes, int64_t sets, const Plan& plan, cudaStream_t s);

// out[t] = the sum over the picks j of row t, in their order, of routes[t * picks + j] (fp32), dead
// picks left out; rounded once.  `width` is a multiple of 8.
int sum_picks(const float* routes, const Indices& indices, int64_t sets, int64_t rows, int picks, int64_t width, void* out, int dtype, cudaStream_t s);

inline bool valid_16bit(int t) { return t == KEEPVQ_F16 || t == KEEPVQ_BF16; }

}  // namespace dense
}  // namespace keepvq
