// Low-rank products chosen per route, added onto a base, and their gradients.  With B = left[e],
// A = right[e] of a route's set e:
//   p = A x,  out = base + scale B p;   q = scale B^T grad,  dx = A^T q,
//   dA = sum q x^T,  dB = scale sum grad p^T
//
// The rank is 8 to 128, so all of it is bound by reading x, grad, base and the factors once; what there
// is to multiply stays on mma.sync, whose fragments are made of 16-byte pieces as they lie in memory (the
// order of a contraction is free, so a lane's eight neighbouring values serve two instructions).  Every lane
// copies the pieces that it will want itself to a queue of its own in shared memory, some steps ahead:
// bytes in flight that cost no registers, and nobody to wait for but the copies.
//
// Two products with a vector in between (low_rank_kernel): a cluster of CTAs takes the rows of one set, up
// to 16, and splits the first contraction over its CTAs and their warps; the partial inner vectors meet in
// shared memory, once per CTA and once over the cluster; the CTAs then split the width of the result.  So
// the inner vectors never leave the SMs, and one row of one set still has a whole cluster's loads in
// flight.  Forward: A, then B.  Input gradient: B^T, then A^T, whose fragments are transposed in registers.
//
// Measured on a B200, 4096 -> 4096, bf16: one row of rank 16 6 us on the device, 61 rows of rank 32 11 us cold; 251 tokens with
// six of 384 corrections of rank 8 20 us; 4096 rows of rank 16 / 64 / 128 31 / 45 / 85 us with the plan (56 / 69 / 124 with an
// fp32 base), where x, base and results are 100 MB.  What bounds it then is instructions and latency per 16 rows, not bytes.  Tiles of 64 rows shared
// by the warps through ldmatrix were slower at every rank from 32 on (4096 rows of rank 64: 67 us).
//
// Inner vectors are fp32 sums; for the second product each is split into the sum of two 16-bit values, scaled
// by a power of two per row for fp16 so that neither its range nor its small values are lost.  The low parts' sums are kept apart
// and made finite, so that an infinity of a factor comes through as the high parts have it (rank 16 and 32: no time; 64: 3 %
// forward and 6 % for dx; 128: 9 and 4 %).
#include "switch_plan.cuh"

namespace keepvq {
namespace dense {

constexpr int64_t LR_MAX_PITCH = int64_t{1} << 28;  // of a row, in values: its bytes stay within 32 bits
constexpr int LR_MAX_RANK = 128, LR_WARPS = 8, LR_THREADS = LR_WARPS * 32, CHUNK = 32;

// ---- fragments ------------------------------------------------------------------------------------
template <typename T>
struct Mma;
template <>
struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)); }
  static constexpr bool SCALED = false;  // the range is fp32's
};
template <>
struct Mma<__half> {
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  static constexpr bool SCALED = true;
};
// Two values as the sum of two 16-bit ones.  An infinity has no rest (inf - inf).
template <typename T>
__device__ __forceinline__ void split(float x, float y, uint32_t& high, uint32_t& low) {
  high = Mma<T>::pack(x, y);
  const float2 h = Mma<T>::unpack(high);
  low = Mma<T>::pack(isinf(h.x) ? 0.0f : x - h.x, isinf(h.y) ? 0.0f : y - h.y);
}
// What the low parts add up to, as something that an infinity can be added to: the largest number in the place of an infinity or of
// no value.  A factor's infinity meets both parts of an inner value; with the low one, zero or of the other sign, it would undo
// what the high one makes of it.  (The smaller magnitude, of the one that is a number, with v's sign.)
__device__ __forceinline__ float finite(float v) {
  float f;
  asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(f) : "f"(v), "f"(__uint_as_float(0x7F7FFFFFu)));
  return f;
}
// An 8 x 8 matrix of 16-bit values, a row's pairs in four lanes, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t t;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
  return t;
}
__device__ __forceinline__ uint4 load16(const uint16_t* p, bool there) { return there ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0); }
__device__ __forceinline__ uint2 load8(const uint16_t* p, bool there) { return there ? __ldg(reinterpret_cast<const uint2*>(p)) : make_uint2(0, 0); }
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// A lane's queue: pieces of up to 16 bytes, those of a step in one group of copies.  A piece that is not there is zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy8(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(there ? 8 : 0) : "memory");
}
__device__ __forceinline__ void step_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int STEPS>
__device__ __forceinline__ void all_but() { asm volatile("cp.async.wait_group %0;" ::"n"(STEPS) : "memory"); }
__device__ __forceinline__ uint4 piece16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

// A power of two not below `most` (finite), within what has a reciprocal; 1 for zero.
__device__ __forceinline__ float power_above(float most) {
  const uint32_t e = (__float_as_uint(most) >> 23) & 0xFFu;
  return most == 0.0f ? 1.0f : __uint_as_float(min(max(e + 1u, 2u), 252u) << 23);
}

__device__ __forceinline__ uint32_t lr_cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t lr_cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void lr_cluster_sync() { asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ float peer_float(const float* p, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// ---- one product after the other ---------------------------------------------------------------------

// Inner vectors as the gradients of the factors take them: per block of 16 places, [rank][16 places] of
// bf16, the two whose sum they are apart; a lane's four places of a fragment (2q, 2q + 1, 2q + 8,
// 2q + 9) side by side.  bf16 for fp16 operands too: the rows of a set are summed over, so no power of two
// of a row's own could be taken out again, and one for several rows would lose the smallest.
struct Inner {
  uint16_t *high, *low;
};

struct LowRankArgs {
  const uint16_t* in;      // rows of the first contraction: x, or grad
  int64_t in_ld;           // multiple of 8
  int in_div;              // routes per row of `in`
  const uint16_t* first;   // its factor: right, or left (transposed)
  const uint16_t* second;  // left, or right (transposed); null: no second product
  int64_t depth, width;    // of the first contraction; of the result
  int rank, ranks, sets;   // in memory; of these, those that are no padding
  float first_scale, second_scale;
  const void* base;        // null: zeros
  int64_t base_ld;
  void* out;
  int64_t out_ld;
  int out32;               // base and out are fp32
  int whole;               // their rows can be taken 16 bytes at a time
  int dead_rows;           // rows without a set are the kernel's (their base, or zeros)
  int solo;                // a tile per route, no plan
  Indices indices;
  Plan plan;
  Inner keep;              // where to leave the inner vectors; null: nowhere
};

// A route without a set: its base, bit for bit.
__device__ __forceinline__ void low_rank_plain_row(const LowRankArgs& a, int64_t r) {
  const int tid = threadIdx.x;
  const int size = a.out32 ? 4 : 2;
  char* to = static_cast<char*>(a.out) + r * a.out_ld * size;
  const char* from = a.base ? static_cast<const char*>(a.base) + r * a.base_ld * size : nullptr;
  if (a.whole) {
    const int n = static_cast<int>(a.width * size / 16);
#pragma unroll 4
    for (int i = tid; i < n; i += LR_THREADS) reinterpret_cast<uint4*>(to)[i] = from ? reinterpret_cast<const uint4*>(from)[i] : make_uint4(0, 0, 0, 0);
  } else if (size == 4) {
    for (int i = tid; i < a.width; i += LR_THREADS) reinterpret_cast<uint32_t*>(to)[i] = from ? reinterpret_cast<const uint32_t*>(from)[i] : 0u;
  } else {
    for (int i = tid; i < a.width; i += LR_THREADS) reinterpret_cast<uint16_t*>(to)[i] = from ? reinterpret_cast<const uint16_t*>(from)[i] : static_cast<uint16_t>(0);
  }
}

// The inner vectors of a tile for the gradients of the factors.
template <int RP, int ROWS>
__device__ __forceinline__ void keep_inner(const LowRankArgs& a, const float* inner, int start, int size) {
  for (int i = threadIdx.x; i < ROWS * RP / 2; i += LR_THREADS) {  // two neighbouring places of a rank
    const int block = i / (RP * 8), j = i / 8 % RP, pair = i % 8;
    const int r0 = block * 16 + pair / 2 * 2 + (pair & 1) * 8;
    if (r0 >= (size + 15) / 16 * 16) continue;
    uint32_t high, low;
    split<__nv_bfloat16>(r0 < size ? inner[r0 * RP + j] : 0.0f, r0 + 1 < size ? inner[(r0 + 1) * RP + j] : 0.0f, high, low);
    const int64_t at = (static_cast<int64_t>(start / 16 + block) * RP + j) * 8 + pair;
    reinterpret_cast<uint32_t*>(a.keep.high)[at] = high;
    reinterpret_cast<uint32_t*>(a.keep.low)[at] = low;
  }
}

// `own`, this CTA's part of the sums of all rows, becomes `inner`, the cluster's (in the order of its CTAs), with a
// power of two per row for fp16.
template <typename T, int RP, int ROWS>
__device__ __forceinline__ void meet(const float* own, float* inner, float* unit, int ctas) {
  const int tid = threadIdx.x;
  if (ctas > 1) lr_cluster_sync();
  else __syncthreads();
  for (int i = tid; i < ROWS * RP; i += LR_THREADS) {
    float sum = own[i];
    if (ctas > 1) {
      sum = 0.0f;
      for (int c = 0; c < ctas; ++c) sum += peer_float(own + i, c);
    }
    inner[i] = sum;
  }
  __syncthreads();
  if (Mma<T>::SCALED) {
    if (tid < ROWS) {
      float most = 0.0f;
      for (int j = 0; j < RP; ++j) {  // of those that are numbers: beside an infinity the others still have to fit
        const float v = fabsf(inner[tid * RP + (j + tid) % RP]);
        if (!isinf(v)) most = fmaxf(most, v);
      }
      unit[tid] = power_above(most);
    }
    __syncthreads();
  }
}

// RP: the rank rounded up (zeros).  BACK: both factors are used transposed.
template <int RP, bool BACK>
struct LowRankShape {
  static constexpr int ROWS = 16, RT = RP / 8, KC = RP / 16, V = RP >= 32 ? 8 : 4, CC = RP / (4 * V);  // V: neighbouring ranks a lane holds
  static constexpr int FACTOR1 = BACK ? 4 * CC : RT, FACTOR2 = BACK ? 2 * KC : 4 * CC;  // pieces of a step: the factor's, and two of the rows
  static constexpr int PIECES = 2 + (FACTOR1 > FACTOR2 ? FACTOR1 : FACTOR2), STEP_BYTES = PIECES * 32 * 16;
  static constexpr bool SMALL = RP <= 16;  // three CTAs on an SM instead of two: calls of many sets with a few rows each
  static constexpr int BUDGET = SMALL ? 9 * 1024 : 12 * 1024, STEPS = BUDGET / STEP_BYTES < 2 ? 2 : BUDGET / STEP_BYTES;  // per warp; some 200 KB in flight on an SM
  static constexpr int QUEUES = LR_WARPS * STEPS * STEP_BYTES;
  static constexpr int BYTES = QUEUES + 2 * ROWS * RP * 4 + 2 * ROWS * 4;  // (the warps' partial sums lie where the queues were)
  static constexpr int CTAS = SMALL ? 3 : BYTES + 1024 <= 114 * 1024 ? 2 : 1;  // on an SM
  static_assert(CTAS * (BYTES + 1024) <= 228 * 1024, "");
  static_assert(LR_WARPS * ROWS * RP * 4 <= QUEUES, "");
};

template <typename T, int RP, bool BACK>
__global__ void __launch_bounds__(LR_THREADS, LowRankShape<RP, BACK>::CTAS) low_rank_kernel(LowRankArgs a) {
  grid_wait();
  using S = LowRankShape<RP, BACK>;
  constexpr int ROWS = S::ROWS, RT = S::RT, V = S::V, KC = S::KC, CC = S::CC, STEPS = S::STEPS;
  extern __shared__ __align__(16) float sm[];
  float* part = sm;                                     // [warps][ROWS][RP], behind the queues of the first product
  float* own = sm + S::QUEUES / 4;                      // [ROWS][RP] of this CTA; then of the cluster
  float* unit = own + 2 * ROWS * RP;                    // [ROWS]
  int* route_of = reinterpret_cast<int*>(unit + ROWS);  // [ROWS]
  float* inner = own + ROWS * RP;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int ctas = static_cast<int>(lr_cluster_size()), rank = static_cast<int>(lr_cluster_rank());
  const int tile = blockIdx.x / ctas;
  const uint32_t queue = static_cast<uint32_t>(__cvta_generic_to_shared(sm)) + warp * (STEPS * S::STEP_BYTES) + lane * 16;
  auto slot = [&](int step, int piece) { return queue + static_cast<uint32_t>((step * S::PIECES + piece) * 512); };

  auto plain_row = [&](int64_t r) { low_rank_plain_row(a, r); };
  int set, start = 0, size = 1;
  if (a.solo) {
    set = a.indices.set_of(tile, a.sets);
    if (set < 0) {  // uniform over the cluster
      if (rank == 0 && a.dead_rows) plain_row(tile);
      return;
    }
    if (tid < ROWS) route_of[tid] = tile;
  } else {
    if (a.dead_rows)
      for (int p = blockIdx.x; p < *a.plan.dead_count; p += gridDim.x) plain_row(a.plan.dead[p]);
    if (tile >= *a.plan.tiles) return;
    const int4 t = a.plan.tile[tile];
    set = t.x; start = t.y; size = t.z;
    if (tid < ROWS) route_of[tid] = a.plan.order[start + min(tid, size - 1)];  // rows past the last repeat it and are not stored
  }
  __syncthreads();

  // ---- the first product: rows [ROWS, depth] times the factor -> [ROWS, RP]
  {
    float acc[RT][4];
#pragma unroll
    for (int n = 0; n < RT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
    int row[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) row[h] = route_of[h * 8 + g] / a.in_div;
    // (rows and ranks times row lengths in bytes are 32 x 32 bit products: one instruction an address)
    const int depth = static_cast<int>(a.depth), in_ld = static_cast<int>(a.in_ld), in_bytes = in_ld * 2, stride = ctas * LR_WARPS * CHUNK, k_first = (rank * LR_WARPS + warp) * CHUNK;
    const char* in_k = reinterpret_cast<const char*>(a.in + k_first + q * 8);
    const int factor_bytes = BACK ? a.rank * 2 : depth * 2;
    const char* factor_k = reinterpret_cast<const char*>(a.first + static_cast<int64_t>(set) * a.rank * depth) +
                           (BACK ? static_cast<int64_t>(k_first + 8 * (g >> 1) + (g & 1)) * factor_bytes + q * V * 2 : static_cast<int64_t>(g) * factor_bytes + (k_first + q * 8) * 2);
    int k_fill = k_first;
    // the pieces of the next 32 values of the contraction, to the queue's step `at`
    auto fill = [&](int at) {
      const bool there = k_fill + q * 8 < in_ld;  // (values of `in` between depth and in_ld are zeros)
#pragma unroll
      for (int h = 0; h < 2; ++h) copy16(slot(at, h), in_k + static_cast<int64_t>(row[h]) * in_bytes, there);
      if (!BACK) {
#pragma unroll
        for (int n = 0; n < RT; ++n) copy16(slot(at, 2 + n), factor_k + static_cast<int64_t>(n * 8) * factor_bytes, there && n * 8 + g < a.rank);
        factor_k += stride * 2;
      } else {
        // the factor's rows lie along the contraction: 8 x 8 blocks of it are transposed in registers.  Row i of a
        // block is the contraction index that the other operand's lane order wants there.
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int more = 4 * (i >> 1) + 2 * (i & 1);
          const bool is = k_fill + 8 * (g >> 1) + (g & 1) + more < depth;
#pragma unroll
          for (int c = 0; c < CC; ++c) {
            const char* from = factor_k + static_cast<int64_t>(more) * factor_bytes + c * 4 * V * 2;
            if (V == 8) copy16(slot(at, 2 + i * CC + c), from, is && c * 4 * V + q * V < a.rank);
            else copy8(slot(at, 2 + i * CC + c), from, is && c * 4 * V + q * V < a.rank);
          }
        }
        factor_k += static_cast<int64_t>(stride) * factor_bytes;
      }
      in_k += stride * 2;
      k_fill += stride;
    };
#pragma unroll
    for (int i = 0; i < STEPS - 1; ++i) {
      if (k_fill < depth) fill(i);
      step_issued();
    }
    int at = 0;
    for (int k0 = k_first; k0 < depth; k0 += stride) {
      if (k_fill < depth) fill(at == 0 ? STEPS - 1 : at - 1);
      step_issued();
      all_but<STEPS - 1>();
      uint4 v[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) v[h] = piece16(slot(at, h));
      if (!BACK) {
#pragma unroll
        for (int n = 0; n < RT; ++n) {
          const uint4 w = piece16(slot(at, 2 + n));
          const uint32_t a0[4] = {v[0].x, v[1].x, v[0].y, v[1].y}, a1[4] = {v[0].z, v[1].z, v[0].w, v[1].w};
          Mma<T>::run(acc[n], a0, w.x, w.y);
          Mma<T>::run(acc[n], a1, w.z, w.w);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int c = 0; c < CC; ++c) {
            const uint4 w0 = piece16(slot(at, 2 + 2 * j * CC + c)), w1 = piece16(slot(at, 2 + (2 * j + 1) * CC + c));
#pragma unroll
            for (int t = 0; t < V / 2; ++t) {
              const uint32_t b0 = transpose8(word(w0, t)), b1 = transpose8(word(w1, t));
              const uint32_t av[4] = {j ? v[0].z : v[0].x, j ? v[1].z : v[1].x, j ? v[0].w : v[0].y, j ? v[1].w : v[1].y};
              Mma<T>::run(acc[c * (V / 2) + t], av, b0, b1);
            }
          }
        }
      }
      if (++at == STEPS) at = 0;
    }
    all_but<0>();
    __syncthreads();  // the queues make room for the partial sums
    // a lane's ranks of tile n: 8 n + 2 q and the next; transposed: c * 4 V + V q + 2 t and the next
#pragma unroll
    for (int n = 0; n < RT; ++n) {
      const int j = BACK ? n / (V / 2) * 4 * V + V * q + 2 * (n % (V / 2)) : 8 * n + 2 * q;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float2*>(part + (warp * ROWS + h * 8 + g) * RP + j) = make_float2(acc[n][2 * h], acc[n][2 * h + 1]);
    }
  }
  __syncthreads();
  for (int i = tid; i < ROWS * RP; i += LR_THREADS) {
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < LR_WARPS; ++w) sum += part[w * ROWS * RP + i];
    own[i] = i % RP < a.ranks ? sum * a.first_scale : 0.0f;  // (a row's infinity times the zeros of ranks that are not there is no zero)
  }
  meet<T, RP, ROWS>(own, inner, unit, ctas);
  if (a.keep.high && rank == 0) keep_inner<RP, ROWS>(a, inner, start, size);

  // ---- the second product: [ROWS, RP] times the factor -> [ROWS, width], 32 columns per warp and step
  if (a.second) {
    const bool queued_base = a.base && a.whole && !a.out32;
    const int width = static_cast<int>(a.width), stride = ctas * LR_WARPS * 32, n_first = (rank * LR_WARPS + warp) * 32, size_of = a.out32 ? 4 : 2;
    const int factor_bytes = BACK ? width * 2 : a.rank * 2, base_bytes = static_cast<int>(a.base_ld) * size_of, out_bytes = static_cast<int>(a.out_ld) * size_of;
    const char* factor_n = reinterpret_cast<const char*>(a.second + static_cast<int64_t>(set) * a.rank * width) +
                           (BACK ? static_cast<int64_t>((V == 8 ? 8 : 4) * (g >> 1) + (g & 1)) * factor_bytes + (n_first + 8 * q) * 2 : static_cast<int64_t>(n_first + 8 * (g >> 1) + (g & 1)) * factor_bytes + q * V * 2);
    const char* base_n = static_cast<const char*>(a.base) + (n_first + 8 * q) * 2;
    char* out_n = static_cast<char*>(a.out) + (n_first + 8 * q) * size_of;
    int route[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) route[h] = route_of[h * 8 + g];
    int n_fill = n_first;
    // the pieces of the next 32 columns: the factor by RP, whose column c of tile t is 8 (c / 2) + 2 t + c % 2, so that a
    // lane's results are neighbours; and the base of all rows
    auto fill = [&](int at) {
      if (!BACK) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const bool is = n_fill + 8 * (g >> 1) + 2 * t + (g & 1) < width;
#pragma unroll
          for (int c = 0; c < CC; ++c) {
            const char* src = factor_n + static_cast<int64_t>(2 * t) * factor_bytes + c * 4 * V * 2;
            if (V == 8) copy16(slot(at, t * CC + c), src, is && c * 4 * V + q * V < a.rank);
            else copy8(slot(at, t * CC + c), src, is && c * 4 * V + q * V < a.rank);
          }
        }
        factor_n += static_cast<int64_t>(stride) * factor_bytes;
      } else {
        const bool is = n_fill + 8 * q < width;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int more = (V == 8 ? c / 2 * 32 + 4 * (c & 1) : 0) + 2 * i;
            copy16(slot(at, 2 * c + i), factor_n + static_cast<int64_t>(more) * factor_bytes, is && (V == 8 ? 8 : 4) * (g >> 1) + (g & 1) + more < a.rank);
          }
        factor_n += stride * 2;
      }
      if (queued_base) {
#pragma unroll
        for (int h = 0; h < 2; ++h) copy16(slot(at, S::FACTOR2 + h), base_n + static_cast<int64_t>(route[h]) * base_bytes, h * 8 + g < size && n_fill + 8 * q < width);
        base_n += stride * 2;
      }
      n_fill += stride;
    };
#pragma unroll
    for (int i = 0; i < STEPS - 1; ++i) {
      if (n_fill < width) fill(i);
      step_issued();
    }
    uint32_t high[KC][4], low[KC][4];
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = (i & 1) * 8 + g;
        const int j = V == 8 ? c / 2 * 32 + 8 * q + 4 * (c & 1) + 2 * (i >> 1) : 4 * q + 2 * (i >> 1);
        const float2 v = *reinterpret_cast<const float2*>(inner + r * RP + j);
        const float u = Mma<T>::SCALED ? 1.0f / unit[r] : 1.0f;  // (a power of two)
        split<T>(v.x * u, v.y * u, high[c][i], low[c][i]);
      }
    int at = 0;
    for (int n0 = n_first; n0 < width; n0 += stride, out_n += stride * size_of) {
      if (n_fill < width) fill(at == 0 ? STEPS - 1 : at - 1);
      step_issued();
      all_but<STEPS - 1>();
      uint32_t b[4][KC][2];
      if (!BACK) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int c = 0; c < CC; ++c) {
            const uint4 w = piece16(slot(at, t * CC + c));
            b[t][(2 * c) % KC][0] = w.x; b[t][(2 * c) % KC][1] = w.y;
            if (V == 8) { b[t][(2 * c + 1) % KC][0] = w.z; b[t][(2 * c + 1) % KC][1] = w.w; }
          }
      } else {
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint4 w = piece16(slot(at, 2 * c + i));
#pragma unroll
            for (int t = 0; t < 4; ++t) b[t][c][i] = transpose8(word(w, t));
          }
      }
      const int n = n0 + 8 * q;
      float d[4][4], e[4][4];  // of the high parts, and of the low ones
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) d[t][i] = e[t][i] = 0.0f;
      }
#pragma unroll
      for (int c = 0; c < KC; ++c) {
#pragma unroll
        for (int t = 0; t < 4; ++t) Mma<T>::run(e[t], low[c], b[t][c][0], b[t][c][1]);
#pragma unroll
        for (int t = 0; t < 4; ++t) Mma<T>::run(d[t], high[c], b[t][c][0], b[t][c][1]);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) d[t][i] += finite(e[t][i]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = h * 8 + g;
        if (r >= size) continue;
        char* to = out_n + static_cast<int64_t>(route[h]) * out_bytes;
        const float s = Mma<T>::SCALED ? a.second_scale * unit[r] : a.second_scale;
        float y[8];
#pragma unroll
        for (int t = 0; t < 4; ++t) { y[2 * t] = s * d[t][2 * h]; y[2 * t + 1] = s * d[t][2 * h + 1]; }
        if (a.whole) {
          if (n >= width) continue;
          if (a.out32) {
            float v[8] = {};
            if (a.base) load8_as_float(static_cast<const float*>(a.base) + route[h] * a.base_ld + n, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += y[i];
            store8_from_float(reinterpret_cast<float*>(to), v);
          } else {
            if (a.base) {
              const uint4 rest = piece16(slot(at, S::FACTOR2 + h));
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 v = Mma<T>::unpack(word(rest, i));
                y[2 * i] += v.x;
                y[2 * i + 1] += v.y;
              }
            }
            store8_from_float(reinterpret_cast<T*>(to), y);
          }
        } else {
          const int dtype = a.out32 ? KEEPVQ_F32 : Mma<T>::SCALED ? KEEPVQ_F16 : KEEPVQ_BF16;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (n + i < width) store_from_float(to, dtype, i, y[i] + (a.base ? load_as_float(a.base, dtype, route[h] * a.base_ld + n + i) : 0.0f));
        }
      }
      if (++at == STEPS) at = 0;
    }
    all_but<0>();
  }
  if (ctas > 1) lr_cluster_sync();  // the others may still be reading this CTA's partial sums
}

// ---- gradients of the factors --------------------------------------------------------------------------

struct FactorGradArgs {
  const uint16_t* in;  // rows: x (for right), grad (for left)
  int64_t in_ld;
  int in_div;
  int64_t width;       // in_dim, out_dim
  int rank, row_parts; // row_parts: warps that share a set's rows, 1, 2, 4 or 8
  float scale;
  Plan plan;
  Inner inner;
  uint16_t* out;
};

// The gradients of a warp's 32 columns and RH ranks that have no value, once more from the high parts alone: an infinity times a
// low part (zero, or of the other sign) undoes what it makes of the high one, which is the definition's.  Plain sums, four ranks
// at a time, up to where none of them can have a value any more; a call whose inputs are finite never comes here.
template <typename T, int RP, bool LEFT>
__device__ __noinline__ void factor_grad_undefined(const FactorGradArgs& a, int set, int64_t col0, int j0, int ranks) {
  const int64_t col = col0 + (threadIdx.x & 31);
  const bool mine = col < a.width;
  const int start = a.plan.offset[set], size = a.plan.count[set];
  T* out = reinterpret_cast<T*>(a.out) + static_cast<int64_t>(set) * a.rank * a.width + (LEFT ? col * a.rank : col);
  const T* in = reinterpret_cast<const T*>(a.in) + (mine ? col : 0);
  for (int j = j0; j < a.rank && j < j0 + ranks; j += 4) {
    bool undefined[4], some = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) some |= undefined[i] = mine && isnan(static_cast<float>(out[(j + i) * (LEFT ? 1 : a.width)]));
    if (!__any_sync(0xFFFFFFFFu, some)) continue;
    float sum[4] = {};
    for (int block = 0; block < size; block += 16) {
      const int place = a.plan.order[start + block + (threadIdx.x & 15)];
      const uint4* inner = reinterpret_cast<const uint4*>(a.inner.high + (static_cast<int64_t>((start + block) / 16) * RP + j) * 16);
      float x[16];
      uint4 parts[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) parts[i] = __ldg(inner + i);
#pragma unroll
      for (int p = 0; p < 16; ++p) {
        const int route = __shfl_sync(0xFFFFFFFFu, place, p);
        x[p] = static_cast<float>(in[static_cast<int64_t>(max(route, 0) / a.in_div) * a.in_ld]);
        if (route < 0) x[p] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int w = 0; w < 8; ++w) {  // (the order of Inner: places 2 (w / 2) + 8 (w % 2) and the next)
          const uint32_t two = word(parts[2 * i + w / 4], w % 4);
          const int p = w / 2 * 2 + w % 2 * 8;
          sum[i] = fmaf(__uint_as_float(two & 0xFFFF0000u), x[p + 1], fmaf(__uint_as_float(two << 16), x[p], sum[i]));
        }
      bool open = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) open |= undefined[i] && !isnan(sum[i]);
      if (!__any_sync(0xFFFFFFFFu, open)) break;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (undefined[i]) out[(j + i) * (LEFT ? 1 : a.width)] = static_cast<T>(a.scale * sum[i]);
  }
}

// A warp has 32 columns of x (or grad) and RH ranks, and walks the set's rows 16 at a time; the warps that share
// them add their sums up in shared memory in their order.
//   right: D[rank][column] = inner^T rows       left: D[column][rank] = rows^T inner
template <typename T, int RP, bool LEFT>
__device__ __forceinline__ void factor_grad(const FactorGradArgs& a, int set, int slab, int half, float* sm) {
  constexpr bool SPLIT = Mma<T>::SCALED;  // fp16
  constexpr int RH = RP > 64 ? 64 : RP, SUMS = RH;  // ranks of a CTA; sums of a lane: 32 columns x RH / 32 lanes
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int part = warp % a.row_parts, slabs = LR_WARPS / a.row_parts;
  const int64_t col0 = (static_cast<int64_t>(slab) * slabs + warp / a.row_parts) * 32, col = col0 + 8 * q;
  const int j0 = half * RH;
  float acc[SUMS / 4][4];
#pragma unroll
  for (int i = 0; i < SUMS; ++i) acc[i / 4][i % 4] = 0.0f;
  const int start = a.plan.offset[set], size = a.plan.count[set], blocks = (size + 15) / 16;
  const bool there = col < a.in_ld;
  // BATCH blocks' rows and inner vectors on their way together, the places of the next ones read meanwhile: what counts is
  // that no load waits for another one's use (8192 rows of rank 16: 47 us a block at a time)
  constexpr int BATCH = RP <= 16 ? 4 : RP <= 32 ? 2 : 1, PIECES = RH / 8;  // of the inner vectors, high and low, for a block
  int route[BATCH][2];
  auto look_up = [&](int b0) {
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) route[u][h] = b0 + u * a.row_parts < blocks ? __ldg(a.plan.order + start + (b0 + u * a.row_parts) * 16 + h * 8 + g) : -1;
  };
  look_up(part);
  for (int b0 = part; b0 < blocks; b0 += BATCH * a.row_parts) {
    uint4 values[BATCH][2];
    uint2 high[BATCH][PIECES], low[BATCH][PIECES];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int b = b0 + u * a.row_parts;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = route[u][h];
        values[u][h] = load16(a.in + static_cast<int64_t>(r < 0 ? 0 : r / a.in_div) * a.in_ld + col, there && r >= 0);
      }
      const int64_t block = (static_cast<int64_t>(start / 16) + b) * RP;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        // right: ranks of the rows of fragment i / 2, then 8 further.  left: column c of tile i is rank RH / 4 (c / 2) + 2 i + c % 2, so
        // that a lane's ranks are neighbours
        const int j = j0 + (LEFT ? (g >> 1) * (RH / 4) + 2 * i + (g & 1) : i * 8 + g);
        high[u][i] = load8(a.inner.high + (block + j) * 16 + 4 * q, b < blocks);
        low[u][i] = load8(a.inner.low + (block + j) * 16 + 4 * q, b < blocks);
      }
    }
    look_up(b0 + BATCH * a.row_parts);
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      // tile t: columns col0 + 8 (c / 2) + 2 t + c % 2, the rows in pairs; fp16 values as the sum of two bf16 ones (exactly)
      uint32_t x[4][2], x_low[SPLIT ? 4 : 1][2];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t v = transpose8(word(values[u][h], t));
          if (SPLIT) {
            const float2 f = Mma<T>::unpack(v);
            split<__nv_bfloat16>(f.x, f.y, x[t][h], x_low[t][h]);
          } else x[t][h] = v;
        }
      using M = Mma<__nv_bfloat16>;
      if (!LEFT) {
#pragma unroll
        for (int m = 0; m < RH / 16; ++m) {
          const uint32_t hi[4] = {high[u][2 * m].x, high[u][2 * m + 1].x, high[u][2 * m].y, high[u][2 * m + 1].y};
          const uint32_t lo[4] = {low[u][2 * m].x, low[u][2 * m + 1].x, low[u][2 * m].y, low[u][2 * m + 1].y};
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            float(&d)[4] = acc[m * 4 + t];
            M::run(d, lo, x[t][0], x[t][1]);
            if (SPLIT) M::run(d, hi, x_low[t % (SPLIT ? 4 : 1)][0], x_low[t % (SPLIT ? 4 : 1)][1]);
            M::run(d, hi, x[t][0], x[t][1]);
          }
        }
      } else {
#pragma unroll
        for (int n = 0; n < RH / 8; ++n)
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            float(&d)[4] = acc[n * 2 + m];
            const uint32_t rows[4] = {x[2 * m][0], x[2 * m + 1][0], x[2 * m][1], x[2 * m + 1][1]};
            M::run(d, rows, low[u][n].x, low[u][n].y);
            if (SPLIT) {
              constexpr int L = SPLIT ? 4 : 1;
              const uint32_t rest[4] = {x_low[2 * m % L][0], x_low[(2 * m + 1) % L][0], x_low[2 * m % L][1], x_low[(2 * m + 1) % L][1]};
              M::run(d, rest, high[u][n].x, high[u][n].y);
            }
            M::run(d, rows, high[u][n].x, high[u][n].y);
          }
      }
    }
  }
  if (a.row_parts > 1) {
#pragma unroll
    for (int i = 0; i < SUMS; ++i) sm[(warp * SUMS + i) * 32 + lane] = acc[i / 4][i % 4];
    __syncthreads();
    if (part != 0) return;
    for (int p = 1; p < a.row_parts; ++p)
#pragma unroll
      for (int i = 0; i < SUMS; ++i) acc[i / 4][i % 4] += sm[((warp + p) * SUMS + i) * 32 + lane];
  }
  float any = 0.0f;
#pragma unroll
  for (int i = 0; i < SUMS; ++i) any += acc[i / 4][i % 4];
  if (!LEFT) {
#pragma unroll
    for (int m = 0; m < RH / 16; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = j0 + m * 16 + h * 8 + g;
        float y[8];
#pragma unroll
        for (int t = 0; t < 4; ++t) { y[2 * t] = a.scale * acc[m * 4 + t][2 * h]; y[2 * t + 1] = a.scale * acc[m * 4 + t][2 * h + 1]; }
        if (j < a.rank && col < a.width) store8_from_float(reinterpret_cast<T*>(a.out) + (static_cast<int64_t>(set) * a.rank + j) * a.width + col, y);
      }
  } else {
    constexpr int MINE = RH / 4;  // neighbouring ranks of a lane
    const int j = j0 + q * MINE;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // rows of the fragment: tile 2 m, then 2 m + 1
        const int64_t n = col0 + 8 * (g >> 1) + 2 * (2 * m + h) + (g & 1);
        if (n >= a.width) continue;
        T* row = reinterpret_cast<T*>(a.out) + (static_cast<int64_t>(set) * a.width + n) * a.rank;
        uint32_t packed[MINE / 2];
#pragma unroll
        for (int t = 0; t < RH / 8; ++t) packed[t] = Mma<T>::pack(a.scale * acc[t * 2 + m][2 * h], a.scale * acc[t * 2 + m][2 * h + 1]);
#pragma unroll
        for (int w = 0; w < MINE / 2; w += 2)
          if (j + 2 * w < a.rank) *reinterpret_cast<uint2*>(row + j + 2 * w) = make_uint2(packed[w], packed[w + 1]);
      }
  }
  if (__any_sync(0xFFFFFFFFu, isnan(any))) {
    __syncwarp();  // (values that other lanes stored)
    factor_grad_undefined<T, RP, LEFT>(a, set, col0, j0, RH);
  }
}

template <typename T, int RP>
__global__ void __launch_bounds__(LR_THREADS) factor_grad_kernel(const __grid_constant__ FactorGradArgs right, const __grid_constant__ FactorGradArgs left, int right_slabs) {
  extern __shared__ __align__(16) float sm[];
  const int slab = blockIdx.x;
  if (slab < right_slabs) factor_grad<T, RP, false>(right, blockIdx.y, slab, blockIdx.z, sm);
  else factor_grad<T, RP, true>(left, blockIdx.y, slab - right_slabs, blockIdx.z, sm);
}

// ---- host -------------------------------------------------------------------------------------------------

static int rank_pad(int64_t rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

struct LowRankPlan {
  int rp, ctas;
  bool solo;
  int64_t tiles;  // at most
};
// One row per tile while there are no more rows than SMs: no plan to wait for, and rows that share a set
// read it from the cache (64 rows of four adapters of rank 16: 15 us, grouped 18).  Else tiles of 16 rows; clusters
// while there are not tiles enough for two CTAs on every SM.
static LowRankPlan plan_low_rank(int64_t routes, int64_t sets, int64_t rank, bool grads) {
  LowRankPlan p;
  p.rp = rank_pad(rank);
  p.solo = !grads && routes <= 148;
  const int64_t used = routes < sets ? routes : sets;
  p.tiles = p.solo ? routes : max_tiles(routes, sets, ROW_STEP);
  const int64_t expected = p.solo ? routes : routes / ROW_STEP + used / 2 + 1;
  p.ctas = 1;
  while (p.ctas < 8 && 2 * p.ctas * expected <= 296) p.ctas *= 2;
  return p;
}

// `configured`: a bit per device, the shared-memory opt-in is a per-device attribute of the function.
static int launch_low_rank_kernel(void (*kernel)(LowRankArgs), int bytes, uint64_t& configured, const LowRankArgs& a, const LowRankPlan& p, cudaStream_t s) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !((configured >> dev) & 1ull)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return note_cuda_error(e);
    if (dev >= 0 && dev < 64) configured |= 1ull << dev;
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(p.tiles * p.ctas));
  config.blockDim = dim3(LR_THREADS);
  config.dynamicSmemBytes = bytes;
  config.stream = s;
  cudaLaunchAttribute attribute = {};
  if (p.ctas > 1) {  // (no early start of clusters, switch_matmul.cu)
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = static_cast<unsigned>(p.ctas);
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  } else {
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
  }
  config.attrs = &attribute;
  config.numAttrs = p.ctas > 1 || p.tiles <= EARLY_LAUNCH_MAX_BLOCKS ? 1 : 0;  // (common.cuh; 20,000 rows of 1024: 1 to 2 us of 48 for it)
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, a);
  return e == cudaSuccess ? KEEPVQ_OK : note_cuda_error(e);
}
template <typename T, int RP, bool BACK>
static int launch_low_rank(const LowRankArgs& a, const LowRankPlan& p, cudaStream_t s) {
  static uint64_t configured = 0;
  return launch_low_rank_kernel(low_rank_kernel<T, RP, BACK>, LowRankShape<RP, BACK>::BYTES, configured, a, p, s);
}
template <typename T, bool BACK>
static int launch_low_rank_of(const LowRankArgs& a, const LowRankPlan& p, cudaStream_t s) {
  if (p.rp == 16) return launch_low_rank<T, 16, BACK>(a, p, s);
  if (p.rp == 32) return launch_low_rank<T, 32, BACK>(a, p, s);
  if (p.rp == 64) return launch_low_rank<T, 64, BACK>(a, p, s);
  return launch_low_rank<T, 128, BACK>(a, p, s);
}
static int launch_low_rank_any(int dtype, bool back, const LowRankArgs& a, const LowRankPlan& p, cudaStream_t s) {
  if (dtype == KEEPVQ_BF16) return back ? launch_low_rank_of<__nv_bfloat16, true>(a, p, s) : launch_low_rank_of<__nv_bfloat16, false>(a, p, s);
  return back ? launch_low_rank_of<__half, true>(a, p, s) : launch_low_rank_of<__half, false>(a, p, s);
}

template <typename T, int RP>
static int launch_factor_grads(const FactorGradArgs& right, const FactorGradArgs& left, int64_t sets, cudaStream_t s) {
  constexpr int RH = RP > 64 ? 64 : RP, SMEM = LR_WARPS * RH * 32 * 4;
  auto kernel = factor_grad_kernel<T, RP>;
  if (SMEM > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return note_cuda_error(e);
  }
  const int64_t cols = 32 * (LR_WARPS / right.row_parts);
  const int64_t of_right = (right.width + cols - 1) / cols, of_left = (left.width + cols - 1) / cols;
  const dim3 grid(static_cast<unsigned>(of_right + of_left), static_cast<unsigned>(sets), RP / RH);
  kernel<<<grid, LR_THREADS, right.row_parts > 1 ? SMEM : 0, s>>>(right, left, static_cast<int>(of_right));
  KEEPVQ_CHECK_LAUNCH();
  return KEEPVQ_OK;
}
template <typename T>
static int launch_factor_grads_of(int rp, const FactorGradArgs& right, const FactorGradArgs& left, int64_t sets, cudaStream_t s) {
  if (rp == 16) return launch_factor_grads<T, 16>(right, left, sets, s);
  if (rp == 32) return launch_factor_grads<T, 32>(right, left, sets, s);
  if (rp == 64) return launch_factor_grads<T, 64>(right, left, sets, s);
  return launch_factor_grads<T, 128>(right, left, sets, s);
}

struct LowRankLayout {
  Plan plan;
  Inner inner, back;  // A x, and scale B^T grad
  float* route_dx;    // [routes, in_dim], where a row has several picks
  int64_t bytes;
};
static LowRankLayout lay_out_low_rank(void* base, int64_t routes, int64_t sets, int64_t in_dim, int64_t rank, int x_div, bool grads) {
  Scratch s{static_cast<char*>(base)};
  const LowRankPlan p = plan_low_rank(routes, sets, rank, grads);
  const int64_t blocks = max_places(routes, sets) / ROW_STEP + 1, values = grads ? blocks * ROW_STEP * p.rp : 0;
  LowRankLayout l = {};
  if (p.solo) return l;  // (nothing to keep: 0 bytes)
  l.plan = take_plan(s, routes, sets, ROW_STEP);
  for (Inner* i : {&l.inner, &l.back}) {
    i->high = s.take<uint16_t>(values);
    i->low = s.take<uint16_t>(values);
  }
  l.route_dx = grads && x_div > 1 ? s.take<float>(routes * in_dim) : nullptr;
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
  if (a.grad_ld > LR_MAX_PITCH || a.out_ld > LR_MAX_PITCH || a.base_ld > LR_MAX_PITCH) return KEEPVQ_ERR_CAPACITY;
  if (a.routes > 0 && (!a.x || !a.left || !a.right || !a.indices || (grads ? !a.grad : !a.out))) return KEEPVQ_ERR_NULL;
  for (const void* p : {a.x, a.left, a.right, a.grad, static_cast<const void*>(a.dx), static_cast<const void*>(a.dleft), static_cast<const void*>(a.dright)})
    if (!aligned_to(p, 16)) return KEEPVQ_ERR_ALIGN;
  if (!aligned_to(a.workspace, 256) || !aligned_to(a.indices, a.index_bits / 8) || !aligned_to(a.base, dtype_size(a.out_dtype)) || !aligned_to(a.out, dtype_size(a.out_dtype))) return KEEPVQ_ERR_ALIGN;
  return KEEPVQ_OK;
}

}  // namespace dense
}  // namespace keepvq

extern "C" {

int64_t keepvq_switch_low_rank_workspace_bytes(int64_t routes, int64_t sets, int64_t out_dim, int64_t in_dim, int64_t rank, int32_t x_div, int32_t grads) {
  using namespace keepvq::dense;
  if (const int rc = check_low_rank_sizes(routes, sets, out_dim, in_dim, rank, x_div)) return rc;
  return lay_out_low_rank(nullptr, routes, sets, in_dim, rank, x_div, grads != 0).bytes;
}

int keepvq_switch_low_rank_padded(const keepvq_switch_low_rank_args* args, int32_t ranks, void* stream) {
  using namespace keepvq::dense;
  if (!args) return KEEPVQ_ERR_NULL;
  const keepvq_switch_low_rank_args& a = *args;
  if (const int rc = check_low_rank(a, false)) return rc;
  if (ranks <= 0 || ranks > a.rank) return KEEPVQ_ERR_SHAPE;
  const LowRankLayout l = lay_out_low_rank(a.workspace, a.routes, a.sets, a.in_dim, a.rank, a.x_div, false);
  if (l.bytes > a.workspace_bytes) return KEEPVQ_ERR_CAPACITY;
  if (l.bytes > 0 && !a.workspace) return KEEPVQ_ERR_NULL;
  if (a.routes == 0) return KEEPVQ_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const LowRankPlan p = plan_low_rank(a.routes, a.sets, a.rank, false);
  LowRankArgs k = {};
  k.indices = {a.indices, a.index_bits};
  k.plan = l.plan;
  if (!p.solo)
    if (const int rc = make_plan(k.indices, a.routes, a.sets, ROW_STEP, ROW_STEP, l.plan, s)) return rc;
  k.in = static_cast<const uint16_t*>(a.x);
  k.in_ld = k.depth = a.in_dim;
  k.in_div = a.x_div;
  k.first = static_cast<const uint16_t*>(a.right);
  k.second = static_cast<const uint16_t*>(a.left);
  k.width = a.out_dim;
  k.rank = static_cast<int>(a.rank);
  k.ranks = ranks;
  k.sets = static_cast<int>(a.sets);
  k.first_scale = 1.0f;
  k.second_scale = a.scale;
  k.base = a.base;
  k.base_ld = a.base_ld;
  k.out = a.out;
  k.out_ld = a.out_ld;
  k.out32 = a.out_dtype == KEEPVQ_F32;
  k.whole = a.out_dim % 8 == 0 && keepvq::aligned_to(a.out, 16) && a.out_ld % 8 == 0 && keepvq::aligned_to(a.base, 16) && (!a.base || a.base_ld % 8 == 0);
  k.dead_rows = 1;
  k.solo = p.solo;
  return launch_low_rank_any(a.dtype, false, k, p, s);
}

int keepvq_switch_low_rank_grads_padded(const keepvq_switch_low_rank_args* args, int32_t ranks, void* stream) {
  using namespace keepvq::dense;
  if (!args) return KEEPVQ_ERR_NULL;
  const keepvq_switch_low_rank_args& a = *args;
  if (const int rc = check_low_rank(a, true)) return rc;
  if (ranks <= 0 || ranks > a.rank) return KEEPVQ_ERR_SHAPE;
  const LowRankLayout l = lay_out_low_rank(a.workspace, a.routes, a.sets, a.in_dim, a.rank, a.x_div, true);
  if (l.bytes > a.workspace_bytes) return KEEPVQ_ERR_CAPACITY;
  if (l.bytes > 0 && !a.workspace) return KEEPVQ_ERR_NULL;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.routes == 0) {
    for (void* p : {a.dleft, a.dright}) {
      const cudaError_t e = p ? cudaMemsetAsync(p, 0, a.sets * a.rank * (p == a.dleft ? a.out_dim : a.in_dim) * 2, s) : cudaSuccess;
      if (e != cudaSuccess) return keepvq::note_cuda_error(e);
    }
    return KEEPVQ_OK;
  }
  const LowRankPlan p = plan_low_rank(a.routes, a.sets, a.rank, true);
  const bool weights = a.dleft || a.dright;
  LowRankArgs k = {};
  k.indices = {a.indices, a.index_bits};
  k.plan = l.plan;
  if (const int rc = make_plan(k.indices, a.routes, a.sets, ROW_STEP, ROW_STEP, l.plan, s)) return rc;
  k.rank = static_cast<int>(a.rank);
  k.ranks = ranks;
  k.sets = static_cast<int>(a.sets);
  // q = scale B^T grad, and dx = A^T q
  k.in = static_cast<const uint16_t*>(a.grad);
  k.in_ld = a.grad_ld;
  k.in_div = 1;
  k.first = static_cast<const uint16_t*>(a.left);
  k.depth = a.out_dim;
  k.first_scale = a.scale;
  k.second = a.dx ? static_cast<const uint16_t*>(a.right) : nullptr;
  k.second_scale = 1.0f;
  k.width = k.out_ld = a.in_dim;
  k.out = l.route_dx ? static_cast<void*>(l.route_dx) : a.dx;
  k.out32 = l.route_dx != nullptr;
  k.whole = 1;
  k.dead_rows = a.dx && !l.route_dx;
  if (weights) k.keep = l.back;
  LowRankArgs inner = k;  // p = A x
  inner.in = static_cast<const uint16_t*>(a.x);
  inner.in_ld = inner.depth = a.in_dim;
  inner.in_div = a.x_div;
  inner.first = static_cast<const uint16_t*>(a.right);
  inner.first_scale = 1.0f;
  inner.second = nullptr;
  inner.dead_rows = 0;
  inner.keep = l.inner;
  if (a.dx || a.dright)
    if (const int rc = launch_low_rank_any(a.dtype, true, k, p, s)) return rc;
  if (a.dleft)
    if (const int rc = launch_low_rank_any(a.dtype, false, inner, p, s)) return rc;
  if (a.dx && l.route_dx)
    if (const int rc = sum_picks(l.route_dx, k.indices, a.sets, a.routes / a.x_div, a.x_div, a.in_dim, a.dx, a.dtype, s)) return rc;
  if (!weights) return KEEPVQ_OK;
  const int64_t mean = a.routes / (a.routes < a.sets ? a.routes : a.sets);
  const int row_parts = mean <= 16 ? 1 : mean <= 64 ? 2 : mean <= 256 ? 4 : 8;  // a part has one to four blocks of 16 rows, more beyond 512 rows
  FactorGradArgs right{static_cast<const uint16_t*>(a.x), a.in_dim, a.x_div, a.dright ? a.in_dim : 0, static_cast<int>(a.rank), row_parts, 1.0f, l.plan, l.back, static_cast<uint16_t*>(a.dright)};
  FactorGradArgs left{static_cast<const uint16_t*>(a.grad), a.grad_ld, 1, a.dleft ? a.out_dim : 0, static_cast<int>(a.rank), row_parts, a.scale, l.plan, l.inner, static_cast<uint16_t*>(a.dleft)};
  return a.dtype == KEEPVQ_BF16 ? launch_factor_grads_of<__nv_bfloat16>(p.rp, right, left, a.sets, s) : launch_factor_grads_of<__half>(p.rp, right, left, a.sets, s);
}

int keepvq_switch_low_rank(const keepvq_switch_low_rank_args* args, void* stream) {
  return keepvq_switch_low_rank_padded(args, args ? static_cast<int32_t>(args->rank) : 0, stream);
}

int keepvq_switch_low_rank_grads(const keepvq_switch_low_rank_args* args, void* stream) {
  return keepvq_switch_low_rank_grads_padded(args, args ? static_cast<int32_t>(args->rank) : 0, stream);
}

}  // extern "C"
