// Products over 16-bit experts chosen per route, and their gradients, on the 5th-generation tensor
// cores.
//
//   forward   out[r]    = W[e_r] x[r / x_div]
//   dx        dx[r]     = W[e_r]^T grad[r], summed over a row's picks in fp32
//   dweight   dW[e]     = sum over e's routes of grad[r] x[r / x_div]^T
//
// One kernel for the three: a tile of 128 values along a result's rows (the M operand: weight rows,
// weight columns, columns of x) times up to N_MAX result rows (the N operand: a set's routes, or columns
// of grad).  The routes are the N operand because N is free in steps of 16: a set of five routes costs one
// such step of the tensor core and its own rows of shared memory, not a tile of 128.
//
//            M operand [128]                      N operand [<= N_MAX]                 contraction
//   forward  W[e] rows        (K-major box)       x rows, gathered     (K-major)       in_dim
//   dx       W[e] columns     (MN-major box)      grad rows, gathered  (K-major)       out_dim
//   dweight  x columns, rows gathered (MN-major)  grad columns, rows gathered (MN-major)  e's routes
//
// Two forms:
//   FEW   few routes per set, the time is reading weights: one CTA per tile, up to 64 result rows, the
//         set's rows gathered by TMA, four at a time by their index, straight from the caller's matrix
//   MANY  two CTAs (of one TPC) per tile of 256 x 256, whose tensor cores work as one: each loads half of
//         both operands.  Rows are first copied into the sets' order, so that they come as boxes of neighbouring rows
//         (gathered by TMA here too, 768 routes an expert took 375 us where copy and products take 42 + 278)
//
// Measured on a B200: 32 experts of 4096 x 2048 with 768 routes each, 280 us of products = 1.47 PFLOP/s, the tensor pipe 91 %
// active, and 42 us of copies; both gradients of 2048 x 4096, 310 + 303 us; 192 experts of 2304 x 5120 with 32 routes each,
// 717 us = 6.3 TB/s of weights; a token's six experts 24 us = 4.2 TB/s: the tiles of 96 CTAs, each as fast as its 128 KB in flight
// allow.  dweight of few routes is bound by writing (64 experts, 94 routes each: 312 us; a plain fill of those bytes 275).
#include "async_copy.cuh"
#include "switch_plan.cuh"

namespace keepvq {
namespace dense {

using fast::elect_one;
using fast::global_timer_ns;
using fast::mbar_complete;
using fast::mbar_expect_tx;
using fast::mbar_init;
using fast::smem_addr;

enum { FORWARD = 0, INPUT_GRAD = 1, WEIGHT_GRAD = 2 };
constexpr int M_TILE = 128, K_BLOCK = 64, N_STEP = 16, BOX_ROWS = 32;  // M_TILE: of a CTA; K_BLOCK: 128 bytes, a swizzled row
constexpr int OUT_WARPS = 8, MM_THREADS = 128 + OUT_WARPS * 32;
enum { WARP_M = 0, WARP_N = 1, WARP_MMA = 2, WARP_OUT = 4 };  // loaders of the two operands, the issuer; the warps of the epilogue
constexpr uint64_t MM_WAIT_NS = 2000000000ull;

// ---- instructions ---------------------------------------------------------------------------------
// PAIR: the barrier may be the first CTA's, the copy's target is this CTA's.
template <bool PAIR>
__device__ __forceinline__ void tma_box_3d(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z, uint32_t bar) {
  if (PAIR) asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];"
                         ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
  else asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                    ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
// Four rows of a matrix, 128 bytes of each from column x on.  The map's box is one row high.
__device__ __forceinline__ void tma_rows4(uint32_t dst, const CUtensorMap* map, int32_t x, const int4& rows, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(rows.x), "r"(rows.y), "r"(rows.z), "r"(rows.w), "r"(bar) : "memory");
}
// A box from shared memory to the matrix; what lies outside it is not written.
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, int32_t x, int32_t y, int32_t z, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];"
               ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(src) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// At most N of this thread's stores still have to read their source.
template <int N>
__device__ __forceinline__ void tma_stores_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
template <bool PAIR>
__device__ __forceinline__ void mma_16bit(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  if (PAIR) asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                         "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                         ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
  else asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                    "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                    ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// An arrival, when the products issued so far are done, on this barrier (of both CTAs of a pair).
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if (PAIR) asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
  else asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t of_first_cta(uint32_t addr) {
  uint32_t mapped;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(mapped) : "r"(addr));
  return mapped;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// PAIR: the barrier may be the other CTA's.  (Nothing but the copies themselves is ordered by this arrival;
// with .release.cluster it cost more than a K block's products.)
template <bool PAIR>
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  if (PAIR) asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
  else mbar_expect_tx(bar, bytes);
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t columns) {
  if (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns) {
  if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
  else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}
// 32 columns of this thread's lane of tensor memory.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                 "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
                 "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
               : "r"(taddr) : "memory");
}

// 16 lanes by 32 columns as fragments: of every 8 lanes x 8 columns a thread has lane thread / 4, columns
// 2 (thread % 4) and the next; v[4 c] .. v[4 c + 1] are those of columns 8 c .. 8 c + 7, + 2 the lanes 8 further.
__device__ __forceinline__ void tmem_ld_fragments(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                 "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(taddr) : "memory");
}
// Four 8 x 8 matrices of 16-bit values to shared memory, transposed; a lane has the address of one row.
__device__ __forceinline__ void store_transposed(uint32_t row, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(row), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Operand tiles with the 128-byte swizzle.  K-major: rows of 128 bytes along the contraction, groups of
// eight 1024 bytes apart.  MN-major: 64 values of M or N in 128 bytes, a row per step of the contraction,
// groups of eight 1024 bytes apart, the next 64 values one box (64 rows) on.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, bool mn_major) {
  const uint64_t lead = mn_major ? (K_BLOCK * 128) >> 4 : 1;
  return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (lead << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// Of this device: 1 since a wait of any call ran out, until asked for (keepvq_switch_matmul_wait_expired).  A call's own status word
// lies in its workspace, which a caller need not keep.
__device__ int32_t some_wait_expired;

// Wait of a whole warp, bounded by time: false after wait_ns in this wait (a call as a whole may take longer), or when
// another warp gave up.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint64_t wait_ns) {
  uint64_t deadline = 0;
  for (uint32_t spin = 0;; ++spin) {
    if (__all_sync(0xFFFFFFFFu, mbar_complete(bar, parity))) return true;
    if ((spin & 31u) == 31u) {
      if (__any_sync(0xFFFFFFFFu, *abort_flag)) return false;
      if (!deadline) deadline = global_timer_ns() + wait_ns;
      else if (__any_sync(0xFFFFFFFFu, global_timer_ns() > deadline)) { *abort_flag = 1; return false; }
    }
  }
}

template <uint32_t STAGES>
struct Ring {
  uint32_t index = 0, phase = 0;
  __device__ __forceinline__ void advance() {
    if (++index == STAGES) { index = 0; phase ^= 1u; }
  }
};

template <bool MANY>
struct Shape {
  static constexpr int N_MAX = MANY ? 256 : 64, N_CTA = MANY ? 128 : 64;  // result rows of a tile; of its N operand in a CTA
  static constexpr int PAD = MANY ? 32 : N_STEP;                           // what the number of result rows is rounded up to
  static constexpr uint32_t A_BYTES = M_TILE * K_BLOCK * 2, STAGE_BYTES = A_BYTES + N_CTA * K_BLOCK * 2;
  static constexpr uint32_t STAGES = 192 * 1024 / STAGE_BYTES;  // 6 or 8
  static constexpr uint32_t OUT_BYTES = (MANY ? 2 : 1) * OUT_WARPS * 32 * 32 * 2;  // 32 x 32 pieces of the result for each warp of the epilogue
  static constexpr uint32_t SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + OUT_BYTES;
  static constexpr uint32_t TMEM_COLS = 2 * N_MAX;              // two accumulators: one is written while the other is drained
};

struct MatmulArgs {
  int x_div, sets, dtype;
  int64_t out_dim, in_dim;
  void* out;        // result rows
  float* route_dx;  // dx before the pick sum, or null
  Plan plan;
  uint64_t wait_ns;  // limit of one wait
  int stall;         // the self-test's: the loader of the N operand leaves after its first tile
};

__device__ __forceinline__ uint32_t round_pair(uint32_t x, uint32_t y, bool bf16) {
  if (bf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(x), __uint_as_float(y));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(__uint_as_float(x), __uint_as_float(y));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// One tile of the result, or a CTA's half of it.
struct Item {
  int set, start, size;  // size: routes (the N operand's rows, or the contraction of dweight); start: their first place
  int m0, n0;            // first value along a result's row; first result row (dweight)
  int n, n_pad;          // result rows; rounded up
  int k_blocks;
};

template <int MODE, bool MANY>
__global__ void __launch_bounds__(MM_THREADS, 1) switch_matmul_kernel(MatmulArgs a, const __grid_constant__ CUtensorMap m_map, const __grid_constant__ CUtensorMap n_map,
                                                                      const __grid_constant__ CUtensorMap out_map) {
  using S = Shape<MANY>;
  static_assert(MANY || MODE != WEIGHT_GRAD, "the rows of dweight's operands are copied first");
  constexpr uint32_t STAGES = S::STAGES;
  constexpr bool M_MN = MODE != FORWARD, N_MN = MODE == WEIGHT_GRAD;
  constexpr int CTAS = MANY ? 2 : 1, N_MAX = S::N_MAX;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[2 * STAGES + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  // MANY neither starts early nor lets its successor: with thousands of blocks started early behind it, calls enqueued one
  // after the other stopped their stream, for a reason that is not known, and have not since
  if (!MANY) grid_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = MANY ? static_cast<int>(cluster_rank()) : 0;  // in the pair; the first CTA issues for both
  const uint32_t ring = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const uint32_t full = smem_addr(bars), empty = full + 8 * STAGES, acc_full = empty + 8 * STAGES, acc_empty = acc_full + 16;
  if (tid == 0) {
    abort_flag = 0;
    for (uint32_t s = 0; s < STAGES; ++s) { mbar_init(full + 8 * s, 2 * CTAS); mbar_init(empty + 8 * s, 1); }
    for (uint32_t s = 0; s < 2; ++s) { mbar_init(acc_full + 8 * s, 1); mbar_init(acc_empty + 8 * s, OUT_WARPS * CTAS); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == WARP_MMA) tmem_alloc<MANY>(smem_addr(&tmem_slot), S::TMEM_COLS);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (MANY) cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  if (!MANY) grid_wait();
  volatile int* aborted = &abort_flag;
  // the first CTA's barriers that both CTAs of a pair arrive on
  const uint32_t full0 = MANY ? of_first_cta(full) : full, acc_empty0 = MANY ? of_first_cta(acc_empty) : acc_empty;

  const int cols = static_cast<int>(MODE == FORWARD ? a.out_dim : a.in_dim);  // of a result row
  const int m_tiles = (cols + CTAS * M_TILE - 1) / (CTAS * M_TILE);
  const int n_tiles = MODE == WEIGHT_GRAD ? static_cast<int>((a.out_dim + N_MAX - 1) / N_MAX) : 1;
  const int depth_blocks = static_cast<int>(((MODE == FORWARD ? a.in_dim : a.out_dim) + K_BLOCK - 1) / K_BLOCK);
  const int items = m_tiles * (MODE == WEIGHT_GRAD ? n_tiles * a.sets : *a.plan.tiles);  // (below 2^31, check_sizes)
  const int first_item = blockIdx.x / CTAS, item_step = gridDim.x / CTAS;
  // Every role walks the same items on its own clock.
  auto item_at = [&](int i) {
    Item it;
    const int outer = static_cast<int>(static_cast<uint32_t>(i) / static_cast<uint32_t>(m_tiles));
    it.m0 = ((i - outer * m_tiles) * CTAS + rank) * M_TILE;
    if (MODE == WEIGHT_GRAD) {
      it.set = static_cast<int>(static_cast<uint32_t>(outer) / static_cast<uint32_t>(n_tiles));
      it.n0 = (outer - it.set * n_tiles) * N_MAX;
      it.start = a.plan.offset[it.set];
      it.size = a.plan.count[it.set];
      it.n = min(N_MAX, static_cast<int>(a.out_dim) - it.n0);
      it.k_blocks = (it.size + K_BLOCK - 1) / K_BLOCK;
    } else {
      const int4 t = a.plan.tile[outer];
      it.set = t.x; it.start = t.y; it.size = t.z;
      it.n0 = 0;
      it.n = it.size;
      it.k_blocks = depth_blocks;
    }
    it.n_pad = (it.n + S::PAD - 1) / S::PAD * S::PAD;
    return it;
  };
  bool ok = true, mma_issued = false;

  if (warp == WARP_M || warp == WARP_N) {
    // ================= the loaders ===============================================================
    Ring<STAGES> r;
    const uint32_t tile = ring + (warp == WARP_N ? S::A_BYTES : 0);
    const CUtensorMap* map = warp == WARP_M ? &m_map : &n_map;
    int left = a.stall && warp == WARP_N ? 1 : -1;  // tiles until this loader leaves; -1: it does not
    for (int i = first_item; i < items && ok; i += item_step) {
      const Item it = item_at(i);
      const int half = it.n_pad / CTAS;  // of the N operand, in this CTA
      int4 rows;
      if (!MANY && warp == WARP_N && lane * 4 < it.size) {  // rows past the last route repeat it: nobody looks at their columns
        const int div = MODE == FORWARD ? a.x_div : 1, last = it.size - 1, q = lane * 4;
        auto row_at = [&](int p) { return a.plan.order[it.start + min(p, last)] / div; };
        rows = make_int4(row_at(q), row_at(q + 1), row_at(q + 2), row_at(q + 3));
      }
      for (int kb = 0; kb < it.k_blocks; ++kb) {
        ok = left != 0 && wait_for(empty + 8 * r.index, r.phase ^ 1u, aborted, a.wait_ns);
        if (!ok) break;
        if (left > 0) --left;
        const uint32_t bar = full0 + 8 * r.index, dst = tile + r.index * S::STAGE_BYTES;
        if (!MANY && warp == WARP_N) {
          if (lane == 0) expect_bytes<MANY>(bar, static_cast<uint32_t>((it.size + 3) / 4 * 512));
          __syncwarp();
          if (lane * 4 < it.size) tma_rows4(dst + lane * 512, map, kb * K_BLOCK, rows, bar);
        } else if (elect_one()) {
          if (MODE == WEIGHT_GRAD) {  // 64 places of the set's routes (those behind the last are not multiplied) by 64 columns
            const int boxes = warp == WARP_M ? 2 : (half + 63) / 64, col0 = warp == WARP_M ? it.m0 : it.n0 + rank * half;
            expect_bytes<MANY>(bar, static_cast<uint32_t>(boxes * (K_BLOCK * 128)));
            for (int b = 0; b < boxes; ++b) tma_box_3d<MANY>(dst + b * (K_BLOCK * 128), map, col0 + b * 64, it.start + kb * K_BLOCK, 0, bar);
          } else if (warp == WARP_N) {
            const int boxes = (half + BOX_ROWS - 1) / BOX_ROWS;  // (rows behind the tile's: nobody looks at their columns)
            expect_bytes<MANY>(bar, static_cast<uint32_t>(boxes * (BOX_ROWS * 128)));
            for (int b = 0; b < boxes; ++b) tma_box_3d<MANY>(dst + b * (BOX_ROWS * 128), map, kb * K_BLOCK, it.start + rank * half + b * BOX_ROWS, 0, bar);
          } else {
            expect_bytes<MANY>(bar, S::A_BYTES);
            if (MODE == FORWARD) tma_box_3d<MANY>(dst, map, kb * K_BLOCK, it.m0, it.set, bar);
            else
              for (int b = 0; b < 2; ++b) tma_box_3d<MANY>(dst + b * (K_BLOCK * 128), map, it.m0 + b * 64, kb * K_BLOCK, it.set, bar);
          }
        }
        __syncwarp();
        r.advance();
      }
    }
  } else if (warp == WARP_MMA && rank == 0) {
    // ================= the issuer =================================================================
    Ring<STAGES> r;
    Ring<2> acc;
    // fp32 accumulator, fp16 or bf16 operands
    const uint32_t format = a.dtype == KEEPVQ_BF16 ? 1u : 0u;
    const uint32_t idesc0 = (1u << 4) | (format << 7) | (format << 10) | (static_cast<uint32_t>(M_MN) << 15) | (static_cast<uint32_t>(N_MN) << 16) | ((CTAS * M_TILE >> 4) << 24);
    for (int i = first_item; i < items && ok; i += item_step) {
      const Item it = item_at(i);
      if (it.k_blocks == 0) continue;  // (an expert without routes: the epilogue writes zeros)
      ok = wait_for(acc_empty + 8 * acc.index, acc.phase ^ 1u, aborted, a.wait_ns);
      const uint32_t idesc = idesc0 | (static_cast<uint32_t>(it.n_pad >> 3) << 17);
      for (int kb = 0; kb < it.k_blocks && ok; ++kb) {
        ok = wait_for(full + 8 * r.index, r.phase, aborted, a.wait_ns);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const int steps = MODE == WEIGHT_GRAD ? min(4, (it.size - kb * K_BLOCK + ROW_STEP - 1) / ROW_STEP) : 4;  // of 16
        if (elect_one()) {
          const uint32_t stage = ring + r.index * S::STAGE_BYTES;
          const uint64_t ad = operand_desc(stage, M_MN), bd = operand_desc(stage + S::A_BYTES, N_MN);
          for (int k = 0; k < steps; ++k)  // 16 of the contraction: 32 bytes of a row, or 16 rows of 128
            mma_16bit<MANY>(tmem + acc.index * N_MAX, ad + k * (M_MN ? 128 : 2), bd + k * (N_MN ? 128 : 2), idesc, (kb | k) != 0);
          mma_commit<MANY>(empty + 8 * r.index);
          if (kb == it.k_blocks - 1) mma_commit<MANY>(acc_full + 8 * acc.index);
        }
        __syncwarp();
        mma_issued = true;
        r.advance();
      }
      acc.advance();
    }
  } else if (warp >= WARP_OUT) {
    // ================= the epilogue ================================================================
    // a warp reaches a quarter of the accumulators' lanes; two share it, 32 result rows in turn (one warp alone took longer
    // to drain 256 of them, 530 cycles for 32, than the products of six K blocks)
    const int quadrant = warp & 3, turn = (warp - WARP_OUT) >> 2;
    constexpr int TURN = OUT_WARPS / 4 * 32;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quadrant * 32) << 16);
    const uint32_t piece = ring + STAGES * S::STAGE_BYTES + (warp - WARP_OUT) * (S::OUT_BYTES / OUT_WARPS);
    uint32_t flip = 0;  // which of this warp's two pieces is next (dweight)
    const bool bf16 = a.dtype == KEEPVQ_BF16;
    const bool whole = cols % 8 == 0;
    Ring<2> acc;
    if (MODE == FORWARD || (MODE == INPUT_GRAD && !a.route_dx)) {  // rows of dead routes
      for (int p = blockIdx.x * OUT_WARPS + warp - WARP_OUT; p < *a.plan.dead_count; p += gridDim.x * OUT_WARPS) {
        uint16_t* row = static_cast<uint16_t*>(a.out) + static_cast<int64_t>(a.plan.dead[p]) * cols;
        if (whole)
          for (int c = lane * 8; c < cols; c += 256) *reinterpret_cast<uint4*>(row + c) = make_uint4(0, 0, 0, 0);
        else
          for (int c = lane; c < cols; c += 32) row[c] = 0;
      }
    }
    for (int i = first_item; i < items && ok; i += item_step) {
      const Item it = item_at(i);
      if (it.k_blocks > 0) {
        ok = wait_for(acc_full + 8 * acc.index, acc.phase, aborted, a.wait_ns);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      }
      const int col = it.m0 + quadrant * 32;
      if (MODE == INPUT_GRAD && a.route_dx) {  // fp32, to be summed over the picks
        for (int c0 = turn * 32; c0 < it.n; c0 += TURN) {
          uint32_t v[32];
          const int n = min(32, it.n - c0), row = lane < n ? a.plan.order[it.start + c0 + lane] : 0;
          tmem_ld32(lanes + acc.index * N_MAX + c0, v);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const int64_t to = __shfl_sync(0xFFFFFFFFu, row, j);
            if (j < n && col + lane < cols) a.route_dx[to * cols + col + lane] = __uint_as_float(v[j]);
          }
        }
      } else {
        // 32 result rows at a time: fragments of tensor memory, rounded, transposed by the store to shared memory, where
        // a result row's 32 values of this warp become 64 bytes in four pieces (piece c of row r at c ^ (r / 2) % 4: no
        // bank twice); the next 32 rows' fragments are on their way meanwhile.  dweight's rows are neighbours: a store of the
        // whole piece by TMA, which has the same swizzle, from two pieces in turn
        const uint32_t from = lanes + acc.index * N_MAX;
        const int row8 = lane >> 2, c = col + (lane & 3) * 8;
        const uint32_t st_row = piece + (lane & 7) * 64 + (((lane >> 3) ^ ((lane >> 1) & 3)) << 4), ld_row = piece + row8 * 64 + (((lane & 3) ^ ((row8 >> 1) & 3)) << 4);
        uint32_t low[16], high[16];
        auto load = [&](int c0) {
          if (it.k_blocks > 0) {
            tmem_ld_fragments(from + c0, low);
            tmem_ld_fragments(from + (16u << 16) + c0, high);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) low[i] = high[i] = 0;
          }
        };
        if (turn * 32 < it.n) load(turn * 32);
        for (int c0 = turn * 32; c0 < it.n; c0 += TURN) {
          int64_t to[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int j = c0 + u * 8 + row8;
            to[u] = MODE == WEIGHT_GRAD || j >= it.n ? -1 : a.plan.order[it.start + j];
          }
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          uint32_t pair[4][4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            pair[u][0] = round_pair(low[4 * u], low[4 * u + 1], bf16);
            pair[u][1] = round_pair(low[4 * u + 2], low[4 * u + 3], bf16);
            pair[u][2] = round_pair(high[4 * u], high[4 * u + 1], bf16);
            pair[u][3] = round_pair(high[4 * u + 2], high[4 * u + 3], bf16);
          }
          if (c0 + TURN < it.n) load(c0 + TURN);
          if (MODE == WEIGHT_GRAD) {
            // a piece is written, and the turn passed on, only with a store of its own: "all but the last store have read"
            // then always means the store from this piece, also where a tile's columns end in front of this warp's
            if (col < cols) {
              if (lane == 0) tma_stores_read<1>();
              __syncwarp();
#pragma unroll
              for (int u = 0; u < 4; ++u) store_transposed(st_row + flip + u * 512, pair[u][0], pair[u][1], pair[u][2], pair[u][3]);
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
              if (lane == 0) tma_store_3d(&out_map, col, it.n0 + c0, it.set, piece + flip);
              flip ^= 32 * 64;
            }
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) store_transposed(st_row + u * 512, pair[u][0], pair[u][1], pair[u][2], pair[u][3]);
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              uint32_t w[4];
              asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(ld_row + u * 512) : "memory");
              uint16_t* dst = static_cast<uint16_t*>(a.out) + to[u] * cols + c;
              if (to[u] < 0) continue;
              if (whole) {
                if (c < cols) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
              } else {
#pragma unroll
                for (int d = 0; d < 8; ++d)
                  if (c + d < cols) dst[d] = static_cast<uint16_t>(w[d >> 1] >> (16 * (d & 1)));
              }
            }
            __syncwarp();
          }
        }
      }
      if (it.k_blocks > 0) {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive_cluster(acc_empty0 + 8 * acc.index);
        acc.advance();
      }
    }
    if (MODE == WEIGHT_GRAD && lane == 0) tma_stores_read<0>();  // (also of a warp that gave up)
  }

  __syncthreads();  // every role has left its loop
  if (*aborted) {
    // What is in flight is waited for, bounded: the issuer's products by one more commit, copies by time.
    if (tid == 0) { atomicExch(a.plan.status, 1); atomicExch(&some_wait_expired, 1); }
    const uint64_t grace = global_timer_ns() + 20000000ull;
    if (warp == WARP_MMA && mma_issued && elect_one()) mma_commit<MANY>(acc_full);
    while (global_timer_ns() < grace) __nanosleep(1000);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (MANY) cluster_sync();  // nobody arrives here, and nothing reads this CTA's memory, any more
  if (warp == WARP_MMA) tmem_free<MANY>(tmem, S::TMEM_COLS);
}

// ---- host ------------------------------------------------------------------------------------------

// A tensor map of 16-bit values in this GPU's own memory: `sets` matrices [rows, width], boxes of 64 values
// by box_rows rows of one of them (0: single rows, to be gathered), or of 32 values with the swizzle that goes with it.
static int value_map(CUtensorMap* map, const void* base, int dtype, int64_t width, int64_t row_values, int64_t rows, int64_t sets, uint32_t box_rows, uint32_t box_cols = K_BLOCK) {
  typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static EncodeTiled encode = nullptr;
  if (!encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found);
    if (e != cudaSuccess) return note_cuda_error(e);
    if (found != cudaDriverEntryPointSuccess || !fn) return KEEPVQ_ERR_UNSUPPORTED;
    encode = reinterpret_cast<EncodeTiled>(fn);
  }
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(sets)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(row_values * 2), static_cast<cuuint64_t>(row_values * 2 * rows)};
  const cuuint32_t box[3] = {box_cols, box_rows ? box_rows : 1, 1}, steps[3] = {1, 1, 1};
  const CUresult r = encode(map, dtype == KEEPVQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, box_rows ? 3 : 2, const_cast<void*>(base), dims, strides, box,
                            steps, CU_TENSOR_MAP_INTERLEAVE_NONE, box_cols == K_BLOCK ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? KEEPVQ_OK : KEEPVQ_ERR_LAUNCH;
}

// FEW reads the weights as fast as they come while TMA's gather keeps up, some 20 routes per expert (64 experts of 4096 x 2048,
// FEW / MANY: 8 routes each 169 / 185 us, 16 each 174 / 188, 24 each 206 / 192, 32 each 238 / 196); MANY wants tiles enough for its pairs.
static bool many_routes(int64_t routes, int64_t experts) { return routes > 16 * experts && routes >= 256; }

struct Waits {
  uint64_t ns = MM_WAIT_NS;
  int stall = 0;
};
struct Layout {
  Plan plan;
  uint16_t *x, *grad;  // rows in the plan's order (MANY)
  float* route_dx;     // [routes, in_dim], where a row has several picks
  int64_t bytes;
};
static Layout lay_out(void* base, int64_t routes, int64_t experts, int64_t out_dim, int64_t in_dim, int x_div, bool grads) {
  Scratch s{static_cast<char*>(base)};
  const bool many = many_routes(routes, experts);
  const int64_t places = max_places(routes, experts);
  Layout l;
  l.plan = take_plan(s, routes, experts, many ? Shape<true>::N_MAX : Shape<false>::N_MAX);
  l.x = many || grads ? s.take<uint16_t>(places * in_dim) : nullptr;
  l.grad = grads ? s.take<uint16_t>(places * align_up(out_dim, 8)) : nullptr;
  l.route_dx = grads && x_div > 1 ? s.take<float>(routes * in_dim) : nullptr;
  l.bytes = s.used;
  return l;
}

static int check_sizes(int64_t routes, int64_t experts, int64_t out_dim, int64_t in_dim, int32_t x_div) {
  if (routes < 0 || experts <= 0 || out_dim <= 0 || in_dim <= 0 || x_div <= 0 || in_dim % 8 != 0 || routes % x_div != 0) return KEEPVQ_ERR_SHAPE;
  if (routes > MAX_ROUTES || experts > MAX_SETS || out_dim > (1 << 24) || in_dim > (1 << 24)) return KEEPVQ_ERR_CAPACITY;
  // tiles are numbered in 32 bits, with room for a step beyond the last
  const int64_t most = (routes / 64 + experts + 1) * ((out_dim > in_dim ? out_dim : in_dim) / 128 + 1), of_weights = experts * (out_dim / 256 + 1) * (in_dim / 256 + 1);
  if (most > (int64_t{1} << 30) || of_weights > (int64_t{1} << 30)) return KEEPVQ_ERR_CAPACITY;
  return KEEPVQ_OK;
}

template <int MODE, bool MANY>
static int launch_tiles(const keepvq_switch_matmul_args& a, const Layout& l, const Waits& waits, cudaStream_t s) {
  using S = Shape<MANY>;
  MatmulArgs m{a.x_div, static_cast<int>(a.experts), a.dtype, a.out_dim, a.in_dim, MODE == FORWARD ? a.out : MODE == INPUT_GRAD ? a.dx : a.dweight, l.route_dx, l.plan, waits.ns, waits.stall};
  const int64_t places = max_places(a.routes, a.experts), grad_ld = MANY ? align_up(a.out_dim, 8) : a.grad_ld;
  CUtensorMap m_map, n_map, out_map;
  int rc = MODE == WEIGHT_GRAD ? value_map(&m_map, l.x, a.dtype, a.in_dim, a.in_dim, places, 1, K_BLOCK)
                               : value_map(&m_map, a.weight, a.dtype, a.in_dim, a.in_dim, a.out_dim, a.experts, MODE == FORWARD ? M_TILE : K_BLOCK);
  if (rc) return rc;
  const uint32_t box = MODE == WEIGHT_GRAD ? K_BLOCK : MANY ? BOX_ROWS : 0;
  rc = MODE == FORWARD ? value_map(&n_map, MANY ? l.x : a.x, a.dtype, a.in_dim, a.in_dim, MANY ? places : a.routes / a.x_div, 1, box)
                       : value_map(&n_map, MANY ? l.grad : a.grad, a.dtype, a.out_dim, grad_ld, MANY ? places : a.routes, 1, box);
  if (rc) return rc;
  out_map = m_map;
  if (MODE == WEIGHT_GRAD)
    if ((rc = value_map(&out_map, a.dweight, a.dtype, a.in_dim, a.in_dim, a.out_dim, a.experts, 32, 32))) return rc;
  auto kernel = switch_matmul_kernel<MODE, MANY>;
  static uint64_t configured = 0;  // one bit per device: the shared-memory opt-in is a per-device attribute of the function
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !((configured >> dev) & 1ull)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM_BYTES);
    if (e != cudaSuccess) return note_cuda_error(e);
    if (dev >= 0 && dev < 64) configured |= 1ull << dev;
  }
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(MANY ? sms / 2 * 2 : sms);
  config.blockDim = dim3(MM_THREADS);
  config.dynamicSmemBytes = S::SMEM_BYTES;
  config.stream = s;
  cudaLaunchAttribute attribute = {};
  if (MANY) {
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = 2;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  } else {
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
  }
  config.attrs = &attribute;
  config.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, m, m_map, n_map, out_map);
  return e == cudaSuccess ? KEEPVQ_OK : note_cuda_error(e);
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

static int forward_call(const keepvq_switch_matmul_args& a, const Waits& waits, cudaStream_t s) {
  if (const int rc = check_call(a, false)) return rc;
  const Layout l = lay_out(a.workspace, a.routes, a.experts, a.out_dim, a.in_dim, a.x_div, false);
  if (l.bytes > a.workspace_bytes) return KEEPVQ_ERR_CAPACITY;
  if (a.routes == 0) return KEEPVQ_OK;
  const bool many = many_routes(a.routes, a.experts);
  if (const int rc = make_plan({a.indices, a.index_bits}, a.routes, a.experts, many ? Shape<true>::N_MAX : Shape<false>::N_MAX, many ? Shape<true>::PAD : N_STEP, l.plan, s)) return rc;
  if (!many) return launch_tiles<FORWARD, false>(a, l, waits, s);
  const RowCopy x{a.x, l.x, a.in_dim, a.in_dim, a.x_div};
  if (const int rc = copy_rows(&x, 1, a.routes, a.experts, l.plan, s)) return rc;
  return launch_tiles<FORWARD, true>(a, l, waits, s);
}

static int grads_call(const keepvq_switch_matmul_args& a, const Waits& waits, cudaStream_t s) {
  if (const int rc = check_call(a, true)) return rc;
  const Layout l = lay_out(a.workspace, a.routes, a.experts, a.out_dim, a.in_dim, a.x_div, true);
  if (l.bytes > a.workspace_bytes) return KEEPVQ_ERR_CAPACITY;
  if (a.routes == 0) {
    const cudaError_t e = a.dweight ? cudaMemsetAsync(a.dweight, 0, a.experts * a.out_dim * a.in_dim * 2, s) : cudaSuccess;
    return e == cudaSuccess ? KEEPVQ_OK : note_cuda_error(e);
  }
  const Indices indices{a.indices, a.index_bits};
  const bool many = many_routes(a.routes, a.experts);
  if (const int rc = make_plan(indices, a.routes, a.experts, many ? Shape<true>::N_MAX : Shape<false>::N_MAX, many ? Shape<true>::PAD : N_STEP, l.plan, s)) return rc;
  const RowCopy copies[2] = {{a.grad, l.grad, a.grad_ld, align_up(a.out_dim, 8), 1}, {a.x, l.x, a.in_dim, a.in_dim, a.x_div}};
  if (many || a.dweight)
    if (const int rc = copy_rows(copies, a.dweight ? 2 : 1, a.routes, a.experts, l.plan, s)) return rc;
  if (a.dx) {
    if (const int rc = many ? launch_tiles<INPUT_GRAD, true>(a, l, waits, s) : launch_tiles<INPUT_GRAD, false>(a, l, waits, s)) return rc;
    if (l.route_dx)
      if (const int rc = sum_picks(l.route_dx, indices, a.experts, a.routes / a.x_div, a.x_div, a.in_dim, a.dx, a.dtype, s)) return rc;
  }
  return a.dweight ? launch_tiles<WEIGHT_GRAD, true>(a, l, waits, s) : KEEPVQ_OK;
}

__global__ void take_wait_expired(int32_t* word) { *word = atomicExch(&some_wait_expired, 0); }

}  // namespace dense
}  // namespace keepvq

extern "C" {

int64_t keepvq_switch_matmul_workspace_bytes(int64_t routes, int64_t experts, int64_t out_dim, int64_t in_dim, int32_t x_div, int32_t grads) {
  using namespace keepvq::dense;
  if (const int rc = check_sizes(routes, experts, out_dim, in_dim, x_div)) return rc;
  return lay_out(nullptr, routes, experts, out_dim, in_dim, x_div, grads != 0).bytes;
}

int keepvq_switch_matmul(const keepvq_switch_matmul_args* args, void* stream) {
  return args ? keepvq::dense::forward_call(*args, {}, static_cast<cudaStream_t>(stream)) : KEEPVQ_ERR_NULL;
}

int keepvq_switch_matmul_grads(const keepvq_switch_matmul_args* args, void* stream) {
  return args ? keepvq::dense::grads_call(*args, {}, static_cast<cudaStream_t>(stream)) : KEEPVQ_ERR_NULL;
}

int keepvq_switch_matmul_wait_expired(int32_t* word, void* stream) {
  if (!word) return KEEPVQ_ERR_NULL;
  if (!keepvq::aligned_to(word, 4)) return KEEPVQ_ERR_ALIGN;
  keepvq::dense::take_wait_expired<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(word);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? KEEPVQ_OK : keepvq::note_cuda_error(e);
}

int keepvq_switch_matmul_wait_selftest(const keepvq_switch_matmul_args* args, int32_t grads, int64_t wait_ns, void* stream) {
  using namespace keepvq::dense;
  if (!args) return KEEPVQ_ERR_NULL;
  if (wait_ns <= 0 || wait_ns > 1000000000ll) return KEEPVQ_ERR_SHAPE;
  const Waits waits{static_cast<uint64_t>(wait_ns), 1};
  return grads ? grads_call(*args, waits, static_cast<cudaStream_t>(stream)) : forward_call(*args, waits, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
