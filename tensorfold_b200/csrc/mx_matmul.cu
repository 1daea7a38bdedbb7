// Products of microscaled 4-bit rows with microscaled 4-bit weights on the block-scaled tensor-core path:
//
//     out[m, n] = sum over blocks b of 2^(sx[m, b] - 127) 2^(sw[n, b] - 127) sum_{i in b} qx[m, i] qw[n, i]
//
// Products of e2m1 values and powers of two are exact; sums are fp32 in tensor memory.  K runs in `sk` slices, a function of the
// weight's shape only; a slice is one chain of MMAs of 64 inputs, slices are added in order, so a row's bits depend neither on the
// number of rows nor on which of the forms below runs it.
//
// "Swap-AB": the weights are the MMA's A operand (M = 128 output columns a block), the rows its B operand (N = 8 to 192).  Both lie
// in memory as the MMA reads them (mx_layout.h), so a stage of 256 inputs is one bulk copy of 17 KB of weights beside the rows'
// copies; nothing passes through registers.  Scales go from the stage to tensor memory (tcgen05.cp, by the thread that issues the
// MMAs), to columns that belong to the stage's slot: they are free when the slot is.
//
// Forms (template):
//   FUSED    few rows (`fused_pays`, 16 at most): the block quantises bf16 rows itself into shared memory while its weights arrive,
//            one launch in all
//   GROUPED  a tile is a plan's item (expert, first, count) x 128 columns; activations may leave quantised, as the next
//            projection's operands
//   PAIR     prompts: two blocks on an SM pair share 256 columns x up to 192 rows, or an item's 128 (cta_group::2), half of the rows
//            in each one's shared memory.  The second block's copies land on its own barriers and a thread of it tells the first block, which issues
//            the MMAs
//   else     rows come quantised, as operands, in the ring.  `cluster` blocks (one a K slice) share a tile where there are few: each
//            sends its part to the blocks that own the rows, with counted stores through distributed shared memory
//
// Roles: warp 0 makes the barriers and loads weights, warp 1 owns tensor memory and issues the MMAs, warp 2 loads rows, warp 3
// forwards (PAIR); from warp 4 on groups of four drain (FUSED: 4-7 drain, the others but 0 and 1 quantise).
//
// What bounds it: windows by the weights' bytes and a fixed start and end (17408 x 5120 at one row 9.8 us among others, 4.8 TB/s;
// 248320 x 5120 99 us, 6.8 TB/s, where the measured copy runs at 6.55); prompts by shared memory, which takes a stage's copies and
// gives them to the MMAs again at 128 bytes a cycle, and by the stores of the results beside that (2048 rows by 17408 x 5120
// 81 us in bursts, 4.5 PFLOP/s; 9 less without the stores; one block a tile 87).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/tensorfold_b200.h"
#include "mx_layout.h"
#include "mx_quant.cuh"
#include "tf_ptx.cuh"

namespace tf {

int fail_moe(int code, const char* msg);
int cuda_fail_moe(cudaError_t e, const char* what);
int* device_error_word();
cudaError_t mx_rows_launch(const void* x, int64_t ldx, int m, int k, int rows, int tile, int64_t item_bytes, const int* items, const int* counts,
                           const int* members, int slots, int pairs, int max_items, void* out, cudaStream_t stream);

cudaError_t mx_rows_configure();

namespace {

constexpr int MX_RING_MAX = 12;
constexpr int MX_BAR_BYTES = 1024;
constexpr int MX_SMEM_MAX = 232448 - 1024 /* alignment slack */ - MX_BAR_BYTES;
constexpr int MX_FUSED_ROWS = 16;
constexpr int MX_QUANT_COLS = 128;                 // columns of the buffer in which a drain group collects rows to quantise
constexpr int MX_QUANT_ROWS = 16;
__host__ __device__ constexpr int quant_bytes(bool gated) {                     // two buffers in turn; SwiGLU leaves half of the columns
  return 2 * MX_QUANT_ROWS * ((gated ? MX_QUANT_COLS / 2 : MX_QUANT_COLS) + 4) * 4;
}
constexpr int MX_CLUSTER_MAX = 6;
constexpr int MX_TILE_MAX = 192;                   // rows of a tile: two accumulators and five slots' scales fill tensor memory

enum MxEpilogue : int { MX_STORE = 0, MX_RELU2 = 1, MX_SWIGLU = 2 };

struct MxParams {
  const uint8_t* w;
  int64_t sb_bytes, expert_stride;
  int N, M, K, steps, stages;
  int cluster;                  // blocks that share a tile, a K slice each (1: every block runs all slices)
  int sk;
  int bounds[MX_CLUSTER_MAX + 1];   // slice s holds stages bounds[s] .. bounds[s + 1]
  int ring;                     // slots
  int bufs;                     // FUSED: operands held in shared memory (2 with a plan, room permitting)
  int operand_stages;           // FUSED: stages of the longest slice
  // rows: operands (items `item_stride` bytes apart), or bf16 rows (FUSED)
  const uint8_t* b;
  int b_rows;
  int64_t item_stride;
  const __nv_bfloat16* x;
  int64_t ldx;
  int slots;                    // FUSED with a plan: rows of x are pair / slots (0: the pair itself)
  int tile, row_tiles;          // rows of a tile; tiles of rows (dense form)
  int step_cb, step_y;          // dense form: a cluster's next tile, as column blocks and row tiles further
  void* out;
  int64_t ldo;
  int out_f32, epi;
  float limit;
  // result quantised into operands instead (one an item, q_rows rows of q_blocks blocks)
  uint8_t* q;
  int q_rows, q_steps;
  int64_t q_item_stride;
  const int *items, *counts, *members;
  int experts, pairs, max_items;
  int settled;                  // no kernel in flight writes the weights or the plan: they are read before the dependency wait
  int lose;                     // self-test: the drain of cluster rank `lose` - 1 gives up its wait for the accumulator at once (0: none)
  int* err;
};

// Shared-memory matrix descriptors.  K-major, 8-row atoms one after another; swizzle 128 B (a stage's codes), 32 B (the last
// stage's steps), or none (scales: 16-byte lines, 8 to an atom of 128 bytes).
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t atom_bytes, uint32_t swizzle) {
  const uint32_t lo = ((addr >> 4) & 0x3FFFu) | (1u << 16);
  const uint32_t hi = (atom_bytes >> 4) | (1u << 14) | (swizzle << 29);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}
constexpr uint32_t SWIZZLE_NONE = 0, SWIZZLE_128 = 2, SWIZZLE_32 = 6;

// e2m1 x e2m1 with power-of-two scales per 32 inputs, K = 64, M = 128 (256 for a pair).  `half`: which two of a line's four scales.
template <bool PAIR>
__device__ __forceinline__ uint32_t instruction(int n, uint32_t half) {
  return (half * 2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) | ((PAIR ? 2u : 1u) << 27) | (half * 2u << 29);
}

template <bool PAIR>
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
  if constexpr (PAIR) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
  }
}
// 32 lines of 16 bytes to four columns, the same in each of the four lane groups (a pair: each block's own lines to its own columns).
template <bool PAIR>
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t from) {
  if constexpr (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(from) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(from) : "memory");
}
// Arrives once every MMA and copy issued so far is done; for a pair on that barrier of both blocks.
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
  else asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t in_block(uint32_t addr, uint32_t rank) {
  uint32_t to;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(addr), "r"(rank));
  return to;
}
// (A release at cluster scope would wait for the memory system each time; what these arrivals order, landed copies and tensor memory
// that has been read, is ordered by the barrier and the tcgen05 fence before them.)
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool elect_lane() {
  uint32_t one;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(one));
  return one != 0;
}
// Bounded wait by a whole warp.  The polling loop stays out of line: the roles share the instruction caches.
__device__ __noinline__ bool poll(uint32_t bar, uint32_t parity, uint32_t abort_word) {
#pragma unroll 1
  for (uint32_t i = 0; i < WAIT_POLLS; ++i) {
    uint32_t done;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done)
                 : "r"(bar), "r"(parity), "r"(20000u)
                 : "memory");
    if (done) return true;
    if ((i & 255u) == 255u && lds32(abort_word)) return false;
  }
  return false;
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, uint32_t abort_word) {
  if (__all_sync(0xFFFFFFFFu, mbar32_try_wait(bar, parity))) return true;
  return __all_sync(0xFFFFFFFFu, poll(bar, parity, abort_word));
}
// The copy and MMA roles are one thread each: a vote, an election and a reconvergence for each stage would cost more than its work.
__device__ __forceinline__ bool lane_wait(uint32_t bar, uint32_t parity, uint32_t abort_word) {
  return mbar32_try_wait(bar, parity) || poll(bar, parity, abort_word);
}
// One test that does not wait.  Asked for a stage before the one ahead of it is issued, its hundred cycles are hidden.
__device__ __forceinline__ uint32_t lane_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok;
}
// A block of a cluster sends slices into the others' shared memory, so none of them leaves before all have sent theirs or given up:
// every thread arrives once its sends are issued, and waits before the block returns.  Relaxed: the slices are counted by the barrier
// that their owner waits for.
__device__ __forceinline__ void sends_are_issued() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void all_sends_are_issued() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void let_copies_land() {
  for (int i = 0; i < 64; ++i) __nanosleep(20000);
}
__device__ __forceinline__ void tmem_load16(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]),
        "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const float* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "f"(v[0]),
      "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]),
      "f"(v[14]), "f"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Four values into the shared memory of block `rank` of the cluster, counted by that block's barrier.
__device__ __forceinline__ void store_remote(uint32_t addr, uint32_t bar, uint32_t rank, const float* v) {
  uint32_t to, at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(addr), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(bar), "r"(rank));
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to), "r"(__float_as_uint(v[0])),
               "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])), "r"(at)
               : "memory");
}

// Whether `ok` holds in all 128 threads that meet at this barrier.
__device__ __forceinline__ bool agreed(int barrier, bool ok) {
  uint32_t all;
  asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %2, 0;\nbarrier.cta.red.and.pred q, %1, 128, p;\nselp.u32 %0, 1, 0, q;\n}"
               : "=r"(all)
               : "r"(barrier), "r"(static_cast<uint32_t>(ok))
               : "memory");
  return all != 0;
}

// Fours of rows each of the c blocks of a cluster owns when they add their slices.
__host__ __device__ __forceinline__ int quads_of(int rows, int c) { return ((rows + 3) / 4 + c - 1) / c; }

// silu(gate) * up in fp32.  The fast division (2 units in the last place) gives 0 for a denominator past 2^126, which gates below -87.3 have
// and ups may bring back into sight: both sides are quarters, so that 1 + e^-g, finite to 2^128, stays below it.  The exact division
// takes its own subroutine: one routed row 21.0 us in place of 17.2, 391 rows of a 2 x 17408 x 5120 pair 57 in place of 47.
__device__ __forceinline__ float swiglu(float g, float u) { return __fdividef(0.25f * g, fmaf(0.25f, expf(-g), 0.25f)) * u; }

template <int NT, bool FUSED, bool GROUPED, bool PAIR = false>
struct MxShape {
  static constexpr int SBS = (NT + MX_SB - 1) / MX_SB;
  static constexpr int B_ROWS = PAIR ? NT / 2 : NT;                // rows of the tile in this block's shared memory
  static constexpr int B_BYTES = B_ROWS * 128 + SBS * MX_SCALES;
  static constexpr int SLOT = MX_UNIT + (FUSED ? 0 : B_BYTES);
  static constexpr int SF_COLS = 8 + 8 * SBS;                      // scale columns of a slot
  static constexpr int TMEM = FUSED ? 256 : 512;
  // Drain groups of four warps; they take sixteen rows in turn.  With a plan the drain has activations to compute and quantise: a routed
  // layer of 2048 rows takes 239 us with two groups, 237 with three, more with four (they leave a slot less).  2048 dense rows take 81
  // with two and with three, 150 rows 15.4 and 16.0.
  static constexpr int GROUPS = NT == 16 ? 1 : GROUPED ? 3 : 2;
  static constexpr int THREADS = 128 + 128 * (GROUPS > 2 ? GROUPS : 2);
  static constexpr bool SLICED = !GROUPED && NT <= MX_SB;          // may run all K slices itself (experts' and tall tiles' weights have one)
  static constexpr int CHUNKS = (NT / 16 + GROUPS - 1) / GROUPS;   // runs of sixteen rows a group drains
  // Slots: each has scale columns of its own.  (Pairs with seven slots in shared memory and five for scales, whose reuse the MMA
  // thread then waits for, took 94 us for 2048 rows by 17408 x 5120 against 88.)
  static constexpr int RING = (TMEM - 2 * NT) / SF_COLS < MX_RING_MAX ? (TMEM - 2 * NT) / SF_COLS : MX_RING_MAX;
};

// Stages of a block in order: a ring slot, and the parity of its barriers.
struct Ring {
  int slot;
  uint32_t phase;
  __device__ __forceinline__ void next(int ring) {
    if (++slot == ring) slot = 0, phase ^= 1u;
  }
};

template <int NT, bool FUSED, bool GROUPED, bool PAIR>
__global__ void __launch_bounds__(MxShape<NT, FUSED, GROUPED, PAIR>::THREADS, 1) mx_kernel(const MxParams p) {
  using S = MxShape<NT, FUSED, GROUPED, PAIR>;
  static_assert(!PAIR || !FUSED, "pairs are for prompts");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);              // [MX_RING_MAX] the slot's copies have landed
  uint64_t* empty = full + MX_RING_MAX;                            // [MX_RING_MAX] the MMAs that read the slot are done
  uint64_t* acc_full = empty + MX_RING_MAX;                        // [2]
  uint64_t* acc_empty = acc_full + 2;                              // [2]
  uint64_t* op_full = acc_empty + 2;                               // [2] FUSED with a plan: an operand is quantised
  uint64_t* op_empty = op_full + 2;                                // [2]
  uint64_t* parts = op_empty + 2;                                  // cluster: every part of this block's rows has come
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(parts + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t ring0 = smem_addr(smem) + MX_BAR_BYTES;           // slots, FUSED operands, then the exchange buffers
  const uint32_t operand0 = ring0 + p.ring * S::SLOT;
  const uint32_t operand_bytes = FUSED ? p.operand_stages * S::B_BYTES : 0;
  const uint32_t extra_off = MX_BAR_BYTES + p.ring * S::SLOT + (FUSED ? p.bufs * operand_bytes : 0);
  const uint32_t abort_word = smem_addr(const_cast<int*>(abort_flag));
  const uint32_t full32 = smem_addr(full), empty32 = smem_addr(empty), acc_full32 = smem_addr(acc_full), acc_empty32 = smem_addr(acc_empty);

  const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
  const int c = GROUPED || PAIR ? 1 : p.cluster;
  const int full_stages = p.steps >> 2, tail = p.steps & 3;
  uint32_t rank, mine, clusters;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%clusterid.x;" : "=r"(mine));
  asm("mov.u32 %0, %%nclusterid.x;" : "=r"(clusters));
  const int slice0 = c > 1 ? rank : 0, slice1 = c > 1 ? rank + 1 : p.sk;
  const int u0 = p.bounds[slice0], u1 = p.bounds[slice1];          // this block's stages of a tile

  auto give_up = [&](int code) {
    if (lane == 0) {
      *abort_flag = code;
      atomicCAS(p.err, 0, code);
    }
  };
  auto lost = [&](int code) {                                      // one thread gave up
    *abort_flag = code;
    atomicCAS(p.err, 0, code);
  };

  // Tiles: (row tile or item) x 128 columns.  Row tiles fastest, so that a column block's weights are read while they are in L2; with a
  // plan columns fastest.  A cluster takes every clusters-th tile; FUSED with a plan a run of neighbours, so that its rows are
  // quantised once an item.
  if (GROUPED && !p.settled) pdl_wait();                           // the plan may be the previous kernel's output
  constexpr bool RUNS = FUSED && GROUPED;
  const int nsb = (p.N + MX_SB - 1) / MX_SB, ncb = PAIR ? (nsb + 1) / 2 : nsb;
  const int tiles = ncb * (GROUPED ? min(p.counts[0], p.max_items) : p.row_tiles);
  const int first_tile = RUNS ? static_cast<int>(static_cast<int64_t>(tiles) * mine / clusters) : mine;
  const int end_tile = RUNS ? static_cast<int>(static_cast<int64_t>(tiles) * (mine + 1) / clusters) : tiles;
  const int tile_step = RUNS ? 1 : clusters;

  // A tile is looked up one ahead: `after` starts the loads of the plan's item, `settle` uses what they brought.
  struct Tile {
    int t;                                                         // number of the tile
    int y, cb;                                                     // item or row tile, column block (of a pair: two super-blocks)
    int expert, from, count;                                       // the item as it stands in the plan
    int m0, rows, n;                                               // first row (or member), rows, MMA N
    int64_t w;                                                     // offset of the weights
  };
  auto look_up = [&](Tile& ti) {
    if (GROUPED && ti.t < end_tile) {
      const int* item = p.items + 3 * ti.y;
      ti.expert = __ldg(item), ti.from = __ldg(item + 1), ti.count = __ldg(item + 2);
    }
  };
  auto settle = [&](Tile& ti) {
    ti.w = (PAIR ? min(2 * ti.cb + static_cast<int>(rank), nsb - 1) : ti.cb) * p.sb_bytes;
    if (GROUPED) {
      // an item that names an expert outside the table runs against expert 0 with no rows (the weights' thread reports it)
      const bool known = ti.expert >= 0 && ti.expert < p.experts;
      ti.w += (known ? ti.expert : 0) * p.expert_stride;
      ti.m0 = ti.from;
      ti.rows = known ? min(p.tile, ti.count) : 0;
      if (ti.m0 < 0 || ti.rows < 0 || ti.m0 > p.pairs - ti.rows) ti.rows = 0;
    } else {
      ti.m0 = ti.y * p.tile;
      ti.rows = min(p.tile, p.M - ti.m0);
    }
    ti.n = PAIR ? max(16, (ti.rows + 15) & ~15) : max(8, (ti.rows + 7) & ~7);
  };
  auto first = [&]() {
    Tile ti = {};
    ti.t = first_tile;
    if (GROUPED) ti.y = first_tile / ncb, ti.cb = first_tile - ti.y * ncb;
    else if (FUSED) ti.cb = first_tile;
    else if (p.row_tiles == 1) ti.cb = first_tile;
    else ti.cb = first_tile / p.row_tiles, ti.y = first_tile - ti.cb * p.row_tiles;
    look_up(ti);
    settle(ti);
    return ti;
  };
  auto after = [&](Tile ti) {
    ti.t += tile_step;
    if (GROUPED) {
      ti.cb += tile_step;
      while (ti.cb >= ncb) ti.cb -= ncb, ++ti.y;
    } else if (FUSED) {
      ti.cb += tile_step;
    } else {
      ti.y += p.step_y, ti.cb += p.step_cb;
      if (ti.y >= p.row_tiles) ti.y -= p.row_tiles, ++ti.cb;
    }
    look_up(ti);
    return ti;
  };

  // The weights' thread.  `fresh`: the first round of the ring, whose slots are free.
  const uint32_t last_bytes = tail * 4096 + mx_tail_scales(tail);
  Ring wr = {0, 1u};
  uint32_t w_ready = 1u;
  Tile wt = {}, wt_after = {};
  int wu = u0;
  bool w_ok = true;
  auto load_weights = [&](int stages, bool fresh) {
    while (stages-- > 0 && wt.t < end_tile) {
      if (!w_ready && !(w_ok = lane_wait(empty32 + 8 * wr.slot, wr.phase, abort_word))) return;
      const uint32_t bar = full32 + 8 * wr.slot, dst = ring0 + wr.slot * S::SLOT, bytes = wu < full_stages ? MX_UNIT : last_bytes;
      wr.next(p.ring);
      w_ready = fresh ? stages > 0 : lane_test(empty32 + 8 * wr.slot, wr.phase);
      mbar32_expect_tx(bar, bytes);
      bulk_load32(dst, p.w + wt.w + static_cast<int64_t>(wu) * MX_UNIT, bytes, bar);
      if (++wu == u1) {
        wu = u0;
        wt = wt_after;
        settle(wt);
        wt_after = after(wt);
      }
    }
  };

  // Rows w, w + stride, ... of `segments` runs of 1024 inputs each, quantised into the operand at `base`; four 16-byte loads a lane, the
  // next run's in flight meanwhile.  `row_at`: the row of x behind row r of the tile, below 0 for none.
  auto quantize_rows = [&](uint8_t* base, int rows, int w, int stride, auto&& row_at) {
    const int p0 = u0 * 32, pieces = min(p.steps * 8, u1 * 32) - p0;   // 16-byte pieces of a row in this slice (K padded to 64)
    const int segments = (pieces + 127) >> 7;
    int r = 0, seg = w;
    auto wrap = [&]() {
      while (seg >= segments) seg -= segments, ++r;
    };
    auto fetch = [&](uint4 (&v4)[4]) {
      const int64_t row = row_at(r);
      const uint4* from = reinterpret_cast<const uint4*>(p.x + row * p.ldx) + p0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int q = seg * 128 + 32 * j + lane;
        v4[j] = make_uint4(0u, 0u, 0u, 0u);
        if (row >= 0 && q < pieces && (p0 + q) * 8 < p.K) v4[j] = from[q];
      }
    };
    wrap();
    uint4 ahead[4];
    if (r < rows) fetch(ahead);
    while (r < rows) {
      const int at_r = r, q0 = seg * 128 + lane;
      uint4 v4[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v4[j] = ahead[j];
      seg += stride;
      wrap();
      if (r < rows) fetch(ahead);
      uint32_t codes[4], scale[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) codes[j] = quantize_block(v4[j], scale[j]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int q = q0 + 32 * j, b = q >> 2, u = b >> 3;
        if (q < pieces) {
          uint8_t* stage = base + u * S::B_BYTES;
          const uint32_t at = u0 + u < full_stages
                                  ? (at_r >> 3) * 1024 + (at_r & 7) * 128 + (((b & 7) ^ (at_r & 7)) << 4)
                                  : ((b & 7) >> 1) * (NT * 32) + (at_r >> 3) * 256 + (at_r & 7) * 32 + (((b & 1) ^ ((at_r >> 2) & 1)) << 4);
          *reinterpret_cast<uint32_t*>(stage + at + 4 * (q & 3)) = codes[j];
          if ((q & 3) == 0) stage[NT * 128 + ((b & 7) >> 2) * 512 + at_r * 16 + (b & 3)] = static_cast<uint8_t>(scale[j]);
        }
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  };

  // Set-up.  Warp 0 makes the barriers and goes on to load weights, which need nothing of the others (it arrives and does not
  // wait); the drain warps rehearse; where every tile has the same rows, the idle warps quantise them.
  const int group = (warp - 4) >> 2;                                 // drain group (warps 4-7; two or three groups where tiles are taller)
  const bool drains = warp >= 4 && group < S::GROUPS;
  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < MX_RING_MAX; ++i) mbar_init(full + i, FUSED ? 1 : PAIR && rank == 0 ? 3 : 2), mbar_init(empty + i, 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(acc_full + i, 1), mbar_init(acc_empty + i, (PAIR ? 8 : 4) * S::GROUPS);
        mbar_init(op_full + i, 4), mbar_init(op_empty + i, 1);
      }
      mbar_init(parts, 1);
      *abort_flag = 0;
      mbar_fence_init();
      wt = first();
      wt_after = after(wt);
      if (c > 1) {
        const int quads = (wt.rows + 3) / 4, share = quads_of(wt.rows, c);
        mbar32_expect_tx(smem_addr(parts), c * max(0, min(share, quads - static_cast<int>(rank) * share)) * MX_SB * 16);
      }
    }
    __syncwarp();
    asm volatile("barrier.cta.arrive 4, %0;" ::"n"(S::THREADS) : "memory");
    if (RUNS) asm volatile("barrier.cta.arrive 5, %0;" ::"n"(32 + 128) : "memory");
    if (c > 1 || PAIR) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    // ------------------------------------------------------------------ weights
    if (!GROUPED && !p.settled) pdl_wait();
    if (lane == 0) {
      load_weights(p.ring, true);
      load_weights(INT32_MAX, false);
      if (!w_ok) lost(ERR_WAIT_EMPTY), let_copies_land();
      if (GROUPED) {
        for (Tile ti = first(); ti.t < end_tile; ti = after(ti))
          if (ti.expert < 0 || ti.expert >= p.experts) atomicCAS(p.err, 0, ERR_BAD_ITEM);
      }
    }
    __syncwarp();
    if (c > 1 || PAIR) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  } else if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(S::TMEM) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(S::TMEM) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  } else if (FUSED && !GROUPED && !drains) {
    pdl_wait();
    quantize_rows(smem + (operand0 - smem_addr(smem)), p.M, warp >= 8 ? warp - 8 : warp + 2, 6, [](int r) { return static_cast<int64_t>(r); });
  }
  uint32_t tmem = 0;
  auto settle_in = [&]() {                                           // every warp but the first: the barriers and tensor memory are there
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    asm volatile("barrier.cta.sync 4, %0;" ::"n"(S::THREADS) : "memory");
    // The other blocks run, and their barriers are there, before anything is sent to them.  Warp 0's arrival releases the barriers;
    // the others' are relaxed: a release beside the weights' copies took as long as those, 1 to 4 us.
    if (c > 1 || PAIR) {
      asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);
    pdl_launch_dependents();
  };
  // (an item's rows lie behind a chain of look-ups: the warps that quantise them start on it at once, and only their first arrival
  // waits for the barriers: 1 us less a call)
  if (RUNS && warp >= 8) asm volatile("barrier.cta.arrive 4, %0;" ::"n"(S::THREADS) : "memory");
  else if (warp != 0 && !drains) settle_in();

  if (warp == 2 && !FUSED) {
    // ------------------------------------------------------------------ quantised rows
    pdl_wait();
    if (elect_lane()) {
      const int64_t stage_bytes = mx_stage_bytes(p.b_rows);
      bool ok = true;
      Ring r = {0, 1u};
      uint32_t ready = 1u;                                         // (a fresh slot's test passes)
      for (Tile ti = first(), then = after(ti); ti.t < end_tile && ok; ti = then, settle(ti), then = after(ti)) {
        const int sbs = mx_scale_blocks(ti.n);
        const uint8_t* src = p.b + ti.y * p.item_stride + u0 * stage_bytes;
#pragma unroll 1
        for (int u = u0; u < u1; ++u, src += stage_bytes) {
          if (!ready && !(ok = lane_wait(empty32 + 8 * r.slot, r.phase, abort_word))) break;
          const uint32_t bar = full32 + 8 * r.slot, dst = ring0 + r.slot * S::SLOT + MX_UNIT;
          r.next(p.ring);
          ready = lane_test(empty32 + 8 * r.slot, r.phase);
          // a pair: half of the rows to each block, all scales to both
          const int rows_here = PAIR ? ti.n / 2 : ti.n, skip = PAIR ? static_cast<int>(rank) * rows_here : 0;
          if (u < full_stages) {
            mbar32_expect_tx(bar, rows_here * 128 + sbs * MX_SCALES);
            bulk_load32(dst, src + skip * 128, rows_here * 128, bar);
            bulk_load32(dst + S::B_ROWS * 128, src + p.b_rows * 128, sbs * MX_SCALES, bar);
          } else {
            const uint32_t scales = sbs * mx_tail_scales(tail);
            mbar32_expect_tx(bar, rows_here * 32 * tail + scales);
            for (int j = 0; j < tail; ++j) bulk_load32(dst + j * S::B_ROWS * 32, src + (j * p.b_rows + skip) * 32, rows_here * 32, bar);
            bulk_load32(dst + S::B_ROWS * 128, src + tail * p.b_rows * 32, scales, bar);
          }
        }
      }
      if (!ok) lost(ERR_WAIT_EMPTY), let_copies_land();
    }
    __syncwarp();
  } else if (PAIR && warp == 3 && rank == 1) {
    // ------------------------------------------------------------------ this block's copies have landed: tell the first block
    if (elect_lane()) {
      const uint32_t first_full = in_block(full32, 0);
      bool ok = true;
      Ring r = {0, 0u};
      for (Tile ti = first(); ti.t < end_tile && ok; ti = after(ti)) {
#pragma unroll 1
        for (int u = u0; u < u1; ++u) {
          if (!(ok = lane_wait(full32 + 8 * r.slot, r.phase, abort_word))) break;
          arrive_remote(first_full + 8 * r.slot);
          r.next(p.ring);
        }
      }
      if (!ok) lost(ERR_WAIT_FULL);
    }
    __syncwarp();
  } else if (warp == 1 && (!PAIR || rank == 0)) {
    // ------------------------------------------------------------------ MMA issue (a pair's by its first block)
    // Measured on one block: an MMA of N columns takes N / 2 cycles but no less than 40 to issue, a scale copy 10 beside MMAs and
    // 37 alone, a commit 34 alone, a wait that passes 110.  The pipe takes few instructions ahead of it, so what a stage costs this
    // thread beyond them shows: descriptors are kept to adds, the next stage's barrier is tested before this stage's MMAs, and
    // the last stage, whose steps are regions of their own, has code of its own.
    if (elect_lane()) {
      const uint32_t sf0 = tmem + 2 * NT;
      const uint64_t a0 = desc(ring0, 1024, SWIZZLE_128), as0 = desc(ring0 + MX_SB * 128, 128, SWIZZLE_NONE);
      const uint64_t b0 = desc(FUSED ? operand0 : ring0 + MX_UNIT, 1024, SWIZZLE_128);
      const uint64_t bs0 = desc((FUSED ? operand0 : ring0 + MX_UNIT) + S::B_ROWS * 128, 128, SWIZZLE_NONE);
      // of the last stage, whose scales lie behind fewer codes
      const uint64_t a1 = desc(ring0, 256, SWIZZLE_32), as1 = desc(ring0 + tail * 4096, 128, SWIZZLE_NONE);
      const uint64_t b1 = desc(FUSED ? operand0 : ring0 + MX_UNIT, 256, SWIZZLE_32);
      const uint32_t sb_step = (FUSED ? MX_SCALES : mx_tail_scales(tail)) >> 4;
      bool ok = true;
      Ring r = {0, 0u};
      int use = 0, op = GROUPED ? -1 : 0, last_y = -1;
      uint32_t ready = 0;
      for (Tile ti = first(), then = after(ti); ti.t < end_tile && ok; ti = then, settle(ti), then = after(ti)) {
        const int n = ti.n, y = ti.y;
        if (RUNS && y != last_y) {
          last_y = y;
          ++op;
          if (!(ok = lane_wait(smem_addr(op_full + op % p.bufs), (op / p.bufs) & 1, abort_word))) break;
        }
        const int buf = RUNS ? op % p.bufs : 0;
        const uint32_t id0 = instruction<PAIR>(n, 0), id1 = instruction<PAIR>(n, 1);
        for (int s = slice0; s < slice1 && ok; ++s, ++use) {
          const int start = p.bounds[s], end = p.bounds[s + 1], last_whole = min(end, full_stages);
          if (use >= 2 && !(ok = lane_wait(acc_empty32 + 8 * (use & 1), ((use >> 1) - 1) & 1, abort_word))) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t d = tmem + (use & 1) * NT;
          uint32_t more = 0;                                         // 0: the first step of the slice overwrites the accumulator
          uint32_t fused_at = FUSED ? buf * (operand_bytes >> 4) : 0;
#pragma unroll 1
          for (int u = start; u < last_whole; ++u) {
            if (!ready && !(ok = lane_wait(full32 + 8 * r.slot, r.phase, abort_word))) break;
            const uint32_t at = r.slot * (S::SLOT >> 4), bt = FUSED ? fused_at : at, sa = sf0 + r.slot * S::SF_COLS, sb = sa + 8;
            const uint32_t done = empty32 + 8 * r.slot;
            r.next(p.ring);
            ready = lane_test(full32 + 8 * r.slot, r.phase);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              copy_scales<PAIR>(sa + 4 * h, as0 + at + 32 * h);
#pragma unroll
              for (int q = 0; q < S::SBS; ++q) copy_scales<PAIR>(sb + 4 * S::SBS * h + 4 * q, bs0 + bt + (MX_SCALES >> 4) * q + 32 * h);
            }
            mma_mxf4<PAIR>(d, a0 + at, b0 + bt, id0, sa, sb, more);
            mma_mxf4<PAIR>(d, a0 + at + 2, b0 + bt + 2, id1, sa, sb, 1u);
            mma_mxf4<PAIR>(d, a0 + at + 4, b0 + bt + 4, id0, sa + 4, sb + 4 * S::SBS, 1u);
            mma_mxf4<PAIR>(d, a0 + at + 6, b0 + bt + 6, id1, sa + 4, sb + 4 * S::SBS, 1u);
            commit<PAIR>(done);
            more = 1;
            if (FUSED) fused_at += S::B_BYTES >> 4;
          }
          if (!ok) break;
          if (end > full_stages) {                                   // the last stage: `tail` steps, each a region of its own
            if (!ready && !(ok = lane_wait(full32 + 8 * r.slot, r.phase, abort_word))) break;
            const uint32_t at = r.slot * (S::SLOT >> 4), bt = FUSED ? fused_at : at, sa = sf0 + r.slot * S::SF_COLS, sb = sa + 8;
            const uint32_t done = empty32 + 8 * r.slot;
            r.next(p.ring);
            ready = lane_test(full32 + 8 * r.slot, r.phase);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (2 * h >= tail) break;
              copy_scales<PAIR>(sa + 4 * h, as1 + at + 32 * h);
#pragma unroll
              for (int q = 0; q < S::SBS; ++q) copy_scales<PAIR>(sb + 4 * S::SBS * h + 4 * q, bs0 + bt + sb_step * q + 32 * h);
            }
#pragma unroll
            for (int j = 0; j < 3; ++j) {
              if (j >= tail) break;
              mma_mxf4<PAIR>(d, a1 + at + j * (4096 >> 4), b1 + bt + j * (S::B_ROWS * 32 >> 4), j & 1 ? id1 : id0, sa + 4 * (j >> 1),
                             sb + 4 * S::SBS * (j >> 1), j == 0 ? more : 1u);
            }
            commit<PAIR>(done);
          }
          commit<PAIR>(acc_full32 + 8 * (use & 1));
        }
        if (RUNS && ok && (then.t >= end_tile || then.y != y)) commit<PAIR>(smem_addr(op_empty + buf));
      }
      if (!ok) lost(ERR_WAIT_FULL);
    }
    __syncwarp();
  } else if (RUNS && warp >= 8) {
    // ------------------------------------------------------------------ bf16 rows of an item -> operand in shared memory
    pdl_wait();
    bool ok = true;
    int op = -1, last_y = -1;
    for (Tile ti = first(), then = after(ti); ti.t < end_tile; ti = then, settle(ti), then = after(ti)) {
      if (ti.y == last_y) continue;
      last_y = ti.y;
      ++op;
      if (op >= p.bufs && !(ok = warp_wait(smem_addr(op_empty + op % p.bufs), (op / p.bufs - 1) & 1, abort_word))) break;
      const int member = lane < ti.rows ? __ldg(p.members + ti.m0 + lane) : -1;    // of row `lane`: a tile has at most 16
      quantize_rows(smem + (operand0 - smem_addr(smem)) + (op % p.bufs) * operand_bytes, ti.rows, warp - 8, 4, [&](int r) -> int64_t {
        const int pair = __shfl_sync(0xFFFFFFFFu, member, r);
        return pair < 0 || pair >= p.pairs ? -1 : p.slots > 0 ? pair / p.slots : pair;
      });
      __syncwarp();
      if (op == 0) asm volatile("barrier.cta.sync 5, %0;" ::"n"(32 + 128) : "memory");
      if (lane == 0) mbar_arrive(op_full + op % p.bufs);
    }
    if (op < 0) asm volatile("barrier.cta.sync 5, %0;" ::"n"(32 + 128) : "memory");
    if (!ok) give_up(ERR_WAIT_EMPTY);
  }

  if (c > 1 && !drains) sends_are_issued();
  if (drains) {
    // ------------------------------------------------------------------ drain
    const int lg = warp & 3;
    const uint32_t empty_at = PAIR ? in_block(acc_empty32, 0) : acc_empty32;
    auto release = [&](int acc) {                                    // an accumulator has been read
      if constexpr (PAIR) arrive_remote(empty_at + 8 * acc);
      else mbar32_arrive(empty_at + 8 * acc);
    };
    auto block_of = [&](const Tile& ti) { return PAIR ? 2 * ti.cb + static_cast<int>(rank) : ti.cb; };
    const bool gated = p.epi == MX_SWIGLU;
    const int ncols = gated ? p.N / 2 : p.N;
    const bool wide = !p.out_f32 && (ncols & 7) == 0 && (p.ldo & 7) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
    const bool wide32 = p.out_f32 && (ncols & 3) == 0 && (p.ldo & 3) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
    // The output row of row n of the tile, below 0 for none.  With a plan lane l holds the pair of row l of the sixteen at hand.
    int pair16 = -1;
    auto pairs_of = [&](const Tile& ti, int n) {
      int pair = -1;
      if (GROUPED && p.q == nullptr && n + (lane & 15) < ti.rows) pair = __ldg(p.members + ti.m0 + n + (lane & 15));
      return pair;
    };
    auto row_of = [&](const Tile& ti, int n) -> int64_t {
      if (GROUPED) {
        const int pair = __shfl_sync(0xFFFFFFFFu, pair16, n & 15);
        return n < ti.rows && pair < p.pairs ? pair : -1;
      }
      return n < ti.rows ? ti.m0 + n : -1;
    };
    // v[j] = row n + j of the tile in output column `col`, a lane a column; COUNT runs of eight rows, 8 apart.  16-byte stores where the
    // output lets them (fp32 results one by one: second projection of a routed layer of 2048 rows 146 us in place of 106, one row 9.0
    // in place of 7.4)
    auto store = [&](auto count, const Tile& ti, const float* v, int n, int col) {
      constexpr int COUNT = decltype(count)::value;
      if (wide) {
        uint4 o[COUNT];
        int64_t row[COUNT];
#pragma unroll
        for (int h = 0; h < COUNT; ++h) {
          const float t[8] = {v[8 * h], v[8 * h + 1], v[8 * h + 2], v[8 * h + 3], v[8 * h + 4], v[8 * h + 5], v[8 * h + 6], v[8 * h + 7]};
          o[h] = transpose8(t, lane);                                // columns col - l8 .. col - l8 + 7 of row n + 8 h + l8
          row[h] = row_of(ti, n + 8 * h + (lane & 7));
        }
#pragma unroll
        for (int h = 0; h < COUNT; ++h)
          if (row[h] >= 0 && col < ncols) *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + row[h] * p.ldo + (col - (lane & 7))) = o[h];
      } else if (wide32) {
#pragma unroll
        for (int h = 0; h < 2 * COUNT; ++h) {
          const float4 o = transpose4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3], lane);   // columns col - l4 .. col - l4 + 3 of row n + 4 h + l4
          const int64_t row = row_of(ti, n + 4 * h + (lane & 3));
          if (row >= 0 && col < ncols) *reinterpret_cast<float4*>(static_cast<float*>(p.out) + row * p.ldo + (col - (lane & 3))) = o;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8 * COUNT; ++j) {
          const int64_t row = row_of(ti, n + j);
          if (row < 0 || col >= ncols) continue;
          if (p.out_f32) static_cast<float*>(p.out)[row * p.ldo + col] = v[j];
          else static_cast<__nv_bfloat16*>(p.out)[row * p.ldo + col] = __float2bfloat16_rn(v[j]);
        }
      }
    };
    // Activations of sixteen rows.  SwiGLU: gate in lanes 0-15, up in lanes 16-31 of the same outputs; the lower lanes come out
    // with rows 0-7 in v[0..7], the upper ones with rows 8-15.  Clips (limit > 0) are comparisons, not fminf: a NaN goes through; and
    // they stand apart, so that the eight values' chains run side by side.
    auto activate = [&](float* v) {
      if (gated) {
        const bool low = lane < 16;
        float u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float got = __shfl_xor_sync(0xFFFFFFFFu, low ? v[8 + j] : v[j], 16);
          u[j] = low ? got : v[8 + j];
          v[j] = low ? v[j] : got;
        }
        if (p.limit > 0.f) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            v[j] = v[j] > p.limit ? p.limit : v[j];
            u[j] = u[j] > p.limit ? p.limit : u[j] < -p.limit ? -p.limit : u[j];
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = swiglu(v[j], u[j]);
      } else if (p.epi == MX_RELU2) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float u = v[j] < 0.f ? 0.f : v[j];
          v[j] = u * u;
        }
      }
    };
    // Sixteen rows of activations to the next projection's operand: through shared memory, where four lanes see a block.
    int turn = 0;
    auto quantize16 = [&](const Tile& ti, const float* v, int n) {
      const int LINE = (gated ? MX_QUANT_COLS / 2 : MX_QUANT_COLS) + 4;
      // (a warp that writes a buffer again has passed the barrier after which the others read its last contents twice)
      float* rows = reinterpret_cast<float*>(smem + extra_off + group * quant_bytes(gated)) + turn * MX_QUANT_ROWS * LINE;
      turn ^= 1;
      const int shift = gated ? 3 : 4;                               // pieces of eight columns a row: 8 or 16
      if (gated) {
        float* to = rows + (lane < 16 ? 0 : 8) * LINE + lg * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < 8; ++j) to[j * LINE] = v[j];
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) rows[j * LINE + lg * 32 + lane] = v[j];
      }
      named_barrier(1 + group, 128);
      // the tile's blocks lie in one stage of the operand
      const int block0 = block_of(ti) << (shift - 2), u = block0 >> 3;
      uint8_t* op = p.q + ti.y * p.q_item_stride + u * mx_stage_bytes(p.q_rows);
      const bool whole = u < p.q_steps >> 2;
      const int q_tail = p.q_steps & 3;
      uint8_t* scales = op + (whole ? p.q_rows * 128 : p.q_rows * 32 * q_tail);
      for (int t = lg * 32 + lane; t < MX_QUANT_ROWS << shift; t += 128) {
        const int r = t >> shift, piece = t & ((1 << shift) - 1), row = n + r;
        const float4* from = reinterpret_cast<const float4*>(rows + r * LINE + piece * 8);
        const float4 lo = from[0], hi = from[1];
        float w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        uint32_t scale;
        const uint32_t codes = quantize_block(w, scale);
        const int b = (block0 & 7) + (piece >> 2);
        if (row < ti.rows && 8 * u + b < 2 * p.q_steps) {
          const int at = whole ? (row >> 3) * 1024 + (row & 7) * 128 + ((b ^ (row & 7)) << 4)
                               : (b >> 1) * p.q_rows * 32 + (row >> 3) * 256 + (row & 7) * 32 + (((b & 1) ^ ((row >> 2) & 1)) << 4);
          *reinterpret_cast<uint32_t*>(op + at + 4 * (piece & 3)) = codes;
          if ((piece & 3) == 0) scales[(b >> 2) * 512 + (row & 31) * 16 + (row >> 5) * 4 + (b & 3)] = static_cast<uint8_t>(scale);
        }
      }
    };

    // Sixteen rows at a time straight from tensor memory.  The loop is not unrolled and its body is kept small: unrolled over
    // a tile (5900 instructions) the warps mostly waited for instructions, and a tile of 256 rows took 42 us.  For the same reason
    // it runs once over no rows before the first accumulator is ready: its instructions are at hand then.
    bool ok = true, sending = c > 1;
    int use = 0;
    uint32_t lanes = 0;
    Tile ti = first(), then = {};
    if (GROUPED) then = after(ti);
    const int here = ti.rows;
    ti.rows = 0;
    if (ti.t >= end_tile) settle_in();
    for (bool rehearsal = true; ti.t < end_tile && ok;) {
      int pairs_ahead = pairs_of(ti, 16 * group);                    // (c is 1 with a plan)
      if (!rehearsal) {
        if (S::SLICED && slice1 - slice0 > 1) {
          // slices are added in registers, and the sum goes back to where the last one came from
          float acc[S::CHUNKS][16];
          for (int s = slice0; s < slice1; ++s, ++use) {
            ok = warp_wait(acc_full32 + 8 * (use & 1), (use >> 1) & 1, abort_word);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t src = lanes + (use & 1) * NT;
#pragma unroll
            for (int i = 0; i < S::CHUNKS; ++i) {
              if (16 * (S::GROUPS * i + group) >= ti.rows) break;
              float v[16];
              tmem_load16(src + 16 * S::GROUPS * i, v);
              tmem_loaded();
#pragma unroll
              for (int j = 0; j < 16; ++j) acc[i][j] = s == slice0 ? v[j] : acc[i][j] + v[j];
              if (s + 1 == slice1) tmem_store16(src + 16 * S::GROUPS * i, acc[i]);
            }
            if (s + 1 == slice1) {
              asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
              break;                                                 // (the loop below ends this use of the accumulator)
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) release(use & 1);
          }
        } else {
          ok = (c == 1 || p.lose != static_cast<int>(rank) + 1) && warp_wait(acc_full32 + 8 * (use & 1), (use >> 1) & 1, abort_word);
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        if (GROUPED && p.q != nullptr) ok = agreed(1 + group, ok);   // (a group's warps meet at barriers below: all of them or none)
        if (!ok) break;
      }
      const uint32_t src = lanes + (use & 1) * NT;
      const int share = max(1, quads_of(ti.rows, c));
      int n0 = 0;                                                    // first row this block finishes
      if (c > 1) {
        // Part [slice][four rows of the owner][128 columns][4] goes to the shared memory of the block that owns the rows (the host
        // launches one tile a cluster, so a block's buffer is written once).
        const uint32_t part = smem_addr(smem) + extra_off + (lg * 32 + lane) * 16;
#pragma unroll 1
        for (int n = 16 * group; n < ti.rows; n += 16 * S::GROUPS) {
          float v[16];
          tmem_load16(src + n - 16 * group, v);
          tmem_loaded();
          int owner = (n >> 2) / share, at = (n >> 2) - owner * share;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (n + 4 * j < ti.rows) store_remote(part + (rank * share + at) * (MX_SB * 16), smem_addr(parts), owner, v + 4 * j);
            if (++at == share) at = 0, ++owner;
          }
        }
        if (!rehearsal) {
          ok = warp_wait(smem_addr(parts), 0, abort_word);
          sends_are_issued();
          sending = false;
          if (!ok) break;
        }
        n0 = 4 * rank * share;
      }
      Tile own = ti;
      if (c > 1) own.rows = min(ti.rows, n0 + 4 * share);
      float ahead[16];                                               // the next sixteen rows are on their way meanwhile
      if (c == 1 && 16 * group < ti.rows) tmem_load16(src, ahead);
#pragma unroll 1
      for (int n = n0 + 16 * group; n < own.rows || (rehearsal && n < n0 + 16 * S::GROUPS); n += 16 * S::GROUPS) {
        float v[16];
        if (c > 1) {
          const float4* part = reinterpret_cast<const float4*>(smem + extra_off) + lg * 32 + lane;
          const int i = (n - n0) >> 2;
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = 0.f;
#pragma unroll 1
          for (int s = 0; s < c; ++s) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (i + j >= share) break;
              const float4 a = part[(s * share + i + j) * MX_SB];
              if (s == 0) {
                v[4 * j] = a.x, v[4 * j + 1] = a.y, v[4 * j + 2] = a.z, v[4 * j + 3] = a.w;
              } else {
                v[4 * j] += a.x, v[4 * j + 1] += a.y, v[4 * j + 2] += a.z, v[4 * j + 3] += a.w;
              }
            }
          }
        } else {
          tmem_loaded();
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = ahead[j];
          if (n + 16 * S::GROUPS < own.rows) tmem_load16(src + n + 16 * S::GROUPS - 16 * group, ahead);
        }
        pair16 = pairs_ahead;
        pairs_ahead = pairs_of(own, n + 16 * S::GROUPS);
        activate(v);
        if (GROUPED && p.q != nullptr) {
          quantize16(own, v, n);
        } else if (gated) {
          store(std::integral_constant<int, 1>(), own, v, n + (lane < 16 ? 0 : 8), block_of(ti) * 64 + lg * 16 + (lane & 15));
        } else {
          store(std::integral_constant<int, 2>(), own, v, n, block_of(ti) * MX_SB + lg * 32 + lane);
        }
      }
      if (rehearsal) {
        rehearsal = false;
        ti.rows = here;
        settle_in();
        lanes = tmem + (static_cast<uint32_t>(lg * 32) << 16) + 16 * group;
        pdl_wait();                                                  // nothing is written before the previous kernel is done
        continue;
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) release(use & 1);
      ++use;
      if (c > 1) break;                                              // (one tile a cluster)
      ti = GROUPED ? then : after(ti);
      settle(ti);
      if (GROUPED) then = after(ti);
    }
    if (!ok) give_up(ERR_WAIT_FULL);
    if (sending) sends_are_issued();                                 // gave up before it had any
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (PAIR) {                                                        // neither block leaves before both are done
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  } else if (c > 1) {
    all_sends_are_issued();
    if (*abort_flag) let_copies_land();                              // (the last ones sent to a block that did not wait for them)
  }
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM) : "memory");
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------------

int g_mx_sms[64] = {};

int g_mx_pairs[64] = {};            // pairs of blocks a device runs at once

int current_device() {
  int dev = 0;
  return cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 ? 63 : dev;
}
int device_sms() { return g_mx_sms[current_device()]; }

// K slices of an (n, k) weight: the most of 1, 2, 3, 4 and 6 whose blocks run at once as clusters, no slice below two stages (three in
// six slices).  A B200 holds 148, 74, 45, 33 or 22 clusters of that many blocks of this size (fewer than 148 / c: they lie inside a
// processor cluster), and a second round costs more than slices gain: 6144 x 5120 (48 column blocks) at one row takes 6.9, 6.1, 10.0 and
// 9.5 us in one to four slices, 5120 x 17408 (40) 17.6, 12.3, 11.1 and 15.6, 4096 x 4096 (32) 5.9, 5.0, 4.9 and 5.1.  Six slices serve
// windows and cost more rows a little: 1024 x 5120 in four / six, at 13 rows 6.8 / 6.0, at 32 6.9 / 7.0, at 300 9.9 / 10.3.
constexpr int MX_CLUSTERS[MX_CLUSTER_MAX + 1] = {0, 148, 74, 45, 33, 0, 22};
int slices_for(int n, int k) {
  const int blocks = (n + MX_SB - 1) / MX_SB, stages = mx_stages(mx_steps(k));
  int c = MX_CLUSTER_MAX;
  while (c > 1 && (blocks > MX_CLUSTERS[c] || stages < (c > 4 ? 3 : 2) * c)) --c;
  return c;
}

template <int NT, bool FUSED, bool GROUPED, bool PAIR = false>
cudaError_t launch(MxParams& p, int64_t tiles, bool quant_out, int sms, cudaStream_t stream) {
  using S = MxShape<NT, FUSED, GROUPED, PAIR>;
  int extra = quant_out ? S::GROUPS * quant_bytes(p.epi == MX_SWIGLU) : 0;
  if (p.cluster > 1) extra = p.cluster * quads_of(std::min(p.tile, p.M), p.cluster) * MX_SB * 16;
  const int operand = FUSED ? p.operand_stages * S::B_BYTES : 0;
  if (FUSED && p.bufs == 2 && MX_SMEM_MAX - extra - 2 * operand < 4 * S::SLOT) p.bufs = 1;
  const int room = MX_SMEM_MAX - extra - p.bufs * operand;
  p.ring = std::min(S::RING, room / S::SLOT);
  if (p.ring < 2) return cudaErrorInvalidConfiguration;              // (the callers' rules keep shapes that would not fit out)
  for (int i = 0; i <= p.sk; ++i) p.bounds[i] = static_cast<int>(static_cast<int64_t>(p.stages) * i / p.sk);
  const int width = PAIR ? 2 : p.cluster;                            // blocks of a cluster
  const int64_t most = PAIR ? std::max(1, g_mx_pairs[current_device()]) : std::max(1, sms / p.cluster);
  const int64_t clusters = p.cluster > 1 ? tiles : std::min(tiles, most);
  if (p.row_tiles > 0) p.step_cb = static_cast<int>(clusters / p.row_tiles), p.step_y = static_cast<int>(clusters % p.row_tiles);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * width));
  cfg.blockDim = dim3(S::THREADS);
  cfg.dynamicSmemBytes = 1024 + MX_BAR_BYTES + p.ring * S::SLOT + p.bufs * operand + extra;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  int count = 0;
  if (width > 1) {
    attrs[count].id = cudaLaunchAttributeClusterDimension;
    attrs[count].val.clusterDim.x = width, attrs[count].val.clusterDim.y = 1, attrs[count].val.clusterDim.z = 1;
    ++count;
  }
  // always: a block sets up under the previous kernel's end, and reads and writes global memory once that is done (weights and plan
  // earlier where they are settled; with a plan that is not, it waits before its set-up too)
  attrs[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[count].val.programmaticStreamSerializationAllowed = 1;
  ++count;
  cfg.attrs = attrs;
  cfg.numAttrs = count;
  return cudaLaunchKernelEx(&cfg, mx_kernel<NT, FUSED, GROUPED, PAIR>, p);
}

template <int NT, bool FUSED, bool GROUPED, bool PAIR = false>
cudaError_t configure() {
  return cudaFuncSetAttribute(mx_kernel<NT, FUSED, GROUPED, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
}

// Rows come as operands: the kernel whose tiles hold `tile` rows.
cudaError_t launch_rows(MxParams& p, int64_t tiles, int sms, cudaStream_t stream) {
  if (p.tile <= 16) return launch<16, false, false>(p, tiles, false, sms, stream);
  if (p.tile <= 64) return launch<64, false, false>(p, tiles, false, sms, stream);
  if (p.tile <= 128) return launch<128, false, false>(p, tiles, false, sms, stream);
  return launch<192, false, false>(p, tiles, false, sms, stream);
}
// Two blocks on an SM pair share a tile of 256 columns.
cudaError_t launch_pairs(MxParams& p, int64_t row_tiles, int sms, cudaStream_t stream) {
  return launch<MX_TILE_MAX, false, false, true>(p, ((p.N + MX_SB - 1) / MX_SB + 1) / 2 * row_tiles, false, sms, stream);
}
cudaError_t pairs_resident(int* pairs) {
  cudaError_t e = configure<MX_TILE_MAX, false, false, true>();
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2);
  cfg.blockDim = dim3(MxShape<MX_TILE_MAX, false, false, true>::THREADS);
  cfg.dynamicSmemBytes = 232448;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaOccupancyMaxActiveClusters(pairs, mx_kernel<MX_TILE_MAX, false, false, true>, &cfg);
}
// A plan's items.  Pairs take items of prompts where there are many tiles: their rows go to half as many blocks, but a tile begins and
// ends later.  Measured, us a layer of both projections (experts, D, NI, picks; up to 16 tiles an SM go to single blocks): 128, 2688,
// 1856, 6 at 2048 rows 210 in pairs / 216, at 64 rows 166 / 170, at 8000 rows 603 / 609; 64, 2048, 768, 8 at 2048 rows 124.0 / 124.3;
// 16, 4096, 1024, 2 at 512 rows 39.6 / 39.3, at 100 rows 30.0 / 28.8.
constexpr int PAIR_TILES = 16;
cudaError_t launch_items(MxParams& p, int64_t tiles, int sms, cudaStream_t stream) {
  if (p.tile <= 16) return launch<16, false, true>(p, tiles, p.q != nullptr, sms, stream);
  if (tiles < static_cast<int64_t>(PAIR_TILES) * sms) return launch<MX_SB, false, true>(p, tiles, p.q != nullptr, sms, stream);
  return launch<MX_SB, false, true, true>(p, tiles, p.q != nullptr, sms, stream);
}

int round8(int m) { return (m + 7) / 8 * 8; }

// Rows of a tile of an m-row call, blocks that share a tile (all K slices or one), and whether two blocks work as a pair: the fewest
// cycles by a plain model.  What paces a stage is shared memory, 128 bytes a cycle: 17 KB of weights and 136 bytes a row come in, and
// four MMAs read 16 KB and 128 bytes a row again; a pair halves the rows' part, but its stages pass from block to block.  A tile has a
// start and an end besides, and slices that blocks exchange cost by the row.  Tiles in several slices stay below 128 rows: the
// sums of taller ones do not fit the drain's registers.
// Measured, us from graphs on weights that L2 does not hold, as chosen / the other way: pairs 17408 x 5120 at 2048 rows 92 with / 101 without,
// at 700 35.2 with / 36.2, at 150 15.0 without / 18.0, 10240 x 2560 at 1000 19.8 with / 20.9; exchange 5120 x 17408 at 48 rows 14.1 with /
// 18.1 without, 6144 x 5120 at 24 8.2 with / 9.1, at 128 10.4 without / 13.7, 4096 x 4096 at 32 7.3 with / 7.9, at 128 8.9 without / 11.2.
// Where the model is off: 6144 x 5120 at 33 rows 8.9 without exchange / 8.5 with, at 48 9.2 / 8.9; 10240 x 2560 at 256 rows 15.0 without
// pairs / 13.9 with; and pairs are held to eight stages, which measurements do not bear out: 248320 x 1024 (four) at 600 rows 162
// without / 149 with.
struct Tiling {
  int tile, cluster;
  bool pair;
};
Tiling tiling_for(int m, int n, int stages, int sk) {
  constexpr double ENDS = 3200, STAGE = 270, ROW = 2.06, PAIR_ENDS = 2500, PAIR_STAGE = 440, PAIR_ROW = 1.05, SWAP = 300, SWAP_ROW = 60;
  const int64_t ncb = (n + MX_SB - 1) / MX_SB;
  Tiling best = {8, 1, false};
  double cost = 1e30;
  auto offer = [&](int64_t tiles, int at_once, double work, Tiling t) {
    const double here = static_cast<double>((tiles + at_once - 1) / at_once) * work;
    if (here <= cost) cost = here, best = t;
  };
  for (int t = 8; t <= (sk > 1 ? MX_SB : MX_TILE_MAX); t += 8) {
    const int64_t row_tiles = (m + t - 1) / t;
    const double stage = std::max(2.0 * t, STAGE + ROW * t);
    offer(ncb * row_tiles, MX_CLUSTERS[1], stages * stage + ENDS, {t, 1, false});
    if (sk > 1) offer(ncb * row_tiles, MX_CLUSTERS[sk], stages * stage / sk + ENDS + SWAP + SWAP_ROW * t, {t, sk, false});
    if (sk == 1 && t % 16 == 0 && m > MX_SB && stages >= 8)
      offer((ncb + 1) / 2 * row_tiles, MX_CLUSTERS[2], stages * (PAIR_STAGE + PAIR_ROW * t) + PAIR_ENDS, {t, 1, true});
    if (t >= m) break;
  }
  return best;
}

// Whether a block can hold its K slice of sixteen quantised rows beside a ring of four slots.
bool fused_fits(int k, int sk) {
  const int stages = mx_stages(mx_steps(k)), longest = (stages + sk - 1) / sk;
  return static_cast<int64_t>(longest) * MxShape<16, true, true>::B_BYTES + 4 * MX_UNIT + MX_CLUSTER_MAX * 4 * MX_SB * 4 <= MX_SMEM_MAX;
}

// Whether a block should quantise its rows itself: it holds its K slice of them beside a ring of four slots, and its six idle warps
// have few segments of 1024 inputs each.
// Measured, us from graphs on weights that L2 does not hold, in the block / from their own kernel, at 24 segments: 5120 x 17408 (six a row)
// at 4 rows 12.2 / 12.6, 14336 x 4096 (four) at 6 8.7 / 9.1, 6144 x 5120 (three) at 8 7.6 / 7.9, 10240 x 2560 (three) at 8 6.8 / 6.7, 4096 x 8192
// (two) at 12 8.1 / 8.4, 2048 x 8192 (two) at 12 7.6 / 7.2, the worst of nine; at 20 to 22 all nine gain, 1 to 12 %; past 24, 17408 x 5120
// (five) at 6 12.7 / 11.8.
constexpr int FUSED_SEGMENTS = 24;
bool fused_pays(int m, int k, int sk) {
  if (m > MX_FUSED_ROWS || !fused_fits(k, sk)) return false;
  const int longest = (mx_stages(mx_steps(k)) + sk - 1) / sk;
  return m * ((longest + 3) / 4) <= FUSED_SEGMENTS;
}

bool misaligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

}  // namespace

cudaError_t mx_configure(int device, int sms) {
  cudaError_t e = mx_rows_configure();
  if (e == cudaSuccess) e = configure<16, true, false>();
  if (e == cudaSuccess) e = configure<16, true, true>();
  if (e == cudaSuccess) e = configure<16, false, false>();
  if (e == cudaSuccess) e = configure<16, false, true>();
  if (e == cudaSuccess) e = configure<64, false, false>();
  if (e == cudaSuccess) e = configure<128, false, false>();
  if (e == cudaSuccess) e = configure<128, false, true>();
  if (e == cudaSuccess) e = configure<128, false, true, true>();
  if (e == cudaSuccess) e = configure<192, false, false>();
  int pairs = 0;
  if (e == cudaSuccess) e = pairs_resident(&pairs);
  if (e == cudaSuccess && device >= 0 && device < 64) g_mx_sms[device] = sms, g_mx_pairs[device] = pairs;
  return e;
}

}  // namespace tf

using namespace tf;

extern "C" {

int tf_mx_split(int n, int k) { return !mx_sizes(n, k) ? TF_ERR_ARG : slices_for(n, k); }

int64_t tf_mx_matmul_bytes(int m, int n, int k) {
  if (m < 1 || m > MX_LONGEST || !mx_sizes(n, k)) return TF_ERR_ARG;
  if (fused_pays(m, k, slices_for(n, k))) return 0;
  const int steps = mx_steps(k), tile = tiling_for(m, n, mx_stages(steps), slices_for(n, k)).tile;
  return (m + tile - 1) / tile * mx_operand_bytes(tile, steps);
}

static int mx_matmul(const void* x, int64_t ldx, int m, const void* tiled, int n, int k, void* out, int64_t ldo, int out_f32, int epi, float limit,
                     void* work, int64_t work_bytes, int pdl, int lose, void* stream) {
  if (m < 1 || m > MX_LONGEST || !mx_sizes(n, k)) return fail_moe(TF_ERR_ARG, "tf_mx_matmul: K must be a positive multiple of 32, n and m positive");
  if (epi < 0 || epi > 2 || (epi == 2 && n % 32) || (epi != 0 && out_f32)) return fail_moe(TF_ERR_ARG, "tf_mx_matmul: bad epilogue");
  if (!x || !tiled || !out || ldo < (epi == 2 ? n / 2 : n) || ldx < k) return fail_moe(TF_ERR_ARG, "tf_mx_matmul: null pointer or short rows");
  if (misaligned(x, 16) || (m > 1 && ldx % 8)) return fail_moe(TF_ERR_ALIGN, "tf_mx_matmul: x rows must start on 16-byte boundaries");
  if (misaligned(tiled, 16) || misaligned(work, 16)) return fail_moe(TF_ERR_ALIGN, "tf_mx_matmul: tiled weights and work must be 16-byte aligned");
  if (misaligned(out, out_f32 ? 4 : 2)) return fail_moe(TF_ERR_ALIGN, "tf_mx_matmul: out is not aligned to its type");
  const int64_t need = tf_mx_matmul_bytes(m, n, k);
  if (need > 0 && (!work || work_bytes < need)) return fail_moe(TF_ERR_ARG, "tf_mx_matmul: work is smaller than tf_mx_matmul_bytes");
  int* err = device_error_word();
  const int sms = device_sms();
  if (err == nullptr || sms < 1) return fail_moe(TF_ERR_STATE, "tf_mx_matmul: tf_init has not been called for the current device");
  MxParams p = {};
  p.w = static_cast<const uint8_t*>(tiled);
  p.N = n, p.M = m, p.K = k;
  p.steps = mx_steps(k), p.stages = mx_stages(p.steps);
  p.sb_bytes = mx_operand_bytes(MX_SB, p.steps);
  p.sk = slices_for(n, k);
  p.out = out, p.ldo = ldo, p.out_f32 = out_f32, p.epi = epi, p.limit = limit;
  p.err = err;
  p.lose = lose;
  p.bufs = 1;
  const int64_t ncb = (n + MX_SB - 1) / MX_SB;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (need == 0) {
    p.x = static_cast<const __nv_bfloat16*>(x), p.ldx = ldx;
    p.tile = MX_FUSED_ROWS;
    p.cluster = p.sk;
    p.operand_stages = (p.stages + p.sk - 1) / p.sk;
    p.row_tiles = 1;
    p.settled = pdl != 0;
    e = launch<16, true, false>(p, ncb, false, sms, s);
  } else {
    const Tiling t = tiling_for(m, n, p.stages, p.sk);
    p.tile = p.b_rows = t.tile, p.cluster = t.cluster;
    p.b = static_cast<const uint8_t*>(work), p.item_stride = mx_operand_bytes(t.tile, p.steps);
    const int64_t row_tiles = (m + t.tile - 1) / t.tile;
    if (row_tiles > 65535 || ncb * row_tiles > (1 << 28)) return fail_moe(TF_ERR_ARG, "tf_mx_matmul: too many rows");
    e = mx_rows_launch(x, ldx, m, k, t.tile, t.tile, p.item_stride, nullptr, nullptr, nullptr, 0, 0, 0, work, s);
    if (e != cudaSuccess) return cuda_fail_moe(e, "tf_mx_matmul: rows");
    p.settled = 1;                                                   // the rows' kernel waits before it lets this one start
    p.row_tiles = static_cast<int>(row_tiles);
    e = t.pair ? launch_pairs(p, row_tiles, sms, s) : launch_rows(p, ncb * row_tiles, sms, s);
  }
  return e == cudaSuccess ? TF_OK : cuda_fail_moe(e, "tf_mx_matmul");
}

int tf_mx_matmul(const void* x, int64_t ldx, int m, const void* tiled, int n, int k, void* out, int64_t ldo, int out_f32, int epi, float limit,
                 void* work, int64_t work_bytes, int pdl, void* stream) {
  return mx_matmul(x, ldx, m, tiled, n, k, out, ldo, out_f32, epi, limit, work, work_bytes, pdl, 0, stream);
}

int tf_mx_selftest_lost_slice(int slice, const void* x, const void* tiled, int n, int k, void* out, void* stream) {
  if (!mx_sizes(n, k)) return fail_moe(TF_ERR_ARG, "tf_mx_selftest_lost_slice: K must be a positive multiple of 32, n positive");
  const int sk = slices_for(n, k);
  if (sk < 2 || slice < 0 || slice >= sk || !fused_pays(1, k, sk))
    return fail_moe(TF_ERR_ARG, "tf_mx_selftest_lost_slice: one of the slices of a weight that runs in several, and in the block");
  return mx_matmul(x, k, 1, tiled, n, k, out, n, 1, MX_STORE, 0.f, nullptr, 0, 0, slice + 1, stream);
}

int64_t tf_mx_operand_bytes(int rows, int k) {
  if (!mx_sizes(rows, k)) return TF_ERR_ARG;
  return mx_operand_bytes(round8(rows), mx_steps(k));
}

int64_t tf_mx_experts_bytes(int k, int tile, int max_items) {
  if (tile < 8 || tile > MX_SB || max_items < 1 || !mx_sizes(tile, k)) return TF_ERR_ARG;
  return tile <= MX_FUSED_ROWS && fused_fits(k, 1) ? 0 : max_items * mx_operand_bytes(round8(tile), mx_steps(k));
}

int tf_mx_experts(const void* x, int64_t ldx, int slots, const void* tiled, int64_t expert_stride, int experts, int n, int k, const int* items,
                  const int* counts, const int* members, int pairs, int max_items, int tile, void* out, int64_t ldo, int out_f32,
                  void* out_operands, int epi, float limit, void* work, int64_t work_bytes, int pdl, void* stream) {
  if (experts < 1 || !mx_sizes(n, k) || pairs < 1 || max_items < 1 || max_items > 65535 || slots < 0)
    return fail_moe(TF_ERR_ARG, "tf_mx_experts: bad sizes (K a positive multiple of 32)");
  if (tile < 8 || tile > MX_SB || tile % 8) return fail_moe(TF_ERR_ARG, "tf_mx_experts: items of 8 to 128 pairs, in whole eights");
  if (epi < 0 || epi > 2 || (epi == 2 && n % 32)) return fail_moe(TF_ERR_ARG, "tf_mx_experts: bad epilogue");
  if (!tiled || !items || !counts || !members || (out == nullptr) == (out_operands == nullptr))
    return fail_moe(TF_ERR_ARG, "tf_mx_experts: null pointer, or not one of out and out_operands");
  const int ncols = epi == 2 ? n / 2 : n;
  if (out && (ldo < ncols || (epi != 0 && out_f32))) return fail_moe(TF_ERR_ARG, "tf_mx_experts: short rows, or activations in fp32");
  if (out_operands && ncols % MX_BLOCK) return fail_moe(TF_ERR_ARG, "tf_mx_experts: quantised results have a multiple of 32 columns");
  if (x && (ldx < k || misaligned(x, 16) || ldx % 8)) return fail_moe(TF_ERR_ALIGN, "tf_mx_experts: x rows must start on 16-byte boundaries");
  if (misaligned(tiled, 16) || expert_stride % 16 || misaligned(work, 16) || misaligned(out_operands, 16) || misaligned(out, out_f32 ? 4 : 2))
    return fail_moe(TF_ERR_ALIGN, "tf_mx_experts: weights, work and operands must start on 16-byte boundaries");
  const int rows = round8(tile);
  const int64_t operand = mx_operand_bytes(rows, mx_steps(k)), need = x ? tf_mx_experts_bytes(k, tile, max_items) : max_items * operand;
  if (need > 0 && (!work || work_bytes < need)) return fail_moe(TF_ERR_ARG, "tf_mx_experts: work is too small");
  int* err = device_error_word();
  const int sms = device_sms();
  if (err == nullptr || sms < 1) return fail_moe(TF_ERR_STATE, "tf_mx_experts: tf_init has not been called for the current device");
  MxParams p = {};
  p.w = static_cast<const uint8_t*>(tiled);
  p.N = n, p.M = pairs, p.K = k;
  p.steps = mx_steps(k), p.stages = mx_stages(p.steps);
  p.sb_bytes = mx_operand_bytes(MX_SB, p.steps), p.expert_stride = expert_stride;
  p.sk = 1, p.cluster = 1;
  p.out = out, p.ldo = ldo, p.out_f32 = out_f32, p.epi = epi, p.limit = limit;
  if (out_operands) {
    p.q = static_cast<uint8_t*>(out_operands), p.q_rows = rows, p.q_steps = mx_steps(ncols);
    p.q_item_stride = mx_operand_bytes(rows, p.q_steps);
  }
  p.items = items, p.counts = counts, p.members = members, p.experts = experts, p.pairs = pairs, p.max_items = max_items;
  p.err = err;
  p.tile = tile;
  p.settled = pdl != 0;
  const int64_t tiles = static_cast<int64_t>((n + MX_SB - 1) / MX_SB) * max_items;       // upper bound: the plan says how many
  if (tiles > (1 << 28)) return fail_moe(TF_ERR_ARG, "tf_mx_experts: too many tiles");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (x && need == 0) {
    p.x = static_cast<const __nv_bfloat16*>(x), p.ldx = ldx, p.slots = slots;
    // the next item's rows are quantised meanwhile (`launch` takes one buffer where two would leave under four slots).  Measured, us a
    // layer, two / one: 128 experts 2688 / 1856, top 6, 4 rows 35.9 / 37.0, 64 experts 2048 / 768, top 8, 16 rows 34.9 / 36.8
    p.bufs = 2, p.operand_stages = p.stages;
    e = launch<16, true, true>(p, tiles, out_operands != nullptr, sms, s);
  } else {
    if (x) {
      e = mx_rows_launch(x, ldx, 0, k, rows, tile, operand, items, counts, members, slots, pairs, max_items, work, s);
      if (e != cudaSuccess) return cuda_fail_moe(e, "tf_mx_experts: rows");
      p.settled = 1;                                                 // (as in tf_mx_matmul)
    }
    p.b = static_cast<const uint8_t*>(work), p.b_rows = rows, p.item_stride = operand;
    p.bufs = 1;
    e = launch_items(p, tiles, sms, s);
  }
  return e == cudaSuccess ? TF_OK : cuda_fail_moe(e, "tf_mx_experts");
}

}  // extern "C"
