// dense with a table as its activation, gated by a second dense or not (cvmk_dense_lut_*): tensor-core
// products of int8 operands whose int32 sums never leave the chip.
//
// dense_lut_small_kernel: the weights are the 128-row operand of the tensor instructions and the rows of x
// (up to 128 of them) its columns, so a launch is one stream of weights whatever the batch.  A gated tile is
// 64 units: 64 rows of w and under them the same 64 of v, so that one accumulator holds both products of a
// unit; ungated, 128 units of w.  The reduction of a tile can be cut over a cluster of CTAs: every CTA
// writes its partial sums (int32: exact in any order) to its shared memory and each finishes its share of the
// units from all of them.
//
// dense_lut_pair_kernel: more rows.  Two CTAs of a cluster multiply a tile of 256 rows by 256 weight rows together
// (tcgen05 cta_group::2; gated: 128 of w, loaded by the first CTA, and the same 128 of v, loaded by the second), walking
// tiles with the requantisation of one beside the products of the next (two accumulators).
//
// What bounds them (one B200, among other launches): the small kernel the stream of weights (24 rows 4096 -> 16384 gated,
// 134 MB: 24.2 us, 0.85 of the copy rate) or, under 10 us, a trip to memory and the steps of a tile one after another (1 row
// 2048 -> 8192 gated, 33.6 MB: 7.8 us); the pair kernel the tensor pipe (4096 rows 4096 -> 16384 gated: 316 us in a burst, 0.78 of
// the measured rate of its instructions, 366 where a long run meets the power limit), and the requantisation where K is short
// (6000 rows 2048 -> 8192 with a residual: 73 us in a burst, 88 in a long run, 45 for the products alone).
//
// Reproduces dense -> [chain] -> cvm_lut -> broadcast_mul -> [chain] of the reference's operators
// (src/runtime/cpu/ops/ops.cc:34-75, :947-956, cpu/ops/broadcast.cc:33-36) bit for bit.
#include <cuda.h>
#include <cuda_runtime.h>
#include <string.h>
#include <algorithm>
#include "common.cuh"
#include "tc_common.cuh"

namespace cvmk {
namespace {

using namespace tc;

constexpr int THREADS = 320;     // warp 0: TMA, warp 1: MMA + TMEM, warps 2..9: epilogue
constexpr int BLOCK_K = 128;     // bytes of K a ring stage
constexpr int MAX_STAGES = 12;
constexpr int W_BYTES = BLOCK_M * BLOCK_K;          // of a stage: 128 rows of weights
constexpr int TABLE_SMEM_MAX = 16 * 1024;
constexpr int SMALL_SMEM_MAX = 224 * 1024, PAIR_SMEM_MAX = 206 * 1024;   // of a launch; a kernel's static part is less than the rest
constexpr uint32_t FULL_MASK = 0xffffffffu;

// A chain of a rounding shift with clamps, and for the one in front of a table the sum with a constant and the table's
// bounds, in three instructions: max(min(sum + (bias + add), hi), lo) >> shift.  The clamps come before the shift, which
// is monotone.  That is the definition's result where neither sum + bias, which wraps there, nor sum + bias + add overflows:
// for biases from `least` to `most`, which the kernel looks at 32 biases at a time.
struct Requant {
  int on, add, lo, hi, shift, least, most;
};

struct Params {
  void* y;
  long long y_pitch;
  int y_dtype, rows, units;
  int kblocks, gated, params_static;
  int unit_tiles, row_tiles, row_tile;
  int stages, split, split_log2, tmem_cols;
  const void* table;
  int table_len, table_dtype, table_smem;
  const int32_t *bias_w, *bias_v;
  int first_w, first_v;            // first step of the chain behind the bias
  const void* res;                 // operand of chain_y's *_T step, or nullptr
  int res_dtype, res_step;
  int* status;
  Requant qw, qv;
  int table_s_dtype;               // of the copy in shared memory
  DevChain cw, cv, cy;
  int straight;                    // 1: straight_part() takes the chains and the table, and the tensor operand if there is one
  int io;                          // and y, and that operand, go through shared memory by TMA: 1 y in int8, 2 y in int32
  int tail;                        // 1: chain_y ends with an int8 tensor and a clip, which run on packed 16-bit words
  uint32_t tail_lo, tail_hi;       // the clip's bounds in both halves
  DevChain head;                   // chain_y without those two steps
  DevChain ct;                     // ungated: steps of chain_y that the copy of the table has gone through already
};

__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ void cluster_sync() {   // (lanes may come to it apart)
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ int4 load_remote(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, int32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}

// The table's entries at a[j], which lie within it.  `table_s` is its copy in shared memory (table_smem).
template <int V>
__device__ __forceinline__ void look_up(const Params& p, const uint8_t* table_s, int32_t (&a)[V]) {
  if (p.table_smem) {
    if (p.table_s_dtype == CVMK_I8) {
#pragma unroll
      for (int j = 0; j < V; ++j) a[j] = reinterpret_cast<const int8_t*>(table_s)[a[j]];
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) a[j] = reinterpret_cast<const int32_t*>(table_s)[a[j]];
    }
  } else if (p.table_dtype == CVMK_I8) {
#pragma unroll
    for (int j = 0; j < V; ++j) a[j] = reinterpret_cast<const int8_t*>(p.table)[a[j]];
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) a[j] = reinterpret_cast<const int32_t*>(p.table)[a[j]];
  }
}
// The chain in front of the table, and the table.
template <int V>
__device__ __forceinline__ void activate(const Params& p, const uint8_t* table_s, int32_t (&a)[V]) {
  apply_chain<V>(p.cw, a, 0, 0, 0, nullptr, -1, p.first_w);
  const int last = p.table_len - 1;
#pragma unroll
  for (int j = 0; j < V; ++j) a[j] = min(max(a[j], 0), last);
  look_up<V>(p, table_s, a);
}

// N entries of the table, `threads` apart from i0 on, through the steps that are functions of an entry.
template <int N>
__device__ __forceinline__ void copy_entries(const Params& p, uint8_t* table_s, int i0, int threads) {
  int32_t v[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int i = i0 + j * threads;
    v[j] = i >= p.table_len ? 0 : (p.table_dtype == CVMK_I8 ? (int32_t) reinterpret_cast<const int8_t*>(p.table)[i] : reinterpret_cast<const int32_t*>(p.table)[i]);
  }
  apply_chain<N>(p.ct, v, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int i = i0 + j * threads;
    if (i >= p.table_len) break;
    if (p.table_s_dtype == CVMK_I8) reinterpret_cast<int8_t*>(table_s)[i] = (int8_t)v[j];
    else reinterpret_cast<int32_t*>(table_s)[i] = v[j];
  }
}
// The table's copy in shared memory.  A thread with more than one entry requests them together, whole words of 16 bytes where entries
// stay as they are: one after the other each is a trip to memory (10000 entries, a graph of 12 rows 112 -> 112: 22.5 us, now 8.2).
__device__ __forceinline__ void copy_table(const Params& p, uint8_t* table_s, int t, int threads) {
  if (p.table_len <= threads) {
    if (t < p.table_len) copy_entries<1>(p, table_s, t, threads);
    return;
  }
  int i = t;
  if (p.ct.n == 0 && (reinterpret_cast<uintptr_t>(p.table) & 15) == 0) {
    const int words = p.table_len * p.table_dtype >> 4;
    for (int w0 = t; w0 < words; w0 += 4 * threads) {
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (w0 + j * threads < words) v[j] = reinterpret_cast<const uint4*>(p.table)[w0 + j * threads];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (w0 + j * threads < words) reinterpret_cast<uint4*>(table_s)[w0 + j * threads] = v[j];
    }
    i += (words << 4) / p.table_dtype;
  }
  for (; i + threads < p.table_len; i += 8 * threads) copy_entries<8>(p, table_s, i, threads);
  if (i < p.table_len) copy_entries<1>(p, table_s, i, threads);
}

// Whether the bias leaves room for the sum (see Requant).
__device__ __forceinline__ bool in_room(int32_t bias, const Requant& q) { return bias >= q.least && bias <= q.most; }
// One channel's sums; `bias` has q.add in it.
template <int V>
__device__ __forceinline__ void requant_one(int32_t bias, const Requant& q, int32_t (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = max(__viaddmin_s32(v[j], bias, q.hi), q.lo) >> q.shift;
}
// V sums at `at` of every CTA of the cluster, added up.  (A word of another CTA takes a fifth of a microsecond to come: the
// requests go out together.)
template <int V>
__device__ __forceinline__ void sum_ranks(const Params& p, uint32_t at, int32_t (&a)[V]) {
  constexpr int AT_ONCE = 16 / V;   // CTAs
#pragma unroll
  for (int j = 0; j < V; ++j) a[j] = 0;
#pragma unroll
  for (int s0 = 0; s0 < 8; s0 += AT_ONCE) {
    if (s0 >= p.split) break;
    int4 g[AT_ONCE][V / 4];
#pragma unroll
    for (int s = 0; s < AT_ONCE; ++s)
      if (s0 + s < p.split) {
        const uint32_t from = p.split > 1 ? map_rank(at, (uint32_t)(s0 + s)) : at;
#pragma unroll
        for (int q = 0; q < V / 4; ++q) g[s][q] = load_remote(from + 16 * q);
      }
#pragma unroll
    for (int s = 0; s < AT_ONCE; ++s)
      if (s0 + s < p.split) {
#pragma unroll
        for (int q = 0; q < V / 4; ++q) { a[4 * q] += g[s][q].x; a[4 * q + 1] += g[s][q].y; a[4 * q + 2] += g[s][q].z; a[4 * q + 3] += g[s][q].w; }
      }
  }
}

// bytes of one row of partial sums: 16 more than the sums, so that eight rows of one column lie in different banks
__host__ __device__ inline int sums_pitch(int row_tile) { return row_tile * 4 + 16; }
__host__ __device__ inline int small_ring_bytes(int row_tile, int stages) {
  const int ring = stages * (W_BYTES + row_tile * BLOCK_K), sums = BLOCK_M * sums_pitch(row_tile);
  return ring > sums ? ring : sums;
}

// JOB: rows of x that a thread finishes at a time, 4 or 8 (few rows: more threads at work; many: fewer instructions an element:
// 256 rows 256 -> 8192 21.6 us with 4, 13.2 with 8; 8 rows 4096 -> 4096 7.7 and 8.7).
template <int JOB>
__global__ void __launch_bounds__(THREADS)
dense_lut_small_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                       const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar_full[MAX_STAGES];
  __shared__ uint64_t bar_empty[MAX_STAGES];
  __shared__ uint64_t bar_acc;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  __shared__ int32_t bias_s[BLOCK_M];   // of the tile's 128 weight rows

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = uniform((int)(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  const int rank = uniform(p.split > 1 ? (int)cluster_rank() : 0);
  const int tile = (int)blockIdx.x >> p.split_log2;
  const int ut = tile / p.row_tiles, row0 = (tile - ut * p.row_tiles) * p.row_tile;
  const int tile_units = p.gated ? 64 : 128, unit0 = ut * tile_units;
  const int kb0 = (rank * p.kblocks) >> p.split_log2, mine = (((rank + 1) * p.kblocks) >> p.split_log2) - kb0;
  const int stage_bytes = W_BYTES + p.row_tile * BLOCK_K;
  uint8_t* const table_s = smem + small_ring_bytes(p.row_tile, p.stages);

  touch_params(p);
  const bool leader = elect_one();
  const uint32_t ring = smem_u32(smem);
  auto load_weights = [&](int s, int kb) {   // of K block kb0 + kb, and announces all of the stage's bytes
    mbar_expect_tx(&bar_full[s], (uint32_t)stage_bytes);
    const int col = (kb0 + kb) * BLOCK_K;
    tma_load_2d(smem + s * stage_bytes, &tmap_w, &bar_full[s], col, unit0);
    tma_load_2d(smem + s * stage_bytes + W_BYTES / 2, p.gated ? &tmap_v : &tmap_w, &bar_full[s], col, p.gated ? unit0 : unit0 + 64);
  };
  auto load_x = [&](int s, int kb) { tma_load_2d(smem + s * stage_bytes + W_BYTES, &tmap_x, &bar_full[s], (kb0 + kb) * BLOCK_K, row0); };
  const int first = min(p.stages, mine);
  if (warp == 0) {
    if (leader) {
      for (int s = 0; s < p.stages; ++s) {
        mbar_init(&bar_full[s], 1);
        mbar_init(&bar_empty[s], 1);
      }
      mbar_init(&bar_acc, 1);
      abort_flag = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (!p.params_static) pdl_wait();
    if (leader)
      for (int i = 0; i < first; ++i) load_weights(i, i);
    __syncwarp();
  } else if (warp == 1) {
    // (the next kernel may start only once this CTA has its TMEM columns)
    tmem_alloc(&tmem_slot, (uint32_t)p.tmem_cols);
    pdl_trigger();
  } else {
    if (!p.params_static) pdl_wait();
    const int t = (int)threadIdx.x - 64;
    if (t < BLOCK_M) {
      const bool up = p.gated && t >= 64;
      const int u = unit0 + (up ? t - 64 : t);
      const int32_t* b = up ? p.bias_v : p.bias_w;
      bias_s[t] = b && u < p.units ? b[u] : 0;
    }
    if (p.table_smem) copy_table(p, table_s, t, THREADS - 64);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = (uint32_t)uniform((int)tmem_slot);

  if (warp == 0) {
    pdl_wait();
    if (leader) {
      for (int i = 0; i < first; ++i) load_x(i, i);
      int stage = 0;
      uint32_t phase = 0;
      for (int i = p.stages; i < mine; ++i) {
        if (!mbar_wait(&bar_empty[stage], phase, &abort_flag, 1)) break;
        load_weights(stage, i);
        load_x(stage, i);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t idesc = umma_idesc_i8(p.row_tile);
    const uint64_t desc0 = umma_desc(ring, BLOCK_K);
    const uint32_t lo0 = (uint32_t)desc0, hi = (uint32_t)(desc0 >> 32);
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; i < mine; ++i) {
      if (!mbar_wait(&bar_full[stage], phase, &abort_flag, 3)) break;
      tc_fence_after();
      const uint32_t al = lo0 + (uint32_t)(stage * stage_bytes >> 4);
      if (leader) {
        mma_i8_k<4>(tmem_base, al, hi, al + (W_BYTES >> 4), hi, idesc, (uint32_t)i);
        if (i + p.stages < mine) mma_commit(&bar_empty[stage]);   // (nobody waits for the last ones)
      }
      if (++stage == p.stages) { stage = 0; phase ^= 1; }
    }
    if (leader) mma_commit(&bar_acc);
    __syncwarp();
  }

  // Every CTA's partial sums go to its ring, which is idle once the accumulator is complete.
  const int pitch = sums_pitch(p.row_tile);
  if (warp >= 2) {
    const int quarter = warp & 3, half = warp >= 6 ? 1 : 0, row = quarter * 32 + lane;
    const bool ok = __all_sync(0xffffffffu, mbar_wait(&bar_acc, 0u, &abort_flag, 4));
    tc_fence_after();
    for (int c = half * 16; ok && c < p.row_tile; c += 32) {
      int32_t v[16];
      tmem_ld16(tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)c, v);
      int4* dst = reinterpret_cast<int4*>(smem + row * pitch + c * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) dst[j] = make_int4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (p.split > 1) cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, (uint32_t)p.tmem_cols);
  }
  // This CTA's share of the units, JOB rows of x a thread and turn.
  if (!abort_flag) {
    pdl_wait();
    const int share = tile_units >> p.split_log2, jobs = share * ((p.row_tile + JOB - 1) / JOB);
    for (int k = (int)threadIdx.x; k < jobs; k += THREADS) {
      const int q = k / share, ul = rank * share + k - q * share, unit = unit0 + ul, r0 = row0 + JOB * q;
      if (unit >= p.units || r0 >= p.rows) continue;
      const int n = min(JOB, p.rows - r0);
      const long long lin = (long long)r0 * p.y_pitch + unit;
      int32_t a[JOB], b[JOB], pre[JOB] = {};
      if (p.res) {
#pragma unroll
        for (int j = 0; j < JOB; ++j)
          if (j < n) pre[j] = p.res_dtype == CVMK_I8 ? reinterpret_cast<const int8_t*>(p.res)[lin + j * p.y_pitch]
                                                     : reinterpret_cast<const int32_t*>(p.res)[lin + j * p.y_pitch];
      }
      const uint32_t at = ring + (uint32_t)(ul * pitch + 4 * JOB * q), at_v = at + (uint32_t)(64 * pitch);
      const int32_t ba = bias_s[ul], bb = bias_s[p.gated ? ul + 64 : ul];
      sum_ranks(p, at, a);
      if (p.gated) sum_ranks(p, at_v, b);
      if (p.qw.on && in_room(ba, p.qw)) {
        requant_one(ba + p.qw.add, p.qw, a);
        look_up<JOB>(p, table_s, a);
      } else {
#pragma unroll
        for (int j = 0; j < JOB; ++j) a[j] += ba;
        activate<JOB>(p, table_s, a);
      }
      if (p.gated) {
        if (p.qv.on && in_room(bb, p.qv)) {
          requant_one(bb + p.qv.add, p.qv, b);
        } else {
#pragma unroll
          for (int j = 0; j < JOB; ++j) b[j] += bb;
          apply_chain<JOB>(p.cv, b, 0, 0, 0, nullptr, -1, p.first_v);
        }
#pragma unroll
        for (int j = 0; j < JOB; ++j) a[j] = (int32_t)((uint32_t)a[j] * (uint32_t)b[j]);
      }
      apply_chain<JOB, true>(p.cy, a, 0, 0, 0, pre, p.res_step);
#pragma unroll
      for (int j = 0; j < JOB; ++j)
        if (j < n) {
          if (p.y_dtype == CVMK_I8) reinterpret_cast<int8_t*>(p.y)[lin + j * p.y_pitch] = (int8_t)a[j];
          else reinterpret_cast<int32_t*>(p.y)[lin + j * p.y_pitch] = a[j];
        }
    }
  }
  __syncwarp();
  if (p.split > 1) cluster_sync();   // nobody still reads this CTA's memory
  if (abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);   // copies in flight land before shared memory is released
    if (lane == 0 && p.status) atomicOr(p.status, 0x400 | abort_flag);
  }
}

// ---------------------------------------------------------------------------------------------
// Pairs of CTAs
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];" ::
                   "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t bar) {   // of either CTA, an address of the cluster's window
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Both sums of a gated chunk with one wait.
__device__ __forceinline__ void tmem_ld_two(uint32_t ta, uint32_t tb, int32_t (&a)[16], int32_t (&b)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%32];\n"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%33];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]), "=r"(a[8]), "=r"(a[9]), "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15]),
        "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]), "=r"(b[4]), "=r"(b[5]), "=r"(b[6]), "=r"(b[7]), "=r"(b[8]), "=r"(b[9]), "=r"(b[10]), "=r"(b[11]), "=r"(b[12]), "=r"(b[13]), "=r"(b[14]), "=r"(b[15])
      : "r"(ta), "r"(tb)
      : "memory");
}

// 16 values of one row from or to memory that may begin and end anywhere: whole 16-byte words where all `n` = 16 are there
// and the address allows it.
__device__ __forceinline__ void load_run(const void* base, int dtype, long long lin, int n, int32_t (&t)[16]) {
  const uint8_t* at = reinterpret_cast<const uint8_t*>(base) + lin * dtype;
  if (dtype == CVMK_I32 && n == 16 && (reinterpret_cast<uintptr_t>(at) & 15) == 0) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int4 raw = reinterpret_cast<const int4*>(at)[q];
      t[4 * q] = raw.x; t[4 * q + 1] = raw.y; t[4 * q + 2] = raw.z; t[4 * q + 3] = raw.w;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 16; ++j)
    t[j] = j >= n ? 0 : (dtype == CVMK_I8 ? (int32_t) reinterpret_cast<const int8_t*>(at)[j] : reinterpret_cast<const int32_t*>(at)[j]);
}
__device__ __forceinline__ uint4 packed(const int32_t (&t)[16]) {
  return make_uint4(pack4(t[0], t[1], t[2], t[3]), pack4(t[4], t[5], t[6], t[7]), pack4(t[8], t[9], t[10], t[11]), pack4(t[12], t[13], t[14], t[15]));
}
__device__ __forceinline__ void store_run(void* base, int dtype, long long lin, int n, const int32_t (&t)[16]) {
  uint8_t* at = reinterpret_cast<uint8_t*>(base) + lin * dtype;
  if (n == 16 && (reinterpret_cast<uintptr_t>(at) & 15) == 0) {
    if (dtype == CVMK_I8) {
      *reinterpret_cast<uint4*>(at) = packed(t);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) reinterpret_cast<int4*>(at)[q] = make_int4(t[4 * q], t[4 * q + 1], t[4 * q + 2], t[4 * q + 3]);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (j < n) {
      if (dtype == CVMK_I8) reinterpret_cast<int8_t*>(at)[j] = (int8_t)t[j];
      else reinterpret_cast<int32_t*>(at)[j] = t[j];
    }
}
// Values within 8 bits, the int8 operand `r` added to or subtracted from them (or they from it) and a clip, two elements an
// instruction: the low bytes.
__device__ __forceinline__ uint4 packed_tail(const Params& p, const uint4& r, const int32_t (&a)[16]) {
  const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
  const int op = p.cy.s[p.cy.n - 2].op;
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t h0 = __byte_perm((uint32_t)a[4 * q], (uint32_t)a[4 * q + 1], 0x5410), h1 = __byte_perm((uint32_t)a[4 * q + 2], (uint32_t)a[4 * q + 3], 0x5410);
    const uint32_t r0 = prmt(rw[q], 0, 0x9180), r1 = prmt(rw[q], 0, 0xB3A2);   // bytes sign-extended to 16 bits
    if (op == K_ADD_T) {
      h0 = __vmaxs2(__viaddmin_s16x2(h0, r0, p.tail_hi), p.tail_lo);
      h1 = __vmaxs2(__viaddmin_s16x2(h1, r1, p.tail_hi), p.tail_lo);
    } else {
      h0 = __vmaxs2(__vmins2(op == K_SUB_T ? __vsub2(h0, r0) : __vsub2(r0, h0), p.tail_hi), p.tail_lo);
      h1 = __vmaxs2(__vmins2(op == K_SUB_T ? __vsub2(h1, r1) : __vsub2(r1, h1), p.tail_hi), p.tail_lo);
    }
    w[q] = __byte_perm(h0, h1, 0x6420);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void add_bias(const int32_t* bias_s, int32_t (&v)[16]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int4 b = reinterpret_cast<const int4*>(bias_s)[q];
    v[4 * q] += b.x; v[4 * q + 1] += b.y; v[4 * q + 2] += b.z; v[4 * q + 3] += b.w;
  }
}

__device__ __forceinline__ void requant(const int32_t* bias_s, const Requant& q, int32_t (&v)[16]) {   // biases with q.add in them
  const int hi = q.hi, lo = q.lo, sh = q.shift;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int4 b = reinterpret_cast<const int4*>(bias_s)[i];
    v[4 * i] = max(__viaddmin_s32(v[4 * i], b.x, hi), lo) >> sh;
    v[4 * i + 1] = max(__viaddmin_s32(v[4 * i + 1], b.y, hi), lo) >> sh;
    v[4 * i + 2] = max(__viaddmin_s32(v[4 * i + 2], b.z, hi), lo) >> sh;
    v[4 * i + 3] = max(__viaddmin_s32(v[4 * i + 3], b.w, hi), lo) >> sh;
  }
}

constexpr int PAIR_STAGE = 2 * W_BYTES;   // a CTA's 128 rows of x and 128 rows of weights
constexpr int PAIR_COLS = 256;            // of an accumulator
constexpr int PAIR_THREADS = 576;         // warp 0: TMA, warp 1: MMA + TMEM, warps 2..17: epilogue
constexpr int EPI_WARPS = PAIR_THREADS / 32 - 2;

// A warp's columns of a tile: 32 rows (`row` is the lane's) by `columns` units from unit0 on; `t0`: their sums in TMEM, `bias`:
// their biases in shared memory (with Requant::add in them where fast_w, fast_v), `acc_free`: the barrier that hands the accumulator back.
struct Part {
  int row, unit0, columns;
  uint32_t t0, acc_free;
  const int32_t* bias;
  const uint8_t* table_s;
};
__device__ __forceinline__ void hand_back(uint32_t acc_free) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) arrive_at(acc_free);
}

// Everything that the straight forms below do not take: step by step.
__device__ __forceinline__ void general_part(const Params& p, const Part& t, bool fast_w, bool fast_v) {
#pragma unroll 1
  for (int c = 0; c < t.columns; c += 16) {
    const int unit = t.unit0 + c, n = min(16, p.units - unit);
    int32_t a[16], b[16];
    __syncwarp();
    if (p.gated) tmem_ld_two(t.t0 + (uint32_t)c, t.t0 + 128u + (uint32_t)c, a, b);
    else tmem_ld16(t.t0 + (uint32_t)c, a);
    if (c + 16 >= t.columns) hand_back(t.acc_free);
    if (n <= 0 || t.row >= p.rows) continue;
    const long long lin = (long long)t.row * p.y_pitch + unit;
    if (fast_w) {
      requant(t.bias + c, p.qw, a);
      look_up<16>(p, t.table_s, a);
    } else {
      add_bias(t.bias + c, a);
      activate<16>(p, t.table_s, a);
    }
    if (p.gated) {
      if (fast_v) {
        requant(t.bias + 32 + c, p.qv, b);
      } else {
        add_bias(t.bias + 32 + c, b);
        apply_chain<16>(p.cv, b, 0, 0, 0, nullptr, -1, p.first_v);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) a[j] = (int32_t)((uint32_t)a[j] * (uint32_t)b[j]);
    }
    if (p.res) load_run(p.res, p.res_dtype, lin, n, b);
    apply_chain<16, true>(p.cy, a, 0, 0, 0, b, p.res_step);
    store_run(p.y, p.y_dtype, lin, n, a);
  }
  __syncwarp();
}

// The same as a function of its own, for the kernels that need it only where a bias is so large that its sum might overflow.
// (The launch's parameters are then read as memory, not as constants: a third of the speed.)
__device__ __noinline__ void rare_part(const Params& p, const Part t, bool fast_w, bool fast_v) { general_part(p, t, fast_w, fast_v); }

// Both sides in the three-instruction form, and the table in shared memory (T32: in int32): the product of a chunk's sides.
template <bool GATED, bool T32>
__device__ __forceinline__ void straight_chunk(const Params& p, const Part& t, const uint8_t* table_s, int c, int32_t (&a)[16], int32_t (&b)[16]) {
  if (GATED) tmem_ld_two(t.t0 + (uint32_t)c, t.t0 + 128u + (uint32_t)c, a, b);
  else tmem_ld16(t.t0 + (uint32_t)c, a);
  if (c + 16 >= t.columns) hand_back(t.acc_free);
  requant(t.bias + c, p.qw, a);
#pragma unroll
  for (int j = 0; j < 16; ++j) a[j] = T32 ? reinterpret_cast<const int32_t*>(table_s)[a[j]] : (int32_t) reinterpret_cast<const int8_t*>(table_s)[a[j]];
  if (GATED) {
    requant(t.bias + 32 + c, p.qv, b);
#pragma unroll
    for (int j = 0; j < 16; ++j) a[j] = (int32_t)((uint32_t)a[j] * (uint32_t)b[j]);
  }
}
// `staged` is the warp's piece of the tile as it will lie in memory, 32 rows of t.columns bytes in the TMA swizzle of that width;
// RES: there the int8 operand of the tensor step lies already.
// Little code: what a tile's loop holds has to come to the SM's instruction cache.
template <bool GATED, bool RES, bool T32>
__device__ __forceinline__ void straight_part(const Params& p, const Part& t, const uint8_t* table_s, uint8_t* staged) {
  const int lane = threadIdx.x & 31;
  constexpr int COLUMNS = GATED ? 32 : 64;
#pragma unroll 1
  for (int c = 0; c < COLUMNS; c += 16) {
    int32_t a[16], b[16];
    straight_chunk<GATED, T32>(p, t, table_s, c, a, b);
    apply_chain<16>(RES ? p.head : p.cy, a, 0, 0, 0);
    uint4* at = reinterpret_cast<uint4*>(staged + panel_offset(lane, c >> 4, COLUMNS));
    *at = RES ? packed_tail(p, *at, a) : packed(a);
    __syncwarp();
  }
}
// Results in int32: 16 columns at a time leave through `out`, 32 rows of 64 bytes in the TMA swizzle of that width, two
// buffers in turn; `operand`: the int8 operand of the tensor step, as above.
template <bool GATED, bool RES, bool T32>
__device__ __forceinline__ void wide_part(const Params& p, const Part& t, const CUtensorMap* tmap_y, const uint8_t* table_s, const uint8_t* operand, uint8_t* out, bool live) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int c = 0; c < t.columns; c += 16) {
    int32_t a[16], b[16];
    straight_chunk<GATED, T32>(p, t, table_s, c, a, b);
    if (RES) {
      const uint4 r = *reinterpret_cast<const uint4*>(operand + panel_offset(lane, c >> 4, GATED ? 32 : 64));
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int j = 0; j < 16; ++j) b[j] = (int32_t)(int8_t)(w[j >> 2] >> ((j & 3) * 8));
    }
    apply_chain<16, true>(p.cy, a, 0, 0, 0, b, p.res_step);
    uint8_t* const to = out + ((c >> 4) & 1) * 2048;
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");   // (what lay there has left)
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<int4*>(to + panel_offset(lane, q, 64)) = make_int4(a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]);
    fence_async_smem();
    __syncwarp();
    if (lane == 0 && live && t.unit0 + c < p.units) tma_store_2d(tmap_y, to, t.unit0 + c, t.row);
    if (lane == 0) tma_store_commit();
  }
}
// The same where rows of y do not begin on 16 bytes, or the operand is int32.  Lanes read and write along rows (a lane that works
// on its own row touches 32 rows a time): 16 columns of the operand, and of results in int32, are turned through `turn`, two rows
// a time; results in int8 wait in `piece` and leave as whole words, wherever a row begins against four bytes, and a few bytes.
constexpr int TURN_PITCH = 17;   // words of a row of 16, or of 64 bytes
constexpr int TURN_BYTES = 32 * TURN_PITCH * 4;
template <bool GATED, bool RES, bool T32>
__device__ __forceinline__ void turned_part(const Params& p, const Part& t, const uint8_t* table_s, uint32_t* piece, int32_t* turn) {
  constexpr int COLUMNS = GATED ? 32 : 64;
  const int lane = threadIdx.x & 31, col = lane & 15, half = lane >> 4, rows = p.rows - (t.row - lane) - half;   // left, from the lane's first on
  const size_t step = 2 * (size_t)p.y_pitch;
  const bool narrow = p.y_dtype == CVMK_I8;
#pragma unroll 1
  for (int c = 0; c < COLUMNS; c += 16) {
    const int unit = t.unit0 + c + col;
    const size_t lin = (size_t)(t.row - lane + half) * (size_t)p.y_pitch + unit;
    const int mine = unit < p.units ? rows : 0;
    int32_t a[16], b[16];
    if (RES) {   // (the operand travels while the sums are waited for)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        b[i] = 2 * i < mine ? (p.res_dtype == CVMK_I8 ? (int32_t) reinterpret_cast<const int8_t*>(p.res)[lin + i * step]
                                                      : reinterpret_cast<const int32_t*>(p.res)[lin + i * step]) : 0;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i) turn[(2 * i + half) * TURN_PITCH + col] = b[i];
    }
    __syncwarp();
    straight_chunk<GATED, T32>(p, t, table_s, c, a, b);
    if (RES) {
#pragma unroll
      for (int j = 0; j < 16; ++j) b[j] = turn[lane * TURN_PITCH + j];
      __syncwarp();
    }
    apply_chain<16, true>(p.cy, a, 0, 0, 0, b, p.res_step);
    if (narrow) {
      const uint4 w = packed(a);
      uint32_t* const to = piece + lane * TURN_PITCH + (c >> 2);
      to[0] = w.x; to[1] = w.y; to[2] = w.z; to[3] = w.w;
      continue;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) turn[lane * TURN_PITCH + j] = a[j];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (2 * i < mine) reinterpret_cast<int32_t*>(p.y)[lin + i * step] = turn[(2 * i + half) * TURN_PITCH + col];
    __syncwarp();
  }
  __syncwarp();
  const int n = min(COLUMNS, p.units - t.unit0);   // bytes of a row
  if (!narrow || n <= 0) return;
  uint8_t* const y0 = reinterpret_cast<uint8_t*>(p.y) + (size_t)(t.row - lane) * (size_t)p.y_pitch + t.unit0;
  auto bytes_in_front = [](const uint8_t* at) { return (int)(-reinterpret_cast<uintptr_t>(at) & 3); };   // of the first whole word
  uint8_t* at = y0 + (size_t)half * (size_t)p.y_pitch;
  for (int i = 0; i < 16; ++i, at += step) {
    const int head = bytes_in_front(at);
    if (2 * i < rows && 4 * col + 4 <= n - head) {
      const uint32_t* const from = piece + (2 * i + half) * TURN_PITCH + col;
      *reinterpret_cast<uint32_t*>(at + head + 4 * col) = __funnelshift_r(from[0], from[1], 8 * head);
    }
  }
  if (t.row < p.rows) {   // what is left at the ends of the lane's row
    uint8_t* const mine = y0 + (size_t)lane * (size_t)p.y_pitch;
    const uint8_t* const from = reinterpret_cast<const uint8_t*>(piece + lane * TURN_PITCH);
    const int head = min(bytes_in_front(mine), n), tail = head + ((n - head) & ~3);
    for (int e = 0; e < 3; ++e) {
      if (e < head) mine[e] = from[e];
      if (tail + e < n) mine[tail + e] = from[tail + e];
    }
  }
  __syncwarp();
}

// Which of these a kernel runs.  They are kernels of their own: together they need more registers than there are, and as functions
// they read the launch's parameters as memory (6000 rows 2048 -> 8192 with a residual to int32: 192 us).
enum Kind { USUAL, WIDE, TURNED, GENERAL };   // straight_part() with a table of int8; wide_part(), or straight_part() with a table of int32
template <int KIND, bool GATED, bool RES>
__device__ __forceinline__ void run_part(const Params& p, const Part& t, const CUtensorMap* tmap_y, const uint8_t* table_s, uint8_t* staged, bool live) {
  if (KIND == USUAL) {
    straight_part<GATED, RES, false>(p, t, table_s, staged);
  } else if (KIND == WIDE) {
    uint8_t* const out = RES ? staged + 2048 : staged;
    if (p.io == 1) straight_part<GATED, RES, true>(p, t, table_s, staged);
    else if (p.table_s_dtype == CVMK_I8) wide_part<GATED, RES, false>(p, t, tmap_y, table_s, staged, out, live);
    else wide_part<GATED, RES, true>(p, t, tmap_y, table_s, staged, out, live);
  } else if (p.table_s_dtype == CVMK_I8) {
    turned_part<GATED, RES, false>(p, t, table_s, reinterpret_cast<uint32_t*>(staged), reinterpret_cast<int32_t*>(staged + TURN_BYTES));
  } else {
    turned_part<GATED, RES, true>(p, t, table_s, reinterpret_cast<uint32_t*>(staged), reinterpret_cast<int32_t*>(staged + TURN_BYTES));
  }
}

template <int KIND>
__global__ void __launch_bounds__(PAIR_THREADS, 1)
dense_lut_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                      const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_y,
                      const __grid_constant__ CUtensorMap tmap_r, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar_full[MAX_STAGES];       // of the first CTA: the bytes of both have landed
  __shared__ uint64_t bar_empty[MAX_STAGES];
  __shared__ uint64_t bar_acc_full[2];
  __shared__ uint64_t bar_res[EPI_WARPS][2];      // [warp][buffer]: the tensor operand of a tile has landed
  __shared__ uint64_t bar_acc_empty[2];           // of the first CTA: the warps of both have read the accumulator
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  __shared__ __align__(16) int32_t bias_s[EPI_WARPS][64];
  __shared__ __align__(16) uint8_t table_s[TABLE_SMEM_MAX];   // (at a place the compiler knows: no addition per look-up)

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = uniform((int)(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  const int rank = uniform((int)cluster_rank());
  const int first = (int)blockIdx.x >> 1, step = (int)gridDim.x >> 1, tiles = p.unit_tiles * p.row_tiles;
  const int tile_units = p.gated ? 128 : 256;
  const bool leader = elect_one();
  touch_params(p);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&bar_full[s], 1);
      mbar_init(&bar_empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&bar_acc_full[a], 1);
      mbar_init(&bar_acc_empty[a], 2 * EPI_WARPS);
      for (int w = 0; w < EPI_WARPS; ++w) mbar_init(&bar_res[w][a], 1);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    tmem_alloc<2>(&tmem_slot, 2 * PAIR_COLS);   // before this CTA lets the next kernel start
    pdl_trigger();
  }
  if (warp >= 2) {
    if (!p.params_static) pdl_wait();
    if (p.table_smem) copy_table(p, table_s, (int)threadIdx.x - 64, PAIR_THREADS - 64);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // neither CTA signals the other's barriers or writes its TMEM before both have them
  tc_fence_after();
  const uint32_t tmem_base = (uint32_t)uniform((int)tmem_slot);
  const int my_tiles = first < tiles ? (tiles - first + step - 1) / step : 0;
  pdl_wait();

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA
    const uint32_t full0 = map_rank(smem_u32(&bar_full[0]), 0);
    int stage = 0;
    uint32_t phase = 0;
    bool live = leader;
    for (int tile = first; live && tile < tiles; tile += step) {
      const int ut = tile / p.row_tiles, rt = tile - ut * p.row_tiles;
      const int row0 = rt * 256 + rank * 128, unit0 = ut * tile_units + (p.gated ? 0 : rank * 128);
      const CUtensorMap* const weights = p.gated && rank ? &tmap_v : &tmap_w;
      for (int kb = 0; kb < p.kblocks; ++kb) {
        if (!mbar_wait(&bar_empty[stage], phase ^ 1, &abort_flag, 1)) { live = false; break; }
        if (rank == 0) mbar_expect_tx(&bar_full[stage], 2 * PAIR_STAGE);
        const uint32_t dst = smem_u32(smem) + (uint32_t)(stage * PAIR_STAGE), bar = full0 + 8u * (uint32_t)stage;
        load_2d_pair(dst, &tmap_x, bar, kb * BLOCK_K, row0);
        load_2d_pair(dst + W_BYTES, weights, bar, kb * BLOCK_K, unit0);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA, of both CTAs by the first
    if (rank == 0) {
      const uint32_t idesc = umma_idesc_i8(256, 256);
      const uint64_t desc0 = umma_desc(smem_u32(smem), BLOCK_K);
      const uint32_t lo0 = (uint32_t)desc0, hi = (uint32_t)(desc0 >> 32);
      int stage = 0;
      uint32_t phase = 0;
      int refills = my_tiles * p.kblocks - p.stages;   // stages, this one included, that are filled again: nobody waits for the others' commits
      bool live = true;
      for (int i = 0; live && i < my_tiles; ++i) {
        const int acc = i & 1;
        if (!mbar_wait(&bar_acc_empty[acc], (uint32_t)((i >> 1) & 1) ^ 1u, &abort_flag, 2)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * PAIR_COLS);
        for (int kb = 0; kb < p.kblocks; ++kb, --refills) {
          if (!mbar_wait(&bar_full[stage], phase, &abort_flag, 3)) { live = false; break; }
          tc_fence_after();
          const uint32_t al = lo0 + (uint32_t)(stage * (PAIR_STAGE >> 4));
          if (leader) {
            mma_i8_k<4, 2>(d_tmem, al, hi, al + (W_BYTES >> 4), hi, idesc, (uint32_t)kb);
            mma_commit_pair_if(refills > 0, &bar_empty[stage]);
          }
          if (++stage == p.stages) { stage = 0; phase ^= 1; }
        }
        if (live && leader) mma_commit<2>(&bar_acc_full[acc]);
        __syncwarp();
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- epilogue: a row a lane, a quarter of the columns a group of four warps
    const int io = KIND == USUAL ? 1 : (KIND == WIDE ? p.io : 0);
    const int quarter = warp & 3, group = (warp - 2) >> 2, columns = tile_units / 4;   // 32 units, ungated 64
    const uint32_t acc_empty0 = map_rank(smem_u32(&bar_acc_empty[0]), 0);
    int32_t* const bias = bias_s[warp - 2];   // of w's columns, gated: 32 of w's and 32 of v's
    const int32_t* const bias2 = p.gated ? p.bias_v : p.bias_w;
    // the warp's piece of a tile on its way, in one buffer or (tensor operands, which come a tile early) two
    const int piece = 32 * columns;
    uint8_t* const staged0 = smem + p.stages * PAIR_STAGE + (warp - 2) * (io == 1 ? piece * (p.res ? 2 : 1) : (io ? (p.res ? 6144 : 4096) : 2 * TURN_BYTES));
    uint32_t res_phase = 0;
    auto request = [&](int tile, int buffer) {   // (one lane)
      const int ut = tile / p.row_tiles, rt = tile - ut * p.row_tiles;
      const int row = rt * 256 + rank * 128 + quarter * 32, unit = ut * tile_units + group * columns;
      if (row >= p.rows || unit >= p.units) return;
      mbar_expect_tx(&bar_res[warp - 2][buffer], (uint32_t)piece);
      tma_load_2d(staged0 + buffer * piece, &tmap_r, &bar_res[warp - 2][buffer], unit, row);
    };
    if (io && p.res && lane == 0 && first < tiles) request(first, 0);
    int i = 0;
    for (int tile = first; tile < tiles; tile += step, ++i) {
      const int acc = i & 1;
      const int ut = tile / p.row_tiles, rt = tile - ut * p.row_tiles;
      const int warp_row = rt * 256 + rank * 128 + quarter * 32, row = warp_row + lane, unit0 = ut * tile_units + group * columns;
      const uint32_t t0 = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * PAIR_COLS + group * columns);
      // what the tile needs beside the sums travels while the products are computed: the biases, and an int8 residual
      const int u1 = unit0 + lane, u2 = p.gated ? u1 : u1 + 32;
      const int32_t b1 = p.bias_w && u1 < p.units ? p.bias_w[u1] : 0, b2 = bias2 && u2 < p.units ? bias2[u2] : 0;
      // (p.io == 1: the operand of the next tile sets out into the buffer that the last tile's results have left)
      const bool live = warp_row < p.rows && unit0 < p.units;
      if (io == 1 && lane == 0) {
        tma_store_wait_read();
        if (p.res && tile + step < tiles) request(tile + step, (i + 1) & 1);
      }
      const Requant& q2 = p.gated ? p.qv : p.qw;
      bool fast1 = __all_sync(FULL_MASK, in_room(b1, p.qw)) && p.qw.on, fast2 = __all_sync(FULL_MASK, in_room(b2, q2)) && q2.on;
      if (!p.gated) fast1 = fast2 = fast1 && fast2;
      __syncwarp();   // (the last tile's biases have been read)
      bias[lane] = fast1 ? b1 + p.qw.add : b1;
      bias[lane + 32] = fast2 ? b2 + q2.add : b2;
      __syncwarp();
      if (!__all_sync(FULL_MASK, mbar_wait(&bar_acc_full[acc], (uint32_t)((i >> 1) & 1), &abort_flag, 4))) break;
      tc_fence_after();
      const Part part = {row, unit0, columns, t0, acc_empty0 + 8u * (uint32_t)acc, bias, table_s};
      const int buffer = io == 1 && p.res ? acc : 0;
      uint8_t* const staged = staged0 + buffer * piece;
      if (io && p.res && live) {
        if (!__all_sync(FULL_MASK, mbar_wait(&bar_res[warp - 2][buffer], (res_phase >> buffer) & 1u, &abort_flag, 5))) break;
        res_phase ^= 1u << buffer;
      }
      const bool straight = fast1 && fast2 && p.straight;
      if (KIND == GENERAL) general_part(p, part, fast1, fast2);
      else if (!straight) rare_part(p, part, fast1, fast2);
      else if (p.res) p.gated ? run_part<KIND, true, true>(p, part, &tmap_y, table_s, staged, live) : run_part<KIND, false, true>(p, part, &tmap_y, table_s, staged, live);
      else p.gated ? run_part<KIND, true, false>(p, part, &tmap_y, table_s, staged, live) : run_part<KIND, false, false>(p, part, &tmap_y, table_s, staged, live);
      if (KIND == WIDE && io == 2 && p.res) {   // (one buffer: the next operand may come once this one has been read)
        __syncwarp();
        if (lane == 0 && tile + step < tiles) request(tile + step, 0);
      }
      if (straight && io == 1) {
        fence_async_smem();
        __syncwarp();
        if (lane == 0 && live) {
          tma_store_2d(&tmap_y, staged, unit0, warp_row);
          tma_store_commit();
        }
      }
    }
    if (io && lane == 0) tma_store_wait_all();   // (shared memory goes with the CTA)
    __syncwarp();
  }
  if (abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);   // copies in flight land before shared memory is released
    if (lane == 0 && p.status) atomicOr(p.status, 0x400 | abort_flag);
    __syncwarp();
  }
  tc_fence_before();
  cluster_sync();   // every accumulator has been read, and nothing is sent to either CTA any more
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<2>(tmem_base, 2 * PAIR_COLS);
  }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encoder() {
  static EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q);
    return e == cudaSuccess && q == cudaDriverEntryPointSuccess ? (EncodeTiledFn)f : nullptr;
  }();
  return fn;
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  cudaGetLastError();
  return sms;
}

// A row-major matrix of int8 (wide: int32), rows `pitch` elements apart, in boxes of `box_bytes` of `box_rows` rows; zeros outside.
CUresult encode_matrix(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t pitch, int box_rows, CUtensorMapL2promotion promo,
                       int box_bytes = BLOCK_K, bool wide = false) {
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch * (wide ? 4 : 1)};
  cuuint32_t box[2] = {(cuuint32_t)box_bytes / (wide ? 4 : 1), (cuuint32_t)box_rows}, estr[2] = {1, 1};
  return encoder()(map, wide ? CU_TENSOR_MAP_DATA_TYPE_INT32 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : (box_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B), promo, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// The three-instruction form of a lowered chain from step `first` on, in front of a table of `len` entries or not (0).
Requant requant_of(const DevChain& c, int first, int len, int K) {
  Requant q = {0, 0, 0, 0, 0, 0, 0};
  const int left = c.n - first;
  if (left < 1 || left > (len ? 2 : 1) || c.s[first].op != K_RS_CLAMP || (left == 2 && c.s[first + 1].op != K_ADD_S)) return q;
  const DevStep& rs = c.s[first];
  const int64_t moved = (int64_t)(left == 2 ? c.s[first + 1].a : 0) * ((int64_t)1 << rs.d), add = rs.c + moved;
  int64_t lo = rs.a + add, hi = rs.b + add;
  if (len) {
    lo = std::max<int64_t>(lo, 0);
    hi = std::min<int64_t>(hi, ((int64_t)len << rs.d) - 1);
  }
  const int64_t room = (int64_t)INT32_MAX - ((int64_t)K << 14);   // |bias| and |bias + add| up to this; a sum is K * 2^14 at most
  const int64_t least = std::max(-room, -room - add), most = std::min(room, room - add);
  if (lo > hi || lo < INT32_MIN || hi > INT32_MAX || add < INT32_MIN || add > INT32_MAX || least > most) return q;
  return {1, (int)add, (int)lo, (int)hi, rs.d, (int)least, (int)most};
}

// Whether y can be stored by TMA: rows begin on 16 bytes, and they end on them, because a store writes whole 16 bytes where the
// last element of a row lies among them (1000 of 1008 bytes: the other eight came out 0).
bool by_tma(const cvmk_dense_lut_desc& d) {
  return !((uintptr_t)d.y & 15) && d.y_pitch * d.y_dtype % 16 == 0 && (int64_t)d.units * d.y_dtype % 16 == 0;
}

bool is_tensor_step(const cvmk_ep_step& s) { return s.op == CVMK_EP_ADD_T || s.op == CVMK_EP_SUB_T || s.op == CVMK_EP_RSUB_T; }

// Which kernel runs a layer, and how the small one cuts it (rows of x a tile, CTAs that share its reduction): every cut, and the
// pairs of CTAs, are given a time, and the least of them is taken.  The terms, in microseconds of a launch in a chain of launches,
// fitted to 1500 shapes (1 to 8192 rows, 64 to 8192 long, 32 to 16384 units, each cut timed) and checked with 8500 others: what
// is chosen takes 1.9 % longer than the best cut, in the mean:
//   small   2.7 for the launch, 0.058 a row of the tile for its last steps, 0.35 a block of K (a load's latency, a ring of several
//           in flight), all operands and tables at 9.4 MB a microsecond out of L2 and the weights at 6 out of memory, 2.2 for the
//           exchange of partial sums; times the rounds of CTAs (0.5 each beyond the first), two an SM up to 64 rows and one
//           beyond, and of clusters as many as are resident at once (GPCs have 16 to 20 SMs).
//   pairs   5.3 for the launch, 0.1 a block of K to fill the ring, and a round of tiles the longer of 0.42 a block and its last
//           steps: 2.7, or where rows of y do not begin on 16 bytes 3.3, 0.6 more for int32 and 1.2 with a tensor operand; the
//           shorter of the two 1.9 times, in the first and the last round.
// Cut over rows, a layer of few units uses the whole GPU: 128 rows 176 -> 122 14.8 us in one tile of rows and 5.4 in eight, 1000
// rows 1024 -> 250 gated 6.2 in 63 (pairs 11.1).  Cut in K: 8 rows 4096 -> 4096 whole 10.6, in four 7.5.
struct Cut { int row_tile, split; };   // split 0: pairs
Cut choose(const cvmk_dense_lut_desc& d, int kblocks, int sms) {
  const double weights = (double)d.units * d.K * (d.v ? 2 : 1);
  const int64_t pair_tiles = (int64_t)((d.rows + 255) / 256) * ((d.units + (d.v ? 127 : 255)) / (d.v ? 128 : 256)), pairs = sms / 2;
  bool operand = false;
  for (int i = 0; i < d.chain_y.n; ++i) operand = operand || is_tensor_step(d.chain_y.s[i]);
  const double last = by_tma(d) ? 2.7 : 3.3 + (d.y_dtype == CVMK_I32 ? 0.6 : 0.0) + (operand ? 1.2 : 0.0), products = 0.42 * kblocks;
  Cut best = {256, 0};
  double least = 5.3 + 0.1 * kblocks + std::max((pair_tiles + pairs - 1) / pairs * std::max(products, last) + 1.9 * std::min(products, last), weights / 6e6);
  static const int at_once[2][4] = {{148, 74, 33, 15}, {296, 148, 71, 33}};   // clusters of 1, 2, 4 and 8 CTAs, one and two an SM; 148 SMs
  for (const int row_tile : {16, 32, 48, 64, 96, 128}) {
    const int rt = std::min(row_tile, (std::min(d.rows, 128) + 15) & ~15);
    const int64_t tiles = (int64_t)((d.units + (d.v ? 63 : 127)) / (d.v ? 64 : 128)) * ((d.rows + rt - 1) / rt);
    for (int log2 = 0; log2 < 4 && (log2 == 0 || kblocks >= 4 << log2); ++log2) {
      const int split = 1 << log2, per = (kblocks + split - 1) / split;
      const int64_t room = std::max<int64_t>((int64_t)at_once[rt <= 64][log2] * sms / 148, 1), rounds = (tiles + room - 1) / room;
      const double bytes = (double)tiles * split * (per * (W_BYTES + rt * BLOCK_K) + (double)d.table_len * d.table_dtype);
      const double us = 2.7 + 0.058 * rt * rounds + std::max({0.35 * per * rounds, bytes / 9.4e6, weights / 6e6}) + (split > 1 ? 2.2 : 0.0) + 0.5 * (rounds - 1);
      if (us < least) {
        least = us;
        best = {rt, split};
      }
    }
    if (rt < row_tile) break;
  }
  if (const char* e = dev_env("CVM_B200_DL_KERNEL")) best = atoi(e) ? Cut{256, 0} : (best.split ? best : Cut{128, 1});
  if (const char* e = dev_env("CVM_B200_DL_ROWTILE")) best.row_tile = atoi(e);
  if (const char* e = dev_env("CVM_B200_DL_SPLIT")) best.split = atoi(e);
  return best;
}

// Values that a step leaves within 8 bits, whatever it is given.
bool to_int8(const DevStep& s) {
  if (s.op == K_CLIP) return s.a >= -128 && s.b <= 127;
  return s.op == K_RS_CLAMP && (((int64_t)s.a + s.c) >> s.d) >= -128 && (((int64_t)s.b + s.c) >> s.d) <= 127;
}

int encode_operands(cvmk_dense_lut_plan* plan, int x_rows, int w_rows) {
  const cvmk_dense_lut_desc& d = plan->d;
  CUresult r = encode_matrix((CUtensorMap*)plan->tmap_x, d.x, d.rows, d.K, d.x_pitch, x_rows, CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
  if (r == CUDA_SUCCESS) r = encode_matrix((CUtensorMap*)plan->tmap_w, d.w, d.units, d.K, d.w_pitch, w_rows, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (r == CUDA_SUCCESS) r = encode_matrix((CUtensorMap*)plan->tmap_v, d.v ? d.v : d.w, d.units, d.K, d.w_pitch, w_rows, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (r != CUDA_SUCCESS) { set_error("dense_lut_prepare: tensor map rejected (CUresult %d)", (int)r); return CVMK_ERR_CUDA; }
  return CVMK_OK;
}

bool is_tensor_op(int op) { return op == K_ADD_T || op == K_SUB_T || op == K_RSUB_T; }
bool is_type(int t) { return t == CVMK_I8 || t == CVMK_I32; }

const char* refusal(const cvmk_dense_lut_desc& d) {
  if (d.rows < 0 || d.units < 1 || d.K < 1 || d.K >= 1 << 17) return "sizes outside 0 <= rows, 1 <= units, 1 <= K < 2^17";
  if (d.rows > INT32_MAX - 256 || d.units > INT32_MAX - 256 || ((int64_t)d.rows / 16 + 1) * ((int64_t)d.units / 64 + 1) > 1 << 27) return "too many outputs for one launch";
  if (!is_type(d.y_dtype) || !is_type(d.table_dtype)) return "y and the table are int8 or int32";
  if (d.table_len < 1) return "a table has at least one entry";
  if ((d.x_pitch && d.x_pitch < d.K) || (d.w_pitch && d.w_pitch < d.K) || (d.y_pitch && d.y_pitch < d.units)) return "a pitch is shorter than its row";
  if ((d.x_pitch ? d.x_pitch : d.K) % 16 || (d.w_pitch ? d.w_pitch : d.K) % 16) return "rows of x, w and v are multiples of 16 bytes apart";
  if ((d.x_pitch | d.w_pitch) >> 39) return "rows too far apart";
  for (const cvmk_epilogue* c : {&d.chain_w, &d.chain_v, &d.chain_y}) {
    if (c->n < 0 || c->n > CVMK_MAX_EP_STEPS) return "a chain has too many steps";
    if (c == &d.chain_v && !d.v && c->n) return "chain_v without v";
    int tensors = 0;
    for (int i = 0; i < c->n; ++i) {
      if (c->s[i].op == CVMK_EP_ADD_C && (i > 0 || c == &d.chain_y)) return "a bias is the first step of chain_w or chain_v";
      if (is_tensor_step(c->s[i])) {
        if (c != &d.chain_y || ++tensors > 1) return "one tensor step, in chain_y";
        if (!is_type(c->s[i].ptr_dtype)) return "a tensor operand is int8 or int32";
      }
    }
  }
  return nullptr;
}

// What the kernels are given, from a plan whose tile sizes, table_smem and io are set.
int make_params(const cvmk_dense_lut_plan& plan, Params* out) {
  Params& p = *out;
  memset(&p, 0, sizeof(p));
  const cvmk_dense_lut_desc& d = plan.d;
  p.y = d.y; p.y_pitch = d.y_pitch; p.y_dtype = d.y_dtype;
  p.rows = d.rows; p.units = d.units;
  p.kblocks = (d.K + BLOCK_K - 1) / BLOCK_K;
  p.gated = d.v != nullptr;
  p.params_static = d.params_static;
  const bool pair = plan.kernel == 1;
  const int tile_units = (p.gated ? 64 : 128) * (pair ? 2 : 1);
  p.unit_tiles = (d.units + tile_units - 1) / tile_units;
  p.row_tile = plan.row_tile;
  p.row_tiles = (d.rows + p.row_tile - 1) / p.row_tile;
  p.stages = plan.stages;
  p.split = plan.split;
  while ((1 << p.split_log2) < p.split) ++p.split_log2;
  p.tmem_cols = 32;
  while (p.tmem_cols < p.row_tile) p.tmem_cols *= 2;
  p.table = d.table; p.table_len = d.table_len; p.table_dtype = d.table_dtype; p.table_smem = plan.table_smem;
  p.status = d.status;
  int rc = lower_chain(d.chain_w, &p.cw);
  if (!rc) rc = lower_chain(d.chain_v, &p.cv);
  if (!rc) rc = lower_chain(d.chain_y, &p.cy);
  if (rc) return rc;
  if (p.cw.n && p.cw.s[0].op == K_ADD_C) { p.bias_w = (const int32_t*)p.cw.s[0].ptr; p.first_w = 1; }
  if (p.cv.n && p.cv.s[0].op == K_ADD_C) { p.bias_v = (const int32_t*)p.cv.s[0].ptr; p.first_v = 1; }
  p.qw = requant_of(p.cw, p.first_w, d.table_len, d.K);
  p.qv = requant_of(p.cv, p.first_v, 0, d.K);
  // Ungated, the first steps of chain_y are functions of a table entry: the copy of the table goes through them.
  p.table_s_dtype = d.table_dtype;
  if (!p.gated && p.table_smem) {
    while (p.ct.n < p.cy.n && !is_tensor_op(p.cy.s[p.ct.n].op)) { p.ct.s[p.ct.n] = p.cy.s[p.ct.n]; ++p.ct.n; }
    if (p.ct.n) p.table_s_dtype = to_int8(p.ct.s[p.ct.n - 1]) ? CVMK_I8 : CVMK_I32;
    if (p.table_s_dtype * (int64_t)d.table_len > p.table_smem) {   // (wider than the room the plan has for it)
      p.ct.n = 0;
      p.table_s_dtype = d.table_dtype;
    }
    for (int i = p.ct.n; i < p.cy.n; ++i) p.cy.s[i - p.ct.n] = p.cy.s[i];
    p.cy.n -= p.ct.n;
  }
  const int at = p.cy.n - 2;
  if (at >= 0 && is_tensor_op(p.cy.s[at].op) && p.cy.s[at].dt == CVMK_I8 && p.cy.s[at + 1].op == K_CLIP && d.y_dtype == CVMK_I8 &&
      p.cy.s[at + 1].a >= -32767 && p.cy.s[at + 1].b <= 32767 &&
      (at ? to_int8(p.cy.s[at - 1]) : !p.gated && p.table_s_dtype == CVMK_I8)) {
    p.tail = 1;
    p.head = p.cy;
    p.head.n = at;
    p.tail_lo = both_halves(p.cy.s[at + 1].a);
    p.tail_hi = both_halves(p.cy.s[at + 1].b);
  }
  p.res_step = -1;
  for (int i = 0; i < p.cy.n; ++i)
    if (is_tensor_op(p.cy.s[i].op)) {
      p.res = p.cy.s[i].ptr; p.res_dtype = p.cy.s[i].dt; p.res_step = i;
    }

  p.straight = p.qw.on && (!p.gated || p.qv.on) && p.table_smem;
  p.io = p.straight && (plan.io == 2 || (plan.io == 1 && (!p.res || p.tail))) ? plan.io : 0;

  return CVMK_OK;
}

}  // namespace
}  // namespace cvmk

using namespace cvmk;

extern "C" int cvmk_dense_lut_supported(const cvmk_dense_lut_desc* d) { return d && !refusal(*d); }

extern "C" int cvmk_dense_lut_prepare(const cvmk_dense_lut_desc* d, cvmk_dense_lut_plan* plan) {
  if (!d || !plan) { set_error("dense_lut_prepare: null argument"); return CVMK_ERR_ARG; }
  if (const char* why = refusal(*d)) { set_error("dense_lut_prepare: %s", why); return CVMK_ERR_ARG; }
  if ((uintptr_t)plan & 63) { set_error("dense_lut_prepare: the plan must be 64-byte aligned"); return CVMK_ERR_ARG; }
  DevChain c;
  for (const cvmk_epilogue* e : {&d->chain_w, &d->chain_v, &d->chain_y})
    if (const int rc = lower_chain(*e, &c)) return rc;
  memset(plan, 0, sizeof(*plan));
  plan->d = *d;
  cvmk_dense_lut_desc& p = plan->d;
  if (!p.x_pitch) p.x_pitch = p.K;
  if (!p.w_pitch) p.w_pitch = p.K;
  if (!p.y_pitch) p.y_pitch = p.units;
  if (p.rows == 0) return CVMK_OK;   // (nothing to launch)
  if (!p.x || !p.w || !p.y || !p.table) { set_error("dense_lut_prepare: null operand"); return CVMK_ERR_ARG; }
  if (((uintptr_t)p.x & 15) || ((uintptr_t)p.w & 15) || ((uintptr_t)p.v & 15)) {
    set_error("dense_lut_prepare: x, w and v must be 16-byte aligned");
    return CVMK_ERR_ARG;
  }
  uintptr_t odd = ((uintptr_t)p.y & (p.y_dtype - 1)) | ((uintptr_t)p.table & (p.table_dtype - 1));
  for (const cvmk_epilogue* e : {&p.chain_w, &p.chain_v, &p.chain_y})
    for (int i = 0; i < e->n; ++i) {
      if (e->s[i].op == CVMK_EP_ADD_C) odd |= (uintptr_t)e->s[i].ptr & 3;
      if (is_tensor_step(e->s[i])) odd |= (uintptr_t)e->s[i].ptr & (e->s[i].ptr_dtype - 1);
    }
  if (odd) { set_error("dense_lut_prepare: an operand is not aligned to its elements"); return CVMK_ERR_ARG; }
  for (int i = 0; i < p.chain_y.n; ++i)
    if (is_tensor_step(p.chain_y.s[i]) && p.chain_y.s[i].ptr == p.y && p.chain_y.s[i].ptr_dtype != p.y_dtype) {
      set_error("dense_lut_prepare: a tensor operand that is y has y's type");   // (another thread's result would lie on it)
      return CVMK_ERR_ARG;
    }
  if (!encoder()) { set_error("dense_lut_prepare: the driver has no cuTensorMapEncodeTiled"); return CVMK_ERR_CUDA; }

  if (check_cuda(cudaGetDevice(&plan->device), "dense_lut_prepare: cudaGetDevice")) return CVMK_ERR_CUDA;
  const int sms = sm_count(), kblocks = (p.K + BLOCK_K - 1) / BLOCK_K, tile_units = p.v ? 64 : 128;
  const int64_t table_bytes = (int64_t)p.table_len * p.table_dtype;
  plan->table_smem = table_bytes <= TABLE_SMEM_MAX ? (int)table_bytes : 0;
  const int table_room = (plan->table_smem + 15) & ~15;
  const Cut cut = choose(p, kblocks, sms);
  plan->kernel = cut.split == 0;
  if (plan->kernel == 1) {
    plan->row_tile = 256;
    plan->split = 1;
    // y in int8 leaves, and an int8 tensor operand comes, by TMA; a warp's piece of the tile waits in shared memory, twice with
    // an operand, for which the ring gives up two of its six stages
    const int wide = p.y_dtype == CVMK_I32;
    plan->io = by_tma(p) ? 1 + wide : 0;
    const void* operand = nullptr;
    for (int i = 0; i < p.chain_y.n; ++i)
      if (is_tensor_step(p.chain_y.s[i])) {
        operand = p.chain_y.s[i].ptr;
        if (p.chain_y.s[i].ptr_dtype != CVMK_I8 || ((uintptr_t)operand & 15) || p.y_pitch % 16) plan->io = 0;
      }
    Params q;
    if (const int rc = make_params(*plan, &q)) return rc;
    plan->io = q.io;
    const int staged = plan->io == 1 ? 128 * (p.v ? 128 : 256) * (operand ? 2 : 1)
                     : EPI_WARPS * (plan->io ? (operand ? 6144 : 4096) : (q.straight ? 2 * TURN_BYTES : 0));
    plan->stages = std::min(6, (PAIR_SMEM_MAX - 1024 - staged) / PAIR_STAGE);
    // (no other kernel's CTAs fit beside a pair: they could hold TMEM columns and wait for its end)
    plan->smem_bytes = std::max(1024 + plan->stages * PAIR_STAGE + staged, 206 * 1024);
    const int64_t tiles = (int64_t)((p.rows + 255) / 256) * ((p.units + (p.v ? 127 : 255)) / (p.v ? 128 : 256));
    plan->grid = 2 * (int)std::min<int64_t>(tiles, sms / 2);
    if (plan->io) {
      const int columns = p.v ? 32 : 64;
      CUresult r = encode_matrix((CUtensorMap*)plan->tmap_y, p.y, p.rows, p.units, p.y_pitch, 32, CU_TENSOR_MAP_L2_PROMOTION_NONE, wide ? 64 : columns, wide);
      if (r == CUDA_SUCCESS && operand)
        r = encode_matrix((CUtensorMap*)plan->tmap_r, operand, p.rows, p.units, p.y_pitch, 32, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, columns);
      if (r != CUDA_SUCCESS) { set_error("dense_lut_prepare: tensor map rejected (CUresult %d)", (int)r); return CVMK_ERR_CUDA; }
    }
    return encode_operands(plan, 128, 128);
  }
  plan->row_tile = cut.row_tile;
  plan->split = cut.split;
  const int64_t tiles = (int64_t)((p.units + tile_units - 1) / tile_units) * ((p.rows + plan->row_tile - 1) / plan->row_tile);
  // (two CTAs an SM, with a shorter ring: 4835 rows 660 -> 293 in tiles of 64 13.4 us, one an SM 22.3)
  const int limit = plan->row_tile <= 64 ? 112 * 1024 : SMALL_SMEM_MAX;
  auto smem_of = [&](int stages) { return 1024 + small_ring_bytes(plan->row_tile, stages) + table_room; };
  plan->stages = std::min((kblocks + plan->split - 1) / plan->split, MAX_STAGES);
  while (plan->stages > 2 && smem_of(plan->stages) > limit) --plan->stages;
  // The CTAs of a cluster wait for one another while they hold TMEM columns, so the columns of all CTAs that an SM has room for
  // have to be there at once: shared memory in proportion to them (512 columns to 228 KB), whatever kernels run beside this one.
  // (26 KB and more: beside a pair of CTAs of conv_tc_kernel, which takes its columns on two SMs, nothing of this kernel fits.)
  int columns = 32;
  while (columns < plan->row_tile) columns *= 2;
  plan->smem_bytes = std::max({smem_of(plan->stages), 26 * 1024, columns * 460});
  plan->grid = (int)(tiles * plan->split);

  return encode_operands(plan, plan->row_tile, 64);
}

extern "C" int cvmk_dense_lut_launch(const cvmk_dense_lut_plan* plan, cvmk_stream_t stream) {
  if (!plan) { set_error("dense_lut_launch: null plan"); return CVMK_ERR_ARG; }
  const cvmk_dense_lut_desc& d = plan->d;
  if (d.rows == 0) return CVMK_OK;
  Params p;
  if (const int rc = make_params(*plan, &p)) return rc;
  const bool pair = plan->kernel == 1;
  const int tile_units = p.gated ? 64 : 128;   // of the small kernel
  const int kind = !p.straight ? GENERAL : (!p.io ? TURNED : (p.io == 1 && p.table_s_dtype == CVMK_I8 ? USUAL : WIDE));

  static bool attr_of_device[64] = {false};
  int dev = 0;
  if (check_cuda(cudaGetDevice(&dev), "dense_lut_launch: cudaGetDevice")) return CVMK_ERR_CUDA;
  if (dev != plan->device) { set_error("dense_lut_launch: the plan was made for device %d, and %d is current", plan->device, dev); return CVMK_ERR_ARG; }
  if (!attr_of_device[dev & 63]) {
    auto allow = [](auto k, int bytes) {
      const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      return e == cudaSuccess ? cudaFuncSetAttribute(k, cudaFuncAttributePreferredSharedMemoryCarveout, 100) : e;
    };
    if (check_cuda(allow(dense_lut_small_kernel<4>, SMALL_SMEM_MAX), "cudaFuncSetAttribute(dense_lut_small_kernel)") ||
        check_cuda(allow(dense_lut_small_kernel<8>, SMALL_SMEM_MAX), "cudaFuncSetAttribute(dense_lut_small_kernel)") ||
        check_cuda(allow(dense_lut_pair_kernel<USUAL>, PAIR_SMEM_MAX), "cudaFuncSetAttribute(dense_lut_pair_kernel)") ||
        check_cuda(allow(dense_lut_pair_kernel<WIDE>, PAIR_SMEM_MAX), "cudaFuncSetAttribute(dense_lut_pair_kernel)") ||
        check_cuda(allow(dense_lut_pair_kernel<TURNED>, PAIR_SMEM_MAX), "cudaFuncSetAttribute(dense_lut_pair_kernel)") ||
        check_cuda(allow(dense_lut_pair_kernel<GENERAL>, PAIR_SMEM_MAX), "cudaFuncSetAttribute(dense_lut_pair_kernel)"))
      return CVMK_ERR_CUDA;
    attr_of_device[dev & 63] = true;
  }
  CUtensorMap tx, tw, tv, ty, tr;
  memcpy(&ty, plan->tmap_y, sizeof(ty));
  memcpy(&tr, plan->tmap_r, sizeof(tr));
  memcpy(&tx, plan->tmap_x, sizeof(tx));
  memcpy(&tw, plan->tmap_w, sizeof(tw));
  memcpy(&tv, plan->tmap_v, sizeof(tv));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)plan->grid);
  cfg.blockDim = dim3(pair ? PAIR_THREADS : THREADS);
  cfg.dynamicSmemBytes = (size_t)plan->smem_bytes;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = pair ? 2u : (unsigned)plan->split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pair || plan->split > 1 ? 2 : 1;
  if (pair) {
    static void (*const kernels[])(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, Params) = {
        dense_lut_pair_kernel<USUAL>, dense_lut_pair_kernel<WIDE>, dense_lut_pair_kernel<TURNED>, dense_lut_pair_kernel<GENERAL>};
    return check_cuda(cudaLaunchKernelEx(&cfg, kernels[kind], tx, tw, tv, ty, tr, p), "dense_lut_pair_kernel launch");
  }
  return check_cuda(cudaLaunchKernelEx(&cfg, tile_units / p.split * p.row_tile < 8 * THREADS ? dense_lut_small_kernel<4> : dense_lut_small_kernel<8>, tx, tw, tv, p), "dense_lut_small_kernel launch");
}
