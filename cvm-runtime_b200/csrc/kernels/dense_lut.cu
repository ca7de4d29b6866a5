// dense with a table as its activation, gated by a second dense or not (cvmk_dense_lut_*): tensor-core
// products of int8 operands whose int32 sums never leave the chip.
//
// dense_lut_small_kernel: the weights are the 128-row operand of the tensor instructions and the rows of x
// (up to 256 of them) its columns, so a launch is one stream of weights whatever the batch.  A gated tile is
// 64 units: 64 rows of w and under them the same 64 of v, so that one accumulator holds both products of a
// unit; ungated, 128 units of w.  The reduction of a tile can be cut over a cluster of CTAs: every CTA
// writes its partial sums (int32: exact in any order) to its shared memory and each finishes its share of the
// units from all of them.
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
constexpr int SMEM_MAX = 226 * 1024;

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
  DevChain cw, cv, cy;
};

__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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

// The chain in front of the table, and the table: `table_s` is its copy in shared memory, or nullptr.
template <int V>
__device__ __forceinline__ void activate(const Params& p, const uint8_t* table_s, int32_t (&a)[V]) {
  apply_chain<V>(p.cw, a, 0, 0, 0, nullptr, -1, p.first_w);
  const int last = p.table_len - 1;
  const void* t = p.table_smem ? (const void*)table_s : p.table;
  if (p.table_dtype == CVMK_I8) {
#pragma unroll
    for (int j = 0; j < V; ++j) a[j] = reinterpret_cast<const int8_t*>(t)[min(max(a[j], 0), last)];
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) a[j] = reinterpret_cast<const int32_t*>(t)[min(max(a[j], 0), last)];
  }
}

__device__ __forceinline__ void copy_table(const Params& p, uint8_t* table_s, int t, int threads) {
  for (int i = t; i < p.table_len * p.table_dtype; i += threads) table_s[i] = reinterpret_cast<const uint8_t*>(p.table)[i];
}

// bytes of one row of partial sums: 16 more than the sums, so that eight rows of one column lie in different banks
__host__ __device__ inline int sums_pitch(int row_tile) { return row_tile * 4 + 16; }
__host__ __device__ inline int small_ring_bytes(int row_tile, int stages) {
  const int ring = stages * (W_BYTES + row_tile * BLOCK_K), sums = BLOCK_M * sums_pitch(row_tile);
  return ring > sums ? ring : sums;
}

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
  // This CTA's share of the units, four rows of x a thread and turn.
  if (!abort_flag) {
    pdl_wait();
    const int share = tile_units >> p.split_log2, jobs = share * (p.row_tile >> 2);
    for (int k = (int)threadIdx.x; k < jobs; k += THREADS) {
      const int q = k / share, ul = rank * share + k - q * share, unit = unit0 + ul, r0 = row0 + 4 * q;
      if (unit >= p.units || r0 >= p.rows) continue;
      int32_t a[4], b[4];
      const uint32_t at = ring + (uint32_t)(ul * pitch + 16 * q), at_v = at + (uint32_t)(64 * pitch);
      const int32_t ba = bias_s[ul], bb = bias_s[p.gated ? ul + 64 : ul];
#pragma unroll
      for (int j = 0; j < 4; ++j) { a[j] = ba; b[j] = bb; }
      for (int s = 0; s < p.split; ++s) {
        const int4 g = load_remote(p.split > 1 ? map_rank(at, (uint32_t)s) : at);
        a[0] += g.x; a[1] += g.y; a[2] += g.z; a[3] += g.w;
        if (p.gated) {
          const int4 h = load_remote(p.split > 1 ? map_rank(at_v, (uint32_t)s) : at_v);
          b[0] += h.x; b[1] += h.y; b[2] += h.z; b[3] += h.w;
        }
      }
      const int n = min(4, p.rows - r0);
      const long long lin = (long long)r0 * p.y_pitch + unit;
      int32_t pre[4] = {0, 0, 0, 0};
      if (p.res) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < n) pre[j] = p.res_dtype == CVMK_I8 ? reinterpret_cast<const int8_t*>(p.res)[lin + j * p.y_pitch]
                                                     : reinterpret_cast<const int32_t*>(p.res)[lin + j * p.y_pitch];
      }
      activate<4>(p, table_s, a);
      if (p.gated) {
        apply_chain<4>(p.cv, b, 0, 0, 0, nullptr, -1, p.first_v);
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = (int32_t)((uint32_t)a[j] * (uint32_t)b[j]);
      }
      apply_chain<4, true>(p.cy, a, 0, 0, 0, pre, p.res_step);
#pragma unroll
      for (int j = 0; j < 4; ++j)
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

// A row-major int8 matrix, read in boxes of BLOCK_K bytes of `box_rows` rows; zeros outside.
CUresult encode_matrix(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t pitch, int box_rows, CUtensorMapL2promotion promo) {
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch};
  cuuint32_t box[2] = {(cuuint32_t)BLOCK_K, (cuuint32_t)box_rows}, estr[2] = {1, 1};
  return encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, promo, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

bool is_tensor_step(const cvmk_ep_step& s) { return s.op == CVMK_EP_ADD_T || s.op == CVMK_EP_SUB_T || s.op == CVMK_EP_RSUB_T; }
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
  if (!encoder()) { set_error("dense_lut_prepare: the driver has no cuTensorMapEncodeTiled"); return CVMK_ERR_CUDA; }

  const int sms = sm_count(), kblocks = (p.K + BLOCK_K - 1) / BLOCK_K, tile_units = p.v ? 64 : 128;
  const int64_t table_bytes = (int64_t)p.table_len * p.table_dtype;
  plan->table_smem = table_bytes <= TABLE_SMEM_MAX ? (int)table_bytes : 0;
  const int table_room = (plan->table_smem + 15) & ~15;
  const int row_tiles = (p.rows + 255) / 256;
  plan->row_tile = ((p.rows + row_tiles - 1) / row_tiles + 15) & ~15;
  const int64_t unit_tiles = (p.units + tile_units - 1) / tile_units, tiles = unit_tiles * row_tiles;
  const int per_sm = plan->row_tile <= 64 ? 2 : 1, limit = per_sm == 2 ? 112 * 1024 : SMEM_MAX;
  plan->split = 1;
  while (plan->split < 8 && kblocks >= 4 * plan->split && tiles * 2 * plan->split <= (int64_t)per_sm * sms) plan->split *= 2;
  auto smem_of = [&](int stages) { return 1024 + small_ring_bytes(plan->row_tile, stages) + table_room; };
  plan->stages = std::min((kblocks + plan->split - 1) / plan->split, MAX_STAGES);
  while (plan->stages > 2 && smem_of(plan->stages) > limit) --plan->stages;
  // (26 KB and more: beside a pair of CTAs of conv_tc_kernel, which takes its TMEM columns on two SMs, nothing of this kernel fits)
  plan->smem_bytes = std::max(smem_of(plan->stages), 26 * 1024);
  plan->grid = (int)(tiles * plan->split);

  CUresult r = encode_matrix((CUtensorMap*)plan->tmap_x, p.x, p.rows, p.K, p.x_pitch, plan->row_tile, CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
  if (r == CUDA_SUCCESS) r = encode_matrix((CUtensorMap*)plan->tmap_w, p.w, p.units, p.K, p.w_pitch, 64, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (r == CUDA_SUCCESS) r = encode_matrix((CUtensorMap*)plan->tmap_v, p.v ? p.v : p.w, p.units, p.K, p.w_pitch, 64, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (r != CUDA_SUCCESS) { set_error("dense_lut_prepare: tensor map rejected (CUresult %d)", (int)r); return CVMK_ERR_CUDA; }
  return CVMK_OK;
}

extern "C" int cvmk_dense_lut_launch(const cvmk_dense_lut_plan* plan, cvmk_stream_t stream) {
  if (!plan) { set_error("dense_lut_launch: null plan"); return CVMK_ERR_ARG; }
  const cvmk_dense_lut_desc& d = plan->d;
  if (d.rows == 0) return CVMK_OK;
  Params p;
  memset(&p, 0, sizeof(p));
  p.y = d.y; p.y_pitch = d.y_pitch; p.y_dtype = d.y_dtype;
  p.rows = d.rows; p.units = d.units;
  p.kblocks = (d.K + BLOCK_K - 1) / BLOCK_K;
  p.gated = d.v != nullptr;
  p.params_static = d.params_static;
  const int tile_units = p.gated ? 64 : 128;
  p.unit_tiles = (d.units + tile_units - 1) / tile_units;
  p.row_tile = plan->row_tile;
  p.row_tiles = (d.rows + p.row_tile - 1) / p.row_tile;
  p.stages = plan->stages;
  p.split = plan->split;
  while ((1 << p.split_log2) < p.split) ++p.split_log2;
  p.tmem_cols = 32;
  while (p.tmem_cols < p.row_tile) p.tmem_cols *= 2;
  p.table = d.table; p.table_len = d.table_len; p.table_dtype = d.table_dtype; p.table_smem = plan->table_smem;
  p.status = d.status;
  if (lower_chain(d.chain_w, &p.cw) || lower_chain(d.chain_v, &p.cv) || lower_chain(d.chain_y, &p.cy)) return CVMK_ERR_ARG;
  if (p.cw.n && p.cw.s[0].op == K_ADD_C) { p.bias_w = (const int32_t*)p.cw.s[0].ptr; p.first_w = 1; }
  if (p.cv.n && p.cv.s[0].op == K_ADD_C) { p.bias_v = (const int32_t*)p.cv.s[0].ptr; p.first_v = 1; }
  p.res_step = -1;
  for (int i = 0; i < p.cy.n; ++i)
    if (p.cy.s[i].op == K_ADD_T || p.cy.s[i].op == K_SUB_T || p.cy.s[i].op == K_RSUB_T) {
      p.res = p.cy.s[i].ptr; p.res_dtype = p.cy.s[i].dt; p.res_step = i;
    }

  static bool attr_of_device[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_of_device[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(dense_lut_small_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(dense_lut_small_kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    if (check_cuda(e, "cudaFuncSetAttribute(dense_lut_small_kernel)")) return CVMK_ERR_CUDA;
    attr_of_device[dev & 63] = true;
  }
  CUtensorMap tx, tw, tv;
  memcpy(&tx, plan->tmap_x, sizeof(tx));
  memcpy(&tw, plan->tmap_w, sizeof(tw));
  memcpy(&tv, plan->tmap_v, sizeof(tv));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)plan->grid);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = (size_t)plan->smem_bytes;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)plan->split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = plan->split > 1 ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, dense_lut_small_kernel, tx, tw, tv, p), "dense_lut_small_kernel launch");
}
