// Sampling with temperature, top-k, min-p and top-p from given random numbers, in whole numbers (cvmk_sample).
//
// A row belongs to one CTA, or to a cluster of them with a contiguous slice each.  A slice is read once, by a bulk
// copy into shared memory; every later pass over it (maximum, the histograms of a cut, the draw) reads it there.
// A cut (the k-th place, or the place where the running weight reaches the top_p share) is found digit by digit: a
// histogram of the next ten bits of d = max - x over the elements that share the bits before, summed over the cluster,
// and the bin in which the running count or weight reaches the target.  What is left of a row is then all elements with
// d < D and the first `ties` ones, in index order, with d = D: neither a sort nor a list.
// Counts and weights are whole numbers, so their order of summation changes nothing.
#include <cuda_runtime.h>
#include "common.cuh"

namespace cvmk {
namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int DIGIT = 10, BINS = 1 << DIGIT;
constexpr int TABLE_SMEM_MAX = 4096;   // entries
constexpr int SMEM_MAX = 226 * 1024;
constexpr uint32_t FULL = 0xffffffffu;

struct Params {
  cvmk_sample_desc d;
  int split, slice;        // CTAs of a row; elements of a CTA, a multiple of 4
  int table_smem;          // 1: the table is copied to shared memory
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
  uint32_t d;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(smem_addr(p)), "r"(rank));
  return d;
}
__device__ __forceinline__ uint32_t load32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t load64(uint32_t addr) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}
__device__ __forceinline__ uint64_t warp_scan(uint64_t v) {   // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t t = __shfl_up_sync(FULL, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// What a thread knows of its row.
struct Row {
  const int32_t* x;      // the slice in shared memory
  const int32_t* table;
  int first, last;       // valid places of the slice: first <= j < last
  int32_t top;           // the largest score
  uint32_t scale, last_entry;
  uint64_t min_weight;   // weights below this over 2^30 are filtered out
  uint32_t split;
  __device__ __forceinline__ uint32_t dist(int j) const { return (uint32_t)top - (uint32_t)x[j]; }
  __device__ __forceinline__ uint32_t raw_weight(uint32_t d) const {
    const uint64_t q = (uint64_t)d * scale >> 16;
    const int32_t w = table[q < last_entry ? (uint32_t)q : last_entry];
    return (uint32_t)max(w, 0);
  }
  __device__ __forceinline__ uint32_t weight(uint32_t d) const {   // 0 where min_p filters it out
    const uint32_t w = raw_weight(d);
    return ((uint64_t)w << 30) >= min_weight ? w : 0u;
  }
  __device__ __forceinline__ void sync() const {
    if (split > 1) asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
  }
};

struct Shared {
  uint32_t hist[2][2][BINS];   // [buffer][low 16 bits and rest of a weight | count, -][bin]
  uint64_t scan[WARPS];
  uint64_t mass[WARPS];        // of this CTA's warps: weight of what lies in front of the cut
  uint32_t ties[WARPS], kept[WARPS];
  int32_t lo[WARPS], hi[WARPS];
  int32_t slice_lo, slice_hi;
  uint32_t late;               // the slice has not arrived
  uint64_t cta_mass;
  uint32_t cta_ties, cta_kept;
  uint64_t found_before, found_size, total;
  int found;
  uint64_t bar;
};

// The elements in front of a cut: all with d < D and the first `ties`, in index order, with d = D.
struct Cut {
  uint64_t D;
  uint32_t ties;
};

// One digit: the histogram of `count or weight` over the elements with d < limit whose bits from `shift + bits` on are `prefix`,
// summed over the cluster; buffer alternates from call to call, so that one barrier a call is enough.
template <bool WEIGHT>
__device__ void histogram(const Row& r, Shared& s, int buffer, uint64_t limit, uint32_t prefix, int shift, int bits) {
  uint32_t* h0 = s.hist[buffer][0];
  uint32_t* h1 = s.hist[buffer][1];
  for (int i = threadIdx.x; i < BINS; i += THREADS) h0[i] = h1[i] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int j0 = r.first & ~31; j0 < r.last; j0 += THREADS) {
    const int j = j0 + (int)threadIdx.x;
    bool in = j >= r.first && j < r.last;
    uint32_t d = 0, w = 1;
    if (in) {
      d = r.dist(j);
      in = d < limit && ((uint64_t)d >> (shift + bits)) == prefix;
    }
    if (WEIGHT && in) {
      w = r.weight(d);
      in = w > 0;
    }
    const uint32_t bin = (d >> shift) & ((1u << bits) - 1u);
    const uint32_t mask = __ballot_sync(FULL, in);
    if (in) {
      int same;
      __match_all_sync(mask, bin, &same);
      if (same) {   // one bin for the whole warp
        const uint32_t a = WEIGHT ? __reduce_add_sync(mask, w & 0xffffu) : (uint32_t)__popc(mask);
        const uint32_t b = WEIGHT ? __reduce_add_sync(mask, w >> 16) : 0u;
        if (lane == __ffs(mask) - 1) {
          atomicAdd(&h0[bin], a);
          if (WEIGHT && b) atomicAdd(&h1[bin], b);
        }
      } else {
        atomicAdd(&h0[bin], WEIGHT ? w & 0xffffu : 1u);
        if (WEIGHT && w >> 16) atomicAdd(&h1[bin], w >> 16);
      }
    }
  }
  r.sync();
}

// Sums of the cluster's histograms in bins 2t, 2t + 1 (t: the thread) and the running sum in front of them.
template <bool WEIGHT>
__device__ void running(const Row& r, Shared& s, int buffer, uint64_t (&own)[2], uint64_t& before, uint64_t& total) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  own[0] = own[1] = 0;
  for (uint32_t c = 0; c < r.split; ++c) {
    const uint64_t a = load64(r.split > 1 ? remote(&s.hist[buffer][0][2 * t], c) : smem_addr(&s.hist[buffer][0][2 * t]));
    own[0] += (uint32_t)a;
    own[1] += a >> 32;
    if (WEIGHT) {
      const uint64_t b = load64(r.split > 1 ? remote(&s.hist[buffer][1][2 * t], c) : smem_addr(&s.hist[buffer][1][2 * t]));
      own[0] += (uint64_t)(uint32_t)b << 16;
      own[1] += b >> 32 << 16;
    }
  }
  const uint64_t sum = own[0] + own[1], inc = warp_scan(sum);
  if (lane == 31) s.scan[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const uint64_t v = lane < WARPS ? s.scan[lane] : 0, all = warp_scan(v);
    if (lane < WARPS) s.scan[lane] = all - v;
    if (lane == WARPS - 1) s.total = all;
  }
  __syncthreads();
  before = s.scan[warp] + inc - sum;
  total = s.total;
}

// Where, in the order of d, the count (or the weight) of the elements with d < limit reaches need(total); `fallback` is the
// cut if the total is less than that.
template <bool WEIGHT, typename Need>
__device__ Cut find_cut(const Row& r, Shared& s, int& buffer, uint64_t limit, int range_bits, const Need& need_of, const Cut& whole, uint32_t tie_weight) {
  int bits = min(range_bits, DIGIT), shift = range_bits - bits;
  uint32_t prefix = 0;
  uint64_t need = 0;
  for (bool first = true;; first = false) {
    histogram<WEIGHT>(r, s, buffer, limit, prefix, shift, bits);
    uint64_t own[2], before, total;
    running<WEIGHT>(r, s, buffer, own, before, total);
    buffer ^= 1;
    if (first) {
      need = need_of(total);
      if (need > total) {   // the cut lies among the ties of `whole`
        Cut c = whole;
        if (tie_weight) c.ties = (uint32_t)min((uint64_t)whole.ties, (need - total + tie_weight - 1) / tie_weight);
        return c;
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (before < need && need <= before + own[k]) {
        s.found = 2 * (int)threadIdx.x + k;
        s.found_before = before;
        s.found_size = own[k];
      }
      before += own[k];
    }
    __syncthreads();
    const uint64_t rest = need - s.found_before, size = s.found_size;
    prefix = (prefix << bits) | (uint32_t)s.found;
    __syncthreads();
    Cut c;
    if (rest == size) {   // all of the bin, as far as it lies in front of the limit
      c.D = min(((uint64_t)prefix + 1) << shift, limit);
      c.ties = 0;
      return c;
    }
    if (shift == 0) {
      const uint32_t w = WEIGHT ? r.weight(prefix) : 1u;
      c.D = prefix;
      c.ties = (uint32_t)((rest + w - 1) / w);
      return c;
    }
    need = rest;
    bits = min(shift, DIGIT);
    shift -= bits;
  }
}

__global__ void __launch_bounds__(THREADS) sample_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = p.split > 1 ? (int)cluster_rank() : 0, row = (int)blockIdx.x / p.split;
  int32_t* const x = reinterpret_cast<int32_t*>(smem_raw);
  int32_t* const table_s = x + p.slice;
  const cvmk_sample_desc& d = p.d;
  const int vocab = d.vocab;
  const int32_t* src = d.logits + (size_t)row * (size_t)d.pitch;
  // Places are counted from the 16-byte boundary at or in front of the row, so that slices begin on one.
  const int skew = (int)((reinterpret_cast<uintptr_t>(src) >> 2) & 3);
  const int begin = rank * p.slice;                       // this slice's place 0
  Row r;
  r.x = x;
  r.first = min(max(skew - begin, 0), p.slice);
  r.last = min(max(skew + vocab - begin, r.first), p.slice);
  r.split = (uint32_t)p.split;

  pdl_trigger();
  if (tid == 0) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_addr(&s.bar)));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  // whole 16-byte words by the bulk engine, the ragged ends by threads
  const int b0 = min((r.first + 3) & ~3, r.last), b1 = max(b0, r.last & ~3);
  const int32_t* at = src - skew + begin;                 // of place 0
  if (tid == 0) {
    const uint32_t bytes = (uint32_t)(b1 - b0) * 4u;
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(&s.bar)), "r"(bytes) : "memory");
    if (bytes)
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_addr(x + b0)),
                   "l"(at + b0), "r"(bytes), "r"(smem_addr(&s.bar))
                   : "memory");
  }
  if (tid >= 32 && tid < 35 && r.first + tid - 32 < b0) x[r.first + tid - 32] = at[r.first + tid - 32];
  if (tid >= 35 && tid < 38 && b1 + tid - 35 < r.last) x[b1 + tid - 35] = at[b1 + tid - 35];
  if (p.table_smem)
    for (int i = tid; i < d.table_len; i += THREADS) table_s[i] = d.table[i];
  r.table = p.table_smem ? table_s : d.table;
  r.last_entry = (uint32_t)d.table_len - 1u;
  r.scale = (uint32_t)max(d.scale[row], 0);
  const int k = d.top_k ? d.top_k[row] : 0;
  const uint64_t one = 1u << 30;
  const uint64_t top_p = d.top_p ? (uint64_t)min(max(d.top_p[row], 0), (int)one) : one;
  const uint64_t min_p = d.min_p ? (uint64_t)min(max(d.min_p[row], 0), (int)one) : 0;
  const uint64_t u = (uint64_t)(d.random[row] & 0x7fffffff);
  __syncthreads();
  // (bounded: the copy is the only thing that is waited for)
  bool landed = false;
  for (uint32_t i = 0; !landed && i < (1u << 19); ++i) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], 0, 2000;\nselp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_addr(&s.bar))
        : "memory");
    landed = ok != 0;
  }

  // ---- the largest and the smallest score
  int32_t lo = INT32_MAX, hi = INT32_MIN;
  for (int j = r.first + tid; j < r.last; j += THREADS) {
    lo = min(lo, x[j]);
    hi = max(hi, x[j]);
  }
  lo = __reduce_min_sync(FULL, lo);
  hi = __reduce_max_sync(FULL, hi);
  if (lane == 0) { s.lo[warp] = lo; s.hi[warp] = hi; }
  __syncthreads();
  if (warp == 0) {
    lo = __reduce_min_sync(FULL, lane < WARPS ? s.lo[lane] : INT32_MAX);
    hi = __reduce_max_sync(FULL, lane < WARPS ? s.hi[lane] : INT32_MIN);
    if (lane == 0) { s.slice_lo = lo; s.slice_hi = hi; s.late = landed ? 0u : 1u; }
  }
  r.sync();
  lo = s.slice_lo;
  hi = s.slice_hi;
  uint32_t late = s.late;
  for (int c = 0; p.split > 1 && c < p.split; ++c) {
    late |= load32(remote(&s.late, (uint32_t)c));
    lo = min(lo, (int32_t)load32(remote(&s.slice_lo, (uint32_t)c)));
    hi = max(hi, (int32_t)load32(remote(&s.slice_hi, (uint32_t)c)));
  }
  if (late) {   // a copy that never came (its wait is bounded): no element is drawn
    if (rank == 0 && tid == 0) d.token[row] = -1;
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
    __syncwarp();
    r.sync();
    return;
  }
  r.top = hi;
  r.min_weight = 0;
  r.min_weight = min_p * (uint64_t)r.raw_weight(0);
  const uint32_t range = (uint32_t)hi - (uint32_t)lo;
  const int range_bits = max(1, 32 - __clz((int)range));

  // ---- the cuts
  Cut cut = {(uint64_t)1 << 32, 0};   // everything
  int buffer = 0;
  if (k >= 1 && k < vocab)
    cut = find_cut<false>(r, s, buffer, (uint64_t)1 << 32, range_bits, [=](uint64_t) { return (uint64_t)k; }, cut, 0u);
  if (top_p < one) {
    const uint32_t w = cut.ties ? r.weight((uint32_t)cut.D) : 0u;
    const uint32_t ties = cut.ties;
    cut = find_cut<true>(r, s, buffer, cut.D, range_bits, [=](uint64_t strict) {
      const uint64_t all = strict + (uint64_t)ties * w;
      const uint64_t need = top_p * (all >> 30) + ((top_p * (all & (one - 1)) + one - 1) >> 30);
      return need > 1 ? need : (uint64_t)1;
    }, cut, w);
  }

  // ---- the draw: every warp sums a contiguous run of the slice
  const uint32_t tie_weight = cut.ties ? r.weight((uint32_t)cut.D) : 0u;
  const int run = ((p.slice + WARPS - 1) / WARPS + 31) & ~31;
  const int j0 = warp * run, j1 = min(j0 + run, r.last);
  uint64_t mass = 0;
  uint32_t ties = 0, kept = 0;
  for (int j = max(j0, r.first & ~31) + lane; j < j1; j += 32) {
    if (j < r.first) continue;
    const uint32_t dj = r.dist(j);
    if (dj < cut.D) {
      const uint32_t w = r.weight(dj);
      mass += w;
      kept += w > 0;
    } else {
      ties += dj == cut.D;
    }
  }
  mass = warp_sum(mass);
  ties = __reduce_add_sync(FULL, ties);
  kept = __reduce_add_sync(FULL, kept);
  if (lane == 0) { s.mass[warp] = mass; s.ties[warp] = ties; s.kept[warp] = kept; }
  __syncthreads();
  if (tid == 0) {
    uint64_t m = 0;
    uint32_t t = 0, n = 0;
    for (int i = 0; i < WARPS; ++i) { m += s.mass[i]; t += s.ties[i]; n += s.kept[i]; }
    s.cta_mass = m; s.cta_ties = t; s.cta_kept = n;
  }
  r.sync();
  uint64_t all = 0, front_mass = 0;
  uint32_t front_ties = 0, all_kept = cut.ties && tie_weight ? cut.ties : 0;
  for (int c = 0; c < p.split; ++c) {
    const uint64_t m = p.split > 1 ? load64(remote(&s.cta_mass, (uint32_t)c)) : s.cta_mass;
    const uint32_t t = p.split > 1 ? load32(remote(&s.cta_ties, (uint32_t)c)) : s.cta_ties;
    const uint32_t n = p.split > 1 ? load32(remote(&s.cta_kept, (uint32_t)c)) : s.cta_kept;
    all += m;
    all_kept += n;
    if (c < rank) { front_mass += m; front_ties += t; }
  }
  all += (uint64_t)cut.ties * tie_weight;
  // of a mass of nothing the first of the order is taken: the first element with d = 0 then weighs 1, all others nothing
  const bool nothing = all == 0;
  const uint64_t target = nothing ? 0 : u * (all >> 31) + ((u * (all & 0x7fffffffu)) >> 31);
  if (nothing) {
    cut.D = 0;
    cut.ties = 1;
  }
  const uint32_t each = nothing ? 1u : tie_weight;
  if (nothing) {   // (rare: the ties of the new cut are counted again)
    uint32_t n = 0;
    for (int j = max(j0, r.first & ~31) + lane; j < j1; j += 32) n += j >= r.first && r.dist(j) == 0;
    n = __reduce_add_sync(FULL, n);
    if (lane == 0) { s.mass[warp] = 0; s.ties[warp] = n; }
    __syncthreads();
    r.sync();   // (nobody still reads the sums of before)
    if (tid == 0) {
      uint32_t t = 0;
      for (int i = 0; i < WARPS; ++i) t += s.ties[i];
      s.cta_ties = t;
    }
    r.sync();
    front_mass = 0;
    front_ties = 0;
    for (int c = 0; c < rank; ++c) front_ties += load32(remote(&s.cta_ties, (uint32_t)c));
  }
  // every warp: the weight in front of its run, and whether the target lies in it
  for (int i = 0; i < warp; ++i) { front_mass += s.mass[i]; front_ties += s.ties[i]; }
  const auto running_at = [&](uint64_t m, uint32_t t) { return m + (uint64_t)min(t, cut.ties) * each; };
  if (running_at(front_mass, front_ties) <= target && target < running_at(front_mass + s.mass[warp], front_ties + s.ties[warp])) {
    for (int j = max(j0, r.first & ~31); j < j1; j += 32) {
      const int at_j = j + lane;
      uint64_t w = 0;
      uint32_t tie = 0;
      if (at_j >= r.first && at_j < j1) {
        const uint32_t dj = r.dist(at_j);
        if (dj < cut.D) w = r.weight(dj);
        else tie = dj == cut.D;
      }
      const uint32_t tie_mask = __ballot_sync(FULL, tie != 0);
      const uint64_t inc = front_mass + warp_scan(w);
      const uint32_t tie_inc = front_ties + (uint32_t)__popc(tie_mask & (FULL >> (31 - lane)));
      const uint32_t hit = __ballot_sync(FULL, running_at(inc, tie_inc) > target);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          d.token[row] = begin + at_j - skew;
          if (d.weight) d.weight[row] = (int32_t)r.raw_weight(r.dist(at_j));
          if (d.mass) d.mass[row] = (int64_t)all;
          if (d.kept) d.kept[row] = (int32_t)all_kept;
        }
        break;
      }
      front_mass = __shfl_sync(FULL, inc, 31);
      front_ties += (uint32_t)__popc(tie_mask);
    }
  }
  __syncwarp();
  if (p.split > 1) r.sync();   // nobody still reads this CTA's memory
}

}  // namespace
}  // namespace cvmk

using namespace cvmk;

extern "C" int cvmk_sample(const cvmk_sample_desc* d, cvmk_stream_t stream) {
  if (!d) { set_error("sample: null argument"); return CVMK_ERR_ARG; }
  if (d->rows < 0 || d->vocab < 1 || d->vocab > CVMK_SAMPLE_MAX_VOCAB || d->table_len < 1) {
    set_error("sample: sizes outside 0 <= rows, 1 <= vocab <= %d, 1 <= table_len", CVMK_SAMPLE_MAX_VOCAB);
    return CVMK_ERR_ARG;
  }
  if (d->pitch && (d->pitch < d->vocab || d->pitch >> 40)) { set_error("sample: bad pitch"); return CVMK_ERR_ARG; }
  if (d->rows == 0) return CVMK_OK;
  if (!d->logits || !d->table || !d->scale || !d->random || !d->token) { set_error("sample: null operand"); return CVMK_ERR_ARG; }
  const uintptr_t odd = (uintptr_t)d->logits | (uintptr_t)d->table | (uintptr_t)d->scale | (uintptr_t)d->top_k | (uintptr_t)d->top_p |
                        (uintptr_t)d->min_p | (uintptr_t)d->random | (uintptr_t)d->token | (uintptr_t)d->weight | (uintptr_t)d->kept;
  if ((odd & 3) || ((uintptr_t)d->mass & 7)) { set_error("sample: an operand is not aligned to its elements"); return CVMK_ERR_ARG; }
  Params p;
  p.d = *d;
  if (!p.d.pitch) p.d.pitch = d->vocab;
  p.table_smem = d->table_len <= TABLE_SMEM_MAX;
  int sms = 148, dev = 0;
  if (check_cuda(cudaGetDevice(&dev), "sample: cudaGetDevice")) return CVMK_ERR_CUDA;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  auto slice_of = [&](int split) { return ((d->vocab + 3 + split - 1) / split + 3) & ~3; };
  auto smem_of = [&](int split) { return slice_of(split) * 4 + (p.table_smem ? d->table_len * 4 : 0); };
  const int room = SMEM_MAX - (int)sizeof(Shared);
  p.split = 1;
  while (p.split < 8 && (smem_of(p.split) > 90 * 1024 || ((int64_t)d->rows * p.split * 2 <= 2 * sms && slice_of(p.split) > 2048))) p.split *= 2;
  p.slice = slice_of(p.split);
  const int smem = smem_of(p.split);
  if (smem > room || (int64_t)d->rows * p.split > INT32_MAX) { set_error("sample: too large"); return CVMK_ERR_ARG; }

  static bool attr_of_device[64] = {false};
  if (!attr_of_device[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, room);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    if (check_cuda(e, "cudaFuncSetAttribute(sample_kernel)")) return CVMK_ERR_CUDA;
    attr_of_device[dev & 63] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(d->rows * p.split));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.split > 1 ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, sample_kernel, p), "sample_kernel launch");
}
