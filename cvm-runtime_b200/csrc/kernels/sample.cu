// Sampling with temperature, top-k, min-p and top-p from given random numbers, in whole numbers (cvmk_sample).
//
// A row belongs to one CTA, or to a cluster of them with a contiguous slice each.  A slice is read once, by a bulk copy into
// shared memory, and every later pass reads it there; or, where there are so many rows that more of them at work are worth more
// than that, each pass reads it from global memory (L2).  What is left of a row after its filters is all elements with
// d = max - x < D and the first `ties` ones, in index order, with d = D: the filters only look for that cut, and neither sort
// nor list the row.
//   top_k   In a CTA, the n-th largest of the maxima of its threads is a lower bound of its n-th largest element (that many
//           threads have one as large); it is bisected to a thousandth of the range of the CTA's scores, downwards.  So the
//           row's k-th is not below the least of the CTAs' bounds for n = k / CTAs.  The elements that are not below it are
//           mostly few more than k; they are put on a list, and one CTA does all the rest on it: a thread holds an element and
//           compares it with every other one, for its rank and the weight in front of it.  Where the list has no room (k beyond
//           it, hundreds of equal scores, or a score far below the others, which makes the range wide: one masked to the type's
//           lowest value) the cut is one by count: 32 rows of 131072, top_k 50, 17 us, with 2000 of each masked 76.
//   top_p   An element's weight is a function of its table index, so the elements of every index are counted; the running
//           sum of count * weight gives the index in which the share is reached and how many of its elements are needed, and
//           the cut among those is one by count again.
//   A cut by count is found digit by digit: a histogram of the next twelve bits of d over the elements that share the bits
//   before, and the bin in which the running count reaches the target.  (With a table too long for shared memory top_p goes
//   that way too, by weight.)
// The draw then sums the weights in blocks of 256 or 512 elements, finds the block, and looks up the element in it.
// Counts and weights are whole numbers, so their order of summation changes nothing.
//
// What bounds it: few rows, the chain of passes and barriers, each a trip to L2 or over a cluster (1 row of 32000 elements, all
// filters: 9.8 us, of which reading its 128 KB is 0.02; 32 rows of 131072: 23 to 26 us, 2.6).  Many rows, the passes themselves: 256 rows
// of 262144 elements take 107 us without cuts (read twice: once from memory, 41 us at the rate of a copy, once from L2), 124 with
// top_k, 251 with top_p, whose counting is an atomic in shared memory for every element above the table's last entry.  More loads
// under way (the next four requested while four are worked on) spill at the 64 registers that two CTAs an SM leave: 190 against
// 184 us over rows of all kinds; three CTAs an SM of 40 registers: 205.
//
// A launch ends whatever its operands do meanwhile: should another stream still write them, tokens mean nothing, but no place is
// looked up outside the arrays, and every CTA of a row takes the same way from barrier to barrier: all go by one reading of the
// row's parameters, by scores that are exchanged, and by counts and sums that each adds up from the same ones.
#include <cuda_runtime.h>
#include "common.cuh"

namespace cvmk {
namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int DIGIT = 12, BINS = 1 << DIGIT;       // of counts
constexpr int WDIGIT = 11, WBINS = 1 << WDIGIT;    // of weights, two words a bin
constexpr int TABLE_SMEM_MAX = 4096;    // entries; with more the table stays where it lies
constexpr int LIST = 512;               // elements on a list
constexpr int MAX_SPLIT = 8;
// Elements of a block of the draw: few, for even shares of the warps and a short search in the one that is hit, where they lie in
// shared memory (32 rows of 131072: 25.9 us with 256, 27.0 with 512); more requests at once where they do not (256 rows of 262144:
// 175 us with 512, 181 with 256).
template <bool RESIDENT>
constexpr int BLOCK_OF = RESIDENT ? 256 : 512;
constexpr int MAX_BLOCKS = CVMK_SAMPLE_MAX_VOCAB / BLOCK_OF<false> + 2;   // (a resident slice has fewer: 56 K elements at most)
static_assert(56 * 1024 / BLOCK_OF<true> + 2 <= MAX_BLOCKS, "room for the blocks of a resident slice");
constexpr uint32_t FULL = 0xffffffffu;
constexpr uint64_t ONE = 1u << 30;
constexpr int RANK_BITS = 10;           // behind a weight: one each for the elements in front

struct Params {
  cvmk_sample_desc d;
  int split, slice;        // CTAs of a row; elements of a CTA, a multiple of 4
  int table_smem;          // 1: the table is copied to shared memory
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
// The cluster's barrier, for warps whose lanes may come to it apart (behind a loop that polls, or a branch of some lanes): its
// aligned form is undefined for such a warp.
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The address, in the cluster's shared window, of `p` in the CTA of rank `rank` (of a cluster of one as well).
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
__device__ __forceinline__ uint64_t warp_scan(uint64_t v) {   // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t t = __shfl_up_sync(FULL, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

__device__ __forceinline__ void store128(uint32_t addr, uint4 v) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void store32(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ uint4 load128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
// The sums over the cluster of four words at p.  A word of another CTA takes a fifth of a microsecond to come: four requests
// are under way at a time.
__device__ __forceinline__ uint4 sum_of_cluster(const uint32_t* p, uint32_t split) {
  if (split == 1) return *reinterpret_cast<const uint4*>(p);
  uint4 sum = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int c0 = 0; c0 < MAX_SPLIT; c0 += 4) {
    if (c0 >= (int)split) break;
    uint4 v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = c0 + c < (int)split ? load128(remote(p, (uint32_t)(c0 + c))) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int c = 0; c < 4; ++c) { sum.x += v[c].x; sum.y += v[c].y; sum.z += v[c].z; sum.w += v[c].w; }
  }
  return sum;
}

// The same where the sums may not fit 32 bits.
__device__ __forceinline__ void sum_of_cluster(const uint32_t* p, uint32_t split, uint64_t (&sum)[4]) {
  sum[0] = sum[1] = sum[2] = sum[3] = 0;
  for (uint32_t c = 0; c < split; ++c) {
    const uint4 v = split > 1 ? load128(remote(p, c)) : *reinterpret_cast<const uint4*>(p);
    sum[0] += v.x; sum[1] += v.y; sum[2] += v.z; sum[3] += v.w;
  }
}

// The elements in front of a cut: all with d < D and the first `ties`, in index order, with d = D.
struct Cut {
  uint64_t D;
  uint32_t ties;
};

struct Shared {
  union {
    alignas(16) uint32_t hist[BINS];   // counts by digit or table index; weights by digit: the low 32 bits, and the high ones
    struct {                           // (a row whose cuts are found on its list needs no histogram behind it)
      alignas(16) uint4 all[LIST];     // of the row's elements: index, distance, and 64 bits to be added up
      union {
        alignas(16) int2 list[LIST];     // of the slice's: score and index
        uint2 sorted[LIST];              // those that stay, by rank: index and weight
      };
    };
  };
  union {
    struct {
      uint64_t block_mass[MAX_BLOCKS];
      uint32_t block_ties[MAX_BLOCKS];
    };
    uint64_t sums_of_list[32 * WARPS];
  };
  uint64_t mass, mass_left;               // of the list behind top_k, and behind top_p
  uint32_t left;                          // elements of it then
  uint64_t scan[WARPS];
  int32_t lo[WARPS], hi[WARPS];
  uint32_t kept[WARPS];
  uint32_t listed;
  // what every CTA of the cluster says of its slice, sent here by it
  alignas(16) int4 scores[MAX_SPLIT];     // smallest, largest, bound
  alignas(16) uint4 answer;
  alignas(16) uint4 sums[MAX_SPLIT];      // weight (low, high), ties, kept
  uint32_t late;                          // a slice has not arrived
  uint32_t tie_weight;
  uint32_t min_weight;
  alignas(16) uint4 row;                  // the row's top_k, top_p, scale and random number, as they were read
  alignas(16) uint4 row_of_all;           // by the first CTA
  uint64_t found_before, found_size;
  int found;
  uint32_t counts[MAX_SPLIT];             // elements on the CTAs' lists
  uint64_t bar;
};

extern __shared__ __align__(16) uint8_t dynamic_smem[];   // the slice, if it is resident, and the table
__device__ __forceinline__ const int32_t* resident() { return reinterpret_cast<const int32_t*>(dynamic_smem); }

// What a thread knows of its row.
struct Row {
  const int32_t* x;
  const int32_t* table;
  int first, last;       // valid places: first <= j < last
  int32_t top;           // the largest score
  uint32_t scale, last_entry, saturated;
  uint32_t min_weight;   // lighter elements are filtered out; 0 where the table has gone through that already
  uint32_t split;
  bool wide;             // the table lies in global memory
  int table_at;          // else at this place of the dynamic shared memory (known to be that: a look-up in a pointer's memory is twice as slow)
  __device__ __forceinline__ const int32_t* in_smem() const { return reinterpret_cast<const int32_t*>(dynamic_smem) + table_at; }
  // entry() in fewer instructions where scale <= 2^16 and the table lies in shared memory: distances above `far` have the last
  // entry, as `far` has, and far * scale is less than 2^31.
  bool gentle;
  uint32_t far;
  __device__ __forceinline__ uint32_t entry_of(int32_t v) const { return min((uint32_t)top - (uint32_t)v, far) * scale >> 16; }
  __device__ __forceinline__ uint32_t dist(int32_t v) const { return (uint32_t)top - (uint32_t)v; }
  // min((d * scale) >> 16, last_entry): a table in shared memory has less than 2^15 entries, and every d above
  // saturated = (2^32 - 1) / scale has a product above 2^31.
  __device__ __forceinline__ uint32_t entry(uint32_t d) const { return min(min(d, saturated) * scale >> 16, last_entry); }
  __device__ __forceinline__ uint32_t weight(uint32_t d) const {   // 0 where min_p filters it out
    if (!wide) return (uint32_t)in_smem()[entry(d)];
    const uint64_t q = (uint64_t)d * scale >> 16;
    const int32_t w = table[q < last_entry ? (uint32_t)q : last_entry];
    return w > 0 && (uint32_t)w >= min_weight ? (uint32_t)w : 0u;
  }
  // The smallest d whose entry is e or more, e <= last_entry (2^32: none).
  __device__ __forceinline__ uint64_t first_of(uint32_t e) const {
    if (e == 0) return 0;
    if (scale == 0) return (uint64_t)1 << 32;
    return min((((uint64_t)e << 16) + scale - 1) / scale, (uint64_t)1 << 32);
  }
  __device__ __forceinline__ void sync() const {
    if (split > 1) {
      cluster_arrive();
      cluster_wait();
    } else {
      __syncthreads();
    }
  }
  // The values at places j .. j + 3, j a multiple of 4 (zeros, or what lies there in shared memory, outside the valid ones).
  template <bool RESIDENT>
  __device__ __forceinline__ int4 four(int j, bool all_valid) const {
    if (RESIDENT) return all_valid || j < last ? *reinterpret_cast<const int4*>(resident() + j) : make_int4(0, 0, 0, 0);
    if (all_valid || (j >= first && j + 4 <= last)) return *reinterpret_cast<const int4*>(x + j);
    int4 v = make_int4(0, 0, 0, 0);   // (nothing outside the row is read)
    if (j >= first && j < last) v.x = x[j];
    if (j + 1 >= first && j + 1 < last) v.y = x[j + 1];
    if (j + 2 >= first && j + 2 < last) v.z = x[j + 2];
    if (j + 3 >= first && j + 3 < last) v.w = x[j + 3];
    return v;
  }
  // Calls f(value, place) for the thread's share of the valid elements: whole groups of four, and the ragged ends by a few threads.
  template <bool RESIDENT, typename F>
  __device__ __forceinline__ void each(const F& f) const {
    const int g0 = (first + 3) >> 2, g1 = last >> 2, tid = threadIdx.x;
    const int32_t* const at = RESIDENT ? resident() : x;
    if (g0 > g1) {   // (less than a group)
      if (first + tid < last) f(at[first + tid], first + tid);
      return;
    }
    const auto four = [&](const int4& v, int g) {
      f(v.x, 4 * g);
      f(v.y, 4 * g + 1);
      f(v.z, 4 * g + 2);
      f(v.w, 4 * g + 3);
    };
    constexpr int UNDER_WAY = RESIDENT ? 4 : 8;
    constexpr int step = THREADS;
    int g = g0 + tid;
    for (; g + (UNDER_WAY - 1) * step < g1; g += UNDER_WAY * step) {
      int4 v[UNDER_WAY];
#pragma unroll
      for (int i = 0; i < UNDER_WAY; ++i) v[i] = reinterpret_cast<const int4*>(at)[g + i * step];
#pragma unroll
      for (int i = 0; i < UNDER_WAY; ++i) four(v[i], g + i * step);
    }
    for (; g < g1; g += step) four(reinterpret_cast<const int4*>(at)[g], g);
    if (first + tid < 4 * g0) f(at[first + tid], first + tid);
    if (4 * g1 + tid < last) f(at[4 * g1 + tid], 4 * g1 + tid);
  }
};

// Sum over the warp of numbers below 2^45.
__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
  return __reduce_add_sync(FULL, (uint32_t)v & 0xfffffu) + ((uint64_t)__reduce_add_sync(FULL, (uint32_t)(v >> 20)) << 20);
}

// Exclusive sum of v over the threads of the CTA, and the sum of all.
__device__ __forceinline__ uint64_t block_scan(Shared& s, uint64_t v, uint64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t inc = warp_scan(v);
  __syncthreads();   // (the scan before has been read)
  if (lane == 31) s.scan[warp] = inc;
  __syncthreads();
  const uint64_t w = lane < WARPS ? s.scan[lane] : 0, sums = warp_scan(w);
  total = __shfl_sync(FULL, sums, 31);
  return __shfl_sync(FULL, sums - w, warp) + inc - v;
}

// (no CTA still reads what was there: `r`, whose histogram it was)
__device__ __forceinline__ void clear(const Row& r, uint32_t* hist) {
  r.sync();
  for (int i = threadIdx.x; i < BINS / 4; i += THREADS) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
}
// The cut that leaves `need` of the elements with from <= d < to (there are as many), and all in front of them.
template <bool RESIDENT>
__device__ Cut cut_by_count(const Row& r, Shared& s, uint64_t need, uint64_t from, uint64_t to) {
  uint32_t base = (uint32_t)from, span = (uint32_t)(to - 1 - from);   // the elements with d - base <= span (distances are 32 bits wide)
  while (true) {
    const int all_bits = max(1, 32 - __clz((int)span)), bits = min(all_bits, DIGIT), shift = all_bits - bits;
    uint32_t* const hist = s.hist;
    clear(r, hist);
    const uint32_t top = (uint32_t)r.top - base;
    r.each<RESIDENT>([&](int32_t v, int) {
      const uint32_t t = top - (uint32_t)v;
      if (t <= span) atomicAdd(&hist[t >> shift], 1u);
    });
    r.sync();
    constexpr int per = BINS / THREADS;
    static_assert(per == 8, "two loads a thread");
    const int bin0 = per * (int)threadIdx.x;
    uint32_t own[per];
    const uint4 none = make_uint4(0, 0, 0, 0);   // (the last digit has fewer bits)
    const uint4 a = bin0 < 1 << bits ? sum_of_cluster(hist + bin0, r.split) : none;
    const uint4 b = bin0 + 4 < 1 << bits ? sum_of_cluster(hist + bin0 + 4, r.split) : none;
    own[0] = a.x; own[1] = a.y; own[2] = a.z; own[3] = a.w; own[4] = b.x; own[5] = b.y; own[6] = b.z; own[7] = b.w;
    uint64_t sum = 0, total;
#pragma unroll
    for (int k = 0; k < per; ++k) sum += own[k];
    uint64_t before = block_scan(s, sum, total);
    if (total < need) return {to, 0};   // (scores that change)
    if (before < need && need <= before + sum) {
#pragma unroll
      for (int k = 0; k < per; ++k) {
        if (before < need && need <= before + own[k]) {
          s.found = bin0 + k;
          s.found_before = before;
          s.found_size = own[k];
        }
        before += own[k];
      }
    }
    __syncthreads();
    need -= s.found_before;
    const uint64_t at = (uint64_t)base + ((uint64_t)(uint32_t)s.found << shift), behind = min(at + ((uint64_t)1 << shift), (uint64_t)base + span + 1);
    if (need == s.found_size) return {behind, 0};   // all of the bin
    if (shift == 0) return {at, (uint32_t)need};
    base = (uint32_t)at;
    span = (uint32_t)(behind - 1 - at);
  }
}

// Where, in the order of d, the weight of the elements with d < limit reaches need(total); if the total is less than that, a
// cut among the ties of `whole`, of tie_weight each.
template <bool RESIDENT, typename Need>
__device__ Cut cut_by_weight(const Row& r, Shared& s, int range_bits, const Need& need_of, const Cut& whole, uint32_t tie_weight) {
  int bits = min(range_bits, WDIGIT), shift = range_bits - bits;
  uint32_t prefix = 0;
  uint64_t need = 0;
  for (bool first = true;; first = false) {
    uint32_t* const hist = s.hist;
    clear(r, hist);
    r.each<RESIDENT>([&](int32_t v, int) {
      const uint32_t d = r.dist(v);
      if (d < whole.D && (uint64_t)d >> (shift + bits) == prefix) {
        // 64 bits a bin, whatever a slice holds: the low word as it wraps, and how often it did.  (Two additions of half a weight,
        // which need no answer, hold 65537 elements a bin, and slices are longer.  256 rows of 262144, 8192 entries: 514 us, with those 501.)
        const uint32_t w = r.weight(d), bin = (d >> shift) & ((1u << bits) - 1u);
        if (w && atomicAdd(&hist[bin], w) > 0xffffffffu - w) atomicAdd(&hist[WBINS + bin], 1u);
      }
    });
    r.sync();
    static_assert(WBINS / THREADS == 4, "one load a thread and half of a bin");
    const int bin0 = 4 * (int)threadIdx.x;
    uint64_t own[4], high[4];
    sum_of_cluster(hist + bin0, r.split, own);
    sum_of_cluster(hist + WBINS + bin0, r.split, high);
#pragma unroll
    for (int k = 0; k < 4; ++k) own[k] += high[k] << 32;
    uint64_t total, before = block_scan(s, own[0] + own[1] + own[2] + own[3], total);
    if (first) {
      need = need_of(total);
      if (need > total) {
        Cut c = whole;
        if (tie_weight) c.ties = (uint32_t)min((uint64_t)whole.ties, (need - total + tie_weight - 1) / tie_weight);
        return c;
      }
    } else if (total < need) {   // (scores that change)
      return whole;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (before < need && need <= before + own[k]) {
        s.found = bin0 + k;
        s.found_before = before;
        s.found_size = own[k];
      }
      before += own[k];
    }
    __syncthreads();
    need -= s.found_before;
    prefix = (prefix << bits) | (uint32_t)s.found;
    if (need == s.found_size) return {min(((uint64_t)prefix + 1) << shift, whole.D), 0};   // all of the bin
    if (shift == 0) {
      const uint32_t w = r.weight(prefix);
      return {prefix, (uint32_t)((need + w - 1) / w)};
    }
    bits = min(shift, WDIGIT);
    shift -= bits;
  }
}

// Puts the elements with d <= last, of all CTAs, on the list s.all of the first CTA: their number, in every CTA, or -1 if they
// are more than LIST.  `index0`: the index of place 0.
template <bool RESIDENT>
__device__ int collect(const Row& r, Shared& s, uint32_t last, int rank, int index0) {
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  r.each<RESIDENT>([&](int32_t v, int j) {
    if (r.dist(v) <= last && *reinterpret_cast<volatile uint32_t*>(&s.listed) <= LIST) {   // (not one after the other when there are too many)
      const uint32_t at = atomicAdd(&s.listed, 1u);
      if (at < LIST) s.list[at] = make_int2(v, index0 + j);
    }
  });
  __syncthreads();
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < r.split) store32(remote(&s.counts[rank], threadIdx.x), s.listed);
  r.sync();
  const uint32_t mine = lane < (int)r.split ? s.counts[lane] : 0u;
  const uint32_t in_all = __reduce_add_sync(FULL, min(mine, LIST + 1u));
  if (in_all == 0 || in_all > LIST) return -1;   // (none: scores that change)
  const uint32_t sums = (uint32_t)warp_scan(mine);
  // (a warp for every CTA's list)
  const uint32_t c = threadIdx.x >> 5, count = __shfl_sync(FULL, mine, (int)(c & 31)), at = __shfl_sync(FULL, sums - mine, (int)(c & 31));
  if (rank == 0 && c < r.split)
    for (uint32_t i = lane; i < count; i += 32) {
      const uint32_t from = remote(&s.list[i], c), index = load32(from + 4), d = r.dist((int32_t)load32(from));
      const uint64_t add = (uint64_t)r.weight(d) << RANK_BITS | 1u;
      s.all[at + i] = make_uint4(index, d, (uint32_t)add, (uint32_t)(add >> 32));
    }
  r.sync();   // (the lists have been read)
  return (int)in_all;
}

// For the thread's element of n (tid < n): what f(sum, its own, j) adds up for all j < n.  n * n turns of a few
// instructions, a warp for 32 elements and, where warps are left, for a part of the others (200 elements and 512 threads:
// 1.8 us; a search for both sums by halving took 6).
template <typename Own, typename F>
__device__ __forceinline__ uint64_t against_all(Shared& s, int n, const Own& own_of, const F& f) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blocks = (n + 31) >> 5, parts = WARPS / blocks, part = warp / blocks, t = (warp - part * blocks) * 32 + lane;
  if (part < parts) {
    const auto own = own_of(min(t, n - 1));
    const int end = n * (part + 1) / parts;
    uint64_t sum = 0;
#pragma unroll 8
    for (int j = n * part / parts; j < end; ++j) f(sum, own, j);
    s.sums_of_list[part * 32 * blocks + t] = sum;
  }
  __syncthreads();
  uint64_t sum = 0;
  if ((int)threadIdx.x < n)
    for (int i = 0; i < parts; ++i) sum += s.sums_of_list[i * 32 * blocks + threadIdx.x];
  return sum;
}

// The weights of the blocks b0, b0 + WARPS, .. < end of a row without a cut, all of whose places are valid, with a table of
// weights below 2^27 (sixteen of them fit 32 bits) and above 0; returns how many elements the lane has seen.  A function of its
// own, so that the registers hold the next block, on its way from global memory, and not what the kernel needs later.
template <bool RESIDENT>
__device__ __noinline__ uint32_t sum_blocks(const Row r, Shared& s, int b0, int end) {
  constexpr int BLOCK = BLOCK_OF<RESIDENT>, GROUPS = BLOCK / 128;
  const int lane = threadIdx.x & 31;
  const int4* const at = reinterpret_cast<const int4*>(RESIDENT ? resident() : r.x);
  const int32_t* const table = r.in_smem();
  int4 next[GROUPS];
  const auto request = [&](int b) {
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) next[i] = at[b * (BLOCK / 4) + i * 32 + lane];
  };
  uint32_t seen = 0;
  if (b0 < end) request(b0);
  for (int b = b0; b < end; b += WARPS) {
    int4 v[GROUPS];
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) v[i] = next[i];
    if (b + WARPS < end) request(b + WARPS);
    uint32_t sum = 0;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i)
      sum += (uint32_t)(table[r.entry_of(v[i].x)] + table[r.entry_of(v[i].y)]) + (uint32_t)(table[r.entry_of(v[i].z)] + table[r.entry_of(v[i].w)]);
    const uint64_t mass = warp_sum(sum);
    if (lane == 0) {
      s.block_mass[b] = mass;
      s.block_ties[b] = 0;
    }
    seen += BLOCK / 32;
  }
  __syncwarp();
  return seen;
}

__device__ __forceinline__ int bits_of(uint64_t range) { return max(1, 64 - __clzll((long long)range)); }   // of the largest distance

template <bool RESIDENT>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const __grid_constant__ Params p) {
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = p.split > 1 ? (int)cluster_rank() : 0, row = (int)blockIdx.x / p.split;
  int32_t* const slice_s = reinterpret_cast<int32_t*>(dynamic_smem);
  int32_t* const table_s = slice_s + (RESIDENT ? p.slice : 0);
  const cvmk_sample_desc& d = p.d;
  const int vocab = d.vocab;
  const int32_t* src = d.logits + (size_t)row * (size_t)d.pitch;
  // Places are counted from the 16-byte boundary at or in front of the row, so that slices begin on one.
  const int skew = (int)((reinterpret_cast<uintptr_t>(src) >> 2) & 3);
  const int begin = rank * p.slice;                       // this slice's place 0
  Row r;
  const int32_t* const at = src - skew + begin;           // of place 0
  const int32_t* const x = RESIDENT ? slice_s : at;
  r.x = x;
  r.first = min(max(skew - begin, 0), p.slice);
  r.last = min(max(skew + vocab - begin, r.first), p.slice);
  r.split = (uint32_t)p.split;

  pdl_trigger();
  if (tid == 0) {
    s.late = 0;
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_addr(&s.bar)));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (p.split > 1) cluster_arrive();   // (waited for before anything is sent)
  pdl_wait();
  // (what the set-up needs of global memory is requested at once: a trip each would be longer than the slice takes)
  constexpr int EARLY = TABLE_SMEM_MAX / THREADS;
  int32_t entry[EARLY];
#pragma unroll
  for (int i = 0; i < EARLY; ++i) entry[i] = p.table_smem && tid + i * THREADS < d.table_len ? d.table[tid + i * THREADS] : 0;
  // whole 16-byte words by the bulk engine, the ragged ends by threads
  const int b0 = min((r.first + 3) & ~3, r.last), b1 = max(b0, r.last & ~3);
  if (RESIDENT && tid == 0) {
    const uint32_t bytes = (uint32_t)(b1 - b0) * 4u;
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(&s.bar)), "r"(bytes) : "memory");
    if (bytes)
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_addr(slice_s + b0)),
                   "l"(at + b0), "r"(bytes), "r"(smem_addr(&s.bar))
                   : "memory");
  }
  if (RESIDENT && tid >= 32 && tid < 35 && r.first + tid - 32 < b0) slice_s[r.first + tid - 32] = at[r.first + tid - 32];
  if (RESIDENT && tid >= 35 && tid < 38 && b1 + tid - 35 < r.last) slice_s[b1 + tid - 35] = at[b1 + tid - 35];
  const uint64_t min_p = d.min_p ? (uint64_t)min(max(d.min_p[row], 0), (int)ONE) : 0;
  const uint32_t min_weight = (uint32_t)((min_p * (uint64_t)max(d.table[0], 0) + ONE - 1) >> 30);
  if (tid == 64) {
    s.row = make_uint4(d.top_k ? (uint32_t)d.top_k[row] : 0u, d.top_p ? (uint32_t)min(max(d.top_p[row], 0), (int)ONE) : (uint32_t)ONE,
                       (uint32_t)max(d.scale[row], 0), (uint32_t)d.random[row] & 0x7fffffffu);
    s.min_weight = min_weight;
  }
  r.last_entry = (uint32_t)d.table_len - 1u;
  r.wide = !p.table_smem;
  r.table = d.table;
  r.table_at = RESIDENT ? p.slice : 0;
  bool plain = true;   // all entries are above 0 and below 2^27
#pragma unroll
  for (int i = 0; i < EARLY; ++i)
    if (p.table_smem && tid + i * THREADS < d.table_len) {
      const int32_t w = (uint32_t)max(entry[i], 0) >= min_weight ? max(entry[i], 0) : 0;
      table_s[tid + i * THREADS] = w;
      plain = plain && w > 0 && w < 1 << 27;
    }
  const bool plain_table = __syncthreads_and(plain) && p.table_smem;
  uint4 of_row = s.row;
  r.min_weight = s.min_weight;
  // (bounded: the copy is the only thing that is waited for)
  bool landed = !RESIDENT;
  for (uint32_t i = 0; !landed && i < (1u << 19); ++i) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], 0, 2000;\nselp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_addr(&s.bar))
        : "memory");
    landed = ok != 0;
  }

  if (p.split > 1) cluster_wait();

  // ---- the largest and the smallest score, and the bound of the k-th largest
  int32_t lo = INT32_MAX, hi = INT32_MIN;
  const auto cut_by_k = [&]() { return (int32_t)of_row.x >= 1 && (int32_t)of_row.x < vocab; };
  if (cut_by_k() || of_row.y < ONE) {
    r.each<RESIDENT>([&](int32_t v, int) {
      lo = min(lo, v);
      hi = max(hi, v);
    });
  } else {   // (the smallest is not asked for)
    r.each<RESIDENT>([&](int32_t v, int) { hi = max(hi, v); });
    lo = INT32_MIN;
  }
  const bool some = lo <= hi;   // the thread has seen an element
  const int32_t mine = hi;
  lo = __reduce_min_sync(FULL, lo);
  hi = __reduce_max_sync(FULL, hi);
  if (lane == 0) { s.lo[warp] = lo; s.hi[warp] = hi; }
  __syncthreads();
  lo = __reduce_min_sync(FULL, lane < WARPS ? s.lo[lane] : INT32_MAX);
  hi = __reduce_max_sync(FULL, lane < WARPS ? s.hi[lane] : INT32_MIN);
  int32_t bound = INT32_MIN;
  const int part = ((int32_t)of_row.x - 1) / p.split + 1;   // of top_k, for a CTA
  if (cut_by_k() && part <= THREADS && __syncthreads_count(some) >= part) {
    const uint32_t far = (uint32_t)hi - (uint32_t)mine;
    uint32_t from = 0, to = (uint32_t)hi - (uint32_t)lo;
    for (int i = 0; i < 10 && from < to; ++i) {   // (to a thousandth of the range: 1 row of 32000 9.6 us, 10.0 with fourteen turns)
      const uint32_t mid = from + (to - from) / 2;
      if (__syncthreads_count(some && far <= mid) >= part) to = mid;
      else from = mid + 1;
    }
    bound = (int32_t)((uint32_t)hi - to);
  }
  if (warp == 0 && lane < p.split) {   // (a lane for every CTA)
    store128(remote(&s.scores[rank], (uint32_t)lane), make_uint4((uint32_t)lo, (uint32_t)hi, (uint32_t)bound, 0));
    if (rank == 0) store128(remote(&s.row_of_all, (uint32_t)lane), of_row);
    if (!landed) store32(remote(&s.late, (uint32_t)lane), 1u);
  }
  r.sync();
  of_row = s.row_of_all;
  const int k = (int)of_row.x;
  const bool by_count = cut_by_k();
  const uint64_t top_p = of_row.y, u = of_row.w;
  r.scale = of_row.z;
  r.saturated = r.scale ? 0xffffffffu / r.scale : 0xffffffffu;
  const bool late = s.late != 0;
  {
    const int4 v = s.scores[min(lane, p.split - 1)];
    lo = __reduce_min_sync(FULL, v.x);
    hi = __reduce_max_sync(FULL, v.y);
    bound = __reduce_min_sync(FULL, v.z);
  }
  if (late) {   // a copy that never came (its wait is bounded): no element is drawn
    if (rank == 0 && tid == 0) d.token[row] = -1;
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
    __syncwarp();
    r.sync();
    return;
  }
  r.top = hi;
  r.gentle = !r.wide && r.scale <= 65536;
  r.far = (uint32_t)min(r.first_of(r.last_entry), ((uint64_t)1 << 32) - 1);
  const int range_bits = bits_of((uint32_t)hi - (uint32_t)lo);

  // ---- the cuts
  const uint64_t end = (uint64_t)1 << 32;
  Cut cut = {end, 0};   // everything
  const auto share_of = [=](uint64_t all) {
    const uint64_t need = top_p * (all >> 30) + ((top_p * (all & (ONE - 1)) + ONE - 1) >> 30);
    return need > 1 ? need : (uint64_t)1;
  };
  if (by_count) {
    const uint32_t last = r.dist(bound);
    const int n = collect<RESIDENT>(r, s, last, rank, begin - skew);
    if (n >= 0) {
      if (rank != 0) return;   // (everything else is done on the list)
      const bool mine = tid < n;
      // ranks, and the weights in front, in the order of the cuts: of (distance, index)
      const uint64_t in_front = against_all(s, n, [&](int t) { return (uint64_t)s.all[t].y << 32 | s.all[t].x; }, [&](uint64_t& sum, uint64_t own, int j) {
        const uint4 e = s.all[j];
        if (((uint64_t)e.y << 32 | e.x) < own) sum += (uint64_t)e.w << 32 | e.z;
      });
      const uint32_t place = (uint32_t)in_front & ((1u << RANK_BITS) - 1u);
      const uint4 e = s.all[mine ? tid : 0];
      const uint32_t weight = (uint32_t)(((uint64_t)e.w << 32 | e.z) >> RANK_BITS);
      const uint64_t before = in_front >> RANK_BITS;
      bool left = mine && place < (uint32_t)k;
      if (mine && (int)place == min(k, n) - 1) {   // the last one that top_k leaves
        s.mass = s.mass_left = before + weight;
        s.left = place + 1;
      }
      __syncthreads();
      const uint64_t mass = s.mass;
      if (top_p < ONE && mass) {
        const uint64_t need = share_of(mass);
        left = left && before < need;
        if (left && before + weight >= need) {   // the last one that top_p leaves
          s.mass_left = before + weight;
          s.left = place + 1;
        }
      }
      if (left) s.sorted[place] = make_uint2(e.x, weight);
      const uint32_t kept = (uint32_t)__syncthreads_count(left && weight > 0);
      const uint64_t all = s.mass_left, target = u * (all >> 31) + ((u * (all & 0x7fffffffu)) >> 31);
      const int m = (int)s.left;
      const uint64_t up_to = against_all(s, m, [&](int t) { return s.sorted[t].x; }, [&](uint64_t& sum, uint32_t own, int j) {
        const uint2 e = s.sorted[j];
        if (e.x <= own) sum += e.y;
      });
      const uint2 drawn = s.sorted[tid < m ? tid : 0];
      // (where nothing weighs anything, the first of the order)
      if (tid < m && (all ? up_to > target && up_to - drawn.y <= target : tid == 0)) {
        d.token[row] = (int32_t)drawn.x;
        if (d.weight) d.weight[row] = (int32_t)drawn.y;
        if (d.mass) d.mass[row] = (int64_t)all;
        if (d.kept) d.kept[row] = (int32_t)kept;
      }
      return;
    }
    cut = cut_by_count<RESIDENT>(r, s, (uint64_t)k, 0, (uint64_t)r.dist(lo) + 1);   // (the list had no room)
  }
  if (top_p < ONE) {
    if (r.wide) {
      const uint32_t ties = cut.ties;
      if (ties) {   // (by one reading of the table)
        if (rank == 0 && tid < p.split) store32(remote(&s.tie_weight, (uint32_t)tid), r.weight((uint32_t)cut.D));
        r.sync();
      }
      const uint32_t w = ties ? s.tie_weight : 0u;
      cut = cut_by_weight<RESIDENT>(r, s, range_bits, [=](uint64_t strict) { return share_of(strict + (uint64_t)ties * w); }, cut, w);
    } else {
      // the elements that are left, by table entry
      uint32_t* const hist = s.hist;
      clear(r, hist);
      if (tid == 0) s.answer = make_uint4(0xffffffffu, 0, 0, 0);
      uint32_t last = 0;   // (of the last entry, which elements far behind the first one share: counted in registers)
      const uint32_t left = (uint32_t)min(cut.D, end - 1);
      const bool beyond = cut.D == end;
      if (beyond && r.gentle) {
        r.each<RESIDENT>([&](int32_t v, int) {
          const uint32_t e = r.entry_of(v);
          if (e == r.last_entry) ++last;
          else atomicAdd(&hist[e], 1u);
        });
      } else {
        r.each<RESIDENT>([&](int32_t v, int) {
          const uint32_t dj = r.dist(v), e = r.entry(dj);
          if (beyond || dj < left) {
            if (e == r.last_entry) ++last;
            else atomicAdd(&hist[e], 1u);
          }
        });
      }
      last = __reduce_add_sync(FULL, last);
      if (lane == 0 && last) atomicAdd(&hist[r.last_entry], last);
      if (tid == 0 && cut.ties && rank == 0) atomicAdd(&hist[r.entry((uint32_t)cut.D)], cut.ties);
      r.sync();
      // Every CTA adds up its share of the entries (a cluster's counts of all of them are 128 KB to fetch: 4 us), tells the
      // others its weight, and the one in whose share the target lies finds the entry for all.
      const int parts = (int)r.split, part = parts > 1 ? rank : 0, share = BINS / parts, per = max(4, share / THREADS);
      const uint32_t e0 = (uint32_t)(part * share + per * tid);
      const bool here = per * tid < share;
      const uint4 none = make_uint4(0, 0, 0, 0), a = here ? sum_of_cluster(hist + e0, r.split) : none;
      const uint4 b = here && per > 4 ? sum_of_cluster(hist + e0 + 4, r.split) : none;
      const uint32_t n[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      uint64_t mass = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n[i]) mass += (uint64_t)n[i] * (uint32_t)table_s[e0 + i];   // (entries behind the table are not counted)
      uint64_t all, before = block_scan(s, mass, all);
      if (parts > 1) {
        if (warp == 0 && lane < parts) store128(remote(&s.sums[rank], (uint32_t)lane), make_uint4((uint32_t)all, (uint32_t)(all >> 32), 0, 0));
        r.sync();
        const uint4 v = lane < parts ? s.sums[lane] : none;
        const uint64_t m = v.x | (uint64_t)v.y << 32, sums = warp_scan(m);
        before += __shfl_sync(FULL, sums - m, rank);
        all = __shfl_sync(FULL, sums, 31);
      }
      const uint64_t need = share_of(all);
      if (before < need && need <= before + mass) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (!n[i]) continue;
          const uint64_t w = (uint32_t)table_s[e0 + i], weight = n[i] * w;
          if (before < need && need <= before + weight) {   // the entry, the elements of it that are needed, and that it has
            const uint4 answer = make_uint4(e0 + i, (uint32_t)((need - before + w - 1) / w), n[i], 0);
            for (int c = 0; c < parts; ++c) store128(parts > 1 ? remote(&s.answer, (uint32_t)c) : smem_addr(&s.answer), answer);
          }
          before += weight;
        }
      }
      r.sync();
      const int e = (int)s.answer.x;
      const uint64_t wanted = s.answer.y, size = s.answer.z;
      if (e >= 0) {   // (else nothing weighs anything, and no cut is needed)
        const uint64_t from = r.first_of((uint32_t)e);
        const uint64_t to = min((uint32_t)e == r.last_entry ? end : r.first_of((uint32_t)e + 1), cut.D + (cut.ties ? 1 : 0));
        if (wanted < size && to - from == 1) {
          cut = {from, (uint32_t)wanted};
        } else if (wanted < size) {
          // (one digit, mostly: an entry is 2^16 / scale distances wide)
          cut = cut_by_count<RESIDENT>(r, s, wanted, from, min(to, max((uint64_t)r.dist(lo) + 1, from + 1)));
        } else if (to <= cut.D) {   // (all of the entry; the cut that was there may lie in it)
          cut = {to, 0};
        }
      }
    }
  }

  // ---- the draw: weights and ties of every block of the slice
  constexpr int BLOCK = BLOCK_OF<RESIDENT>, GROUPS = BLOCK / 128;
  const int blocks = (r.last + BLOCK - 1) / BLOCK;
  uint32_t kept = 0;
  const uint32_t D32 = (uint32_t)min(cut.D, end - 1);
  const bool beyond = cut.D == end;
  // (whole blocks from `whole0` to `whole1`)
  const int whole0 = (r.first + BLOCK - 1) / BLOCK, whole1 = r.last / BLOCK;
  const bool straight = beyond && r.gentle && plain_table;
  if (straight) {
    const int b0 = whole0 + (warp - whole0 % WARPS + WARPS) % WARPS;   // the warp's first of them
    kept += sum_blocks<RESIDENT>(r, s, b0, whole1);
  }
  for (int b = warp; b < blocks; b += WARPS) {
    const bool whole = b >= whole0 && b < whole1;
    if (straight && whole) continue;
    uint64_t mass = 0;
    uint32_t ties = 0;
    int4 v[GROUPS];
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) v[i] = r.four<RESIDENT>(b * BLOCK + 4 * (i * 32 + lane), whole);
    if (whole && beyond) {
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) {
        const uint32_t w0 = r.weight(r.dist(v[i].x)), w1 = r.weight(r.dist(v[i].y)), w2 = r.weight(r.dist(v[i].z)), w3 = r.weight(r.dist(v[i].w));
        mass += w0;
        mass += w1;
        mass += w2;
        mass += w3;
        kept += min(w0, 1u) + min(w1, 1u) + min(w2, 1u) + min(w3, 1u);
      }
    } else {
      bool some_in = false;   // (behind a cut hardly any element is)
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) {
        const int32_t e[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int q = 0; q < 4; ++q) some_in |= beyond || r.dist(e[q]) <= D32;
      }
      if (__any_sync(FULL, some_in)) {
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
          const int j = b * BLOCK + 4 * (i * 32 + lane);
          const int32_t e[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const bool valid = j + q >= r.first && j + q < r.last;
            const uint32_t dj = r.dist(e[q]);
            if (valid && (beyond || dj < D32)) {
              const uint32_t w = r.weight(dj);
              mass += w;
              kept += min(w, 1u);
            } else {
              ties += valid && dj == D32;
            }
          }
        }
      }
    }
    __syncwarp();
    mass = warp_sum(mass);
    ties = cut.ties ? __reduce_add_sync(FULL, ties) : 0u;
    if (lane == 0) {
      s.block_mass[b] = mass;
      s.block_ties[b] = ties;
    }
  }
  kept = __reduce_add_sync(FULL, kept);
  if (lane == 0) s.kept[warp] = kept;
  __syncthreads();
  const int per_lane = (blocks + 31) / 32;      // blocks of a lane of warp 0
  uint64_t mass_in_front = 0;
  uint32_t ties_in_front = 0;                   // of the lane's blocks
  auto scan_blocks = [&]() {
    uint64_t m = 0, t = 0;
    for (int b = lane * per_lane; b < min((lane + 1) * per_lane, blocks); ++b) { m += s.block_mass[b]; t += s.block_ties[b]; }
    const uint64_t mi = warp_scan(m), ti = cut.ties ? warp_scan(t) : 0;
    mass_in_front = mi - m;
    ties_in_front = cut.ties ? (uint32_t)(ti - t) : 0u;
    const uint64_t mass = __shfl_sync(FULL, mi, 31);
    const uint32_t ties = __shfl_sync(FULL, (uint32_t)ti, 31);
    if (lane < p.split) store128(remote(&s.sums[rank], (uint32_t)lane), make_uint4((uint32_t)mass, (uint32_t)(mass >> 32), ties, kept));
    if (rank == 0 && lane < p.split) store32(remote(&s.tie_weight, (uint32_t)lane), cut.ties ? r.weight((uint32_t)cut.D) : 0u);
  };
  if (warp == 0) {
    kept = __reduce_add_sync(FULL, lane < WARPS ? s.kept[lane] : 0u);
    scan_blocks();
  }
  r.sync();
  uint64_t all, front_mass;
  uint32_t front_ties, all_kept;
  auto add_up = [&]() {   // over the CTAs, and over those in front of this one
    all = front_mass = 0;
    front_ties = all_kept = 0;
#pragma unroll
    for (int c = 0; c < MAX_SPLIT; ++c) {
      if (c >= p.split) break;
      const uint4 v = s.sums[c];
      const uint64_t m = v.x | (uint64_t)v.y << 32;
      all += m;
      all_kept += v.w;
      if (c < rank) { front_mass += m; front_ties += v.z; }
    }
  };
  add_up();
  uint32_t tie_weight = s.tie_weight;
  if (cut.ties && tie_weight) all_kept += cut.ties;
  all += (uint64_t)cut.ties * tie_weight;
  const uint64_t target = u * (all >> 31) + ((u * (all & 0x7fffffffu)) >> 31);
  if (all == 0) {
    // Nothing weighs anything: the first of the order is taken, as if the first element with d = 0 weighed 1 and all others
    // nothing (rare: the ties are counted again).
    cut = {0, 1};
    tie_weight = 1;
    r.sync();   // (nobody still reads the sums of before)
    for (int b = warp; b < blocks; b += WARPS) {
      uint32_t ties = 0;
      for (int j = max(b * BLOCK, r.first & ~31) + lane; j < min((b + 1) * BLOCK, r.last); j += 32) ties += j >= r.first && r.dist(x[j]) == 0;
      __syncwarp();
      ties = __reduce_add_sync(FULL, ties);
      if (lane == 0) { s.block_mass[b] = 0; s.block_ties[b] = ties; }
    }
    __syncthreads();
    if (warp == 0) scan_blocks();
    r.sync();
    add_up();
  }
  if (warp == 0) {
    // the lane and the block of it in which the running weight passes the target
    const auto passed = [&](uint64_t m, uint32_t t) { return m + (uint64_t)min(t, cut.ties) * tie_weight > target; };
    uint64_t m = front_mass + mass_in_front;
    uint32_t t = front_ties + ties_in_front;
    int hit = -1;
    if (!passed(m, t)) {
      for (int b = lane * per_lane; b < min((lane + 1) * per_lane, blocks); ++b) {
        if (passed(m + s.block_mass[b], t + s.block_ties[b])) { hit = b; break; }
        m += s.block_mass[b];
        t += s.block_ties[b];
      }
    }
    __syncwarp();
    const uint32_t who = __ballot_sync(FULL, hit >= 0);   // one lane of one CTA
    if (who) {
      const int from = __ffs(who) - 1;
      const int b = __shfl_sync(FULL, hit, from);
      m = __shfl_sync(FULL, m, from);
      t = __shfl_sync(FULL, t, from);
      // its elements, four of every 128 a lane
      uint32_t w[GROUPS][4], tie[GROUPS];
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) {
        const int j = b * BLOCK + 4 * (i * 32 + lane);
        const int4 v = r.four<RESIDENT>(j, false);
        const int32_t e[4] = {v.x, v.y, v.z, v.w};
        tie[i] = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const bool valid = j + q >= r.first && j + q < r.last;
          const uint32_t dj = r.dist(e[q]);
          w[i][q] = valid && dj < cut.D ? r.weight(dj) : 0u;
          tie[i] |= (valid && dj == cut.D ? 1u : 0u) << q;
        }
      }
      // the 128 of them, and among these the lane
      bool done = false;
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) {
        if (done) continue;
        const uint64_t mine_mass = (uint64_t)w[i][0] + w[i][1] + w[i][2] + w[i][3];
        const uint32_t mine_ties = (uint32_t)__popc(tie[i]);
        const uint64_t mass_to = m + warp_sum(mine_mass);
        const uint32_t ties_to = t + (cut.ties ? __reduce_add_sync(FULL, mine_ties) : 0u);
        done = passed(mass_to, ties_to);
        if (!done) {
          m = mass_to;
          t = ties_to;
          continue;
        }
        uint64_t m1 = m + warp_scan(mine_mass) - mine_mass;
        uint32_t t1 = t + (cut.ties ? (uint32_t)warp_scan(mine_ties) - mine_ties : 0u);
        if (!passed(m1, t1) && passed(m1 + mine_mass, t1 + mine_ties)) {
          int place = -1;
          uint32_t weight = 0;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t one_tie = tie[i] >> q & 1u;
            m1 += w[i][q];
            t1 += one_tie;
            if (place < 0 && passed(m1, t1)) {
              place = q;
              weight = one_tie ? (all ? tie_weight : 0u) : w[i][q];
            }
          }
          d.token[row] = begin + b * BLOCK + 4 * (i * 32 + lane) + place - skew;
          if (d.weight) d.weight[row] = (int32_t)weight;
          if (d.mass) d.mass[row] = (int64_t)all;
          if (d.kept) d.kept[row] = (int32_t)all_kept;
        }
      }
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
  if (d->rows > INT32_MAX / 8) { set_error("sample: too many rows for one launch"); return CVMK_ERR_ARG; }
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
  // How many CTAs a row is cut over, and whether its slices are kept in shared memory.  The choice is by sizes, and by whether
  // rows may be cut (top_k or top_p given); of 14000 drawn sizes (1 to 512 rows, 300 to 262144 elements) it takes 2 % longer than
  // the best, in the mean.  us of one call in a chain of calls, kept (k) or read again from L2 (g), CTAs a row:
  //   - as many CTAs a row as are resident at once, two an SM (of clusters of eight 33, not 37: GPCs have 16 to 20 SMs), each with
  //     4000 elements or more, with cuts 7000.  50021 elements, 64 rows, with cuts: k4 25, k8 38, g2 35; 150 rows without: g1 23,
  //     g2 30, k4 30.
  //   - with cuts rows differ in how long they take, and more and shorter CTAs even that out: slices of 90000 at most, and long
  //     ones may be more than are resident at once.  262144 elements, 256 rows: g1 260, g2 223, g4 201, g8 256; 131072, 150 rows:
  //     g1 102, g2 78, g4 82; 147285, 39 rows: g4 43, k8 29; 100000, 180 rows: g1 90, g2 71; but 50021, 200 rows: g1 55, g2 58.
  //   - kept where two slices fit an SM, or one where no SM has two.  131072 elements, 8 rows with cuts: k8 22, g8 28; 262144:
  //     k8 23, g8 28.  Where that many CTAs have an SM each, no more are made: 48375 elements, 129 rows without cuts k1 12, k2 17;
  //     but with cuts only for one CTA a row: 131072 elements, 32 rows with top_k in all k4 14, k8 20, with top_p alone in
  //     every third k4 32, k8 27.
  const int room = 226 * 1024 - (int)sizeof(Shared), half = 113 * 1024 - (int)sizeof(Shared) - 1024;
  const bool cuts = d->top_k || d->top_p;
  static const int two_an_sm[4] = {296, 148, 71, 33}, one_an_sm[4] = {148, 74, 33, 15};   // clusters of 1, 2, 4 and 8 CTAs; 148 SMs
  const auto at_work = [&](int log) {
    const int slice = slice_of(1 << log);
    return (int64_t)two_an_sm[log] * sms / 148 * (!cuts || slice < 12000 ? 100 : (slice < 30000 ? 120 : 150)) / 100;
  };
  const auto alone = [&](int log) { return d->rows <= (int64_t)one_an_sm[log] * sms / 148; };
  int log2 = 0;
  while (log2 < 3 && d->rows <= at_work(log2 + 1) && slice_of(2 << log2) >= (cuts ? 7000 : 4000) &&
         !((!cuts || log2 == 0) && alone(log2) && !alone(log2 + 1) && smem_of(1 << log2) <= room)) ++log2;
  while (cuts && log2 < 3 && slice_of(1 << log2) > 90000) ++log2;
  p.split = 1 << log2;
  bool resident = smem_of(p.split) <= half || (smem_of(p.split) <= room && alone(log2));
  if (const char* e = dev_env("CVM_B200_SAMPLE_SPLIT")) p.split = atoi(e);
  if (const char* e = dev_env("CVM_B200_SAMPLE_STREAM")) resident = atoi(e) == 0;
  p.slice = slice_of(p.split);
  const int smem = resident ? smem_of(p.split) : (p.table_smem ? d->table_len * 4 : 0);

  static bool attr_of_device[64] = {false};
  if (!attr_of_device[dev & 63]) {
    for (auto k : {sample_kernel<true>, sample_kernel<false>}) {
      cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, room);
      if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
      if (check_cuda(e, "cudaFuncSetAttribute(sample_kernel)")) return CVMK_ERR_CUDA;
    }
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
  return check_cuda(cudaLaunchKernelEx(&cfg, resident ? sample_kernel<true> : sample_kernel<false>, p), "sample_kernel launch");
}
