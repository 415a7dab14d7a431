// What a row of logits answers: its top log-probabilities, and a token drawn from it.
#include <cfloat>
#include <string>

#include "ws_guard.h"
#include "ws_rows.h"

namespace ws {
namespace {

namespace cg = cooperative_groups;

// ------------------------------------------------------------ top log-probabilities
//
// One pass over the row gives its maximum m and S = sum exp((x - m) / t), and keeps in shared memory the
// maximum of every thread's logits in every group of steps, 16 bits of its order key (up to kGroups
// groups: one step each for a row of 2^17 16-bit logits). The k-th largest of the threads' maxima over the whole
// row (for records of more than kFewMaxima, of four parts of it) is a lower bound of the k-th
// largest logit, and a close one: about 1.15 k logits of a row reach it. So the pass itself costs a logit a share of one
// comparison, and behind it the few groups whose maximum reaches the bound are read once more, out of
// L2, for the logits that do.
//
// A candidate is 64 bits, the order key of its logit above the complement of its id, so that no two are equal and the
// larger one comes first in the record. The list has room for k candidates and all that one unit of each thread
// gives. A row of which more logits reach the bound (ascending or equal ones) is taken again unit
// by unit, dropping all but the k largest before each: slow, and right for any row.
//
// 64 of 2048 x 128256 bf16 take 110 us (4.8 TB/s) on the device, of 64 rows 14 us with four blocks each. Many rows are bound by
// instructions, about 37000 a warp-wide row of which a third come behind the pass; few by latency, a microsecond or two for each of the
// pass, the bound, the candidates and the exchange.
constexpr uint32_t kTopDepth = 2;  // steps in flight (2048 x 128256 bf16: 110, 115 and 129 us with 2, 3 and 4)
constexpr uint32_t kGroups = 16;
constexpr uint32_t kFewMaxima = 64;
constexpr uint32_t kCandidates = WS_TOP_MAX_K + kRowThreads * 8;
constexpr uint32_t kCounted = 128;  // candidates that are put in order by counting
constexpr uint32_t kSorted = 512;   // and by sorting
constexpr uint32_t kMostCollected = 1200;  // of 4096 maxima in a row of 16 groups: 1420 logits reach the bound; of 2048: 1810

struct TopShared {
  uint64_t sorted[WS_TOP_MAX_K];  // the block's k largest in order
  uint16_t maxima[kGroups][kRowThreads];
  uint32_t bins[kRowThreads];
  uint2 keys[kRowWarps], votes[2][kRowWarps];
  uint32_t sums[kRowWarps];
  float2 soft[kRowWarps];
  uint32_t count, queued, sorted_count, bin, key;
};
static_assert(kCandidates * sizeof(uint64_t) + kGroups * kRowThreads * sizeof(uint16_t) <= kTopDepth * kStepBytes,
              "the list and the queue take the ring's place");

// What the blocks of a cluster tell each other of their shares of a row.
struct TopTold {
  uint64_t lists[RowCluster::kMost][WS_TOP_MAX_K];
  uint32_t counts[RowCluster::kMost];
  float2 soft[RowCluster::kMost];
};

__device__ __forceinline__ uint64_t candidate(float x, uint32_t id) { return ((uint64_t)order_key(x) << 32) | (0xFFFFFFFFu - id); }
__device__ __forceinline__ float candidate_value(uint64_t v) { return key_value((uint32_t)(v >> 32)); }

// Keeps the k largest of the first n > k candidates (in no order) and returns the smallest of these.
__device__ __noinline__ uint64_t keep_largest(TopShared& s, uint64_t* list, uint32_t n, uint32_t k) {
  constexpr uint32_t kMine = (kCandidates + kRowThreads - 1) / kRowThreads;
  uint64_t mine[kMine];
#pragma unroll
  for (uint32_t i = 0; i < kMine; ++i) {
    const uint32_t at = i * kRowThreads + threadIdx.x;
    mine[i] = at < n ? list[at] : 0;
  }
  // The k-th largest by bisection, two bits a round: how many reach each of three trials.
  uint64_t edge = 0;
#pragma unroll 1
  for (int bit = 62; bit >= 0; bit -= 2) {
    uint32_t low = 0, high = 0;  // trials 1 and 2, and trial 3
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) {
      low += (mine[i] >= (edge | (1ull << bit)) ? 1u : 0u) + (mine[i] >= (edge | (2ull << bit)) ? 0x10000u : 0u);
      high += mine[i] >= (edge | (3ull << bit)) ? 1u : 0u;
    }
    low = __reduce_add_sync(0xFFFFFFFFu, low);
    high = __reduce_add_sync(0xFFFFFFFFu, high);
    uint2* votes = s.votes[(bit >> 1) & 1];  // the other half may still be read
    if ((threadIdx.x & 31u) == 0) votes[threadIdx.x >> 5] = make_uint2(low, high);
    __syncthreads();
    low = high = 0;
#pragma unroll
    for (uint32_t w = 0; w < kRowWarps; ++w) {
      low += votes[w].x;
      high += votes[w].y;
    }
    const uint64_t step = high >= k ? 3u : (low >> 16) >= k ? 2u : (low & 0xFFFFu) >= k ? 1u : 0u;
    edge |= step << bit;
  }
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < kMine; ++i)
    if (mine[i] >= edge) list[atomicAdd(&s.count, 1u)] = mine[i];
  __syncthreads();
  return edge;
}

// All of units [first, last) that reach `bound`, unit by unit, with the list cut down to the k largest before each.
template <class T>
__device__ __noinline__ void top_by_units(TopShared& s, uint64_t* list, const RowWalk<T> walk, uint32_t first, uint32_t last, uint32_t k,
                                          float bound) {
  __syncthreads();
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
  uint64_t least = 0;
  for (uint32_t u0 = first; u0 < last; u0 += kRowThreads) {
    if (s.count > k) least = keep_largest(s, list, s.count, k);
    __syncthreads();
    const uint32_t u = u0 + threadIdx.x;
    if (u < last) {
      float f[kUnit<T>];
      walk.load(u, f);
#pragma unroll
      for (uint32_t i = 0; i < kUnit<T>; ++i) {
        if (f[i] >= bound) {
          const uint64_t v = candidate(f[i], u * kUnit<T> + i - walk.head);
          if (v > least) list[atomicAdd(&s.count, 1u)] = v;
        }
      }
    }
    __syncthreads();
  }
}

// A logit that at least k of the block's maxima (N of each thread) reach, close to the k-th largest of them; the lowest finite
// number where fewer than k are above -inf. The maxima are counted into bins between the largest and the smallest; the bound is the
// smallest of those in the bins that hold the first k, which holds whatever the bins are.
template <uint32_t N>
__device__ __forceinline__ float kth_of_maxima(TopShared& s, const float (&most)[N], uint32_t k) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  uint32_t key[N], hi = 0, lo = ~0u;
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) {
    key[j] = most[j] > -INFINITY ? order_key(most[j]) : 0;  // 0: none
    hi = max(hi, key[j]);
    lo = min(lo, key[j] ? key[j] : ~0u);
  }
  hi = __reduce_max_sync(0xFFFFFFFFu, hi);
  lo = __reduce_min_sync(0xFFFFFFFFu, lo);
  if (lane == 0) s.keys[warp] = make_uint2(hi, lo);
  s.bins[threadIdx.x] = 0;
  if (threadIdx.x == 0) s.key = ~0u;
  __syncthreads();
#pragma unroll
  for (uint32_t w = 0; w < kRowWarps; ++w) {
    hi = max(hi, s.keys[w].x);
    lo = min(lo, s.keys[w].y);
  }
  const float m = key_value(hi), scale = (float)(kRowThreads - 1) / fmaxf(m - key_value(lo), 1e-30f);
  uint32_t bin[N];
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) {
    bin[j] = key[j] ? (uint32_t)fmaxf(fminf((m - most[j]) * scale, (float)(kRowThreads - 1)), 0.f) : ~0u;
    if (key[j]) atomicAdd(&s.bins[bin[j]], 1u);
  }
  __syncthreads();
  const uint32_t own = s.bins[threadIdx.x];
  uint32_t all;
  const uint32_t before = block_scan(own, s.sums, &all);
  if (all < k) return -FLT_MAX;  // the same for the whole block
  if (before < k && before + own >= k) s.bin = threadIdx.x;
  __syncthreads();
  const uint32_t last = s.bin;
  uint32_t least = ~0u;
#pragma unroll
  for (uint32_t j = 0; j < N; ++j)
    if (key[j] && bin[j] <= last) least = min(least, key[j]);
  least = __reduce_min_sync(0xFFFFFFFFu, least);
  if (lane == 0) atomicMin(&s.key, least);
  __syncthreads();
  return fmaxf(key_value(s.key), -FLT_MAX);
}

// Up to kSorted candidates in descending order: the k largest into s.sorted. A bitonic network, two neighbours to a thread: exchanges
// over up to 32 places stay within a warp. Counting larger ones instead takes n^2 comparisons: as fast at 128 candidates, 2.5 times as
// long at 300.
__device__ __noinline__ void sort_largest(TopShared& s, uint64_t* list, uint32_t n, uint32_t k) {
  const uint32_t t = threadIdx.x, places = n <= kSorted / 2 ? kSorted / 2 : kSorted;
  __syncthreads();
  uint64_t a = 2 * t < n ? list[2 * t] : 0, b = 2 * t + 1 < n ? list[2 * t + 1] : 0;
#pragma unroll 1
  for (uint32_t size = 2; size <= places; size *= 2) {
    const bool down = (2 * t & size) == 0;
#pragma unroll 1
    for (uint32_t far = size / 2; far > 32; far /= 2) {
      __syncthreads();
      list[t] = a;
      list[kRowThreads + t] = b;
      __syncthreads();
      const uint64_t oa = list[t ^ (far / 2)], ob = list[kRowThreads + (t ^ (far / 2))];
      const bool larger = ((2 * t & far) == 0) == down;
      a = (a > oa) == larger ? a : oa;
      b = (b > ob) == larger ? b : ob;
    }
#pragma unroll
    for (uint32_t far = 32; far > 1; far /= 2) {
      if (far >= size) continue;
      const uint64_t oa = __shfl_xor_sync(0xFFFFFFFFu, a, far / 2), ob = __shfl_xor_sync(0xFFFFFFFFu, b, far / 2);
      const bool larger = ((2 * t & far) == 0) == down;
      a = (a > oa) == larger ? a : oa;
      b = (b > ob) == larger ? b : ob;
    }
    const uint64_t high = a > b ? a : b, low = a > b ? b : a;
    a = down ? high : low;
    b = down ? low : high;
  }
  if (2 * t < k) s.sorted[2 * t] = a;
  if (2 * t + 1 < k) s.sorted[2 * t + 1] = b;
}

// The k largest logits of the units [first, last) that a block reads step by step. Where these are few (kGroups units a thread
// or fewer), the groups are the units themselves.
template <class T>
struct TopCollector {
  using B = Batch<T>;
  TopShared& s;
  uint32_t k, each, left, group = 0;  // steps a group has (0: it is a unit), and is still to get
  float here = -INFINITY, most[B::kUnits];

  __device__ __forceinline__ TopCollector(TopShared& shared, uint32_t k_, uint32_t first, uint32_t last) : s(shared), k(k_) {
    const uint32_t steps = (last - first + B::kSpan - 1) / B::kSpan;
    each = left = steps * B::kUnits <= kGroups ? 0 : (steps + kGroups - 1) / kGroups;
#pragma unroll
    for (uint32_t j = 0; j < B::kUnits; ++j) most[j] = -INFINITY;
  }
  // The next step; all: the largest of the thread's logits in it.
  __device__ __forceinline__ void add(const B& b, float all) {
    if (each == 0) {
#pragma unroll
      for (uint32_t j = 0; j < B::kUnits; ++j) {
        const float top = word_top<T>(unit_word<T>(b.raw[j]));
        most[j] = fmaxf(most[j], top);
        put(top);
      }
    } else {
      here = fmaxf(here, all);
      if (--left == 0) close();
    }
  }
  // Behind the last step: the k largest, and some others that come close, in `list`, room for kCandidates that the ring has left; s.count of
  // them (more than kCandidates: not all were written down). k up to kMostCollected.
  __device__ __forceinline__ float collect(uint64_t* list, const RowWalk<T>& walk, uint32_t first, uint32_t last) {
    if (left != each) close();
    if (threadIdx.x == 0) s.count = s.queued = 0;
    uint16_t* queue = reinterpret_cast<uint16_t*>(list + kCandidates);
    float bound;
    if (k > WS_TOP_MAX_K) {
      float every[kGroups];
#pragma unroll
      for (uint32_t g = 0; g < kGroups; ++g) every[g] = g < group ? fmaxf(key_value((uint32_t)s.maxima[g][threadIdx.x] << 16), -INFINITY) : -INFINITY;
      bound = kth_of_maxima(s, every, k);
    } else if (k > kFewMaxima) {
      bound = kth_of_maxima(s, most, k);
    } else {
      const float one[1] = {fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]))};
      bound = kth_of_maxima(s, one, k);
    }
    const uint16_t key = (uint16_t)(order_key(bound) >> 16);
    // The groups that reach it, in a queue that all threads work off.
    __syncthreads();  // every thread is done with the ring
    for (uint32_t g = 0; g < group; ++g)
      if (s.maxima[g][threadIdx.x] >= key) queue[atomicAdd(&s.queued, 1u)] = (uint16_t)(g * kRowThreads + threadIdx.x);
    __syncthreads();
    // Of a hit of several units, a thread takes one after the other.
    const uint32_t parts = each ? each * B::kUnits : 1, work = s.queued * parts;
    for (uint32_t i = threadIdx.x; i < work; i += kRowThreads) {
      const uint32_t hit = queue[i / parts], part = i % parts, g = hit / kRowThreads, who = hit % kRowThreads;
      const uint32_t step = each ? g * each + part / B::kUnits : g / B::kUnits, j = (each ? part : g) % B::kUnits;
      const uint32_t u = first + step * B::kSpan + (who >> 5) * B::kWarpSpan + j * 32 + (who & 31u);
      if (u < last) {
        float f[kUnit<T>];
        walk.load(u, f);
        take(list, f, u * kUnit<T> - walk.head, bound);
      }
    }
    __syncthreads();
    return bound;
  }
  // s.sorted_count (at most k <= WS_TOP_MAX_K) candidates in s.sorted, in order; visible behind the next barrier.
  __device__ __forceinline__ void finish(uint64_t* list, const RowWalk<T>& walk, uint32_t first, uint32_t last) {
    const float bound = collect(list, walk, first, last);
    if (s.count > kCandidates) top_by_units<T>(s, list, walk, first, last, k, bound);
    if (s.count > kSorted) keep_largest(s, list, s.count, k);  // k <= WS_TOP_MAX_K <= kSorted remain
    const uint32_t n = s.count;
    if (threadIdx.x == 0) s.sorted_count = min(n, k);
    if (n > kCounted) {
      sort_largest(s, list, n, k);
      return;
    }
    // A candidate's place is the number of larger ones. The list is read eight at a time, up to 0s behind its end.
    if (threadIdx.x < 8) list[n + threadIdx.x] = 0;
    __syncthreads();
    if (threadIdx.x < n) {
      const uint64_t v = list[threadIdx.x];
      uint32_t place = 0;
      for (uint32_t q = 0; q < n; q += 8) {
        ulonglong2 o[4];
#pragma unroll
        for (uint32_t h = 0; h < 4; ++h) o[h] = reinterpret_cast<const ulonglong2*>(list + q)[h];
#pragma unroll
        for (uint32_t h = 0; h < 4; ++h) place += (o[h].x > v) + (o[h].y > v);
      }
      if (place < k) s.sorted[place] = v;
    }
  }

 private:
  __device__ __forceinline__ void put(float top) { s.maxima[group++][threadIdx.x] = (uint16_t)(order_key(top) >> 16); }
  __device__ __forceinline__ void close() {
#pragma unroll
    for (uint32_t j = 0; j < B::kUnits; ++j)
      if (group % B::kUnits == j) most[j] = fmaxf(most[j], here);
    put(here);
    here = -INFINITY;
    left = each;
  }
  __device__ __forceinline__ void take(uint64_t* list, const float (&f)[kUnit<T>], uint32_t id, float bound) const {
    uint32_t mask = 0;
#pragma unroll
    for (uint32_t i = 0; i < kUnit<T>; ++i) mask |= (f[i] >= bound ? 1u : 0u) << i;
    if (!mask) return;
    uint32_t at = atomicAdd(&s.count, (uint32_t)__popc(mask));
#pragma unroll
    for (uint32_t i = 0; i < kUnit<T>; ++i) {
      if (mask >> i & 1u) {
        if (at < kCandidates) list[at] = candidate(f[i], id + i);
        ++at;
      }
    }
  }
};

// The place of this block's i-th candidate in the cluster's record: i and how many of the other blocks' are larger. The
// lists are searched side by side.
__device__ __forceinline__ uint32_t cluster_place(const RowCluster& cluster, const TopTold& told, uint32_t k, uint32_t i, uint64_t v) {
  uint32_t at[RowCluster::kMost], n[RowCluster::kMost];
#pragma unroll
  for (uint32_t b = 0; b < RowCluster::kMost; ++b) {
    at[b] = 0;
    n[b] = b < cluster.blocks && b != cluster.rank ? told.counts[b] : 0;
  }
  for (uint32_t step = 1u << (31 - __clz(k)); step; step >>= 1) {
#pragma unroll
    for (uint32_t b = 0; b < RowCluster::kMost; ++b) {
      const uint32_t next = at[b] + step;
      const uint64_t o = told.lists[b][min(next, (uint32_t)WS_TOP_MAX_K) - 1];  // read in any case: the searches do not wait for one another
      at[b] = next <= n[b] && o > v ? next : at[b];
    }
  }
  uint32_t place = i;
#pragma unroll
  for (uint32_t b = 0; b < RowCluster::kMost; ++b) place += at[b];
  return place;
}

// The block's sorted candidates into every block's `told`; between ready() and told().
__device__ __forceinline__ void tell_top(const RowCluster& cluster, const TopShared& s, TopTold* told) {
  const uint32_t n = s.sorted_count;
  for (uint32_t b = 0; b < cluster.blocks; ++b) {
    if (b == cluster.rank) {
      if (threadIdx.x == 0) told->counts[b] = n;
      continue;
    }
    TopTold* to = cluster.of(told, b);
    if (threadIdx.x < n) to->lists[cluster.rank][threadIdx.x] = s.sorted[threadIdx.x];
    if (threadIdx.x == 0) to->counts[cluster.rank] = n;
  }
}

template <class T>
__global__ void __launch_bounds__(kRowThreads, 4)
    top_kernel(RowSet x, uint32_t k, float c, float inv_t, int64_t* __restrict__ ids, float* __restrict__ logprobs) {
  // The ring, and behind it, where the row has several blocks, what they tell each other.
  extern __shared__ __align__(16) uint8_t memory[];
  __shared__ TopShared s;
  const RowCluster cluster;
  cluster.started();
  const uint32_t row = cluster.row();
  const RowWalk<T> walk(row_ptr<T>(x, row), x.vocab);
  uint32_t first, last;
  split_units(walk.units, cluster.rank, cluster.blocks, first, last);
  Ring<T, kTopDepth> ring(memory, walk, first, last);
  TopCollector<T> top(s, k, first, last);
  Soft soft;
  for (uint32_t u0 = first; u0 < last; u0 += Batch<T>::kSpan) {
    Batch<T> b;
    ring.read(b);
    const float all = step_max(b);
    soft.add(b, all, c);
    top.add(b, all);
    ring.advance();
  }
  top.finish(reinterpret_cast<uint64_t*>(memory), walk, first, last);
  soft = block_soft(soft, c, s.soft);  // a barrier behind s.sorted, too
  uint32_t n = s.sorted_count;
  TopTold* told = reinterpret_cast<TopTold*>(memory + kTopDepth * kStepBytes);
  if (cluster.blocks > 1) {
    cluster.ready();
    tell_soft(cluster, soft, told->soft);
    tell_top(cluster, s, told);
    cluster.told();
    soft = told_soft(cluster, c, told->soft);
    n = 0;
    for (uint32_t b = 0; b < cluster.blocks; ++b) n += told->counts[b];
  }
  const double log_s = log((double)soft.s);
  const size_t out = (size_t)row * k;
  if (threadIdx.x < s.sorted_count) {
    const uint64_t v = s.sorted[threadIdx.x];
    const uint32_t place = cluster.blocks > 1 ? cluster_place(cluster, *told, k, threadIdx.x, v) : threadIdx.x;
    if (place < k) {
      ids[out + place] = (int64_t)(0xFFFFFFFFu - (uint32_t)v);
      logprobs[out + place] = (float)(((double)candidate_value(v) - (double)soft.m) * (double)inv_t - log_s);
    }
  }
  if (cluster.rank == 0) {
    for (uint32_t i = n + threadIdx.x; i < k; i += kRowThreads) {
      ids[out + i] = -1;
      logprobs[out + i] = isnan(soft.s) ? NAN : -INFINITY;
    }
  }
}

// ------------------------------------------------------------ sampling
//
// The tokens that top-k, top-p and min-p keep are a prefix of the row's order, so they are named by the
// smallest logit kept and by how many of the tokens with that very logit are kept (those
// with the lowest ids). Weights are 2^42 exp((x - m) / t) rounded to integers: 2^20 of
// them fit 64 bits, sums are exact whatever their order, and what rounding leaves off is 2^-43 of the
// largest weight a token.
//
// One pass over the row gives (m, s) of every chunk (a warp's share of a step), in fp32, and, where tokens
// are to be dropped, the largest logits as for a record. Most rows are decided by these:
//   - all tokens kept: u times the total falls into a chunk, and within the chunk
//     between two tokens, whose weights are computed as integers;
//   - else, if the tokens kept are all among the largest ones at hand, these
//     alone are weighed, as integers.
// The total from fp32 sums is off by at most kSumError, relative (the exponential by 2^-22; its exponent by three
// roundings, on exponents of at most 40 as far as they matter, 5e-6; 22 additions in a chain, 1.3e-6). Where
// a border lies closer than that allows, and where more tokens are kept than are at hand, the row is
// decided by exact_token, which weighs every token as an integer.
//
// 1024 x 100003 fp16 with top-k 50 and top-p 0.95 take 66 us (3.1 TB/s): the pass, and the order of the candidates. A
// row of 128256 that exact_token weighs takes a block 50 us without truncation, bound by 64-bit arithmetic, and 200 us with a
// top-p that keeps thousands, bound by additions in shared memory.
constexpr uint32_t kBins = 1024;
constexpr uint32_t kChunkUnits = Batch<float>::kWarpSpan;  // of any type
template <class T>
constexpr uint32_t kChunk = kChunkUnits * kUnit<T>;
constexpr uint32_t kChunks = WS_MAX_VOCAB / kChunk<float> + 1;
constexpr double kWeightOne = 4398046511104.0;  // 2^42
constexpr double kSumError = 1.0 / 131072;
constexpr uint32_t kNucleus = 200;  // tokens at hand where top-k does not say: of 256, some 290 candidates would have to be sorted in 512 places
constexpr double kNoWeight = -16.0 * 1075.0;  // 16 log2 of what 64 bits round to 0

struct Bins {
  uint32_t count[kBins];
  unsigned long long mass[kBins];
};
struct ChunkSums {
  unsigned long long mass[kChunks];
  uint32_t ties[kChunks];
};
// What exact_token has in the ring's place: the tokens of the block's part that may be kept, once they are few, and the counts of a pass.
struct ExactShared {
  uint64_t list[kCandidates];
  Bins bins;
};
static_assert(sizeof(ExactShared) <= kTopDepth * kStepBytes && sizeof(ChunkSums) <= kTopDepth * kStepBytes, "they take the ring's place");

struct SampleShared {
  TopShared top;
  struct {
    unsigned long long mass;
    uint32_t ties;
  } mine;  // for the other blocks of the cluster
  unsigned long long scan[kRowWarps];
  double sums[kRowWarps];
  unsigned long long weight[WS_TOP_MAX_K];
  uint64_t merged[WS_TOP_MAX_K];  // the row's largest, in order, where it has several blocks
  double roots[16];
  double chunk_before;
  uint32_t chunk;
  uint32_t key_lo, key_hi;
  uint32_t found_bin, found_count;
  unsigned long long found_before;
  uint64_t token;  // token and the order key of its logit, in the lower half
};

__device__ __forceinline__ int64_t top_k_of(const ws_sampling& p, uint32_t row) {
  if (!p.top_k_each) return p.top_k;
  return p.top_k_is_int64 ? ((const int64_t*)p.top_k_each)[row] : (int64_t)((const int32_t*)p.top_k_each)[row];
}

// A row's settings; what is left of a temperature of 0 and of a top_p of 0 is top_k = 1.
struct SampleSettings {
  float t, top_p, min_p;
  int64_t top_k;
  double u, log_min_p;

  __device__ __forceinline__ SampleSettings(const ws_sampling& p, const float* uniform, uint32_t row) {
    t = p.temperature_each ? p.temperature_each[row] : p.temperature;
    top_p = p.top_p_each ? p.top_p_each[row] : p.top_p;
    min_p = fminf(p.min_p_each ? p.min_p_each[row] : p.min_p, 1.f);
    top_k = top_k_of(p, row);
    u = (double)uniform[row];
    log_min_p = min_p > 0.f ? 16.0 * log2((double)min_p) : 0.0;
    if (!(t > 0.f)) {
      t = 1.f;
      top_k = 1;
    }
    if (!(top_p > 0.f)) top_k = 1;
  }
  // A uniform number of 0 takes the first token of any weight, below 2^-43, too.
  __device__ __forceinline__ bool first() const { return !(u > 0.0); }
  // The cumulative weight that the token reaches first.
  __device__ __forceinline__ unsigned long long need(unsigned long long total) const {
    return first() ? 1 : min((unsigned long long)fmin(u * (double)total, 9e18) + 1, total);
  }
};

// The tokens that may still be kept, if they are in `list`; all of the block's part otherwise.
struct Few {
  const uint64_t* list = nullptr;
  uint32_t n = 0;
};

// A row under its temperature; one block's part of it, in units [first, last).
template <class T>
struct SampleRow {
  RowWalk<T> walk;
  uint32_t first, last;
  float m;
  double inv_t, log2_t, log2_m;  // 1 and 16 log2(e) over the temperature, and the latter times -m
  const double* roots;   // 2^(i / 16) for i from 0 to 15

  // 16 log2 of a token's weight. In 64 bits nothing is lost by taking the products before the difference: logits that are not equal differ by
  // 2^-24 of their size, the products are off by 2^-53 of it.
  __device__ __forceinline__ double log_weight(float v) const {
    // v in 64 bits by its bits, which are quicker than a conversion; 0 and what lies next to it become 2^-127, infinities 2^128.
    const uint32_t u = __float_as_uint(v);
    const double x = __hiloint2double((int)((u & 0x80000000u) | ((u & 0x7FFFFFFFu) >> 3) + 0x38000000u), (int)(u << 29));
    return v == m ? 0.0 : fma(x, log2_t, log2_m);
  }
  // 2^(y / 16 + 42) rounded to an integer, y <= 0. With n next to y, 2^(y / 16) = 2^(n / 16) 2^(f / 16) with |f| <= 1/2, and 2^(f / 16) is
  // e^(f ln 2 / 16) by its series up to the 5th power, off by 2e-13, less than 2^-42. Adding 2^10 leaves the multiple of 2^-42 in the sum's
  // lower bits. No branch, so that several go on at once: it is 12 operations in 64 bits, one behind the other.
  __device__ __forceinline__ unsigned long long fixed(double y) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: behind it a sum has no fraction
    constexpr double kStep = 0.693147180559945309417 / 16;
    const double k = y + kRound;
    const int n = __double2loint(k);
    const double f = y - (k - kRound);
    double p = kStep * kStep * kStep * kStep * kStep / 120;
    p = fma(p, f, kStep * kStep * kStep * kStep / 24);
    p = fma(p, f, kStep * kStep * kStep / 6);
    p = fma(p, f, kStep * kStep / 2);
    p = fma(p, f, kStep);
    p = fma(p, f, 1.0) * roots[n & 15];
    p = __hiloint2double(__double2hiint(p) + (n >> 4) * (1 << 20), __double2loint(p)) + 1024.0;
    const unsigned long long w = (unsigned long long)(__double_as_longlong(p) - __double_as_longlong(1024.0));
    return y > -704.0 ? w : 0;  // 2^-44 rounds to 0
  }
  __device__ __forceinline__ unsigned long long fixed_of(float v) const { return fixed(log_weight(v)); }
  // As it counts when the token is drawn.
  __device__ __forceinline__ unsigned long long kept(float v, const SampleSettings& p) const {
    const double y = log_weight(v);
    unsigned long long w = fixed(y);
    if (p.first() && w == 0 && y > kNoWeight) w = 1;
    if (p.min_p > 0.f && !(y >= p.log_min_p)) w = 0;
    return w;
  }
  // visit(logits, id) for the units of the block's part, or for the candidates in `few`, where there are some: an array of logits,
  // those that are not there as -inf, and a function from its index to a token's id. Four units a thread are on their way at once.
  template <class F>
  __device__ __forceinline__ void each(const Few& few, F&& visit) const {
    if (few.list) {
      for (uint32_t i = threadIdx.x; i < few.n; i += kRowThreads) {
        const float f[1] = {candidate_value(few.list[i])};
        visit(f, [&](uint32_t) { return 0xFFFFFFFFu - (uint32_t)few.list[i]; });
      }
      return;
    }
    for (uint32_t u0 = first; u0 < last; u0 += Batch<T>::kSpan) {
      uint4 raw[Batch<T>::kUnits];
      const bool inside = u0 * kUnit<T> >= walk.head && u0 + Batch<T>::kSpan <= last && (u0 + Batch<T>::kSpan) * kUnit<T> <= walk.end;
#pragma unroll
      for (uint32_t j = 0; j < Batch<T>::kUnits; ++j) {
        const uint32_t u = Batch<T>::unit(u0, j);
        raw[j] = inside ? __ldg(reinterpret_cast<const uint4*>(walk.aligned) + u) : load_edge(walk, u < last ? u : ~0u);
      }
#pragma unroll
      for (uint32_t j = 0; j < Batch<T>::kUnits; ++j) {
        float f[kUnit<T>];
        unpack<T>(raw[j], f);
        const uint32_t id = Batch<T>::unit(u0, j) * kUnit<T> - walk.head;
        visit(f, [&](uint32_t i) { return id + i; });
      }
    }
  }
};

// Which tokens are kept: those with a logit above `edge`, and the first `ties` of those equal to it.
struct Kept {
  float edge = -INFINITY;
  uint32_t ties = 0;
};

// The token of a chunk at which hit(weight before it, weight up to it), both counted from the chunk's begin, holds: into s.token.
// `tied`: tokens equal to the edge before the chunk. The whole block calls it, and a barrier has to follow.
template <class T, class H>
__device__ __forceinline__ void find_in_chunk(SampleShared& s, const SampleRow<T>& row, const SampleSettings& p, uint32_t chunk,
                                              const Kept& kept, uint32_t tied, H&& hit) {
  constexpr uint32_t kMine = kChunk<T> / kRowThreads;
  const uint32_t p0 = chunk * kChunk<T> + threadIdx.x * kMine;
  const bool edged = kept.edge > -INFINITY;
  float v[kMine];
  uint32_t equal = 0;
#pragma unroll
  for (uint32_t i = 0; i < kMine; ++i) {
    v[i] = p0 + i >= row.walk.head && p0 + i < row.walk.end ? row.walk.at(p0 + i) : -INFINITY;
    equal += edged && v[i] == kept.edge;
  }
  uint32_t nth = tied, ties_all;
  if (edged) nth += block_scan(equal, s.top.sums, &ties_all);
  unsigned long long w[kMine], sum = 0, all;
#pragma unroll
  for (uint32_t i = 0; i < kMine; ++i) {
    const bool tie = edged && v[i] == kept.edge;
    w[i] = v[i] > kept.edge || (tie && nth < kept.ties) ? row.kept(v[i], p) : 0;
    nth += tie;
    sum += w[i];
  }
  unsigned long long before = block_scan(sum, s.scan, &all);
#pragma unroll
  for (uint32_t i = 0; i < kMine; ++i) {
    if (w[i] && hit(before, before + w[i])) s.token = ((uint64_t)(p0 + i - row.walk.head) << 32) | order_key(v[i]);
    before += w[i];
  }
}

// *p += w in shared memory, by its halves: two additions of 32 bits, the second one often 0, take less than one of 64, which is a
// loop of exchanges.
__device__ __forceinline__ void add_shared(unsigned long long* p, unsigned long long w) {
  uint32_t* half = reinterpret_cast<uint32_t*>(p);
  const uint32_t low = (uint32_t)w, old = atomicAdd(half, low);
  const uint32_t high = (uint32_t)(w >> 32) + (old + low < old ? 1u : 0u);
  if (high) atomicAdd(half + 1, high);
}

// One counting pass: digit(logit) in [0, kBins) for those that take part, or -1; in every bin how many they are or, where
// `weigh`, their weight. Finds the lowest digit at which the running total (of counts, or of weights where `weigh`) reaches
// target(total of all): s.found_*. A target of 0 asks for none. Returns the total. The last bin, which may take most of a row, is
// counted in registers.
template <class T, class D, class G>
__device__ __forceinline__ unsigned long long find_bin(SampleShared& s, Bins& bins, const SampleRow<T>& row, const Few& few, bool weigh,
                                                       G&& target, D&& digit) {
  cg::cluster_group cluster = cg::this_cluster();
  for (uint32_t i = threadIdx.x; i < kBins; i += kRowThreads) {
    bins.count[i] = 0;
    bins.mass[i] = 0;
  }
  __syncthreads();
  uint32_t tail_count = 0;
  unsigned long long tail_mass = 0;
  row.each(few, [&](const auto& f, auto) {
    constexpr uint32_t n = sizeof(f) / sizeof(float);
    int d[n];
#pragma unroll
    for (uint32_t i = 0; i < n; ++i) {
      d[i] = digit(f[i]);
      tail_count += d[i] == (int)kBins - 1;
    }
    if (weigh) {
      unsigned long long w[n];
#pragma unroll
      for (uint32_t i = 0; i < n; ++i) {
        w[i] = row.fixed_of(f[i]);
        tail_mass += d[i] == (int)kBins - 1 ? w[i] : 0;
      }
#pragma unroll
      for (uint32_t i = 0; i < n; ++i)
        if ((uint32_t)d[i] < kBins - 1 && w[i]) add_shared(&bins.mass[d[i]], w[i]);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < n; ++i)
        if ((uint32_t)d[i] < kBins - 1) atomicAdd(&bins.count[d[i]], 1u);
    }
  });
  tail_count = (uint32_t)block_sum((unsigned long long)tail_count, s.scan);
  tail_mass = block_sum(tail_mass, s.scan);
  if (threadIdx.x == 0) {
    bins.count[kBins - 1] = tail_count;
    bins.mass[kBins - 1] = tail_mass;
  }
  cluster.sync();
  // Thread i takes bins 4i .. 4i + 3 of all blocks.
  constexpr uint32_t kMine = kBins / kRowThreads;
  uint32_t count[kMine];
  unsigned long long mass[kMine], sum = 0, all;
#pragma unroll
  for (uint32_t j = 0; j < kMine; ++j) {
    count[j] = 0;
    mass[j] = 0;
    for (uint32_t b = 0; b < cluster.num_blocks(); ++b) {
      const Bins* o = cluster.map_shared_rank(&bins, b);
      count[j] += o->count[threadIdx.x * kMine + j];
      mass[j] += o->mass[threadIdx.x * kMine + j];
    }
    sum += weigh ? mass[j] : count[j];
  }
  unsigned long long before = block_scan(sum, s.scan, &all);
  const unsigned long long goal = target(all);
#pragma unroll
  for (uint32_t j = 0; j < kMine; ++j) {
    const unsigned long long in = weigh ? mass[j] : count[j];
    if (before < goal && before + in >= goal) {
      s.found_bin = threadIdx.x * kMine + j;
      s.found_before = before;
    }
    before += in;
  }
  cluster.sync();  // found_* is there, and no block reads these bins any more
  return all;
}

// The logit at which the total over the row in descending order reaches `target`, among logits above `floor`, and how many of the tokens
// with this very logit it takes. target(total of all above the floor) is at most that total; where it is 0, there is no edge to find and
// `kept` stays.
template <class T, class G>
__device__ __forceinline__ void find_edge(SampleShared& s, ExactShared& m, const SampleRow<T>& row, Few& few, bool weigh, float floor,
                                          Kept& kept, G&& target) {
  cg::cluster_group cluster = cg::this_cluster();
  // First by distance from the maximum, 1/64 of a temperature a bin and one for all that is 16 below.
  const float scale = fminf((float)(64.0 * row.inv_t), 3e38f);
  auto coarse = [&](float v) { return v == row.m ? 0 : (int)fminf((row.m - v) * scale, (float)(kBins - 1)); };
  unsigned long long goal = 0;
  find_bin(s, m.bins, row, few, weigh, [&](unsigned long long all) { return goal = target(all); }, [&](float v) { return v > floor ? coarse(v) : -1; });
  if (goal == 0) return;  // the same for the whole cluster
  const int bin = (int)s.found_bin;
  goal -= s.found_before;
  // Nothing below this bin is kept: if what is above is few in this block, the passes to come need not go over the row; if only the bin's own
  // tokens are, those of this function need not. The edge lies above the floor, so that tokens at the floor itself are not kept. The list has
  // the counts of up to kBins chunks beside it.
  Few in_bin = few;
  for (int only = 0; only < 2 && !in_bin.list; ++only) {
    if (threadIdx.x == 0) s.top.count = 0;
    __syncthreads();
    row.each(few, [&](const auto& f, auto id) {
      constexpr uint32_t n = sizeof(f) / sizeof(float);
      uint32_t mask = 0;
#pragma unroll
      for (uint32_t i = 0; i < n; ++i) mask |= (f[i] > floor && (only ? coarse(f[i]) == bin : coarse(f[i]) <= bin) ? 1u : 0u) << i;
      if (!mask || s.top.count > kCandidates) return;  // too many already
      uint32_t i0 = atomicAdd(&s.top.count, (uint32_t)__popc(mask));
#pragma unroll
      for (uint32_t i = 0; i < n; ++i) {
        if (mask >> i & 1u) {
          if (i0 < kCandidates) m.list[i0] = candidate(f[i], id(i));
          ++i0;
        }
      }
    });
    __syncthreads();
    if (s.top.count <= kCandidates) in_bin = Few{m.list, s.top.count};
    if (in_bin.list && !only && row.last - row.first <= kBins * kChunkUnits) few = in_bin;
    __syncthreads();  // the count is read
  }
  // Then by the order keys of the bin's logits, from the first bit in which they differ.
  uint32_t lo = 0xFFFFFFFFu, hi = 0;
  row.each(in_bin, [&](const auto& f, auto) {
#pragma unroll
    for (uint32_t i = 0; i < sizeof(f) / sizeof(float); ++i) {
      const bool in = f[i] > floor && coarse(f[i]) == bin;
      const uint32_t k = order_key(f[i]);
      lo = min(lo, in ? k : 0xFFFFFFFFu);
      hi = max(hi, in ? k : 0u);
    }
  });
  lo = __reduce_min_sync(0xFFFFFFFFu, lo);
  hi = __reduce_max_sync(0xFFFFFFFFu, hi);
  if (threadIdx.x == 0) {
    s.key_lo = 0xFFFFFFFFu;
    s.key_hi = 0;
  }
  __syncthreads();
  if ((threadIdx.x & 31u) == 0) {
    atomicMin(&s.key_lo, lo);
    atomicMax(&s.key_hi, hi);
  }
  cluster.sync();
  lo = 0xFFFFFFFFu;
  hi = 0;
  for (uint32_t b = 0; b < cluster.num_blocks(); ++b) {
    lo = min(lo, cluster.map_shared_rank(&s, b)->key_lo);
    hi = max(hi, cluster.map_shared_rank(&s, b)->key_hi);
  }
  cluster.sync();
  int left = lo == hi ? 0 : 32 - __clz(lo ^ hi);  // low bits still open
  uint32_t prefix = left == 32 ? 0 : hi >> left;  // those above
#pragma unroll 1
  while (left > 0) {
    const int step = min(left, 8);
    const int shift = left - step;
    // The largest digit first: digits are counted from the top.
    find_bin(s, m.bins, row, in_bin, weigh, [&](unsigned long long) { return goal; }, [&](float v) {
      const uint32_t k = order_key(v);
      const bool in = v > floor && coarse(v) == bin && (left == 32 || (k >> left) == prefix);
      return in ? (int)((1u << step) - 1u - ((k >> shift) & ((1u << step) - 1u))) : -1;
    });
    goal -= s.found_before;
    prefix = (left == 32 ? 0u : prefix << step) | ((1u << step) - 1u - s.found_bin);
    left = shift;
    __syncthreads();  // found_* is read
  }
  kept.edge = key_value(prefix);
  // What is left of the target lies within the weight of the tokens at the edge, which all weigh the same.
  const unsigned long long one = row.fixed_of(kept.edge);
  kept.ties = (uint32_t)(weigh ? (goal + one - 1) / max(one, 1ull) : goal);
}

// The row's token from integer weights of all its tokens, by the whole cluster: into s.token of the block that holds it.
// `memory`: what the ring left, for the counts. `few`: the block's part of the first top-k, if they are known.
template <class T>
__device__ __noinline__ void exact_token(SampleShared& s, void* memory, const SampleRow<T> row, const SampleSettings p, Few few, uint32_t vocab) {
  cg::cluster_group cluster = cg::this_cluster();
  ExactShared& m = *reinterpret_cast<ExactShared*>(memory);
  Kept kept;
  if (p.top_k == 1) {
    kept.edge = row.m;
    kept.ties = 1;
  } else if (p.top_k > 1 && p.top_k < (int64_t)vocab) {
    const unsigned long long most = (unsigned long long)p.top_k;
    find_edge(s, m, row, few, false, -INFINITY, kept, [&](unsigned long long all) { return all > most ? most : 0; });
  }
  if (p.top_p < 1.f && p.top_k != 1) {
    const float floor = kept.edge;
    const unsigned long long one = floor > -INFINITY ? row.fixed_of(floor) : 0;
    uint32_t ties = kept.ties;
    find_edge(s, m, row, few, true, floor, kept, [&](unsigned long long above) {
      const unsigned long long total = above + one * ties;
      unsigned long long goal = (unsigned long long)ceil((double)p.top_p * (double)total);
      goal = min(max(goal, 1ull), total);
      if (goal <= above) return goal;
      ties = min(ties, (uint32_t)((goal - above + one - 1) / max(one, 1ull)));  // it ends among those at the floor
      return 0ull;
    });
    if (kept.edge == floor) kept.ties = ties;
  }

  // Weights of the tokens kept, in id order: by chunks, then within the chunk that holds the token.
  // By chunk of the block's part; beside the list, where there is one (find_edge sees to it that they fit).
  const bool edged = kept.edge > -INFINITY;
  const unsigned long long one = edged ? row.kept(kept.edge, p) : 0;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t chunk0 = row.first / kChunkUnits;
  const uint32_t chunk1 = row.first < row.last ? (row.last + kChunkUnits - 1) / kChunkUnits : chunk0;
  unsigned long long* chunk_mass = few.list ? m.bins.mass : reinterpret_cast<ChunkSums*>(memory)->mass;
  uint32_t* chunk_ties = few.list ? m.bins.count : reinterpret_cast<ChunkSums*>(memory)->ties;
  unsigned long long mass = 0;
  uint32_t tied = 0;
  const bool plain = !p.first() && !(p.min_p > 0.f);  // kept() is fixed_of()
  __syncthreads();
  if (few.list) {
    for (uint32_t c = threadIdx.x; c < chunk1 - chunk0; c += kRowThreads) {
      chunk_mass[c] = 0;
      chunk_ties[c] = 0;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < few.n; i += kRowThreads) {
      const float v = candidate_value(few.list[i]);
      const uint32_t c = (0xFFFFFFFFu - (uint32_t)few.list[i] + row.walk.head) / kChunk<T> - chunk0;
      if (v > kept.edge) {
        const unsigned long long w = row.kept(v, p);
        add_shared(&chunk_mass[c], w);
        mass += w;
      } else if (v == kept.edge) {
        atomicAdd(&chunk_ties[c], 1u);
        ++tied;
      }
    }
  } else {
    for (uint32_t ch = chunk0 + warp; ch < chunk1; ch += kRowWarps) {
      unsigned long long w = 0;
      uint32_t e = 0;
      uint4 raw[Batch<T>::kUnits];
      const uint32_t u0 = ch * kChunkUnits;
      const bool inside = u0 * kUnit<T> >= row.walk.head && u0 + kChunkUnits <= row.last && (u0 + kChunkUnits) * kUnit<T> <= row.walk.end;
#pragma unroll
      for (uint32_t j = 0; j < Batch<T>::kUnits; ++j) {
        const uint32_t u = u0 + j * 32 + lane;
        raw[j] = inside ? __ldg(reinterpret_cast<const uint4*>(row.walk.aligned) + u) : load_edge(row.walk, u < row.last ? u : ~0u);
      }
#pragma unroll
      for (uint32_t j = 0; j < Batch<T>::kUnits; ++j) {
        float f[kUnit<T>];
        unpack<T>(raw[j], f);
#pragma unroll
        for (uint32_t i = 0; i < kUnit<T>; ++i) e += edged && f[i] == kept.edge;
        if (plain) {
          unsigned long long one_w[kUnit<T>];
#pragma unroll
          for (uint32_t i = 0; i < kUnit<T>; ++i) one_w[i] = row.fixed_of(f[i]);
#pragma unroll
          for (uint32_t i = 0; i < kUnit<T>; ++i) w += f[i] > kept.edge ? one_w[i] : 0;
        } else {
#pragma unroll
          for (uint32_t i = 0; i < kUnit<T>; ++i) w += f[i] > kept.edge ? row.kept(f[i], p) : 0;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xFFFFFFFFu, w, o);
      e = __reduce_add_sync(0xFFFFFFFFu, e);
      if (lane == 0) {
        chunk_mass[ch - chunk0] = w;
        chunk_ties[ch - chunk0] = e;
        mass += w;
        tied += e;
      }
    }
  }
  mass = block_sum(mass, s.scan);
  tied = (uint32_t)block_sum((unsigned long long)tied, s.scan);
  if (threadIdx.x == 0) {
    s.mine.mass = mass;
    s.mine.ties = tied;
  }
  cluster.sync();
  unsigned long long before = 0, total = 0, mine = 0;
  uint32_t ties_before = 0, seen = 0;
  for (uint32_t b = 0; b < cluster.num_blocks(); ++b) {
    const SampleShared* o = cluster.map_shared_rank(&s, b);
    const uint32_t next = seen + o->mine.ties;
    const unsigned long long w = o->mine.mass + one * (min(next, kept.ties) - min(seen, kept.ties));
    if (b == cluster.block_rank()) {
      before = total;
      ties_before = seen;
      mine = w;
    }
    total += w;
    seen = next;
  }
  const unsigned long long need = p.need(total);
  if (before < need && need <= before + mine) {  // the same for the whole block
    // Thread i takes chunks i * each .. of the block's.
    const uint32_t n = chunk1 - chunk0, each = (n + kRowThreads - 1) / kRowThreads;
    const uint32_t c0 = min(threadIdx.x * each, n), c1 = min(c0 + each, n);
    uint32_t e = 0, all_ties;
    for (uint32_t c = c0; c < c1; ++c) e += chunk_ties[c];
    uint32_t tie = ties_before + block_scan(e, s.top.sums, &all_ties);
    const uint32_t tie0 = tie;
    unsigned long long w = 0, all;
    for (uint32_t c = c0; c < c1; ++c) {
      w += chunk_mass[c] + one * (min(tie + chunk_ties[c], kept.ties) - min(tie, kept.ties));
      tie += chunk_ties[c];
    }
    unsigned long long at = before + block_scan(w, s.scan, &all);
    tie = tie0;
    for (uint32_t c = c0; c < c1; ++c) {
      const unsigned long long own = chunk_mass[c] + one * (min(tie + chunk_ties[c], kept.ties) - min(tie, kept.ties));
      if (at < need && need <= at + own) {
        s.chunk = chunk0 + c;
        s.found_before = at;
        s.found_count = tie;
      }
      at += own;
      tie += chunk_ties[c];
    }
    __syncthreads();
    const unsigned long long base = s.found_before;
    find_in_chunk(s, row, p, min(s.chunk, chunk1 - 1), kept, s.found_count,
                  [&](unsigned long long b, unsigned long long a) { return base + b < need && need <= base + a; });
  }
  cluster.sync();  // the blocks' shared memory is read until here, and s.token is there
}

// The token from the row's largest logits, `n` in order in `list`, where they hold all that is kept; false: they may not. The
// same answer in every block. `all_there`: the row has no others above -inf. total: of the row, in units of
// the largest weight, off by at most kSumError.
template <class T>
__device__ __forceinline__ bool token_of_largest(SampleShared& s, const SampleRow<T>& row, const SampleSettings& p, const uint64_t* list,
                                                 uint32_t n, bool all_there, uint32_t vocab, double total) {
  const uint32_t i = threadIdx.x;
  const bool limited = p.top_k >= 1 && p.top_k < (int64_t)vocab;
  bool whole = all_there || (limited && p.top_k <= (int64_t)n);  // the list holds all that top-k keeps
  const uint32_t id = i < n ? 0xFFFFFFFFu - (uint32_t)list[i] : 0xFFFFFFFFu;
  const float v = i < n ? candidate_value(list[i]) : -INFINITY;
  const double y = i < n ? row.log_weight(v) : -INFINITY;
  const unsigned long long fixed = row.fixed(y);
  uint32_t keep = n;
  if (p.top_p < 1.f && p.top_k != 1) {
    unsigned long long sum;
    const unsigned long long cum = block_scan(fixed, s.scan, &sum) + fixed;
    if (whole) {
      unsigned long long target = (unsigned long long)ceil((double)p.top_p * (double)sum);
      target = min(max(target, 1ull), sum);
      keep = __syncthreads_count(i < n && cum < target) + 1;
    } else {
      if (limited) return false;
      const double target = (double)p.top_p * total * kWeightOne, off = 2 * kSumError * target + 512.0;
      const uint32_t low = __syncthreads_count(i < n && (double)cum < target - off);
      const uint32_t high = __syncthreads_count(i < n && (double)cum < target + off);
      if (low != high || low >= n) return false;
      keep = low + 1;
      whole = true;
    }
  }
  if (p.min_p > 0.f) {
    const uint32_t heavy = __syncthreads_count(i < keep && y >= p.log_min_p);
    whole = whole || heavy < keep;
    keep = heavy;
  }
  if (!whole) return false;
  const unsigned long long w = i < keep ? (p.first() && fixed == 0 && y > kNoWeight ? 1 : fixed) : 0;
  const unsigned long long sum = block_sum(w, s.scan);
  const unsigned long long need = p.need(sum);
  s.weight[i] = w;
  __syncthreads();
  if (i < keep) {
    unsigned long long cum = 0;
#pragma unroll 4
    for (uint32_t q = 0; q < keep; ++q) cum += 0xFFFFFFFFu - (uint32_t)list[q] <= id ? s.weight[q] : 0;
    if (w && cum >= need && cum - w < need) s.token = ((uint64_t)id << 32) | order_key(v);
  }
  return true;
}

template <class T>
__global__ void __launch_bounds__(kRowThreads, 3)
    sample_kernel(RowSet x, const float* __restrict__ uniform, ws_sampling sampling, int64_t* __restrict__ tokens,
                  float* __restrict__ logprobs) {
  // The ring (then what exact_token counts), (m, s) of the row's chunks, and, where the row has several blocks, what they tell each other.
  extern __shared__ __align__(16) uint8_t memory[];
  __shared__ SampleShared s;
  const RowCluster cluster;
  cluster.started();
  const uint32_t r = cluster.row();
  const SampleSettings p(sampling, uniform, r);
  // Finite and above 0, so that a logit of -inf has no weight at an infinite temperature, either.
  const float c = fmaxf(fminf(kLog2e / p.t, 3e38f), 1.4e-45f);
  const RowWalk<T> walk(row_ptr<T>(x, r), x.vocab);
  const uint32_t chunks = (walk.units + kChunkUnits - 1) / kChunkUnits;
  uint32_t chunk0, chunk1;
  split_units(chunks, cluster.rank, cluster.blocks, chunk0, chunk1);
  SampleRow<T> row{walk, chunk0 * kChunkUnits, min(chunk1 * kChunkUnits, walk.units), 0.f, 1.0 / (double)p.t,
                   16.0 * 1.442695040888963407360 / (double)p.t, 0.0, s.roots};
  row.first = min(row.first, row.last);
  float2* soft = reinterpret_cast<float2*>(memory + kTopDepth * kStepBytes);
  TopTold* told = reinterpret_cast<TopTold*>(soft + ((chunks + 1) & ~1u));
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const bool dropping = (p.top_k >= 1 && p.top_k < (int64_t)x.vocab) || p.top_p < 1.f || p.min_p > 0.f;
  // The largest logits, in order: as many as top-k asks for, or kNucleus. A larger top-k is left to exact_token, which up to
  // kMostCollected gets a list.
  const bool many = p.top_k > WS_TOP_MAX_K && p.top_k <= kMostCollected && p.top_k < (int64_t)x.vocab;
  const uint32_t k = p.top_k >= 1 && p.top_k <= kMostCollected ? (uint32_t)p.top_k : kNucleus;
  Few few;

  Ring<T, kTopDepth> ring(memory, walk, row.first, row.last);
  TopCollector<T> top(s.top, k, row.first, row.last);
  if (threadIdx.x == 0) s.token = ~0ull;
  if (threadIdx.x < 16) s.roots[threadIdx.x] = exp2(threadIdx.x / 16.0);
  for (uint32_t u0 = row.first; u0 < row.last; u0 += Batch<T>::kSpan) {
    Batch<T> b;
    ring.read(b);
    const float all = step_max(b);
    const float m = key_value(__reduce_max_sync(0xFFFFFFFFu, order_key(all)));
    float sum = step_sum(b, m, c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    const uint32_t ch = u0 / kChunkUnits + warp;
    if (lane == 0 && ch < chunk1) soft[ch] = make_float2(m, sum);
    if (dropping) top.add(b, all);
    ring.advance();
  }
  if (many) {
    uint64_t* candidates = reinterpret_cast<ExactShared*>(memory)->list;
    top.collect(candidates, walk, row.first, row.last);
    // The list has the counts of up to kBins chunks beside it.
    if (s.top.count <= kCandidates && row.last - row.first <= kBins * kChunkUnits) few = Few{candidates, s.top.count};
  } else if (dropping) {
    top.finish(reinterpret_cast<uint64_t*>(memory), walk, row.first, row.last);
  }
  __syncthreads();
  const uint64_t* list = s.top.sorted;
  const bool sorted = dropping && !many;
  uint32_t n = sorted ? s.top.sorted_count : 0;
  if (cluster.blocks > 1) {
    cluster.ready();
    for (uint32_t b = 0; b < cluster.blocks; ++b) {
      if (b == cluster.rank) continue;
      float2* to = cluster.of(soft, b);
      for (uint32_t i = chunk0 + threadIdx.x; i < chunk1; i += kRowThreads) to[i] = soft[i];
    }
    if (sorted) tell_top(cluster, s.top, told);
    cluster.told();
    if (sorted) {
      const uint32_t own = n;
      n = 0;
      for (uint32_t b = 0; b < cluster.blocks; ++b) n += told->counts[b];
      if (threadIdx.x < own) {
        const uint64_t v = s.top.sorted[threadIdx.x];
        const uint32_t place = cluster_place(cluster, *told, k, threadIdx.x, v);
        if (place < k)
          for (uint32_t b = 0; b < cluster.blocks; ++b) cluster.of(s.merged, b)[place] = v;
      }
      cluster.told();
      list = s.merged;
    }
  }
  const bool all_there = n < k;
  n = min(n, k);

  // The row's maximum and total from its chunks', the same in every block.
  const uint32_t each = (chunks + kRowThreads - 1) / kRowThreads;
  const uint32_t c0 = min(threadIdx.x * each, chunks), c1 = min(c0 + each, chunks);
  float m = -INFINITY;
  for (uint32_t i = c0; i < c1; ++i) m = fmaxf(m, soft[i].x);
  m = block_max(m, reinterpret_cast<float*>(s.sums));
  row.m = m;
  row.log2_m = -(double)m * row.log2_t;
  // 2^((x - m) c) of a chunk in 64 bits, with the c that its sum has.
  auto chunk_sum = [&](uint32_t i) {
    const float2 t = soft[i];
    return t.x == -INFINITY ? (double)t.y : (double)t.y * (t.x == m ? 1.0 : exp2(((double)t.x - (double)m) * (double)c));
  };
  double mine = 0.0, total;
  for (uint32_t i = c0; i < c1; ++i) mine += chunk_sum(i);
  const double before = block_scan(mine, s.sums, &total);
  if (m == -INFINITY) {  // the same for the whole cluster
    if (cluster.rank == 0 && threadIdx.x == 0) {
      tokens[r] = -1;
      if (logprobs) logprobs[r] = isnan(total) ? NAN : -INFINITY;
    }
    return;
  }

  // A total that is no finite number (NaN or +inf logits) and a factor that has left fp32's range leave it to exact_token.
  bool decided = false;
  if (dropping && p.top_k == 1) {
    if (threadIdx.x == 0) s.token = ((uint64_t)(0xFFFFFFFFu - (uint32_t)list[0]) << 32) | (list[0] >> 32);
    decided = true;
  } else if (isfinite(total) && c < 1e30f) {
    if (sorted) {
      decided = token_of_largest(s, row, p, list, n, all_there, x.vocab, total);
    } else if (!dropping && !p.first()) {
      const double target = p.u * total;
      if (threadIdx.x == 0) s.chunk = chunks;
      __syncthreads();
      if (before <= target && target < before + mine) {
        double at = before;
        for (uint32_t i = c0; i < c1; ++i) {
          const double own = chunk_sum(i);
          if (at <= target && target < at + own) {
            s.chunk = i;
            s.chunk_before = at;
          }
          at += own;
        }
      }
      __syncthreads();
      if (s.chunk < chunks) {
        const double base = s.chunk_before * kWeightOne, goal = target * kWeightOne, off = 2 * kSumError * goal + 2048.0;
        find_in_chunk(s, row, p, s.chunk, Kept{}, 0, [&](unsigned long long b, unsigned long long a) {
          return base + (double)b < goal - off && base + (double)a > goal + off;
        });
        __syncthreads();
        decided = s.token != ~0ull;
      }
    }
  }
  const bool here = decided;
  if (!decided) {
    __syncthreads();
    exact_token(s, memory, row, p, few, x.vocab);
  } else {
    __syncthreads();
  }
  // Decided above, every block has the token; exact_token leaves it in the block that holds it (or in none, if logits
  // change while they are read).
  if (threadIdx.x == 0) {
    const uint64_t token = s.token;
    if (here ? cluster.rank == 0 : token != ~0ull) {
      tokens[r] = (int64_t)(token >> 32);
      if (logprobs) logprobs[r] = (float)(((double)key_value((uint32_t)token) - (double)m) * row.inv_t - log(total));
    }
  }
}

int fail(int code, const std::string& msg) {
  set_last_error(msg.c_str());
  return code;
}

int done(cudaError_t e, const char* what) {
  return e == cudaSuccess ? WS_OK : fail(WS_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

}  // namespace
}  // namespace ws

using namespace ws;

extern "C" int ws_top_logprobs(const ws_rows* logits, uint32_t k, float temperature, int64_t* ids, float* logprobs,
                               int device, void* stream) {
  return guarded([&] {
    RowArgs x;
    const int rc = check_rows(logits, "logits", &x);
    if (rc != WS_OK) return rc;
    if (k < 1 || k > WS_TOP_MAX_K || k > x.set.vocab) return fail(WS_ERR_INVALID, "k must be from 1 to 256 and at most the vocabulary");
    if (!(temperature >= 1e-6f && temperature <= 1e6f)) return fail(WS_ERR_INVALID, "temperature must be from 1e-6 to 1e6");
    if (device < 0) return fail(WS_ERR_INVALID, "bad device ordinal");
    if (x.rows == 0) return (int)WS_OK;
    if (!ids || !logprobs) return fail(WS_ERR_INVALID, "null result pointer");
    DeviceGuard guard(device);
    cudaError_t e = guard.error();
    if (e == cudaSuccess)
      e = by_type(x.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const uint32_t blocks = blocks_a_row(x);
        return launch_rows<top_kernel<T>>(x.rows, blocks, kTopDepth * kStepBytes + (blocks > 1 ? sizeof(TopTold) : 0), device, stream,
                                          x.set, k, kLog2e / temperature, 1.f / temperature, ids, logprobs);
      });
    return done(e, "top log-probabilities");
  });
}

extern "C" int ws_sample(const ws_rows* logits, const float* uniform, const ws_sampling* sampling, int64_t* tokens,
                         float* logprobs, int device, void* stream) {
  return guarded([&] {
    RowArgs x;
    const int rc = check_rows(logits, "logits", &x);
    if (rc != WS_OK) return rc;
    if (!sampling) return fail(WS_ERR_INVALID, "null sampling settings");
    if (device < 0) return fail(WS_ERR_INVALID, "bad device ordinal");
    if (x.rows == 0) return (int)WS_OK;
    if (!uniform || !tokens) return fail(WS_ERR_INVALID, "null pointer");
    DeviceGuard guard(device);
    cudaError_t e = guard.error();
    if (e == cudaSuccess)
      e = by_type(x.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        // Where no token is dropped, some rows have all their tokens weighed as integers, 50 us for one block: more blocks for each
        // (256 x 151936 fp32: 99 us with one, 63 with four).
        const bool all_kept = !sampling->temperature_each && !sampling->top_k_each && !sampling->top_p_each && !sampling->min_p_each &&
                              sampling->temperature > 0.f && sampling->top_k <= 0 && sampling->top_p >= 1.f && !(sampling->min_p > 0.f);
        // Settings of each row's own bring such rows, too, and others that need as much, and the call ends with the slowest (128 x 128256
        // bf16, all kinds of settings: 220 us with one block, 115 with four).
        const bool each_own = sampling->temperature_each || sampling->top_k_each || sampling->top_p_each || sampling->min_p_each;
        const uint32_t blocks = blocks_a_row(x, each_own ? 56 : 0, all_kept ? 4 * kFewBlocks : kFewBlocks);
        const uint32_t chunks = (x.set.vocab + 2 * kUnit<T> - 2) / kChunk<T> + 1;  // at most, with the row's head
        return launch_rows<sample_kernel<T>>(x.rows, blocks, kTopDepth * kStepBytes + ((chunks + 1) & ~1u) * sizeof(float2) + (blocks > 1 ? sizeof(TopTold) : 0),
                                             device, stream, x.set, uniform, *sampling, tokens, logprobs);
      });
    return done(e, "sample");
  });
}
