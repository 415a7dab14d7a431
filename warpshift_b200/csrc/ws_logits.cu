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
// One pass over the row gives its maximum m and S = sum exp((x - m) / t), and keeps
// the candidates for the k largest logits in shared memory: a candidate is 64 bits, the order key
// of its logit above the complement of its id, so that no two are equal and the
// larger one comes first in the record.
//
// What a logit costs is one comparison of its unit's maximum with a threshold, below which nothing can be in
// the record. The threshold comes from maxima that are at hand anyway: every thread keeps the maximum of each
// of its kUnits places in a step over all steps, kRowThreads * kUnits logits of different
// ids, the k-th largest of which is a lower bound of the k-th largest logit, and a close one. It is
// found by bisection over the upper 16 bits of the order keys after steps 1, 2, 4, 8, ...
// and at the end, when the list holds few more than k candidates.
//
// The list has room for k candidates and all of a step's that one unit of each thread
// gives. A step that would overflow it (ascending or equal logits) is taken again unit
// by unit, dropping all but the k largest before each: slow, and right for any row.
constexpr uint32_t kCandidates = WS_TOP_MAX_K + kRowThreads * kUnit;
constexpr uint32_t kSorted = 512;  // candidates that are put in order by counting

struct TopShared {
  uint64_t list[kCandidates];
  uint64_t sorted[WS_TOP_MAX_K];  // the block's k largest in order, for the other blocks of the cluster
  uint32_t count, sorted_count;
  uint32_t sums[kRowWarps];
  uint2 votes[2][kRowWarps];
  float2 soft[kRowWarps];
  float2 soft_mine;
};

__device__ __forceinline__ uint64_t candidate(float x, uint32_t id) { return ((uint64_t)order_key(x) << 32) | (0xFFFFFFFFu - id); }
__device__ __forceinline__ float candidate_value(uint64_t v) { return key_value((uint32_t)(v >> 32)); }

// Keeps the k largest of s.list's first n > k candidates (in no order) and returns the smallest of these.
__device__ __noinline__ uint64_t keep_largest(TopShared& s, uint32_t n, uint32_t k) {
  constexpr uint32_t kMine = (kCandidates + kRowThreads - 1) / kRowThreads;
  uint64_t mine[kMine];
#pragma unroll
  for (uint32_t i = 0; i < kMine; ++i) {
    const uint32_t at = i * kRowThreads + threadIdx.x;
    mine[i] = at < n ? s.list[at] : 0;
  }
  uint64_t edge = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const uint64_t trial = edge | (1ull << bit);
    uint32_t c = 0;
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) c += mine[i] >= trial;
    if (block_sum(c, s.sums) >= k) edge = trial;
  }
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < kMine; ++i)
    if (mine[i] >= edge) s.list[atomicAdd(&s.count, 1u)] = mine[i];
  __syncthreads();
  return edge;
}

// A logit that at least k of the block's maxima reach, as large as 16 bits of its order key
// tell; the lowest finite number where fewer than k are above -inf. Two bits a round: the
// counts of three trials by one shuffle-free reduction in the warp, and one barrier.
template <uint32_t N>
__device__ __forceinline__ float kth_of_maxima(TopShared& s, const float (&top)[N], uint32_t k) {
  uint32_t key[N];
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) key[j] = order_key(top[j]) >> 16;
  uint32_t edge = 0;
#pragma unroll
  for (int bit = 14; bit >= 0; bit -= 2) {
    uint32_t low = 0, high = 0;  // counts of trials 1 and 2, and of trial 3
#pragma unroll
    for (uint32_t j = 0; j < N; ++j) {
      low += (key[j] >= (edge | (1u << bit)) ? 1u : 0u) + (key[j] >= (edge | (2u << bit)) ? 0x10000u : 0u);
      high += key[j] >= (edge | (3u << bit)) ? 1u : 0u;
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
    const uint32_t step = high >= k ? 3u : (low >> 16) >= k ? 2u : (low & 0xFFFFu) >= k ? 1u : 0u;
    edge |= step << bit;
  }
  constexpr uint32_t kNone = 0x007Fu;  // upper half of -inf's key
  return edge <= kNone ? -FLT_MAX : key_value(edge << 16);
}

// The statistics and the k largest logits of units [first, last) of a row: s.sorted_count (at most k) candidates in s.sorted, in
// order. Every thread gets the statistics.
template <class T>
__device__ __forceinline__ Soft row_top(const RowWalk<T>& walk, uint32_t first, uint32_t last, float c, uint32_t k, TopShared& s) {
  using B = Batch<T>;
  if (threadIdx.x == 0) s.count = 0;
  Soft soft;
  float most[B::kUnits];
#pragma unroll
  for (uint32_t j = 0; j < B::kUnits; ++j) most[j] = -INFINITY;
  float edge = -FLT_MAX;  // logits below it are of no use; nor are -inf and NaN
  B next;
  if (first < last) next.load(walk, first, last);
  __syncthreads();
  uint32_t step = 1;
  for (uint32_t u0 = first; u0 < last; u0 += B::kSpan, ++step) {
    const B now = next;
    if (u0 + B::kSpan < last) next.load(walk, u0 + B::kSpan, last);
    float top[B::kUnits], all = -INFINITY;
#pragma unroll
    for (uint32_t j = 0; j < B::kUnits; ++j) {
      top[j] = unit_max<T>(now.raw[j]);
      most[j] = fmaxf(most[j], top[j]);
      all = fmaxf(all, top[j]);
    }
    soft.add(now, all, c);
    if ((step & (step - 1)) == 0) edge = fmaxf(edge, kth_of_maxima(s, most, k));
    const uint32_t before = s.count;
    __syncthreads();  // everyone has it
    if (all >= edge) {
#pragma unroll
      for (uint32_t j = 0; j < B::kUnits; ++j) {
        if (top[j] >= edge) {
          float f[kUnit];
          unpack<T>(now.raw[j], f);
          const uint32_t id = (u0 + j * kRowThreads + threadIdx.x) * kUnit - walk.head;
#pragma unroll
          for (uint32_t i = 0; i < kUnit; ++i) {
            if (f[i] >= edge) {
              const uint32_t at = atomicAdd(&s.count, 1u);
              if (at < kCandidates) s.list[at] = candidate(f[i], id + i);
            }
          }
        }
      }
    }
    __syncthreads();
    if (s.count > kCandidates) {
      __syncthreads();
      if (threadIdx.x == 0) s.count = before;
      __syncthreads();
      uint64_t least = 0;
      for (uint32_t j = 0; j < B::kUnits; ++j) {
        if (s.count > k) least = keep_largest(s, s.count, k);
        __syncthreads();
        Raw<T> raw = now.raw[0];
#pragma unroll
        for (uint32_t q = 1; q < B::kUnits; ++q)
          if (q == j) raw = now.raw[q];
        float f[kUnit];
        unpack<T>(raw, f);
        const uint32_t id = (u0 + j * kRowThreads + threadIdx.x) * kUnit - walk.head;
#pragma unroll
        for (uint32_t i = 0; i < kUnit; ++i) {
          if (f[i] >= edge) {
            const uint64_t v = candidate(f[i], id + i);
            if (v > least) s.list[atomicAdd(&s.count, 1u)] = v;
          }
        }
        __syncthreads();
      }
      if (s.count > k) least = keep_largest(s, s.count, k);
      edge = fmaxf(edge, least ? candidate_value(least) : -FLT_MAX);
      __syncthreads();
    }
  }
  // Of the candidates those that reach the last threshold, in order. A thread holds at most kMine of them.
  edge = fmaxf(edge, kth_of_maxima(s, most, k));
  constexpr uint32_t kMine = (kCandidates + kRowThreads - 1) / kRowThreads;
  uint64_t mine[kMine];
  const uint32_t found = s.count;
#pragma unroll
  for (uint32_t i = 0; i < kMine; ++i) {
    const uint32_t at = i * kRowThreads + threadIdx.x;
    mine[i] = at < found ? s.list[at] : 0;
  }
  __syncthreads();
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < kMine; ++i)
    if (mine[i] && candidate_value(mine[i]) >= edge) s.list[atomicAdd(&s.count, 1u)] = mine[i];
  __syncthreads();
  if (s.count > kSorted) keep_largest(s, s.count, k);  // k <= WS_TOP_MAX_K <= kSorted remain
  const uint32_t n = s.count;
  if (threadIdx.x == 0) s.sorted_count = min(n, k);
  for (uint32_t i = threadIdx.x; i < n; i += kRowThreads) {
    const uint64_t v = s.list[i];
    uint32_t place = 0;
#pragma unroll 4
    for (uint32_t q = 0; q < n; ++q) place += s.list[q] > v;
    if (place < k) s.sorted[place] = v;
  }
  return block_soft(soft, c, s.soft);  // with a barrier behind s.sorted
}

// The cluster's record: place of this block's i-th candidate, which is i and how many of the other blocks' are larger.
__device__ __forceinline__ uint32_t cluster_place(TopShared& s, uint32_t i, uint64_t v) {
  cg::cluster_group cluster = cg::this_cluster();
  uint32_t place = i;
  for (uint32_t b = 0; b < cluster.num_blocks(); ++b) {
    if (b == cluster.block_rank()) continue;
    const TopShared* o = cluster.map_shared_rank(&s, b);
    uint32_t lo = 0, hi = o->sorted_count;
    while (lo < hi) {
      const uint32_t mid = (lo + hi) / 2;
      if (o->sorted[mid] > v) lo = mid + 1;
      else hi = mid;
    }
    place += lo;
  }
  return place;
}

template <class T>
__global__ void __launch_bounds__(kRowThreads, 3)
    top_kernel(RowSet x, uint32_t k, float c, float inv_t, int64_t* __restrict__ ids, float* __restrict__ logprobs) {
  __shared__ TopShared s;
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t blocks = cluster.num_blocks(), rank = cluster.block_rank(), row = blockIdx.x / blocks;
  const RowWalk<T> walk(row_ptr<T>(x, row), x.vocab);
  uint32_t first, last;
  split_units(walk.units, rank, blocks, first, last);
  const Soft soft = cluster_soft(row_top(walk, first, last, c, k, s), c, &s.soft_mine);
  const double log_s = log((double)soft.s);
  const size_t out = (size_t)row * k;
  if (threadIdx.x < s.sorted_count) {
    const uint64_t v = s.sorted[threadIdx.x];
    const uint32_t place = blocks > 1 ? cluster_place(s, threadIdx.x, v) : threadIdx.x;
    if (place < k) {
      ids[out + place] = (int64_t)(0xFFFFFFFFu - (uint32_t)v);
      logprobs[out + place] = (float)(((double)candidate_value(v) - (double)soft.m) * (double)inv_t - log_s);
    }
  }
  if (rank == 0) {
    uint32_t n = 0;
    for (uint32_t b = 0; b < blocks; ++b) n += cluster.map_shared_rank(&s, b)->sorted_count;
    for (uint32_t i = n + threadIdx.x; i < k; i += kRowThreads) {
      ids[out + i] = -1;
      logprobs[out + i] = isnan(soft.s) ? NAN : -INFINITY;
    }
  }
  if (blocks > 1) cluster.sync();  // the blocks' shared memory is read until here
}

// ------------------------------------------------------------ sampling
//
// The tokens that top-k, top-p and min-p keep are a prefix of the row's order, so they are named by the
// smallest logit kept and by how many of the tokens with that very logit are kept (those
// with the lowest ids). Weights are 2^42 exp((x - m) / t) rounded to integers: 2^20 of
// them fit 64 bits, sums are exact whatever their order, and what rounding and the 64-bit
// exponential leave off is below 2^-42 of the largest weight a token.
constexpr uint32_t kBins = 1024;
constexpr uint32_t kChunkUnits = 128;  // a warp's piece of the row when tokens are counted in id order
constexpr uint32_t kChunk = kChunkUnits * kUnit;
constexpr uint32_t kChunks = WS_MAX_VOCAB / kChunk + 1;
constexpr double kWeightOne = 4398046511104.0;  // 2^42

struct SampleShared {
  union {
    struct {
      uint32_t count[kBins];
      unsigned long long mass[kBins];
    } bins;
    struct {
      unsigned long long mass[kChunks];
      uint32_t ties[kChunks];
    } chunks;
  };
  struct {
    unsigned long long mass;
    uint32_t ties;
  } mine;  // for the other blocks of the cluster
  unsigned long long sum_scratch[kRowWarps];
  float2 soft_scratch[kRowWarps];
  float2 soft_mine;
  uint32_t key_lo, key_hi;
  uint32_t found_bin;
  unsigned long long found_before, found_mass;
  uint32_t found_count;
};

__device__ __forceinline__ int64_t top_k_of(const ws_sampling& p, uint32_t row) {
  if (!p.top_k_each) return p.top_k;
  return p.top_k_is_int64 ? ((const int64_t*)p.top_k_each)[row] : (int64_t)((const int32_t*)p.top_k_each)[row];
}

// A row under its temperature; one block's part of it, in units [first, last).
template <class T>
struct SampleRow {
  RowWalk<T> walk;
  uint32_t first, last;
  float m;
  double inv_t;

  __device__ __forceinline__ double weight(float v) const { return v == m ? 1.0 : exp(((double)v - (double)m) * inv_t); }
  __device__ __forceinline__ unsigned long long fixed(float v) const {
    return v == m ? (unsigned long long)kWeightOne : __double2ull_rn(weight(v) * kWeightOne);
  }
  // visit(logit, position) for every logit of the block's part above -inf.
  template <class F>
  __device__ __forceinline__ void each(F&& visit) const {
    for (uint32_t u = first + threadIdx.x; u < last; u += kRowThreads) {
      float f[kUnit];
      walk.load(u, f);
#pragma unroll
      for (uint32_t i = 0; i < kUnit; ++i)
        if (f[i] > -INFINITY) visit(f[i], u * kUnit + i);
    }
  }
};

// Sum over the cluster; every thread of it gets it.
template <class T>
__device__ unsigned long long cluster_sum(unsigned long long v, SampleShared& s, const SampleRow<T>&) {
  cg::cluster_group cluster = cg::this_cluster();
  v = block_sum(v, s.sum_scratch);
  if (threadIdx.x == 0) s.mine.mass = v;
  cluster.sync();
  unsigned long long t = 0;
  for (uint32_t b = 0; b < cluster.num_blocks(); ++b) t += cluster.map_shared_rank(&s, b)->mine.mass;
  cluster.sync();
  return t;
}

// One counting pass: digit(logit) in [0, kBins) for those that take part, or -1; in every bin how many they are and, where
// `weigh`, their weight. Finds the lowest digit at which the running total (of counts, or of weights where
// `weigh`) reaches `target`: s.found_*. The last bin, which may take most of a row, is counted in registers.
template <class T, class D>
__device__ void find_bin(SampleShared& s, const SampleRow<T>& row, bool weigh, unsigned long long target, D&& digit) {
  cg::cluster_group cluster = cg::this_cluster();
  for (uint32_t i = threadIdx.x; i < kBins; i += kRowThreads) {
    s.bins.count[i] = 0;
    s.bins.mass[i] = 0;
  }
  __syncthreads();
  uint32_t tail_count = 0;
  unsigned long long tail_mass = 0;
  row.each([&](float v, uint32_t) {
    const int d = digit(v);
    if (d < 0) return;
    const unsigned long long w = weigh ? row.fixed(v) : 0;
    if (d == (int)kBins - 1) {
      ++tail_count;
      tail_mass += w;
    } else {
      atomicAdd(&s.bins.count[d], 1u);
      if (w) atomicAdd(&s.bins.mass[d], w);
    }
  });
  tail_count = (uint32_t)block_sum((unsigned long long)tail_count, s.sum_scratch);
  tail_mass = block_sum(tail_mass, s.sum_scratch);
  if (threadIdx.x == 0) {
    s.bins.count[kBins - 1] = tail_count;
    s.bins.mass[kBins - 1] = tail_mass;
  }
  cluster.sync();
  // Thread i takes bins 4i .. 4i + 3 of all blocks.
  constexpr uint32_t kMine = kBins / kRowThreads;
  uint32_t count[kMine];
  unsigned long long mass[kMine], sum = 0;
#pragma unroll
  for (uint32_t j = 0; j < kMine; ++j) {
    count[j] = 0;
    mass[j] = 0;
    for (uint32_t b = 0; b < cluster.num_blocks(); ++b) {
      const SampleShared* o = cluster.map_shared_rank(&s, b);
      count[j] += o->bins.count[threadIdx.x * kMine + j];
      mass[j] += o->bins.mass[threadIdx.x * kMine + j];
    }
    sum += weigh ? mass[j] : count[j];
  }
  // Sum of the bins before this thread's.
  unsigned long long incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if ((threadIdx.x & 31u) >= (uint32_t)o) incl += up;
  }
  __syncthreads();
  if ((threadIdx.x & 31u) == 31u) s.sum_scratch[threadIdx.x >> 5] = incl;
  __syncthreads();
  unsigned long long before = incl - sum;
  for (uint32_t w = 0; w < (threadIdx.x >> 5); ++w) before += s.sum_scratch[w];
#pragma unroll
  for (uint32_t j = 0; j < kMine; ++j) {
    const unsigned long long in = weigh ? mass[j] : count[j];
    if (before < target && before + in >= target) {
      s.found_bin = threadIdx.x * kMine + j;
      s.found_before = before;
      s.found_count = count[j];
    }
    before += in;
  }
  cluster.sync();  // found_* is there, and no block reads these bins any more
}

// The logit at which the total over the row in descending order reaches `target` (1 <= target <= the
// total), among logits above `floor`: *edge, and in *ties how many of the tokens with this very logit it
// takes.
template <class T>
__device__ void find_edge(SampleShared& s, const SampleRow<T>& row, bool weigh, unsigned long long target, float floor, float* edge,
                          uint32_t* ties) {
  cg::cluster_group cluster = cg::this_cluster();
  // First by distance from the maximum, 1/64 of a temperature a bin and one for all that is 16 below.
  const float scale = fminf((float)(64.0 * row.inv_t), 3e38f);
  auto coarse = [&](float v) { return v == row.m ? 0 : (int)fminf((row.m - v) * scale, (float)(kBins - 1)); };
  find_bin(s, row, weigh, target, [&](float v) { return v > floor ? coarse(v) : -1; });
  const int bin = (int)s.found_bin;
  target -= s.found_before;
  uint32_t at = s.found_count;
  // Then by the order keys of the bin's logits, from the first bit in which they differ.
  uint32_t lo = 0xFFFFFFFFu, hi = 0;
  row.each([&](float v, uint32_t) {
    if (v > floor && coarse(v) == bin) {
      const uint32_t k = order_key(v);
      lo = min(lo, k);
      hi = max(hi, k);
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
  for (uint32_t b = 0; b < cluster.num_blocks(); ++b) {
    lo = min(lo, cluster.map_shared_rank(&s, b)->key_lo);
    hi = max(hi, cluster.map_shared_rank(&s, b)->key_hi);
  }
  cluster.sync();
  int left = lo == hi ? 0 : 32 - __clz(lo ^ hi);  // low bits still open
  uint32_t prefix = left == 32 ? 0 : hi >> left;  // those above
  while (left > 0) {
    const int step = min(left, 8);
    const int shift = left - step;
    // The largest digit first: digits are counted from the top.
    find_bin(s, row, weigh, target, [&](float v) {
      if (!(v > floor) || coarse(v) != bin) return -1;
      const uint32_t k = order_key(v);
      if (left < 32 && (k >> left) != prefix) return -1;
      return (int)((1u << step) - 1u - ((k >> shift) & ((1u << step) - 1u)));
    });
    target -= s.found_before;
    at = s.found_count;
    prefix = (left == 32 ? 0u : prefix << step) | ((1u << step) - 1u - s.found_bin);
    left = shift;
    __syncthreads();  // found_* is read
  }
  *edge = key_value(lo == hi ? lo : prefix);
  const unsigned long long one = row.fixed(*edge);
  *ties = weigh ? (uint32_t)min((unsigned long long)at, (target + one - 1) / max(one, 1ull)) : (uint32_t)target;
}

template <class T>
__global__ void __launch_bounds__(kRowThreads)
    sample_kernel(RowSet x, const float* __restrict__ uniform, ws_sampling sampling, int64_t* __restrict__ tokens,
                  float* __restrict__ logprobs) {
  __shared__ SampleShared s;
  const cg::cluster_group cluster = cg::this_cluster();
  const uint32_t blocks = cluster.num_blocks(), rank = cluster.block_rank(), r = blockIdx.x / blocks;
  float t = sampling.temperature_each ? sampling.temperature_each[r] : sampling.temperature;
  const float top_p = sampling.top_p_each ? sampling.top_p_each[r] : sampling.top_p;
  const float min_p = fminf(sampling.min_p_each ? sampling.min_p_each[r] : sampling.min_p, 1.f);
  int64_t top_k = top_k_of(sampling, r);
  if (rank == 0 && threadIdx.x == 0) tokens[r] = -1;  // the token's block writes it behind a cluster barrier
  if (!(t > 0.f)) {
    t = 1.f;
    top_k = 1;
  }
  if (!(top_p > 0.f)) top_k = 1;
  const float c = fminf(kLog2e / t, 3e38f);
  const RowWalk<T> walk(row_ptr<T>(x, r), x.vocab);
  const uint32_t chunks = (walk.units + kChunkUnits - 1) / kChunkUnits;
  const uint32_t each = (chunks + blocks - 1) / blocks;
  const uint32_t chunk0 = min(rank * each, chunks), chunk1 = min(chunk0 + each, chunks);
  SampleRow<T> row{walk, min(chunk0 * kChunkUnits, walk.units), min(chunk1 * kChunkUnits, walk.units), 0.f, 1.0 / (double)t};
  const Soft soft = cluster_soft(row_soft(walk, row.first, row.last, c, s.soft_scratch), c, &s.soft_mine);
  row.m = soft.m;
  if (soft.m == -INFINITY) {  // the same for the whole cluster
    if (rank == 0 && threadIdx.x == 0 && logprobs) logprobs[r] = isnan(soft.s) ? NAN : -INFINITY;
    if (blocks > 1) cluster.sync();
    return;
  }

  // The prefix of the order that is kept: all above `edge`, and `ties` of those equal to it.
  float edge = -INFINITY;
  uint32_t ties = 0;
  if (top_k == 1) {
    edge = soft.m;
    ties = 1;
  } else if (top_k > 1 && top_k < (int64_t)x.vocab) {
    unsigned long long there = 0;
    row.each([&](float, uint32_t) { ++there; });
    if (cluster_sum(there, s, row) > (unsigned long long)top_k)
      find_edge(s, row, false, (unsigned long long)top_k, -INFINITY, &edge, &ties);
  }
  if (top_p < 1.f && !(edge == soft.m && ties == 1)) {
    unsigned long long above = 0;
    row.each([&](float v, uint32_t) { above += v > edge ? row.fixed(v) : 0; });
    above = cluster_sum(above, s, row);
    const unsigned long long one = edge > -INFINITY ? row.fixed(edge) : 0;
    const unsigned long long total = above + one * ties;
    unsigned long long target = (unsigned long long)ceil((double)top_p * (double)total);
    target = min(max(target, 1ull), total);
    if (target > above)
      ties = min(ties, (uint32_t)((target - above + one - 1) / max(one, 1ull)));
    else
      find_edge(s, row, true, target, edge, &edge, &ties);
  }

  // Weights of the tokens kept, in id order: by chunks, then within the chunk that holds the token.
  // A uniform number of 0 takes the first token of any weight, below 2^-43, too.
  const double u = (double)uniform[r];
  const bool first = !(u > 0.0);
  auto kept = [&](float v) -> unsigned long long {
    if (min_p > 0.f && !(row.weight(v) >= (double)min_p)) return 0;
    const unsigned long long w = row.fixed(v);
    return first && w == 0 && row.weight(v) > 0.0 ? 1 : w;
  };
  const unsigned long long one = edge > -INFINITY ? kept(edge) : 0;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  unsigned long long mass = 0;
  uint32_t tied = 0;
  __syncthreads();
  for (uint32_t ch = chunk0 + warp; ch < chunk1; ch += kRowWarps) {
    unsigned long long w = 0;
    uint32_t e = 0;
    for (uint32_t u = ch * kChunkUnits + lane; u < min((ch + 1) * kChunkUnits, walk.units); u += 32) {
      float f[kUnit];
      walk.load(u, f);
#pragma unroll
      for (uint32_t i = 0; i < kUnit; ++i) {
        if (f[i] > edge) w += kept(f[i]);
        e += f[i] == edge && edge > -INFINITY;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xFFFFFFFFu, w, o);
    e = __reduce_add_sync(0xFFFFFFFFu, e);
    if (lane == 0) {
      s.chunks.mass[ch - chunk0] = w;
      s.chunks.ties[ch - chunk0] = e;
    }
    mass += w;
    tied += e;
  }
  mass = block_sum(lane == 0 ? mass : 0ull, s.sum_scratch);
  tied = (uint32_t)block_sum(lane == 0 ? (unsigned long long)tied : 0ull, s.sum_scratch);
  if (threadIdx.x == 0) {
    s.mine.mass = mass;
    s.mine.ties = tied;
  }
  cluster.sync();
  unsigned long long before = 0, total = 0, mine = 0;
  uint32_t ties_before = 0, seen = 0;
  for (uint32_t b = 0; b < blocks; ++b) {
    const SampleShared* o = cluster.map_shared_rank(&s, b);
    const uint32_t next = seen + o->mine.ties;
    const unsigned long long w = o->mine.mass + one * (min(next, ties) - min(seen, ties));
    if (b == rank) {
      before = total;
      ties_before = seen;
      mine = w;
    }
    total += w;
    seen = next;
  }
  unsigned long long need = !first ? (unsigned long long)fmin(u * (double)total, 9e18) + 1 : 1;
  need = min(need, total);
  if (before < need && need <= before + mine && warp == 0) {
    // 32 chunks at a time.
    uint32_t ch = chunk0;
    unsigned long long base = before;
    uint32_t tie_base = ties_before;
    for (; ch < chunk1; ch += 32) {
      const uint32_t q = ch + lane;
      const uint32_t e = q < chunk1 ? s.chunks.ties[q - chunk0] : 0;
      uint32_t e_incl = e;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, e_incl, o);
        if (lane >= (uint32_t)o) e_incl += up;
      }
      const uint32_t e0 = tie_base + e_incl - e, e1 = tie_base + e_incl;
      unsigned long long w = (q < chunk1 ? s.chunks.mass[q - chunk0] : 0ull) + one * (min(e1, ties) - min(e0, ties));
      const unsigned long long own = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long up = __shfl_up_sync(0xFFFFFFFFu, w, o);
        if (lane >= (uint32_t)o) w += up;
      }
      const uint32_t hit = __ballot_sync(0xFFFFFFFFu, base + w >= need);
      if (hit) {
        const int l = __ffs(hit) - 1;
        base += __shfl_sync(0xFFFFFFFFu, w - own, l);
        tie_base = __shfl_sync(0xFFFFFFFFu, e0, l);
        ch += l;
        break;
      }
      base += __shfl_sync(0xFFFFFFFFu, w, 31);
      tie_base += __shfl_sync(0xFFFFFFFFu, e_incl, 31);
    }
    for (uint32_t p0 = ch * kChunk; p0 < min((ch + 1) * kChunk, walk.end); p0 += 32) {
      const uint32_t p = p0 + lane;
      const float v = p >= walk.head && p < walk.end ? walk.at(p) : -INFINITY;
      const uint32_t equal = __ballot_sync(0xFFFFFFFFu, v == edge && edge > -INFINITY);
      const uint32_t nth = tie_base + __popc(equal & ((1u << lane) - 1u));
      unsigned long long w = 0;
      if (v > edge) w = kept(v);
      if (v == edge && edge > -INFINITY && nth < ties) w = one;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long up = __shfl_up_sync(0xFFFFFFFFu, w, o);
        if (lane >= (uint32_t)o) w += up;
      }
      const uint32_t hit = __ballot_sync(0xFFFFFFFFu, base + w >= need);
      if (hit) {
        if (lane == (uint32_t)(__ffs(hit) - 1)) {
          tokens[r] = (int64_t)(p - walk.head);
          if (logprobs) logprobs[r] = (float)(((double)v - (double)soft.m) * row.inv_t - log((double)soft.s));
        }
        break;
      }
      base += __shfl_sync(0xFFFFFFFFu, w, 31);
      tie_base += __popc(equal);
    }
  }
  if (blocks > 1) cluster.sync();  // the blocks' shared memory is read until here
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
        return launch_rows(top_kernel<T>, x.rows, blocks_a_row(x.rows, x.set.vocab / kUnit), stream, x.set, k, kLog2e / temperature, 1.f / temperature, ids,
                           logprobs);
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
        return launch_rows(sample_kernel<T>, x.rows, blocks_a_row(x.rows, x.set.vocab / kUnit), stream, x.set, uniform, *sampling, tokens, logprobs);
      });
    return done(e, "sample");
  });
}
