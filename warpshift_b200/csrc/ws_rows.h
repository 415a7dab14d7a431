// Rows of logits on the device: addressing, guarded loads, and the online
// softmax statistics that the row operators (ws_logits.cu, ws_distill.cu) share.
//
// A row has V contiguous elements. It is walked in "aligned positions": position
// p = 0 is the last 16-byte boundary at or before the row, so element i sits at
// p = i + head, and every unit of 16 bytes (8 or 4 positions) is one aligned load
// whatever the row's own alignment. The units that reach over either end of the row
// are loaded element by element; nothing outside the row is read.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "../../include/warpshift_b200.h"

namespace ws {

constexpr uint32_t kRowThreads = 256;
constexpr uint32_t kRowWarps = kRowThreads / 32;
template <class T>
constexpr uint32_t kUnit = 16 / sizeof(T);  // elements of a 16-byte unit
constexpr float kLog2e = 1.4426950408889634f;

// Device copy of ws_rows (strides in elements).
struct RowSet {
  char* data;
  int64_t stride_outer, stride_inner;
  uint32_t inner, vocab;
};

template <class T>
__device__ __forceinline__ T* row_ptr(const RowSet& r, uint32_t row) {
  const uint32_t o = row / r.inner, i = row - o * r.inner;
  return reinterpret_cast<T*>(r.data) + (int64_t)o * r.stride_outer + (int64_t)i * r.stride_inner;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }

// A unit's elements, as they lie in memory, as fp32; and back, rounded.
template <class T>
__device__ __forceinline__ void unpack(const uint4& r, float (&f)[kUnit<T>]);
template <>
__device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4& r, float (&f)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
template <>
__device__ __forceinline__ void unpack<__half>(const uint4& r, float (&f)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
template <>
__device__ __forceinline__ void unpack<float>(const uint4& r, float (&f)[4]) {
  f[0] = __uint_as_float(r.x);
  f[1] = __uint_as_float(r.y);
  f[2] = __uint_as_float(r.z);
  f[3] = __uint_as_float(r.w);
}

template <class T>
__device__ __forceinline__ uint4 pack(const float (&f)[kUnit<T>]);
template <>
__device__ __forceinline__ uint4 pack<__nv_bfloat16>(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&p);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ uint4 pack<__half>(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&p);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ uint4 pack<float>(const float (&f)[4]) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}

// One row as a CTA walks it. first/last: its units [first, last) of the row's
// `units`; the CTAs of a cluster split a row in order, in whole chunks.
template <class T>
struct RowWalk {
  const T* aligned;  // position 0; only positions [head, end) belong to the row
  uint32_t head, end, units;

  __device__ __forceinline__ RowWalk(const T* row, uint32_t vocab) {
    head = (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T);
    aligned = row - head;
    end = head + vocab;
    units = (end + kUnit<T> - 1) / kUnit<T>;
  }
  // Whether all positions of unit u belong to the row.
  __device__ __forceinline__ bool whole(uint32_t u) const { return u * kUnit<T> >= head && (u + 1) * kUnit<T> <= end; }
  __device__ __forceinline__ float at(uint32_t p) const { return to_float(aligned[p]); }
  // Unit u; positions outside the row read as -inf.
  __device__ __forceinline__ void load(uint32_t u, float (&f)[kUnit<T>]) const {
    if (whole(u)) {
      unpack<T>(__ldg(reinterpret_cast<const uint4*>(aligned) + u), f);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < kUnit<T>; ++i) {
        const uint32_t p = u * kUnit<T> + i;
        f[i] = (p >= head && p < end) ? at(p) : -INFINITY;
      }
    }
  }
};

// What a thread takes of a row in one step: kUnits units.
template <class T>
struct Batch {
  static constexpr uint32_t kUnits = 4;
  static constexpr uint32_t kWarpSpan = kUnits * 32;          // units of a warp's step, contiguous
  static constexpr uint32_t kSpan = kUnits * kRowThreads;     // units of the block's step
  uint4 raw[kUnits];

  // The thread's j-th unit in the block's step that begins at unit u0.
  static __device__ __forceinline__ uint32_t unit(uint32_t u0, uint32_t j) {
    return u0 + (threadIdx.x >> 5) * kWarpSpan + j * 32 + (threadIdx.x & 31u);
  }
};

// The way of a row's units through shared memory: kDepth steps of asynchronous 16-byte copies in flight. Every
// thread copies and reads units of its own, so that nothing waits for another
// thread. Bytes in flight are what a block that shares its SM with two or three others needs to
// keep HBM busy (about 44 bytes a ns for an SM, for about a microsecond), without
// registers to hold them.
constexpr uint32_t kStepBytes = 64 * kRowThreads;

// A unit that may not be wholly the row's, element by element where it is not (u = ~0: nothing of it is). Out of line: few units need it.
template <class T>
__device__ __noinline__ uint4 load_edge(const RowWalk<T> walk, uint32_t u) {
  float f[kUnit<T>];
  if (u == ~0u) {
#pragma unroll
    for (uint32_t i = 0; i < kUnit<T>; ++i) f[i] = -INFINITY;
  } else {
    walk.load(u, f);
  }
  return pack<T>(f);
}

template <class T, uint32_t kDepth>
class Ring {
 public:
  using B = Batch<T>;

  // `memory`: kDepth * kStepBytes, 16-byte aligned. Units [first, last) are read.
  __device__ __forceinline__ Ring(void* memory, const RowWalk<T>& walk, uint32_t first, uint32_t last)
      : walk_(walk), last_(last), ahead_(first), slot_(0) {
    mine_ = (uint32_t)__cvta_generic_to_shared(memory) + threadIdx.x * 16;
    source_ = reinterpret_cast<const uint4*>(walk.aligned) + B::unit(first, 0);
    // Steps that begin from inside_from_ to inside_to_ are wholly the row's and the range's.
    inside_from_ = walk.head ? 1 : 0;
    const uint32_t whole = min(last, walk.end / kUnit<T>);
    inside_to_ = whole >= B::kSpan ? whole - B::kSpan : 0;
    if (whole < B::kSpan) inside_from_ = ~0u;
#pragma unroll 1
    for (uint32_t d = 0; d < kDepth; ++d) fill(d);
  }
  // Every copy has landed; the memory may be used for something else behind a barrier.
  static __device__ __forceinline__ void drain() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

  // The next step's units, those outside the row or the range as -inf.
  __device__ __forceinline__ void read(B& b) const {
    asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
    fetch(slot_, b);
  }
  // Step `slot` of the first kDepth, which stays where it is as long as no later step is copied over it.
  __device__ __forceinline__ void again(uint32_t slot, B& b) const { fetch(slot, b); }
  // Whether all units of the block's step that begins at unit u0 are wholly the row's.
  __device__ __forceinline__ bool inside(uint32_t u0) const { return u0 >= inside_from_ && u0 <= inside_to_; }
  // To the step after it; to be called when what read() gave has been used.
  __device__ __forceinline__ void advance() {
    fill(slot_);
    slot_ = slot_ + 1 == kDepth ? 0 : slot_ + 1;
  }

 private:
  __device__ __forceinline__ uint32_t at(uint32_t slot, uint32_t j) const { return mine_ + slot * kStepBytes + j * (kRowThreads * 16); }
  __device__ __forceinline__ void fetch(uint32_t slot, B& b) const {
#pragma unroll
    for (uint32_t j = 0; j < B::kUnits; ++j) {
      uint4& v = b.raw[j];
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at(slot, j)) : "memory");
    }
  }
  __device__ __forceinline__ void fill(uint32_t slot) {
    if (ahead_ < last_) {
      if (inside(ahead_)) {
#pragma unroll
        for (uint32_t j = 0; j < B::kUnits; ++j)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at(slot, j)), "l"(source_ + j * 32) : "memory");
      } else {
#pragma unroll 1
        for (uint32_t j = 0; j < B::kUnits; ++j) {
          const uint32_t u = B::unit(ahead_, j);
          if (u < last_ && walk_.whole(u)) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at(slot, j)), "l"(source_ + j * 32) : "memory");
            continue;
          }
          const uint4 r = load_edge(walk_, u < last_ ? u : ~0u);
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at(slot, j)), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w) : "memory");
        }
      }
    }
    ahead_ += B::kSpan;
    source_ += B::kSpan;
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  const RowWalk<T>& walk_;
  const uint4* source_;
  uint32_t last_, ahead_, slot_, mine_, inside_from_, inside_to_;
};

// Pairs of fp32 in one instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}

__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}

// Floats as integers of the same order (-0 is taken as +0 first, so that equal
// logits have equal keys).
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// 2^((x - m) c) takes one multiply-add before the exponential as 2^(x c - r), r = m c rounded, times 2^(r - m c), which is a constant near 1
// that one more multiply-add gives exactly. x c - r is rounded once, so nothing is lost against (x - m) c; but r - m c has to be
// small: with |m| c below kOneStep it is at most 64. Beyond (masks of the type's lowest value, temperatures next to 0) the difference
// comes first.
constexpr float kOneStep = 1e9f;
__device__ __forceinline__ bool one_step(float m, float c) { return fabsf(m) * c < kOneStep; }
__device__ __forceinline__ float one_step_rest(float m, float c, float r) { return ex2(-fmaf(m, c, -r)); }

// Sum of 2^((x - m) c) over a thread's units of a step (m = -inf: all of them are -inf, and the sum is 0).
template <class T>
__device__ __forceinline__ float step_sum(const Batch<T>& b, float m, float c) {
  const float base = m == -INFINITY ? 0.f : m;
  const uint64_t cc = pair(c, c);
  uint64_t sum = 0;
  float scale = 1.f;
  if (one_step(base, c)) {
    const float r = base * c;
    const uint64_t nr = pair(-r, -r);
#pragma unroll
    for (uint32_t j = 0; j < Batch<T>::kUnits; ++j) {
      float f[kUnit<T>];
      unpack<T>(b.raw[j], f);
#pragma unroll
      for (uint32_t i = 0; i < kUnit<T>; i += 2) {
        const float2 e = unpair(fma2(pair(f[i], f[i + 1]), cc, nr));
        sum = add2(sum, pair(ex2(e.x), ex2(e.y)));
      }
    }
    scale = one_step_rest(base, c, r);
  } else {
    const uint64_t nb = pair(-base, -base);
#pragma unroll 1
    for (uint32_t j = 0; j < Batch<T>::kUnits; ++j) {
      uint4 raw = b.raw[0];
#pragma unroll
      for (uint32_t q = 1; q < Batch<T>::kUnits; ++q) raw = q == j ? b.raw[q] : raw;
      float f[kUnit<T>];
      unpack<T>(raw, f);
#pragma unroll
      for (uint32_t i = 0; i < kUnit<T>; i += 2) {
        const float2 e = unpair(mul2(add2(pair(f[i], f[i + 1]), nb), cc));
        sum = add2(sum, pair(ex2(e.x), ex2(e.y)));
      }
    }
  }
  const float2 t = unpair(sum);
  return (t.x + t.y) * scale;
}

// Running maximum m and sum s of 2^((x - m) c), c = log2(e) / temperature. The
// difference x - m is taken before the product, so logits of any size (a mask of
// the type's lowest value, say) give exponents that are exact near the maximum.
// m = -inf: nothing seen but -inf. A NaN or +inf logit makes s NaN.
struct Soft {
  float m = -INFINITY, s = 0.f;

  // One step's logits, of which `top` is the largest. They are added up among themselves first, which
  // keeps the chains of additions short.
  template <class T>
  __device__ __forceinline__ void add(const Batch<T>& b, float top, float c) {
    if (top > m) {
      s *= ex2((m - top) * c);
      m = top;
    }
    s += step_sum(b, m, c);
  }
};

// Sum over the block in a fixed order; every thread gets it. `scratch`: one slot
// for each warp.
template <class V>
__device__ __forceinline__ V block_sum(V v, V* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31u) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  V t = scratch[0];
#pragma unroll
  for (uint32_t w = 1; w < kRowWarps; ++w) t += scratch[w];
  return t;
}

// The block's statistics from its threads', in a fixed order; every thread gets them. The maximum
// first, so that a thread's sum is scaled once.
__device__ __forceinline__ Soft block_soft(Soft t, float c, float2* scratch) {
  const float top = key_value(__reduce_max_sync(0xFFFFFFFFu, order_key(t.m)));
  t.s *= t.m == top ? 1.f : ex2((t.m - top) * c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t.s += __shfl_xor_sync(0xFFFFFFFFu, t.s, o);
  __syncthreads();
  if ((threadIdx.x & 31u) == 0) scratch[threadIdx.x >> 5] = make_float2(top, t.s);
  __syncthreads();
  Soft r;
  r.m = scratch[0].x;
#pragma unroll
  for (uint32_t w = 1; w < kRowWarps; ++w) r.m = fmaxf(r.m, scratch[w].x);
#pragma unroll
  for (uint32_t w = 0; w < kRowWarps; ++w) r.s += scratch[w].y * (scratch[w].x == r.m ? 1.f : ex2((scratch[w].x - r.m) * c));
  return r;
}

// Sum over the threads before this one, in a fixed order; *total: over all.
template <class V>
__device__ __forceinline__ V block_scan(V v, V* scratch, V* total) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  V incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= (uint32_t)o) incl += up;
  }
  __syncthreads();
  if (lane == 31u) scratch[warp] = incl;
  __syncthreads();
  V before = 0, all = 0;
#pragma unroll
  for (uint32_t w = 0; w < kRowWarps; ++w) {
    if (w == warp) before = all;
    all += scratch[w];
  }
  *total = all;
  const V excl = __shfl_up_sync(0xFFFFFFFFu, incl, 1);
  return before + (lane ? excl : V(0));
}

// The largest of the block's values; every thread gets it.
__device__ __forceinline__ float block_max(float v, float* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31u) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = scratch[0];
#pragma unroll
  for (uint32_t w = 1; w < kRowWarps; ++w) t = fmaxf(t, scratch[w]);
  return t;
}

// The blocks of a cluster (1, 2, 4 or 8) share a row and tell each other what they found by storing into each
// other's shared memory, so that a block may leave as soon as it has what it needs:
//   started() at the kernel's begin; ready() before the first store into another block;
//   told() behind the stores: from then on every block's stores to this one are there.
class RowCluster {
 public:
  static constexpr uint32_t kMost = 8;

  __device__ __forceinline__ RowCluster() : blocks(cooperative_groups::this_cluster().num_blocks()), rank(cooperative_groups::this_cluster().block_rank()) {}
  __device__ __forceinline__ void started() const {
    if (blocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  }
  __device__ __forceinline__ void ready() const {
    if (blocks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  __device__ __forceinline__ void told() const {
    telling();
    heard();
  }
  // Its two halves, for work in between that touches none of what is told.
  __device__ __forceinline__ void telling() const {
    if (blocks > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  __device__ __forceinline__ void heard() const {
    if (blocks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
  }
  // `p` of this block's shared memory, in block b's.
  template <class V>
  __device__ __forceinline__ V* of(V* p, uint32_t b) const {
    return cooperative_groups::this_cluster().map_shared_rank(p, b);
  }
  __device__ __forceinline__ uint32_t row() const { return blockIdx.x / blocks; }

  const uint32_t blocks, rank;
};

// The row's statistics from those of the cluster's blocks, which all get them; between ready() and told().
__device__ __forceinline__ void tell_soft(const RowCluster& cluster, const Soft& block, float2* slots) {
  if (threadIdx.x < cluster.blocks) *cluster.of(slots + cluster.rank, threadIdx.x) = make_float2(block.m, block.s);
}
__device__ __forceinline__ Soft told_soft(const RowCluster& cluster, float c, const float2* slots) {
  Soft r;
  float2 v[RowCluster::kMost];
#pragma unroll
  for (uint32_t b = 0; b < RowCluster::kMost; ++b) {
    v[b] = b < cluster.blocks ? slots[b] : make_float2(-INFINITY, 0.f);
    r.m = fmaxf(r.m, v[b].x);
  }
#pragma unroll
  for (uint32_t b = 0; b < RowCluster::kMost; ++b) r.s += v[b].y * (v[b].x == r.m ? 1.f : ex2((v[b].x - r.m) * c));
  return r;
}

// The larger of two words' elements, a NaN giving way to a number: two elements in one instruction where they have 16 bits.
template <class T>
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t word_max<__nv_bfloat16>(uint32_t a, uint32_t b) {
  const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
template <>
__device__ __forceinline__ uint32_t word_max<__half>(uint32_t a, uint32_t b) {
  const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
template <>
__device__ __forceinline__ uint32_t word_max<float>(uint32_t a, uint32_t b) {
  return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
}
template <class T>
__device__ __forceinline__ uint32_t unit_word(const uint4& r) {
  return word_max<T>(word_max<T>(r.x, r.y), word_max<T>(r.z, r.w));
}
// The largest element of a word; -inf if there is no number.
template <class T>
__device__ __forceinline__ float word_top(uint32_t w) {
  if (sizeof(T) == 4) return fmaxf(__uint_as_float(w), -INFINITY);
  float f[kUnit<T>];
  unpack<T>(make_uint4(w, w, w, w), f);
  return fmaxf(fmaxf(f[0], f[1]), -INFINITY);
}
// The largest of a thread's logits in a step.
template <class T>
__device__ __forceinline__ float step_max(const Batch<T>& b) {
  uint32_t w = unit_word<T>(b.raw[0]);
#pragma unroll
  for (uint32_t j = 1; j < Batch<T>::kUnits; ++j) w = word_max<T>(w, unit_word<T>(b.raw[j]));
  return word_top<T>(w);
}

// A thread's statistics of the units that `ring` reads. between(): called once, behind the first step, when what was loaded before the
// ring has come in.
template <class T, uint32_t kDepth, class F>
__device__ __forceinline__ Soft read_soft(Ring<T, kDepth>& ring, uint32_t first, uint32_t last, float c, F&& between) {
  Soft soft;
  for (uint32_t u = first; u < last; u += Batch<T>::kSpan) {
    Batch<T> b;
    ring.read(b);
    soft.add(b, step_max(b), c);
    ring.advance();
    if (u == first) between();
  }
  return soft;
}

// Units of the row that block `rank` of `blocks` walks.
__device__ __forceinline__ void split_units(uint32_t units, uint32_t rank, uint32_t blocks, uint32_t& first, uint32_t& last) {
  const uint32_t each = (units + blocks - 1) / blocks;
  first = min(rank * each, units);
  last = min(first + each, units);
}

// ---------------------------------------------------------------- host side
void set_last_error(const char* msg);

struct RowArgs {
  RowSet set;
  uint32_t rows;
  int dtype;
};

// Checks `rows` (ws_last_error names `what`) and fills `out`.
int check_rows(const ws_rows* rows, const char* what, RowArgs* out);

// Makes `device` current for its lifetime.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) {
    error_ = cudaGetDevice(&previous_);
    if (error_ == cudaSuccess && previous_ != device) {
      error_ = cudaSetDevice(device);
      changed_ = error_ == cudaSuccess;
    }
  }
  ~DeviceGuard() {
    if (changed_) cudaSetDevice(previous_);
  }
  cudaError_t error() const { return error_; }

 private:
  int previous_ = 0;
  bool changed_ = false;
  cudaError_t error_ = cudaSuccess;
};

// f((T*)nullptr) for the element type.
template <class F>
cudaError_t by_type(int dtype, F&& f) {
  switch (dtype) {
    case WS_DTYPE_BF16: return f((__nv_bfloat16*)nullptr);
    case WS_DTYPE_FP16: return f((__half*)nullptr);
    default: return f((float*)nullptr);
  }
}

// How many blocks (a cluster: 1, 2, 4 or 8) share each row. Every block costs some microseconds beside its share of the row, so that
// many rows go to one block each (loss forward of 2048 x 128256 bf16: 84 us, 96 with two blocks a row); kernels that write as much as
// they read gain from smaller shares, down to `share` KiB (backward of these: 175 us with one block, 164 with four). Rows are split further
// until there are `most` blocks, down to 16 KiB a block: two for each of 148 SMs (top 64 of 64 x 128256: 14 us with four blocks a row, 18 with
// one, 21 with eight).
constexpr uint32_t kFewBlocks = 296;
inline uint32_t blocks_a_row(const RowArgs& x, uint32_t share = 0, uint32_t most = kFewBlocks) {
  const uint32_t kib = x.set.vocab / 1024 * (x.dtype == WS_DTYPE_FP32 ? 4u : 2u);
  uint32_t c = 1;
  while (c < 8 && share && kib >= 2 * c * share) c *= 2;
  while (c < 8 && (uint64_t)x.rows * c * 2 <= most && kib >= 2 * c * 16) c *= 2;
  return c;
}

// Launches `rows` clusters of `cluster` blocks of kRowThreads threads with `smem` bytes of dynamic shared memory each.
template <auto kernel, class... A>
cudaError_t launch_rows(uint32_t rows, uint32_t cluster, size_t smem, int device, void* stream, A... args) {
  // More than 48 KiB of shared memory in all has to be asked for, once for a kernel and device.
  static std::atomic<uint64_t> told{0};
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (!(told.load(std::memory_order_relaxed) & bit)) {
    cudaFuncAttributes own;
    cudaError_t e = cudaFuncGetAttributes(&own, kernel);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - (int)own.sharedSizeBytes);
    if (e != cudaSuccess) return e;
    told.fetch_or(bit);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * cluster);
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace ws
