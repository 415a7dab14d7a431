// Rows of logits on the device: addressing, guarded loads, and the online
// softmax statistics that the row operators (ws_logits.cu, ws_distill.cu) share.
//
// A row has V contiguous elements. It is walked in "aligned positions": position
// p = 0 is the last 16-byte boundary at or before the row, so element i sits at
// p = i + head, with head < 8 elements, and every unit of 8 positions is one
// (16-bit types) or two (fp32) aligned 16-byte loads whatever the row's own
// alignment. The units that reach over either end of the row are loaded element by
// element; nothing outside the row is read.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/warpshift_b200.h"

namespace ws {

constexpr uint32_t kRowThreads = 256;
constexpr uint32_t kRowWarps = kRowThreads / 32;
constexpr uint32_t kUnit = 8;  // elements of one load step of a thread
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

// Eight consecutive elements as they lie in memory: one 16-byte word for the
// 16-bit types, two for fp32.
template <class T>
struct Raw {
  uint4 v[sizeof(T) / 2];
};

template <class T>
__device__ __forceinline__ void unpack(const Raw<T>& r, float (&f)[kUnit]);
template <>
__device__ __forceinline__ void unpack<__nv_bfloat16>(const Raw<__nv_bfloat16>& r, float (&f)[kUnit]) {
  const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
template <>
__device__ __forceinline__ void unpack<__half>(const Raw<__half>& r, float (&f)[kUnit]) {
  const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
template <>
__device__ __forceinline__ void unpack<float>(const Raw<float>& r, float (&f)[kUnit]) {
  const uint32_t w[8] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w, r.v[1].x, r.v[1].y, r.v[1].z, r.v[1].w};
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
}

template <class T>
__device__ __forceinline__ Raw<T> pack(const float (&f)[kUnit]);
template <>
__device__ __forceinline__ Raw<__nv_bfloat16> pack<__nv_bfloat16>(const float (&f)[kUnit]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&p);
  }
  return {{make_uint4(w[0], w[1], w[2], w[3])}};
}
template <>
__device__ __forceinline__ Raw<__half> pack<__half>(const float (&f)[kUnit]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&p);
  }
  return {{make_uint4(w[0], w[1], w[2], w[3])}};
}
template <>
__device__ __forceinline__ Raw<float> pack<float>(const float (&f)[kUnit]) {
  Raw<float> r;
  r.v[0] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  r.v[1] = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
  return r;
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
    units = (end + kUnit - 1) / kUnit;
  }
  // Whether all eight positions of unit u belong to the row.
  __device__ __forceinline__ bool whole(uint32_t u) const { return u * kUnit >= head && (u + 1) * kUnit <= end; }
  __device__ __forceinline__ float at(uint32_t p) const { return to_float(aligned[p]); }
  // Unit u; positions outside the row read as -inf.
  __device__ __forceinline__ void load(uint32_t u, float (&f)[kUnit]) const {
    if (whole(u)) {
      Raw<T> r;
      const uint4* v = reinterpret_cast<const uint4*>(aligned + (size_t)u * kUnit);
#pragma unroll
      for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.v[i] = __ldg(v + i);
      unpack<T>(r, f);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < kUnit; ++i) {
        const uint32_t p = u * kUnit + i;
        f[i] = (p >= head && p < end) ? at(p) : -INFINITY;
      }
    }
  }
};

// 16 bytes that are read once: not kept in L1.
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// -inf in every element of a word.
template <class T>
constexpr uint32_t kNegInf = 0xFF800000u;
template <>
constexpr uint32_t kNegInf<__nv_bfloat16> = 0xFF80FF80u;
template <>
constexpr uint32_t kNegInf<__half> = 0xFC00FC00u;

// What a block reads of a row in one step: kBatch units from each thread, thread t's j-th one at
// u0 + j * kRowThreads + t. 64 bytes a thread in flight for either element size.
template <class T>
struct Batch {
  static constexpr uint32_t kUnits = 8 / sizeof(T);
  static constexpr uint32_t kSpan = kUnits * kRowThreads;  // units of the block's step
  Raw<T> raw[kUnits];

  // Units [u0, u0 + kSpan) up to `last`; what lies outside is -inf.
  __device__ __forceinline__ void load(const RowWalk<T>& walk, uint32_t u0, uint32_t last) {
    if (u0 * kUnit >= walk.head && u0 + kSpan <= last && (u0 + kSpan) * kUnit <= walk.end) {
      const T* p = walk.aligned + (size_t)(u0 + threadIdx.x) * kUnit;
#pragma unroll
      for (uint32_t j = 0; j < kUnits; ++j)
#pragma unroll
        for (uint32_t i = 0; i < sizeof(T) / 2; ++i) raw[j].v[i] = load16(p + j * kRowThreads * kUnit + i * (16 / sizeof(T)));
      return;
    }
#pragma unroll
    for (uint32_t j = 0; j < kUnits; ++j) {
      const uint32_t u = u0 + j * kRowThreads + threadIdx.x;
      if (u < last && walk.whole(u)) {
#pragma unroll
        for (uint32_t i = 0; i < sizeof(T) / 2; ++i)
          raw[j].v[i] = load16(walk.aligned + (size_t)u * kUnit + i * (16 / sizeof(T)));
      } else {
        float f[kUnit];
#pragma unroll
        for (uint32_t i = 0; i < kUnit; ++i) {
          const uint32_t p = u * kUnit + i;
          f[i] = u < last && p >= walk.head && p < walk.end ? walk.at(p) : -INFINITY;
        }
        raw[j] = pack<T>(f);
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (uint32_t j = 0; j < kUnits; ++j)
#pragma unroll
      for (uint32_t i = 0; i < sizeof(T) / 2; ++i) raw[j].v[i] = make_uint4(kNegInf<T>, kNegInf<T>, kNegInf<T>, kNegInf<T>);
  }
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
    const float base = m == -INFINITY ? 0.f : m;
    const uint64_t nb = pair(-base, -base), cc = pair(c, c);
    uint64_t sum = 0;
#pragma unroll
    for (uint32_t j = 0; j < Batch<T>::kUnits; ++j) {
      float f[kUnit];
      unpack<T>(b.raw[j], f);
#pragma unroll
      for (uint32_t i = 0; i < kUnit; i += 2) {
        const float2 e = unpair(mul2(add2(pair(f[i], f[i + 1]), nb), cc));
        sum = add2(sum, pair(ex2(e.x), ex2(e.y)));
      }
    }
    const float2 t = unpair(sum);
    s += t.x + t.y;
  }
  __device__ __forceinline__ void merge(float m2, float s2, float c) {
    const float top = fmaxf(m, m2);
    s = s * (m == top ? 1.f : ex2((m - top) * c)) + s2 * (m2 == top ? 1.f : ex2((m2 - top) * c));
    m = top;
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

// The block's statistics from its threads', in a fixed order; every thread gets them.
__device__ __forceinline__ Soft block_soft(Soft t, float c, float2* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xFFFFFFFFu, t.m, o), s2 = __shfl_xor_sync(0xFFFFFFFFu, t.s, o);
    t.merge(m2, s2, c);
  }
  __syncthreads();
  if ((threadIdx.x & 31u) == 0) scratch[threadIdx.x >> 5] = make_float2(t.m, t.s);
  __syncthreads();
  Soft r;
  r.m = scratch[0].x;
  r.s = scratch[0].y;
#pragma unroll
  for (uint32_t w = 1; w < kRowWarps; ++w) r.merge(scratch[w].x, scratch[w].y, c);
  return r;
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

// The row's statistics from those of the cluster's blocks, which all get them. `mine`
// is the block's slot, which no block writes again before the next cluster barrier.
__device__ __forceinline__ Soft cluster_soft(const Soft& block, float c, float2* mine) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  if (cluster.num_blocks() == 1) return block;
  if (threadIdx.x == 0) *mine = make_float2(block.m, block.s);
  cluster.sync();
  Soft r;
  for (uint32_t b = 0; b < cluster.num_blocks(); ++b) {
    const float2 v = *cluster.map_shared_rank(mine, b);
    if (b == 0) {
      r.m = v.x;
      r.s = v.y;
    } else {
      r.merge(v.x, v.y, c);
    }
  }
  return r;
}

template <class T>
__device__ __forceinline__ float unit_max(const Raw<T>& r) {
  float f[kUnit];
  unpack<T>(r, f);
  return fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
}

// Statistics of units [first, last) of a row, for the whole block. The loads of a step are in flight while
// the step before is summed up.
template <class T>
__device__ __forceinline__ Soft row_soft(const RowWalk<T>& walk, uint32_t first, uint32_t last, float c, float2* scratch) {
  Soft soft;
  Batch<T> next;
  if (first < last) next.load(walk, first, last);
  for (uint32_t u = first; u < last; u += Batch<T>::kSpan) {
    const Batch<T> now = next;
    if (u + Batch<T>::kSpan < last) next.load(walk, u + Batch<T>::kSpan, last);
    float top = unit_max<T>(now.raw[0]);
#pragma unroll
    for (uint32_t j = 1; j < Batch<T>::kUnits; ++j) top = fmaxf(top, unit_max<T>(now.raw[j]));
    soft.add(now, top, c);
  }
  return block_soft(soft, c, scratch);
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

// How many blocks (a cluster: 1, 2, 4 or 8) share each of `rows` rows of `units` units.
inline uint32_t blocks_a_row(uint32_t rows, uint32_t units) {
  uint32_t c = 1;
  while (c < 8 && (uint64_t)rows * c * 2 <= 592 && units / c >= 512) c *= 2;
  return c;
}

// Launches `rows` clusters of `cluster` blocks of kRowThreads threads.
template <class... P, class... A>
cudaError_t launch_rows(void (*kernel)(P...), uint32_t rows, uint32_t cluster, void* stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * cluster);
  cfg.blockDim = dim3(kRowThreads);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

}  // namespace ws
