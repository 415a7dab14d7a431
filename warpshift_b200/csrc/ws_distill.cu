// Distillation of a student from a teacher's top log-probabilities: loss and gradient.
//
// For a row x of V student logits at temperature t, with the record's probabilities
// q_j (divided by their sum where the tail is renormalised), Q = sum_j q_j,
// m = max x and S = sum_i exp((x_i - m) / t):
//   loss    = w [ sum_j q_j log q_j - sum_j q_j (x_{id_j} - m) / t + Q log S ]
//   dx_i    = g w / t [ Q exp((x_i - m) / t) / S - sum_{j: id_j = i} q_j ]
// S is summed in fp32 by threads and the record's sums in 64 bits; the gradient is
// computed in fp32 and rounded once. What a row needs is one pass over its logits for
// (m, S); the gradient is one more pass over logits and gradient. The k
// tokens of the record are a correction: the dense part of a row is written first and
// the elements named by the record again behind a block barrier, each once, by the
// first entry that names it.
//
// All three kernels are bound by HBM where rows are many. 4096 x 151936 bf16, k = 32: forward
// 187 us (6.7 TB/s), backward 370 us (6.7 TB/s, read and write). The one-launch kernel
// waits between its passes for the row's sum: 2048 x 128256 bf16 216 us, where reading and writing once
// take 160; its second pass comes from L2, or from shared memory where a block's share is 64 KiB at most.
#include <algorithm>
#include <string>

#include "ws_guard.h"
#include "ws_rows.h"

namespace ws {

int check_rows(const ws_rows* rows, const char* what, RowArgs* out) {
  auto fail = [&](const char* why) {
    set_last_error((std::string(what) + ": " + why).c_str());
    return WS_ERR_INVALID;
  };
  if (!rows) return fail("null rows");
  if (rows->dtype < WS_DTYPE_BF16 || rows->dtype > WS_DTYPE_FP32) return fail("unknown type");
  if (rows->vocab < 1 || rows->vocab > WS_MAX_VOCAB) return fail("a row has 1 to 2^20 elements");
  if (rows->rows > WS_MAX_LOGIT_ROWS) return fail("too many rows");
  if (rows->inner < 1) return fail("inner is at least 1");
  if (rows->stride_outer < 0 || rows->stride_inner < 0) return fail("negative stride");
  if (rows->rows) {
    if (!rows->data) return fail("null pointer");
    if ((uintptr_t)rows->data % (rows->dtype == WS_DTYPE_FP32 ? 4 : 2)) return fail("address is not aligned to the type");
  }
  out->set.data = (char*)rows->data;
  out->set.stride_outer = rows->stride_outer;
  out->set.stride_inner = rows->stride_inner;
  out->set.inner = (uint32_t)std::min<uint64_t>(rows->inner, WS_MAX_LOGIT_ROWS);
  out->set.vocab = (uint32_t)rows->vocab;
  out->rows = (uint32_t)rows->rows;
  out->dtype = rows->dtype;
  return WS_OK;
}

namespace {

struct Record {
  const void* ids;
  const float* logprobs;
  const float* weights;
  uint32_t k;
  int ids32, renormalize;
  float c;      // log2(e) / temperature
  float inv_t;  // 1 / temperature
};

// Steps in flight of the kernels that read a row once (2048 x 128256 bf16, forward: 90, 85 and 90 us with 2, 3 and 4).
constexpr uint32_t kDepth = 3;
constexpr uint32_t kStepDepth = 4;  // of the one that reads it twice: a block's share up to 64 KiB stays

// Every block of a row goes over the whole record: with long ones a row has fewer blocks (333 x 50001 fp32, k = 256, one and two blocks:
// backward 42 and 48 us, both in one launch 55 and 64).
constexpr uint32_t kShortRecord = 64;

// Entry `threadIdx.x` of a row's record and the logit of its token; a token id of -1 has no mass. Loaded in two parts, the second of
// which needs the first, so that a kernel can read its row in between.
struct Entry {
  int id = -1;
  float lp = -INFINITY, x = 0.f;
  int64_t raw = -1;

  __device__ __forceinline__ void load(const Record& r, uint32_t row) {
    if (threadIdx.x >= r.k) return;
    const size_t at = (size_t)row * r.k + threadIdx.x;
    raw = r.ids32 ? ((const int32_t*)r.ids)[at] : ((const int64_t*)r.ids)[at];
    lp = r.logprobs[at];
  }
  template <class T>
  __device__ __forceinline__ void look_up(const T* logits, uint32_t vocab) {
    if (raw >= 0 && raw < (int64_t)vocab && lp > -INFINITY) {
      id = (int)raw;
      x = to_float(logits[raw]);
    }
  }
};

// A record summed up in 64 bits, by warps and then by one thread. Probabilities are taken relative to
// the largest one where they are renormalised (shift = its log-probability, else 0), so that a record far out in
// the teacher's tail neither underflows nor overflows, and logits relative to the largest one of the record, so that
// nothing is lost where logits are huge (a mask of the type's lowest value).
struct RecordSums {
  double q, q_lp, q_x;  // sums of q, q lp and q (x - at), q = exp(lp - shift)
  float shift, at;

  __device__ __forceinline__ void merge(const RecordSums& o) {
    if (o.q == 0.0) return;
    if (q == 0.0) {
      *this = o;
      return;
    }
    const float s = fmaxf(shift, o.shift);
    const double mine = shift == s ? 1.0 : exp((double)shift - (double)s);
    const double his = o.shift == s ? 1.0 : exp((double)o.shift - (double)s);
    q_x = mine * q_x + his * (o.q_x + o.q * ((double)o.at - (double)at));
    q = mine * q + his * o.q;
    q_lp = mine * q_lp + his * o.q_lp;
    shift = s;
  }
};

// A row's record as the block's threads share it.
struct RecordShared {
  RecordSums part[kRowWarps];
  int ids[WS_TOP_MAX_K];
  float lps[WS_TOP_MAX_K];
};

// The thread's entry and, where asked for, the warp's part of the sums into `s`; a barrier has to follow.
__device__ __forceinline__ void put_record(const Record& r, const Entry& e, RecordShared& s, bool sums = true) {
  const uint32_t warp = threadIdx.x >> 5;
  s.ids[threadIdx.x] = e.id;
  s.lps[threadIdx.x] = e.lp;
  if (!sums) return;
  RecordSums t{0.0, 0.0, 0.0, 0.f, 0.f};
  if (warp * 32 < r.k) {
    const uint32_t none = order_key(-INFINITY);
    if (r.renormalize) {
      const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, e.id >= 0 ? order_key(e.lp) : none);
      t.shift = top == none ? 0.f : key_value(top);
    }
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, e.id >= 0 && e.x > -INFINITY ? order_key(e.x) : none);
    t.at = top == none ? 0.f : key_value(top);
    t.q = e.id >= 0 ? exp((double)e.lp - (double)t.shift) : 0.0;
    if (t.q != 0.0) {
      t.q_lp = t.q * (double)e.lp;
      t.q_x = t.q * ((double)e.x - (double)t.at);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      t.q += __shfl_xor_sync(0xFFFFFFFFu, t.q, o);
      t.q_lp += __shfl_xor_sync(0xFFFFFFFFu, t.q_lp, o);
      t.q_x += __shfl_xor_sync(0xFFFFFFFFu, t.q_x, o);
    }
  }
  if ((threadIdx.x & 31u) == 0) s.part[warp] = t;
}

__device__ __forceinline__ RecordSums record_sums(const Record& r, const RecordShared& s) {
  RecordSums t = s.part[0];
  for (uint32_t w = 1; w * 32 < r.k; ++w) t.merge(s.part[w]);
  return t;
}

// The first entry that names a token writes its gradient: for that thread, the sum of exp(lp - its own lp) over all entries that name it;
// 0 for the others and for tokens outside units [first, last).
template <class T>
__device__ __forceinline__ float record_share(const Record& r, const Entry& e, const RecordShared& s, const RowWalk<T>& walk, uint32_t first,
                                              uint32_t last) {
  const uint32_t p = (uint32_t)e.id + walk.head;
  if (e.id < 0 || p < first * kUnit<T> || p >= last * kUnit<T>) return 0.f;
  float share = 0.f;
  bool owner = true;
#pragma unroll 4
  for (uint32_t j = 0; j < r.k; ++j) {
    if (s.ids[j] == e.id) {
      owner = owner && j >= threadIdx.x;
      share += j == threadIdx.x ? 1.f : expf(s.lps[j] - e.lp);
    }
  }
  return owner ? share : 0.f;
}

// What the gradient of a row needs: dense * 2^((x_i - m) c) for every token, and record * exp(lp - shift) less for those on record. dense = 0: the
// row has no gradient, and its logits are not read for it.
struct RowGrad {
  float m = 0.f, dense = 0.f, record = 0.f, shift = 0.f;
};

__device__ __forceinline__ RowGrad row_grad(const Record& r, const RecordSums& t, const Soft& soft, float factor) {
  RowGrad g;
  if (t.q == 0.0 || soft.m == -INFINITY) return g;
  g.m = soft.m;
  g.shift = t.shift;
  g.dense = factor * (r.renormalize ? 1.f / soft.s : (float)(t.q / (double)soft.s));
  g.record = r.renormalize ? (float)((double)factor / t.q) : factor;
  return g;
}

// The row's loss before its weight.
__device__ __forceinline__ float row_loss(const Record& r, const RecordSums& t, const Soft& soft) {
  if (t.q == 0.0) return 0.f;                // no mass on record
  if (soft.m == -INFINITY) return INFINITY;  // no finite logit
  const double log_s = log((double)soft.s);
  const double q_d = (t.q_x + t.q * ((double)t.at - (double)soft.m)) * (double)r.inv_t;
  if (r.renormalize) return (float)((t.q_lp - q_d) / t.q - (log(t.q) + (double)t.shift) + log_s);
  return (float)(t.q_lp - q_d + t.q * log_s);
}

// A unit of a gradient row element by element, what lies outside the row left alone.
template <class T>
__device__ __noinline__ void write_edge(const RowWalk<T> walk, T* out, uint32_t u, uint4 v) {
  float f[kUnit<T>];
  unpack<T>(v, f);
#pragma unroll
  for (uint32_t i = 0; i < kUnit<T>; ++i) {
    const uint32_t p = u * kUnit<T> + i;
    if (p >= walk.head && p < walk.end) out[p] = from_float<T>(f[i]);
  }
}

// The dense part of a gradient row, a 2^((x - m) c).
template <class T>
class DenseGrad {
 public:
  __device__ __forceinline__ DenseGrad(const RowWalk<T>& walk, T* out, uint32_t last, const RowGrad& g, float c)
      : walk_(walk), out_(out), last_(last), m_(g.m), c_(c), a_(g.dense) {
    wide_ = ((uintptr_t)out & 15u) == 0;
    r_ = m_ * c;
    scale_ = a_ * one_step_rest(m_, c, r_);
    one_step_ = one_step(m_, c);
    // For 16-bit gradients the factor goes into the exponent, which is off by 2^-24 of 200 at most then, 8e-6 of the value: far below
    // their own rounding.
    folded_ = sizeof(T) == 2 && a_ > 1e-30f && a_ < 1e30f && fabsf(r_) < 100.f;
    if (folded_) r_ -= log2f(scale_);
  }
  // All steps from unit `first`: read(batch, u0) gives the step's logits, inside(u0) tells whether its units are wholly the row's.
  template <class R, class I>
  __device__ __forceinline__ void write(uint32_t first, R&& read, I&& inside) const {
    if (wide_ && one_step_) {
      if (folded_) write_wide<true>(first, read, inside);
      else write_wide<false>(first, read, inside);
      return;
    }
    for (uint32_t u0 = first; u0 < last_; u0 += Batch<T>::kSpan) {
      Batch<T> b;
      read(b, u0);
#pragma unroll 1
      for (uint32_t j = 0; j < Batch<T>::kUnits; ++j) {
        const uint32_t u = Batch<T>::unit(u0, j);
        if (u >= last_) continue;
        uint4 raw = b.raw[0];
#pragma unroll
        for (uint32_t q = 1; q < Batch<T>::kUnits; ++q) raw = q == j ? b.raw[q] : raw;
        float f[kUnit<T>];
        unpack<T>(raw, f);
#pragma unroll
        for (uint32_t i = 0; i < kUnit<T>; ++i) f[i] = one_step_ ? scale_ * ex2(fmaf(f[i], c_, -m_ * c_)) : a_ * ex2((f[i] - m_) * c_);
        write_edge(walk_, out_, u, pack<T>(f));
      }
    }
  }

 private:
  template <bool kFolded, class R, class I>
  __device__ __forceinline__ void write_wide(uint32_t first, R&& read, I&& inside) const {
    const uint64_t cc = pair(c_, c_), nr = pair(-r_, -r_), aa = pair(scale_, scale_);
    uint4* out = reinterpret_cast<uint4*>(out_) + Batch<T>::unit(first, 0);
    for (uint32_t u0 = first; u0 < last_; u0 += Batch<T>::kSpan, out += Batch<T>::kSpan) {
      Batch<T> b;
      read(b, u0);
#pragma unroll
      for (uint32_t j = 0; j < Batch<T>::kUnits; ++j) {
        float f[kUnit<T>];
        unpack<T>(b.raw[j], f);
#pragma unroll
        for (uint32_t i = 0; i < kUnit<T>; i += 2) {
          float2 e = unpair(fma2(pair(f[i], f[i + 1]), cc, nr));
          e.x = ex2(e.x);
          e.y = ex2(e.y);
          if (!kFolded) e = unpair(mul2(pair(e.x, e.y), aa));
          f[i] = e.x;
          f[i + 1] = e.y;
        }
        b.raw[j] = pack<T>(f);
      }
      if (inside(u0)) {
#pragma unroll
        for (uint32_t j = 0; j < Batch<T>::kUnits; ++j) out[j * 32] = b.raw[j];
      } else {
#pragma unroll 1
        for (uint32_t j = 0; j < Batch<T>::kUnits; ++j) {
          const uint32_t u = Batch<T>::unit(u0, j);
          uint4 raw = b.raw[0];
#pragma unroll
          for (uint32_t q = 1; q < Batch<T>::kUnits; ++q) raw = q == j ? b.raw[q] : raw;
          if (u >= last_) continue;
          if (walk_.whole(u)) out[j * 32] = raw;
          else write_edge(walk_, out_, u, raw);
        }
      }
    }
  }

  const RowWalk<T>& walk_;
  T* out_;
  uint32_t last_;
  float m_, c_, a_, r_, scale_;
  bool wide_, one_step_, folded_;
};

template <class T>
__device__ __forceinline__ void write_zeros(const RowWalk<T>& walk, T* out, bool wide, uint32_t first, uint32_t last) {
  for (uint32_t u = first + threadIdx.x; u < last; u += kRowThreads) {
    if (wide && walk.whole(u)) {
      reinterpret_cast<uint4*>(out)[u] = make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < kUnit<T>; ++i) {
        const uint32_t p = u * kUnit<T> + i;
        if (p >= walk.head && p < walk.end) out[p] = from_float<T>(0.f);
      }
    }
  }
}

// The element that the thread's entry names, if it is its to write; behind the dense part.
template <class T>
__device__ __forceinline__ void write_record(const Record& r, const Entry& e, float share, const RowWalk<T>& walk, T* out, const RowGrad& g) {
  __syncthreads();  // the block's dense part is written
  if (share != 0.f)
    out[(uint32_t)e.id + walk.head] = from_float<T>(g.dense * ex2((e.x - g.m) * r.c) - g.record * (share * expf(e.lp - g.shift)));
}

template <class T>
__global__ void __launch_bounds__(kRowThreads, 4)
    distill_forward_kernel(RowSet x, Record r, float* __restrict__ loss, float* __restrict__ stats) {
  extern __shared__ __align__(16) uint8_t ring_memory[];
  __shared__ float2 soft_scratch[kRowWarps], soft_slots[RowCluster::kMost];
  __shared__ RecordShared record;
  const RowCluster cluster;
  cluster.started();
  const uint32_t row = cluster.row();
  const float w = r.weights ? r.weights[row] : 1.f;
  Entry e;
  if (cluster.rank == 0) e.load(r, row);
  float2* out = reinterpret_cast<float2*>(stats) + row;
  const T* src = row_ptr<T>(x, row);
  const RowWalk<T> walk(src, x.vocab);
  uint32_t first, last;
  split_units(walk.units, cluster.rank, cluster.blocks, first, last);
  Ring<T, kDepth> ring(ring_memory, walk, first, last);  // on its way before the weight is there
  if (w == 0.f) {                                        // the same for the whole cluster
    ring.drain();
    cluster.ready();
    if (cluster.rank == 0 && threadIdx.x == 0) {
      loss[row] = 0.f;
      *out = make_float2(0.f, 0.f);
    }
    return;
  }
  Soft soft = read_soft(ring, first, last, r.c, [&] { e.look_up(src, x.vocab); });
  if (cluster.rank == 0) put_record(r, e, record);
  soft = block_soft(soft, r.c, soft_scratch);
  if (cluster.blocks > 1) {
    cluster.ready();
    tell_soft(cluster, soft, soft_slots);
    cluster.told();
    soft = told_soft(cluster, r.c, soft_slots);
  }
  if (cluster.rank == 0 && threadIdx.x == 0) {
    const RecordSums t = record_sums(r, record);
    loss[row] = w * row_loss(r, t, soft);
    const RowGrad g = row_grad(r, t, soft, 1.f);
    *out = make_float2(g.m, g.dense);
  }
}

template <class T>
__global__ void __launch_bounds__(kRowThreads, 4)
    distill_backward_kernel(RowSet x, Record r, const float* __restrict__ stats, const float* __restrict__ grad_loss,
                            int64_t grad_outer, int64_t grad_inner, RowSet dx) {
  extern __shared__ __align__(16) uint8_t ring_memory[];
  __shared__ RecordShared record;
  const RowCluster cluster;  // its blocks have nothing to tell each other here
  const uint32_t row = cluster.row();
  const float w = r.weights ? r.weights[row] : 1.f;
  const float2 st = reinterpret_cast<const float2*>(stats)[row];
  const uint32_t o = row / x.inner, in = row - o * x.inner;
  const float out_g = grad_loss[(int64_t)o * grad_outer + (int64_t)in * grad_inner];
  Entry e;
  e.load(r, row);
  const T* src = row_ptr<T>(x, row);
  const RowWalk<T> walk(src, x.vocab);
  uint32_t first, last;
  split_units(walk.units, cluster.rank, cluster.blocks, first, last);
  T* out = row_ptr<T>(dx, row) - walk.head;  // by aligned position
  const bool wide = ((uintptr_t)out & 15u) == 0;  // for rows without a gradient
  Ring<T, kDepth> ring(ring_memory, walk, first, last);  // on its way before the factors are there
  const float factor = out_g * w * r.inv_t;
  if (w == 0.f || factor == 0.f || st.y == 0.f) {
    ring.drain();
    write_zeros(walk, out, wide, first, last);
    return;
  }
  RowGrad g{st.x, factor * st.y, factor, 0.f};
  const DenseGrad<T> dense(walk, out, last, g, r.c);
  bool looked_up = false;
  dense.write(first, [&](Batch<T>& b, uint32_t u0) {
    if (u0 != first) {
      ring.advance();
      if (!looked_up) e.look_up(src, x.vocab);
      looked_up = true;
    }
    ring.read(b);
  }, [&](uint32_t u0) { return ring.inside(u0); });
  if (!looked_up) e.look_up(src, x.vocab);
  put_record(r, e, record, r.renormalize);
  __syncthreads();
  const float share = record_share(r, e, record, walk, first, last);
  if (r.renormalize) {
    const RecordSums t = record_sums(r, record);
    g.record = (float)((double)factor / t.q);
    g.shift = t.shift;
  }
  write_record(r, e, share, walk, out, g);
}

template <class T>
__global__ void __launch_bounds__(kRowThreads, 3)
    distill_step_kernel(RowSet x, Record r, float* __restrict__ loss, RowSet dx) {
  extern __shared__ __align__(16) uint8_t ring_memory[];
  __shared__ float2 soft_scratch[kRowWarps], soft_slots[RowCluster::kMost];
  __shared__ RecordShared record;
  const RowCluster cluster;
  cluster.started();
  const uint32_t row = cluster.row();
  const float w = r.weights ? r.weights[row] : 1.f;
  Entry e;
  e.load(r, row);
  const T* src = row_ptr<T>(x, row);
  const RowWalk<T> walk(src, x.vocab);
  uint32_t first, last;
  split_units(walk.units, cluster.rank, cluster.blocks, first, last);
  T* out = row_ptr<T>(dx, row) - walk.head;
  const bool wide = ((uintptr_t)out & 15u) == 0;  // for rows without a gradient
  Ring<T, kStepDepth> ring(ring_memory, walk, first, last);  // on its way before the weight is there
  if (w == 0.f) {                                            // the same for the whole cluster
    ring.drain();
    cluster.ready();
    if (cluster.rank == 0 && threadIdx.x == 0) loss[row] = 0.f;
    write_zeros(walk, out, wide, first, last);
    return;
  }
  Soft soft = read_soft(ring, first, last, r.c, [&] { e.look_up(src, x.vocab); });
  put_record(r, e, record);
  soft = block_soft(soft, r.c, soft_scratch);
  if (cluster.blocks > 1) {
    cluster.ready();
    tell_soft(cluster, soft, soft_slots);
  }
  cluster.telling();
  const float share = record_share(r, e, record, walk, first, last);
  const RecordSums t = record_sums(r, record);
  cluster.heard();
  if (cluster.blocks > 1) soft = told_soft(cluster, r.c, soft_slots);
  const RowGrad g = row_grad(r, t, soft, w * r.inv_t);
  const DenseGrad<T> dense(walk, out, last, g, r.c);
  if (g.dense == 0.f) {
    write_zeros(walk, out, wide, first, last);
  } else if (last - first <= kStepDepth * Batch<T>::kSpan) {
    // The second pass from shared memory, where the block's share still is.
    uint32_t slot = 0;
    dense.write(first, [&](Batch<T>& b, uint32_t) { ring.again(slot++, b); }, [&](uint32_t u0) { return ring.inside(u0); });
  } else {
    Ring<T, kStepDepth> second(ring_memory, walk, first, last);
    dense.write(first, [&](Batch<T>& b, uint32_t u0) {
      if (u0 != first) second.advance();
      second.read(b);
    }, [&](uint32_t u0) { return second.inside(u0); });
  }
  if (g.dense != 0.f) write_record(r, e, share, walk, out, g);
  if (cluster.rank == 0 && threadIdx.x == 0) loss[row] = w * row_loss(r, t, soft);
}

int fail(int code, const std::string& msg) {
  set_last_error(msg.c_str());
  return code;
}

int done(cudaError_t e, const char* what) {
  return e == cudaSuccess ? WS_OK : fail(WS_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

int check_teacher(const ws_teacher* t, uint32_t rows, Record* out) {
  if (!t) return fail(WS_ERR_INVALID, "null teacher record");
  if (t->k < 1 || t->k > WS_TOP_MAX_K) return fail(WS_ERR_INVALID, "a teacher record has 1 to 256 entries a row");
  if (t->tail != WS_TAIL_DROP && t->tail != WS_TAIL_RENORMALIZE) return fail(WS_ERR_INVALID, "unknown tail");
  if (!(t->temperature >= 1e-6f && t->temperature <= 1e6f)) return fail(WS_ERR_INVALID, "temperature must be from 1e-6 to 1e6");
  if (rows && (!t->ids || !t->logprobs)) return fail(WS_ERR_INVALID, "null pointer in the teacher record");
  *out = Record{t->ids, t->logprobs, t->weights, t->k, t->ids_are_int32 != 0, t->tail == WS_TAIL_RENORMALIZE,
                kLog2e / t->temperature, 1.f / t->temperature};
  return WS_OK;
}

int check_grad(const ws_rows* grad, const RowArgs& x, RowArgs* out) {
  const int rc = check_rows(grad, "gradient", out);
  if (rc != WS_OK) return rc;
  if (out->rows != x.rows || out->set.vocab != x.set.vocab || out->dtype != x.dtype)
    return fail(WS_ERR_INVALID, "the gradient has other rows, vocabulary or type than the logits");
  return WS_OK;
}

}  // namespace
}  // namespace ws

using namespace ws;

extern "C" int ws_distill_forward(const ws_rows* logits, const ws_teacher* teacher, float* loss, float* stats, int device,
                                  void* stream) {
  return guarded([&] {
    RowArgs x;
    Record r;
    int rc = check_rows(logits, "logits", &x);
    if (rc == WS_OK) rc = check_teacher(teacher, x.rows, &r);
    if (rc != WS_OK) return rc;
    if (device < 0) return fail(WS_ERR_INVALID, "bad device ordinal");
    if (x.rows == 0) return (int)WS_OK;
    if (!loss || !stats) return fail(WS_ERR_INVALID, "null result pointer");
    if ((uintptr_t)stats % 8) return fail(WS_ERR_INVALID, "stats must be 8-byte aligned");
    DeviceGuard guard(device);
    cudaError_t e = guard.error();
    if (e == cudaSuccess)
      e = by_type(x.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return launch_rows<distill_forward_kernel<T>>(x.rows, blocks_a_row(x), kDepth * kStepBytes, device, stream, x.set, r, loss, stats);
      });
    return done(e, "distill forward");
  });
}

extern "C" int ws_distill_backward(const ws_rows* logits, const ws_teacher* teacher, const float* stats,
                                   const float* grad_loss, int64_t grad_outer, int64_t grad_inner, const ws_rows* grad,
                                   int device, void* stream) {
  return guarded([&] {
    RowArgs x, dx;
    Record r;
    int rc = check_rows(logits, "logits", &x);
    if (rc == WS_OK) rc = check_teacher(teacher, x.rows, &r);
    if (rc == WS_OK) rc = check_grad(grad, x, &dx);
    if (rc != WS_OK) return rc;
    if (device < 0) return fail(WS_ERR_INVALID, "bad device ordinal");
    if (x.rows == 0) return (int)WS_OK;
    if (!stats || !grad_loss) return fail(WS_ERR_INVALID, "null pointer");
    if ((uintptr_t)stats % 8) return fail(WS_ERR_INVALID, "stats must be 8-byte aligned");
    const uint32_t pieces = blocks_a_row(x, r.k <= kShortRecord ? 56 : 112);
    DeviceGuard guard(device);
    cudaError_t e = guard.error();
    if (e == cudaSuccess)
      e = by_type(x.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return launch_rows<distill_backward_kernel<T>>(x.rows, pieces, kDepth * kStepBytes, device, stream, x.set, r, stats, grad_loss, grad_outer, grad_inner, dx.set);
      });
    return done(e, "distill backward");
  });
}

extern "C" int ws_distill_step(const ws_rows* logits, const ws_teacher* teacher, float* loss, const ws_rows* grad,
                               int device, void* stream) {
  return guarded([&] {
    RowArgs x, dx;
    Record r;
    int rc = check_rows(logits, "logits", &x);
    if (rc == WS_OK) rc = check_teacher(teacher, x.rows, &r);
    if (rc == WS_OK) rc = check_grad(grad, x, &dx);
    if (rc != WS_OK) return rc;
    if (device < 0) return fail(WS_ERR_INVALID, "bad device ordinal");
    if (x.rows == 0) return (int)WS_OK;
    if (!loss) return fail(WS_ERR_INVALID, "null result pointer");
    DeviceGuard guard(device);
    cudaError_t e = guard.error();
    if (e == cudaSuccess)
      e = by_type(x.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return launch_rows<distill_step_kernel<T>>(x.rows, blocks_a_row(x, r.k <= kShortRecord ? 96 : 192), kStepDepth * kStepBytes, device, stream, x.set, r, loss, dx.set);
      });
    return done(e, "distill step");
  });
}
