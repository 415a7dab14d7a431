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

namespace cg = cooperative_groups;

struct Record {
  const void* ids;
  const float* logprobs;
  const float* weights;
  uint32_t k;
  int ids32, renormalize;
  float c;      // log2(e) / temperature
  float inv_t;  // 1 / temperature
};

// Entry j of a row's record; a token id of -1 has no mass.
__device__ __forceinline__ void record_entry(const Record& r, uint32_t row, uint32_t j, uint32_t vocab, int& id, float& lp) {
  id = -1;
  lp = -INFINITY;
  if (j >= r.k) return;
  const size_t at = (size_t)row * r.k + j;
  const int64_t raw = r.ids32 ? ((const int32_t*)r.ids)[at] : ((const int64_t*)r.ids)[at];
  lp = r.logprobs[at];
  if (raw >= 0 && raw < (int64_t)vocab && lp > -INFINITY) id = (int)raw;
}

// A row's record summed up. After renormalising, probabilities are taken relative to the
// record's largest one (shift = its log-probability), so that a record far out in the teacher's
// tail neither underflows nor overflows; shift is 0 otherwise.
struct RecordSums {
  double q, q_lp, q_d;  // sums of q, q lp and q (x - m) / t with q = exp(lp - shift)
  float shift;
};

// What the gradient of a row needs: dense part mass_over_s * exp((x_i - m) / t), and q_scale * exp(lp - shift).
struct RowGrad {
  float m, mass_over_s, q_scale;
};

// Entry `threadIdx.x` of the record and the record's shift.
__device__ __forceinline__ float record_shift(const Record& r, int id, float lp, float* scratch) {
  if (!r.renormalize) return 0.f;
  const float top = block_max(id >= 0 ? lp : -INFINITY, scratch);
  return top == -INFINITY ? 0.f : top;
}

template <class T>
__device__ __forceinline__ RecordSums record_sums(const Record& r, uint32_t row, const T* x, uint32_t vocab, float m,
                                                  double* scratch) {
  int id;
  float lp;
  record_entry(r, row, threadIdx.x, vocab, id, lp);
  RecordSums t;
  t.shift = record_shift(r, id, lp, reinterpret_cast<float*>(scratch));
  double q = id >= 0 ? exp((double)lp - (double)t.shift) : 0.0, q_lp = 0.0, q_d = 0.0;
  if (q != 0.0) {
    q_lp = q * (double)lp;
    q_d = q * (((double)to_float(x[id]) - (double)m) * (double)r.inv_t);
  }
  t.q = block_sum(q, scratch);
  t.q_lp = block_sum(q_lp, scratch);
  t.q_d = block_sum(q_d, scratch);
  return t;
}

// The row's loss before its weight, and the gradient's factors (0: no gradient).
__device__ __forceinline__ float finish_loss(const Record& r, const RecordSums& t, const Soft& soft, RowGrad& g) {
  g = RowGrad{soft.m, 0.f, 0.f};
  if (t.q == 0.0) return 0.f;                  // no mass on record
  if (soft.m == -INFINITY) return INFINITY;    // no finite logit
  const double scale = r.renormalize ? 1.0 / t.q : 1.0;
  g.q_scale = (float)scale;
  g.mass_over_s = (float)(t.q * scale / (double)soft.s);
  const double log_s = log((double)soft.s);
  if (r.renormalize) return (float)((t.q_lp - t.q_d) * scale - (log(t.q) + (double)t.shift) + log_s);
  return (float)(t.q_lp - t.q_d + t.q * log_s);
}

// Writes units [first, last) of one gradient row: dense part a * 2^((x - m) c), then the record's
// corrections that fall among them.
template <class T>
__device__ __forceinline__ void write_grad(const Record& r, uint32_t row, const RowWalk<T>& walk, uint32_t first, uint32_t last,
                                           T* grad, uint32_t vocab, float m, float shift, float a, float b, int* ids, float* qs) {
  // a = g w Q / (t S), b = g w q_scale / t, q = exp(lp - shift); both 0: the row has no gradient and its logits are not read.
  const bool none = a == 0.f && b == 0.f;
  T* out = grad - walk.head;  // by aligned position
  const bool same = (((uintptr_t)out) & 15u) == 0;
  const uint64_t nm = pair(-m, -m), cc = pair(r.c, r.c), aa = pair(a, a);
  Batch<T> next;
  if (none) next = Batch<T>{};
  else if (first < last) next.load(walk, first, last);
  for (uint32_t u0 = first; u0 < last; u0 += Batch<T>::kSpan) {
    const Batch<T> now = next;
    if (!none && u0 + Batch<T>::kSpan < last) next.load(walk, u0 + Batch<T>::kSpan, last);
#pragma unroll
    for (uint32_t j = 0; j < Batch<T>::kUnits; ++j) {
      const uint32_t u = u0 + j * kRowThreads + threadIdx.x;
      if (u >= last) continue;
      float f[kUnit];
      unpack<T>(now.raw[j], f);
      if (!none) {
#pragma unroll
        for (uint32_t i = 0; i < kUnit; i += 2) {
          const float2 e = unpair(mul2(add2(pair(f[i], f[i + 1]), nm), cc));
          const float2 g = unpair(mul2(aa, pair(ex2(e.x), ex2(e.y))));
          f[i] = g.x;
          f[i + 1] = g.y;
        }
      }
      if (same && walk.whole(u)) {
        const Raw<T> w = pack<T>(f);
        uint4* v = reinterpret_cast<uint4*>(out + (size_t)u * kUnit);
#pragma unroll
        for (uint32_t i = 0; i < sizeof(T) / 2; ++i) v[i] = w.v[i];
      } else {
#pragma unroll
        for (uint32_t i = 0; i < kUnit; ++i) {
          const uint32_t p = u * kUnit + i;
          if (p >= walk.head && p < walk.end) out[p] = from_float<T>(f[i]);
        }
      }
    }
  }
  if (none) return;  // the same for the whole block
  int id;
  float lp;
  record_entry(r, row, threadIdx.x, vocab, id, lp);
  ids[threadIdx.x] = id;
  qs[threadIdx.x] = id >= 0 ? expf(lp - shift) : 0.f;
  __syncthreads();  // the dense part is written, too
  const uint32_t p = (uint32_t)id + walk.head;
  if (id >= 0 && p >= first * kUnit && p < last * kUnit) {
    float q = 0.f;
    bool owner = true;
    for (uint32_t j = 0; j < r.k; ++j) {
      if (ids[j] == id) {
        owner = owner && j >= threadIdx.x;
        q += qs[j];
      }
    }
    if (owner) out[p] = from_float<T>(a * ex2((walk.at(p) - m) * r.c) - b * q);
  }
}

template <class T>
__global__ void __launch_bounds__(kRowThreads)
    distill_forward_kernel(RowSet x, Record r, float* __restrict__ loss, float* __restrict__ stats) {
  __shared__ float2 soft_scratch[kRowWarps];
  __shared__ float2 mine;
  __shared__ double sums[kRowWarps];
  const cg::cluster_group cluster = cg::this_cluster();
  const uint32_t blocks = cluster.num_blocks(), rank = cluster.block_rank(), row = blockIdx.x / blocks;
  const float w = r.weights ? r.weights[row] : 1.f;
  float2* out = reinterpret_cast<float2*>(stats) + row;
  if (w == 0.f) {  // the same for the whole cluster
    if (rank == 0 && threadIdx.x == 0) {
      loss[row] = 0.f;
      *out = make_float2(0.f, 0.f);
    }
    return;
  }
  const T* src = row_ptr<T>(x, row);
  const RowWalk<T> walk(src, x.vocab);
  uint32_t first, last;
  split_units(walk.units, rank, blocks, first, last);
  const Soft soft = cluster_soft(row_soft(walk, first, last, r.c, soft_scratch), r.c, &mine);
  if (rank == 0) {
    const RecordSums t = record_sums<T>(r, row, src, x.vocab, soft.m, sums);
    if (threadIdx.x == 0) {
      RowGrad g;
      loss[row] = w * finish_loss(r, t, soft, g);
      *out = make_float2(g.m, g.mass_over_s);
    }
  }
  if (blocks > 1) cluster.sync();  // `mine` is read until here
}

template <class T>
__global__ void __launch_bounds__(kRowThreads)
    distill_backward_kernel(RowSet x, Record r, const float* __restrict__ stats, const float* __restrict__ grad_loss,
                            int64_t grad_outer, int64_t grad_inner, RowSet dx) {
  __shared__ int ids[kRowThreads];
  __shared__ float qs[kRowThreads];
  __shared__ double sums[kRowWarps];
  const cg::cluster_group cluster = cg::this_cluster();
  const uint32_t pieces = cluster.num_blocks(), piece = cluster.block_rank(), row = blockIdx.x / pieces;
  const float w = r.weights ? r.weights[row] : 1.f;
  const float2 st = reinterpret_cast<const float2*>(stats)[row];
  const uint32_t o = row / x.inner, in = row - o * x.inner;
  float a = 0.f, b = 0.f, shift = 0.f;
  if (w != 0.f && st.y != 0.f) {
    const float g = grad_loss[(int64_t)o * grad_outer + (int64_t)in * grad_inner] * w * r.inv_t;
    float scale = 1.f;
    if (r.renormalize) {
      int id;
      float lp;
      record_entry(r, row, threadIdx.x, x.vocab, id, lp);
      shift = record_shift(r, id, lp, reinterpret_cast<float*>(sums));
      scale = (float)(1.0 / block_sum(id >= 0 ? exp((double)lp - (double)shift) : 0.0, sums));
    }
    a = g * st.y;
    b = g * scale;
  }
  const RowWalk<T> walk(row_ptr<T>(x, row), x.vocab);
  uint32_t first, last;
  split_units(walk.units, piece, pieces, first, last);
  write_grad<T>(r, row, walk, first, last, row_ptr<T>(dx, row), x.vocab, st.x, shift, a, b, ids, qs);
}

template <class T>
__global__ void __launch_bounds__(kRowThreads)
    distill_step_kernel(RowSet x, Record r, float* __restrict__ loss, RowSet dx) {
  __shared__ float2 soft_scratch[kRowWarps];
  __shared__ float2 mine;
  __shared__ double sums[kRowWarps];
  __shared__ int ids[kRowThreads];
  __shared__ float qs[kRowThreads];
  const cg::cluster_group cluster = cg::this_cluster();
  const uint32_t blocks = cluster.num_blocks(), rank = cluster.block_rank(), row = blockIdx.x / blocks;
  const float w = r.weights ? r.weights[row] : 1.f;
  const T* src = row_ptr<T>(x, row);
  const RowWalk<T> walk(src, x.vocab);
  uint32_t first, last;
  split_units(walk.units, rank, blocks, first, last);
  float m = 0.f, shift = 0.f, a = 0.f, b = 0.f, l = 0.f;
  if (w != 0.f) {  // the same for the whole cluster
    const Soft soft = cluster_soft(row_soft(walk, first, last, r.c, soft_scratch), r.c, &mine);
    const RecordSums t = record_sums<T>(r, row, src, x.vocab, soft.m, sums);
    RowGrad g;
    l = w * finish_loss(r, t, soft, g);
    m = g.m;
    shift = t.shift;
    a = w * r.inv_t * g.mass_over_s;
    b = w * r.inv_t * g.q_scale;
  }
  if (rank == 0 && threadIdx.x == 0) loss[row] = l;
  write_grad<T>(r, row, walk, first, last, row_ptr<T>(dx, row), x.vocab, m, shift, a, b, ids, qs);
  if (blocks > 1) cluster.sync();  // `mine` is read until here
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
        return launch_rows(distill_forward_kernel<T>, x.rows, blocks_a_row(x.rows, x.set.vocab / kUnit), stream, x.set, r, loss, stats);
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
    const uint32_t pieces = blocks_a_row(x.rows, x.set.vocab / kUnit);
    DeviceGuard guard(device);
    cudaError_t e = guard.error();
    if (e == cudaSuccess)
      e = by_type(x.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return launch_rows(distill_backward_kernel<T>, x.rows, pieces, stream, x.set, r, stats, grad_loss, grad_outer, grad_inner, dx.set);
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
        return launch_rows(distill_step_kernel<T>, x.rows, blocks_a_row(x.rows, x.set.vocab / kUnit), stream, x.set, r, loss, dx.set);
      });
    return done(e, "distill step");
  });
}
