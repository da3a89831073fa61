// Distillation from a teacher's top logits: the k largest logits of each row with the row's
// log-sum-exp (the teacher's side), and the divergence of the student's softmax from the
// distribution they give, with its gradient (the student's side).
//
// Loss of a row, s = z / tau, entries e with class id_e and probability p_e, O the classes that no
// entry names, lse the log-sum-exp of s over all classes and lse_O over O:
//   L = sum_e p_e (ln p_e - s_e + lse) + rho (ln rho - lse_O + lse)
//   dL/ds_c = (P + rho) q_c - p_c                            c named by an entry
//           = ((P + rho) q_O - rho) exp(s_c - lse_O)         c in O
// with P = sum_e p_e, q_c = exp(s_c - lse), q_O = exp(lse_O - lse). The sums over O are taken
// without the entries instead of as a difference from the sum over all classes, which would
// cancel when the student agrees with the teacher.
//
// Exponentials are powers of two of (z - m) log2(e) / tau with the difference taken first, so a
// row of the type's lowest value stays finite. Maxima propagate NaN, so a NaN logit reaches the
// row's loss and gradient.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/splax_b200.h"
#include "common.cuh"
#include "kernels.h"
#include "rows.cuh"

namespace splax {
namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;

__device__ __forceinline__ float load_value(const void* p, int dtype, int64_t i) {
  if (dtype == SPLAX_F32) return static_cast<const float*>(p)[i];
  if (dtype == SPLAX_BF16) return to_f(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_f(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ int32_t load_id(const void* p, bool wide, int64_t i, int32_t classes) {
  const int64_t c = wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
  return c >= 0 && c < classes ? static_cast<int32_t>(c) : -1;
}

template <typename Op>
__device__ __forceinline__ float block_reduce(float x, float* s_red, Op op) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x = op(x, __shfl_xor_sync(0xffffffffu, x, off));
  __syncthreads();  // s_red may still be read from the reduction before
  if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = x;
  __syncthreads();
  x = s_red[0];
  for (int w = 1; w < kRowWarps; ++w) x = op(x, s_red[w]);
  return x;
}

struct LossParams {
  const void* logits;
  int64_t rows, row_stride;
  int32_t classes, k;
  const void* top_values;
  const void* top_ids;
  const float* top_lse;
  const float* weights;
  int value_dtype;
  bool wide_ids;
  double inv_tau;
  float scale2;            // log2(e) / tau
  float inv_hi, inv_lo;    // 1 / tau
  float grad_scale;        // tau / denom
  const float* v_loss;
  void* grad;
  double* partials;
};

// One CTA per row: the named classes as a bitmap in shared memory, then a pass for the maximum
// over O, one for its sum and one for the gradient.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) distill_kernel(LossParams a) {
  pdl_enter();
  extern __shared__ uint32_t s_named[];
  __shared__ float s_red[kRowWarps];
  __shared__ float s_p[kDistillMaxK], s_z[kDistillMaxK], s_x[kDistillMaxK];
  __shared__ int32_t s_id[kDistillMaxK];
  __shared__ float s_bc[4];
  const int tid = threadIdx.x;
  const float ninf = neg_inf();
  const int words = (a.classes + 31) / 32;
  for (int i = tid; i < words; i += kRowThreads) s_named[i] = 0u;
  double total = 0.0;
  const float cot = a.v_loss ? *a.v_loss : 1.0f;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* z = static_cast<const T*>(a.logits) + r * a.row_stride;
    T* g = a.grad ? static_cast<T*>(a.grad) + r * a.classes : nullptr;
    const float w = a.weights ? a.weights[r] : 1.0f;
    __syncthreads();
    if (tid < a.k) {
      const int32_t id = load_id(a.top_ids, a.wide_ids, r * a.k + tid, a.classes);
      s_id[tid] = id;
      s_x[tid] = id < 0 ? ninf : load_value(a.top_values, a.value_dtype, r * a.k + tid);
      s_z[tid] = id < 0 ? ninf : to_f(z[id]);
      if (id >= 0) atomicOr(&s_named[id >> 5], 1u << (id & 31));
    }
    __syncthreads();
    // teacher (one thread: the entries are few)
    if (tid == 0) {
      float vmax = ninf;
      for (int e = 0; e < a.k; ++e) vmax = max_nan(vmax, s_x[e]);
      float norm = 0.0f, mass = 0.0f, ment = ninf;
      bool live = true;
      if (a.top_lse) {
        norm = a.top_lse[r];
        live = !(norm == ninf);
      } else {
        live = !(vmax == ninf);
        float sum = 0.0f;
        for (int e = 0; e < a.k; ++e)
          if (s_x[e] != ninf) sum += expf((s_x[e] - vmax) * a.inv_hi);
        norm = logf(sum);
      }
      for (int e = 0; e < a.k; ++e) {
        float x = ninf;
        if (s_x[e] != ninf)
          x = a.top_lse ? fmaf(s_x[e], a.inv_lo, fmaf(s_x[e], a.inv_hi, -norm))
                        : (s_x[e] - vmax) * a.inv_hi - norm;
        s_x[e] = x;  // ln p
        s_p[e] = expf(x);
        mass += s_p[e];
        ment = max_nan(ment, s_z[e]);
      }
      s_bc[0] = mass;
      s_bc[1] = ment;
      s_bc[2] = live && w != 0.0f ? 1.0f : 0.0f;
    }
    __syncthreads();
    const float mass = s_bc[0], ment = s_bc[1];
    bool live = s_bc[2] != 0.0f;
    float mo = ninf, zo = 0.0f;
    auto outside = [&](int c) { return ((s_named[c >> 5] >> (c & 31)) & 1u) == 0u; };
    if (live) {
      for (int c = tid; c < a.classes; c += kRowThreads)
        if (outside(c)) mo = max_nan(mo, to_f(z[c]));
      mo = block_reduce(mo, s_red, max_nan);
      if (mo != ninf) {
        for (int c = tid; c < a.classes; c += kRowThreads)
          if (outside(c)) zo += exp2f((to_f(z[c]) - mo) * a.scale2);
        zo = block_reduce(zo, s_red, [](float x, float y) { return x + y; });
      }
    }
    const float m = max_nan(mo, ment);
    live = live && !(m == ninf);
    const float rho = live && a.top_lse && mo != ninf ? fmaxf(0.0f, 1.0f - mass) : 0.0f;
    if (live && tid == 0) {
      float sum = mo == ninf ? 0.0f : zo * exp2f((mo - m) * a.scale2);
      for (int e = 0; e < a.k; ++e) {
        bool first = s_id[e] >= 0;
        for (int j = 0; j < e; ++j) first = first && s_id[j] != s_id[e];
        if (first) sum += exp2f((s_z[e] - m) * a.scale2);
      }
      const float lsum = log2f(sum);
      // in 64 bits: the logit of an entry may be the type's lowest value
      const double ln_sum = static_cast<double>(kLn2) * lsum;
      double loss = 0.0;
      for (int e = 0; e < a.k; ++e)
        if (s_p[e] != 0.0f)
          loss += s_p[e] * (s_x[e] - ((static_cast<double>(s_z[e]) - m) * a.inv_tau - ln_sum));
      const double lqo = logf(zo) + (static_cast<double>(mo) - m) * a.inv_tau - ln_sum;
      if (rho > 0.0f) loss += rho * (logf(rho) - lqo);
      total += w * loss;
      s_bc[3] = lsum;
      s_bc[1] = mo == ninf ? 0.0f : ((mass + rho) * expf(static_cast<float>(lqo)) - rho) / zo;
    }
    __syncthreads();
    if (g) {
      if (!live) {
        for (int c = tid; c < a.classes; c += kRowThreads) g[c] = from_f<T>(0.0f);
      } else {
        const float lsum = s_bc[3], coef = s_bc[1];
        const float gs = w * a.grad_scale * cot;
        for (int c = tid; c < a.classes; c += kRowThreads)
          if (outside(c))
            g[c] = from_f<T>(mo == ninf ? 0.0f
                                        : gs * (coef * exp2f((to_f(z[c]) - mo) * a.scale2)));
        if (tid < a.k && s_id[tid] >= 0) {
          float p = 0.0f;
          bool first = true;
          for (int j = 0; j < a.k; ++j)
            if (s_id[j] == s_id[tid]) {
              first = first && j >= tid;
              p += s_p[j];
            }
          if (first)
            g[s_id[tid]] =
                from_f<T>(gs * ((mass + rho) * exp2f((s_z[tid] - m) * a.scale2 - lsum) - p));
        }
      }
    }
    __syncthreads();
    if (tid < a.k && s_id[tid] >= 0) s_named[s_id[tid] >> 5] = 0u;
  }
  if (tid == 0 && a.partials) a.partials[blockIdx.x] = total;
}


// What the entries of one row say, worked out by the threads of one CTA.
struct Entries {
  float p[kDistillMaxK];    // probability
  float x[kDistillMaxK];    // ln p (-inf: the entry is empty)
  float z[kDistillMaxK];    // the student's logit
  int32_t id[kDistillMaxK];
  int32_t first[kDistillMaxK];  // no earlier entry names the class
  float mass;               // sum of p
  float m;                  // maximum of z
  int32_t live;             // the row counts, as far as the teacher and its weight say
};

// Warp 0: probabilities and sums. top_lse NULL: the entries are renormalised, and their mass is
// one by definition.
__device__ __forceinline__ void entry_stats(Entries& s, int k, const float* top_lse, int64_t r,
                                            float w, float inv_hi, float inv_lo) {
  const int lane = threadIdx.x & 31;
  const float ninf = neg_inf();
  auto warp_max = [](float x) {
    for (int off = 16; off > 0; off >>= 1) x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, off));
    return x;
  };
  auto warp_sum = [](float x) {
    for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
    return x;
  };
  float vmax = ninf, zmax = ninf;
  for (int e = lane; e < k; e += 32) {
    vmax = max_nan(vmax, s.x[e]);
    zmax = max_nan(zmax, s.z[e]);
  }
  vmax = warp_max(vmax);
  zmax = warp_max(zmax);
  float norm;
  bool live;
  if (top_lse) {
    norm = top_lse[r];
    live = !(norm == ninf);
  } else {
    live = !(vmax == ninf);
    float sum = 0.0f;
    for (int e = lane; e < k; e += 32)
      if (s.x[e] != ninf) sum += expf((s.x[e] - vmax) * inv_hi);
    norm = logf(warp_sum(sum));
  }
  float mass = 0.0f;
  for (int e = lane; e < k; e += 32) {
    const float v = s.x[e];
    float x = ninf;
    if (v != ninf)
      x = top_lse ? fmaf(v, inv_lo, fmaf(v, inv_hi, -norm)) : (v - vmax) * inv_hi - norm;
    const float p = expf(x);
    s.x[e] = x;
    s.p[e] = p;
    mass += p;
  }
  mass = top_lse ? warp_sum(mass) : 1.0f;
  if (lane == 0) {
    s.mass = mass;
    s.m = zmax;
    s.live = live && w != 0.0f;
  }
}

// Long rows: a cluster per row, each CTA with its share in shared memory, so the logits are read
// from memory once for the sum and the gradient. The share arrives by one bulk copy while the
// entries are worked out (by every CTA of the cluster, which saves exchanging them); the entries'
// places are then set to -inf, so the pass over the share needs no test for them. One pass takes
// the maximum and the sum over O together; the CTAs exchange those two numbers, and the second
// pass turns the share into the gradient, stored as 16-byte vectors where the gradient's rows lie
// to 16 bytes as the logits' do, otherwise through shared memory in consecutive elements.
template <typename T>
__global__ void __launch_bounds__(512)
distill_row_kernel(LossParams a) {
  extern __shared__ uint4 s_buf[];
  __shared__ Entries s;
  __shared__ __align__(8) uint64_t s_bar;
  __shared__ MaxSum s_warp[16];
  __shared__ MaxSum s_part[2][8];  // by parity: a CTA may be a row ahead of its cluster
  __shared__ float s_out[3];       // log2 of the sum over all classes, coefficient over O, rho
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const float ninf = neg_inf();
  if (tid == 0) mbar_init(&s_bar, 1);
  pdl_enter();
  const float cot = a.v_loss ? *a.v_loss : 1.0f;
  double total = 0.0;
  uint32_t phase = 0, parity = 0;
  __syncthreads();
  for (int64_t r = blockIdx.x / size; r < a.rows; r += gridDim.x / size) {
    const T* z = static_cast<const T*>(a.logits) + r * a.row_stride;
    T* g = a.grad ? static_cast<T*>(a.grad) + r * a.classes : nullptr;
    const RowShare<T> share = row_share(z, a.classes, rank, size);
    const int n = share.v1 - share.v0;
    const float w = a.weights ? a.weights[r] : 1.0f;
    bool live = w != 0.0f, late = false;
    float coef = 0.0f, mo = ninf;
    if (live) {
      load_share(share, a.classes, s_buf, &s_bar);
      if (tid < a.k) {
        const int32_t id = load_id(a.top_ids, a.wide_ids, r * a.k + tid, a.classes);
        s.id[tid] = id;
        s.x[tid] = id < 0 ? ninf : load_value(a.top_values, a.value_dtype, r * a.k + tid);
        s.z[tid] = id < 0 ? ninf : to_f(z[id]);
      }
      __syncthreads();
      if (warp == 0) {
        entry_stats(s, a.k, a.top_lse, r, w, a.inv_hi, a.inv_lo);
      } else if (warp <= 4) {
        const int e = tid - 32;
        if (e < a.k) {
          bool first = s.id[e] >= 0;
          for (int j = 0; j < e; ++j) first = first && s.id[j] != s.id[e];
          s.first[e] = first;
        }
      }
      late = !mbar_wait(&s_bar, phase);
      phase ^= 1;
      if (tid < a.k && s.id[tid] >= 0) {
        const int at = s.id[tid] - share.cls0;
        if (at >= 0 && at < n * kVec<T>) reinterpret_cast<T*>(s_buf)[at] = from_f<T>(ninf);
      }
      __syncthreads();
      MaxSum acc{ninf, 0.0f};
      for (int v = tid; v < n; v += threads) {
        float x[kVec<T>];
        unpack(s_buf[v], x, T{});
        add(acc, x, a.scale2);
      }
      for (int off = 16; off > 0; off >>= 1)
        acc = join(acc, {__shfl_xor_sync(0xffffffffu, acc.m, off),
                         __shfl_xor_sync(0xffffffffu, acc.s, off)}, a.scale2);
      if (lane == 0) s_warp[warp] = acc;
      __syncthreads();
      if (warp == 0) {
        acc = lane < threads / 32 ? s_warp[lane] : MaxSum{ninf, 0.0f};
        for (int off = 8; off > 0; off >>= 1)
          acc = join(acc, {__shfl_xor_sync(0xffffffffu, acc.m, off),
                           __shfl_xor_sync(0xffffffffu, acc.s, off)}, a.scale2);
        if (lane < static_cast<int>(size)) {
          const uint32_t to = cluster_addr(&s_part[parity][rank], lane);
          cluster_store(to, acc.m);
          cluster_store(to + 4, acc.s);
        }
      }
      __syncwarp();
      if (size > 1) cluster_sync();
      if (warp == 0) {
        MaxSum o{ninf, 0.0f};
        for (uint32_t q = 0; q < size; ++q) o = join(o, s_part[parity][q], a.scale2);
        const float m = max_nan(o.m, s.m);
        float sum = 0.0f;
        for (int e = lane; e < a.k; e += 32)
          if (s.first[e]) sum += ex2_approx((s.z[e] - m) * a.scale2);
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const bool some = !(o.m == ninf);
        if (some) sum += o.s * ex2_approx((o.m - m) * a.scale2);
        const float lsum = log2f(sum);
        const float rho = a.top_lse && some ? fmaxf(0.0f, 1.0f - s.mass) : 0.0f;
        // in 64 bits: a logit may be the type's lowest value
        const double ln_sum = static_cast<double>(kLn2) * lsum;
        double loss = 0.0;
        for (int e = lane; e < a.k; e += 32)
          if (s.p[e] != 0.0f)
            loss += s.p[e] * (s.x[e] - ((static_cast<double>(s.z[e]) - m) * a.inv_tau - ln_sum));
        for (int off = 16; off > 0; off >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, off);
        const double lqo = logf(o.s) + (static_cast<double>(o.m) - m) * a.inv_tau - ln_sum;
        if (rho > 0.0f) loss += rho * (logf(rho) - lqo);
        const bool counts = s.live && !(m == ninf);
        if (late) loss = static_cast<double>(__int_as_float(0x7fc00000));
        __syncwarp();
        if (lane == 0) {
          if (counts) total += w * loss;
          s.live = counts;
          s.m = m;
          s_out[0] = late ? __int_as_float(0x7fc00000) : lsum;
          s_out[1] = some ? ((s.mass + rho) * expf(static_cast<float>(lqo)) - rho) / o.s : 0.0f;
          s_out[2] = rho;
          s_warp[0].m = o.m;
        }
      }
      parity ^= 1;
      __syncthreads();
      live = s.live;
      mo = s_warp[0].m;
      coef = s_out[1];
    }
    if (g) {
      const float gs = w * a.grad_scale * cot;
      const float c0 = live ? gs * coef : 0.0f;
      const float base = mo == ninf ? 0.0f : mo;
      const bool even = ((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(z)) & 15u) == 0;
      T* out = g + share.cls0;
      for (int v = tid; v < n; v += threads) {
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (live) {
          float x[kVec<T>];
          unpack(s_buf[v], x, T{});
#pragma unroll
          for (int i = 0; i < kVec<T>; ++i) x[i] = c0 * ex2_approx((x[i] - base) * a.scale2);
          u = pack(x, T{});
        }
        const int c = share.cls0 + v * kVec<T>;
        if (even && c >= 0 && c + kVec<T> <= a.classes)
          __stcs(reinterpret_cast<uint4*>(out + v * kVec<T>), u);
        else
          s_buf[v] = u;
      }
      __syncthreads();
      const int lo = share.cls0 < 0 ? -share.cls0 : 0;
      const int hi = min(n * kVec<T>, a.classes - share.cls0);
      const T* e = reinterpret_cast<const T*>(s_buf);
      if (!even) {
        for (int i = lo + tid; i < hi; i += threads) out[i] = e[i];
      } else if (n > 0) {  // the ends of the row
        const int head = lo > 0 ? min(kVec<T>, hi) : 0, tail = max(head, hi / kVec<T> * kVec<T>);
        if (tid >= lo && tid < head) out[tid] = e[tid];
        if (tail + tid < hi) out[tail + tid] = e[tail + tid];
      }
      if (live) {
        __syncthreads();  // an entry's place was stored above
        if (tid < a.k && s.first[tid]) {
          const int at = s.id[tid] - share.cls0;
          if (at >= 0 && at < n * kVec<T>) {
            float p = 0.0f;
            for (int j = tid; j < a.k; ++j)
              if (s.id[j] == s.id[tid]) p += s.p[j];
            const float q = ex2_approx((s.z[tid] - s.m) * a.scale2 - s_out[0]);
            g[s.id[tid]] = from_f<T>(gs * ((s.mass + s_out[2]) * q - p));
          }
        }
      }
    }
    fence_async();  // the next row's copy into the share comes after these accesses
    __syncthreads();
  }
  if (tid == 0 && rank == 0 && a.partials) a.partials[blockIdx.x / size] = total;
}

// The loss from the CTAs' partial sums, in index order for a result that does not depend on
// which CTA finished first.
__global__ void __launch_bounds__(256)
distill_finish_kernel(const double* partials, int count, double scale, float* loss) {
  pdl_enter();
  __shared__ double s[256];
  double t = 0.0;
  for (int i = threadIdx.x; i < count; i += 256) t += partials[i];
  s[threadIdx.x] = t;
  __syncthreads();
  for (int st = 128; st > 0; st >>= 1) {
    if (threadIdx.x < st) s[threadIdx.x] += s[threadIdx.x + st];
    __syncthreads();
  }
  if (threadIdx.x == 0) *loss = static_cast<float>(s[0] * scale);
}

template <typename T>
__global__ void __launch_bounds__(256)
distill_scale_kernel(T* grad, int64_t count, const float* v_loss) {
  pdl_enter();
  const float v = *v_loss;
  if (v == 1.0f) return;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += stride)
    grad[i] = from_f<T>(to_f(grad[i]) * v);
}

// One CTA per row: the log-sum-exp, then k passes for the largest key below the one before.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
top_kernel(const T* logits, int64_t rows, int64_t row_stride, int32_t classes, int32_t k,
           float scale2, float inv_tau, T* values, int32_t* ids, float* lse) {
  pdl_enter();
  __shared__ float s_red[kRowWarps];
  __shared__ unsigned long long s_key[kRowWarps];
  const int tid = threadIdx.x;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* z = logits + r * row_stride;
    float m = neg_inf(), sum = 0.0f;
    for (int c = tid; c < classes; c += kRowThreads) m = max_nan(m, to_f(z[c]));
    m = block_reduce(m, s_red, max_nan);
    for (int c = tid; c < classes; c += kRowThreads) sum += exp2f((to_f(z[c]) - m) * scale2);
    sum = block_reduce(sum, s_red, [](float x, float y) { return x + y; });
    if (tid == 0) lse[r] = m == neg_inf() ? m : fmaf(m, inv_tau, logf(sum));
    uint64_t last = ~0ull;
    for (int e = 0; e < k; ++e) {
      unsigned long long best = 0;
      for (int c = tid; c < classes; c += kRowThreads) {
        const uint64_t key = order_key(to_f(z[c]), c);
        if ((e == 0 || key < last) && key > best) best = key;
      }
      for (int off = 16; off > 0; off >>= 1) {
        const unsigned long long o = __shfl_xor_sync(0xffffffffu, best, off);
        best = o > best ? o : best;
      }
      __syncthreads();
      if ((tid & 31) == 0) s_key[tid >> 5] = best;
      __syncthreads();
      for (int w = 0; w < kRowWarps; ++w) best = s_key[w] > best ? s_key[w] : best;
      last = best;
      if (tid == 0) {
        const int32_t c = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(best));
        ids[r * k + e] = c;
        values[r * k + e] = z[c];
      }
    }
  }
}


// The largest k of the candidates in s_cand[0, count), sorted, to s_kept: each candidate counts
// those before it. k <= kDistillMaxK.
constexpr int kCandidates = 1024;
__device__ __forceinline__ void keep_largest(const uint64_t* s_cand, int count, int k,
                                             uint64_t* s_kept) {
  for (int i = threadIdx.x; i < k; i += blockDim.x)
    if (i >= count) s_kept[i] = 0;
  for (int i = threadIdx.x; i < count; i += blockDim.x) {
    const uint64_t key = s_cand[i];
    int rank = 0;
    for (int j = 0; j < count; ++j) rank += s_cand[j] > key;
    if (rank < k) s_kept[rank] = key;
  }
}

// Long rows: a cluster per row, each CTA with its share in shared memory. One pass takes each
// thread's maximum and sum; the k-th largest of the maxima of 2k or more groups of threads is a
// bound that at least k logits reach and few more do (about 1.4 k of a row in no particular order),
// so the second pass collects those few and they are sorted by counting. Rows where more than
// kCandidates reach the bound (many equal values) find the k-th largest by bisection of the value
// and then of the class. The CTAs' lists are joined by the cluster's first.
template <typename T>
__global__ void __launch_bounds__(512)
top_row_kernel(const T* logits, int64_t rows, int64_t row_stride, int32_t classes, int32_t k,
               float scale2, float inv_tau, T* values, int32_t* ids, float* lse) {
  extern __shared__ uint4 s_buf[];
  __shared__ uint64_t s_cand[kCandidates];
  __shared__ uint64_t s_kept[kDistillMaxK];
  __shared__ __align__(8) uint64_t s_bar;
  __shared__ __align__(8) MaxSum s_sum;
  __shared__ MaxSum s_warp[16];
  __shared__ float s_group[512];
  __shared__ float s_bound;
  __shared__ int s_count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const float ninf = neg_inf();
  if (tid == 0) mbar_init(&s_bar, 1);
  pdl_enter();
  uint32_t phase = 0;
  // groups of `span` threads, 2k of them or as many as there are threads
  int span = threads;
  while (span > 1 && threads / span < 2 * k) span /= 2;
  const int groups = threads / span;
  __syncthreads();
  for (int64_t r = blockIdx.x / size; r < rows; r += gridDim.x / size) {
    const T* z = logits + r * row_stride;
    const RowShare<T> share = row_share(z, classes, rank, size);
    const int n = share.v1 - share.v0;
    load_share(share, classes, s_buf, &s_bar);
    if (tid == 0) {
      s_count = 0;
      s_bound = ninf;
    }
    const bool late = !mbar_wait(&s_bar, phase);
    phase ^= 1;
    __syncthreads();
    MaxSum acc{ninf, 0.0f};
    for (int v = tid; v < n; v += threads) {
      float x[kVec<T>];
      unpack(s_buf[v], x, T{});
      add(acc, x, scale2);
    }
    float gm = acc.m;
    for (int off = 1; off < span && off < 32; off <<= 1)
      gm = max_nan(gm, __shfl_xor_sync(0xffffffffu, gm, off));
    if (span <= 32) {
      if ((lane & (span - 1)) == 0) s_group[tid / span] = gm;
    } else if (lane == 0) {
      s_group[warp] = gm;
    }
    for (int off = 16; off > 0; off >>= 1)
      acc = join(acc, {__shfl_xor_sync(0xffffffffu, acc.m, off),
                       __shfl_xor_sync(0xffffffffu, acc.s, off)}, scale2);
    if (lane == 0) s_warp[warp] = acc;
    __syncthreads();
    if (warp == 0) {
      acc = lane < threads / 32 ? s_warp[lane] : MaxSum{ninf, 0.0f};
      for (int off = 8; off > 0; off >>= 1)
        acc = join(acc, {__shfl_xor_sync(0xffffffffu, acc.m, off),
                         __shfl_xor_sync(0xffffffffu, acc.s, off)}, scale2);
      if (late) acc.s = __int_as_float(0x7fc00000);
      if (lane == 0) s_sum = acc;
    }
    const int have = span <= 32 ? groups : threads / 32;  // maxima in s_group
    for (int i = tid; i < have; i += threads) {
      const uint32_t b = order_bits(s_group[i]);
      int before = 0;
      for (int j = 0; j < have; ++j) {
        const uint32_t o = order_bits(s_group[j]);
        before += o > b || (o == b && j < i);
      }
      if (before == k - 1) s_bound = s_group[i];
    }
    __syncthreads();
    // NaN is above the bound, and a bound of NaN lets all through
    const float bound = s_bound;
    for (int v = tid; v < n; v += threads) {
      float x[kVec<T>];
      unpack(s_buf[v], x, T{});
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i)
        if (!(x[i] < bound)) {
          const int c = share.cls0 + v * kVec<T> + i;
          if (c >= 0 && c < classes) {
            const int at = atomicAdd(&s_count, 1);
            if (at < kCandidates) s_cand[at] = order_key(x[i], c);
          }
        }
    }
    __syncthreads();
    if (s_count > kCandidates) {
      // number of the share's logits with a key at or above `low`
      auto reach = [&](uint64_t low) {
        int c = 0;
        for (int v = tid; v < n; v += threads) {
          float x[kVec<T>];
          unpack(s_buf[v], x, T{});
#pragma unroll
          for (int i = 0; i < kVec<T>; ++i) {
            const int cls = share.cls0 + v * kVec<T> + i;
            c += cls >= 0 && cls < classes && order_key(x[i], cls) >= low;
          }
        }
        return c;
      };
      auto total = [&](uint64_t low) {
        __syncthreads();
        if (tid == 0) s_count = 0;
        const int mine = reach(low);
        __syncthreads();
        const int w = __reduce_add_sync(0xffffffffu, mine);
        if (lane == 0) atomicAdd(&s_count, w);
        __syncthreads();
        return s_count;
      };
      // the largest 64-bit bound that k keys reach: keys differ, so exactly k do
      uint64_t low = 0;
      for (int bit = 63; bit >= 0; --bit) {
        const uint64_t at = low | (1ull << bit);
        if (total(at) >= k) low = at;
      }
      __syncthreads();
      if (tid == 0) s_count = 0;
      __syncthreads();
      for (int v = tid; v < n; v += threads) {
        float x[kVec<T>];
        unpack(s_buf[v], x, T{});
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) {
          const int c = share.cls0 + v * kVec<T> + i;
          if (c >= 0 && c < classes && order_key(x[i], c) >= low)
            s_cand[atomicAdd(&s_count, 1)] = order_key(x[i], c);
        }
      }
      __syncthreads();
    }
    keep_largest(s_cand, s_count, k, s_kept);
    __syncthreads();
    if (size > 1) {
      cluster_sync();  // every CTA's list and sum are there
      if (rank == 0) {
        for (int i = tid; i < static_cast<int>(size) * k; i += threads)
          s_cand[i] = cluster_load(cluster_addr(&s_kept[i % k], i / k));
        if (tid == 0) {
          MaxSum all = s_sum;
          for (uint32_t q = 1; q < size; ++q) {
            const uint64_t u = cluster_load(cluster_addr(&s_sum, q));
            all = join(all, {__uint_as_float(static_cast<uint32_t>(u)),
                             __uint_as_float(static_cast<uint32_t>(u >> 32))}, scale2);
          }
          s_sum = all;
        }
      }
      cluster_sync();  // the lists are read
      if (rank == 0) {
        keep_largest(s_cand, static_cast<int>(size) * k, k, s_kept);
        __syncthreads();
      }
    }
    if (rank == 0) {
      if (tid < k) {
        const int32_t c = key_class(s_kept[tid]);
        const bool good = c >= 0 && c < classes;  // always, unless a copy was late
        ids[r * k + tid] = good ? c : -1;
        values[r * k + tid] = good ? z[c] : from_f<T>(__int_as_float(0x7fc00000));
      }
      if (tid == 0) lse[r] = s_sum.m == ninf ? ninf : fmaf(s_sum.m, inv_tau, logf(s_sum.s));
    }
    fence_async();
    __syncthreads();
  }
}

unsigned row_grid(int64_t rows) {
  return static_cast<unsigned>(rows < kDistillMaxPartials ? rows : kDistillMaxPartials);
}

// Rows of more classes than this have a cluster each.
constexpr int kShortRow = 1024;

// Threads of a CTA for a share of `vecs` vectors: a few vectors each. At least 160: warps 1 to 4
// look at the entries while warp 0 sums them.
unsigned row_threads(int vecs) { return vecs > 2048 ? 512u : 256u; }

template <typename T>
int launch_distill_t(const DistillArgs& a, cudaStream_t stream) {
  const double inv = 1.0 / a.temperature;
  LossParams p{a.logits,      a.rows,
               a.row_stride,  a.classes,
               a.k,           a.top_values,
               a.top_ids,     a.top_lse,
               a.weights,     a.value_dtype,
               a.wide_ids,    inv,           static_cast<float>(1.4426950408889634 * inv),
               static_cast<float>(inv), static_cast<float>(inv - static_cast<float>(inv)),
               static_cast<float>(a.temperature / a.denom), a.v_loss,
               a.grad,        a.partials};
  int launched = 0;
  const unsigned grid = row_grid(a.rows);
  if (grid > 0 && a.classes > kShortRow) {
    const int64_t bytes = a.classes * static_cast<int64_t>(sizeof(T));
    const unsigned size = row_cluster(a.rows, bytes, sm_count());
    const int vecs = row_share_vecs(a.classes, kVec<T>, size);
    launch_clusters(distill_row_kernel<T>, grid, size, row_threads(vecs), 16 * vecs, stream, p);
    ++launched;
  } else if (grid > 0) {
    launch_pdl(distill_kernel<T>, grid, kRowThreads, 4 * ((a.classes + 31) / 32), stream, p);
    ++launched;
  }
  if (a.loss) {
    launch_pdl(distill_finish_kernel, 1, 256, 0, stream, a.partials, static_cast<int>(grid),
               a.temperature * a.temperature / a.denom, a.loss);
    ++launched;
  }
  return launched;
}

template <typename T>
int launch_top_t(const TopLogitsArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return 0;
  const double inv = 1.0 / a.temperature;
  if (a.classes > kShortRow) {
    const int64_t bytes = a.classes * static_cast<int64_t>(sizeof(T));
    const unsigned size = row_cluster(a.rows, bytes, sm_count());
    const int vecs = row_share_vecs(a.classes, kVec<T>, size);
    const unsigned clusters = static_cast<unsigned>(a.rows < (1 << 20) ? a.rows : 1 << 20);
    launch_clusters(top_row_kernel<T>, clusters, size, row_threads(vecs), 16 * vecs, stream,
                    static_cast<const T*>(a.logits), a.rows, a.row_stride, a.classes, a.k,
                    static_cast<float>(1.4426950408889634 * inv), static_cast<float>(inv),
                    static_cast<T*>(a.values), a.ids, a.lse);
    return 1;
  }
  launch_pdl(top_kernel<T>, static_cast<unsigned>(a.rows < 65536 ? a.rows : 65536), kRowThreads,
             0, stream, static_cast<const T*>(a.logits), a.rows, a.row_stride, a.classes, a.k,
             static_cast<float>(1.4426950408889634 * inv), static_cast<float>(inv),
             static_cast<T*>(a.values), a.ids, a.lse);
  return 1;
}

}  // namespace

int launch_distill(const DistillArgs& a, cudaStream_t stream) {
  if (a.dtype == SPLAX_F32) return launch_distill_t<float>(a, stream);
  if (a.dtype == SPLAX_BF16) return launch_distill_t<__nv_bfloat16>(a, stream);
  return launch_distill_t<__half>(a, stream);
}

void launch_distill_scale(void* grad, int dtype, int64_t count, const float* v_loss,
                          cudaStream_t stream) {
  const int64_t want = (count + 2047) / 2048;
  const unsigned grid = static_cast<unsigned>(want < 2368 ? want : 2368);
  if (dtype == SPLAX_F32)
    launch_pdl(distill_scale_kernel<float>, grid, 256, 0, stream, static_cast<float*>(grad),
               count, v_loss);
  else if (dtype == SPLAX_BF16)
    launch_pdl(distill_scale_kernel<__nv_bfloat16>, grid, 256, 0, stream,
               static_cast<__nv_bfloat16*>(grad), count, v_loss);
  else
    launch_pdl(distill_scale_kernel<__half>, grid, 256, 0, stream, static_cast<__half*>(grad),
               count, v_loss);
}

int launch_top_logits(const TopLogitsArgs& a, cudaStream_t stream) {
  if (a.dtype == SPLAX_F32) return launch_top_t<float>(a, stream);
  if (a.dtype == SPLAX_BF16) return launch_top_t<__nv_bfloat16>(a, stream);
  return launch_top_t<__half>(a, stream);
}

}  // namespace splax
