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

namespace splax {
namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;
constexpr float kLn2 = 0.693147180559945309f;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) {
  return __float2bfloat16(x);
}
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half(x); }

// Maximum that returns NaN if either operand is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

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

// Order of the kept logits as one 64-bit number: the value (NaN above all, the two zeros alike),
// then the lower class.
__device__ __forceinline__ uint64_t order_key(float v, int32_t c) {
  uint32_t u = __float_as_uint(v + 0.0f);
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  if (v != v) u = 0xffffffffu;
  return (static_cast<uint64_t>(u) << 32) | (0xffffffffu - static_cast<uint32_t>(c));
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

unsigned row_grid(int64_t rows) {
  return static_cast<unsigned>(rows < kDistillMaxPartials ? rows : kDistillMaxPartials);
}

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
  if (grid > 0) {
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
