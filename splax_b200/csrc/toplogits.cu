// The k largest logits of each row, with their classes and the row's log-sum-exp: what
// distillation keeps of a teacher.
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
    if (tid == 0) load_share(share, classes, s_buf, &s_bar);
    if (warp == 1) store_ends(load_ends(share, classes), s_buf);
    if (tid == 0) {
      s_count = 0;
      s_bound = ninf;
    }
    const bool late = !mbar_wait(&s_bar, phase);
    phase ^= 1;
    __syncthreads();
    Running run;
    for (int v = tid; v < n; v += threads) {
      const uint4 u = s_buf[v];
      float x[kVec<T>];
      unpack(u, x, T{});
      run.add(x, vec_max(u, x, T{}), scale2);
    }
    MaxSum acc = run.get();
    float gm = acc.m;
    for (int off = 1; off < span && off < 32; off <<= 1)
      gm = max_nan(gm, __shfl_xor_sync(0xffffffffu, gm, off));
    if (span <= 32) {
      if ((lane & (span - 1)) == 0) s_group[tid / span] = gm;
    } else if (lane == 0) {
      s_group[warp] = gm;
    }
    acc = warp_join(acc, scale2);
    if (lane == 0) s_warp[warp] = acc;
    __syncthreads();
    if (warp == 0) {
      acc = lane < threads / 32 ? s_warp[lane] : MaxSum{ninf, 0.0f};
      acc = warp_join(acc, scale2);
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

// Rows of more classes than this have a cluster each.
constexpr int kShortRow = 1024;

// Threads of a CTA for a share of `vecs` vectors: a few vectors each. At least 160: warps 1 to 4
// look at the entries while warp 0 sums them.
unsigned row_threads(int vecs) { return vecs > 2048 ? 512u : 256u; }

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

int launch_top_logits(const TopLogitsArgs& a, cudaStream_t stream) {
  if (a.dtype == SPLAX_F32) return launch_top_t<float>(a, stream);
  if (a.dtype == SPLAX_BF16) return launch_top_t<__nv_bfloat16>(a, stream);
  return launch_top_t<__half>(a, stream);
}

}  // namespace splax
