// The k largest logits of each row, with their classes and the row's log-sum-exp: what
// distillation keeps of a teacher.
//
// Bound: the logits are read once. Three kernels, by the length and the number of the rows:
//   up to 2047 classes    top_tile_kernel, a warp on tiles of rows in shared memory
//   longer, few rows      top_share_kernel, a cluster of CTAs on a row
//   longer, many rows     top_ring_kernel, a CTA on a row in chunks
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

// Keys above all but the k largest of a list in shared memory, by the threads that share it. `sync`
// is a barrier of theirs.
//
// Each of count <= kCounted keys counts those before it: the k largest go to `kept`, in order.
constexpr int kCounted = 512;
template <int THREADS>
__device__ __forceinline__ void sort_kept(const uint64_t* list, int count, int k, uint64_t* kept) {
  for (int i = threadIdx.x; i < count; i += THREADS) {
    const uint64_t key = list[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < count; ++j) rank += list[j] > key;
    if (rank < k) kept[rank] = key;
  }
}
// Any number of keys, k or more of them: the k-th largest by bisection, then the k largest go to
// the list's beginning in any order. `word` is shared; ends after a barrier.
template <int THREADS, typename Sync>
__device__ __forceinline__ void prune(uint64_t* list, int count, int k, uint64_t* kept, int* word,
                                      Sync sync) {
  uint64_t low = 0;  // keys differ, so exactly k reach the largest bound that k reach
  for (int bit = 63; bit >= 0; --bit) {
    const uint64_t at = low | (1ull << bit);
    sync();
    if (threadIdx.x == 0) *word = 0;
    sync();
    int n = 0;
    for (int i = threadIdx.x; i < count; i += THREADS) n += list[i] >= at;
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) atomicAdd(word, n);
    sync();
    if (*word >= k) low = at;
  }
  sync();
  if (threadIdx.x == 0) *word = 0;
  sync();
  for (int i = threadIdx.x; i < count; i += THREADS)
    if (list[i] >= low) kept[atomicAdd(word, 1)] = list[i];
  sync();
  for (int i = threadIdx.x; i < k; i += THREADS) list[i] = kept[i];
  sync();
}
// The logit of a key, exact but for the sign of a zero.
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = static_cast<uint32_t>(key >> 32);
  return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}

// Bound that at least k of the logits behind the threads' maxima `m` reach and few more do: the k-th
// largest of the maxima of 2 k groups of threads, or of as many as there are. -inf if fewer than k
// groups have one. `groups`: a float per group; ends after a barrier.
template <int THREADS, typename Sync>
__device__ __forceinline__ float kth_of_groups(float m, int k, float* groups, float* bound,
                                               Sync sync) {
  if (m != m) m = __int_as_float(0x7f800000);  // NaN counts as the largest
  int span = 32;  // threads of a group
  while (span > 1 && THREADS / span < 2 * k) span /= 2;
  const int have = THREADS / span;
  for (int off = 1; off < span; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if ((threadIdx.x & (span - 1)) == 0) groups[threadIdx.x / span] = m;
  if (threadIdx.x == 0) *bound = neg_inf();
  sync();
  for (int i = threadIdx.x; i < have; i += THREADS) {
    const float mine = groups[i];
    int before = 0;
#pragma unroll 4
    for (int j = 0; j < have; ++j) before += groups[j] > mine || (groups[j] == mine && j < i);
    if (before == k - 1) *bound = mine;
  }
  sync();
  return *bound;
}

// Of N vectors `stride` apart, the first one's first class being `cls`, what reaches the bound, or
// exceeds it where `strict`, to the list; `room` keys of it, the count goes on. NaN passes either
// test. Few vectors come here: a mask first, then its bits one by one from memory again.
template <typename T, int N>
__device__ __forceinline__ void push(const uint4* at, int stride, int cls, int classes,
                                     float bound, bool strict, uint64_t* list, int room,
                                     int* count) {
  constexpr int V = kVec<T>;
  uint32_t pass = 0;
#pragma unroll
  for (int q = 0; q < N; ++q) {
    float x[V];
    unpack(at[q * stride], x, T{});
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (strict ? !(x[i] <= bound) : !(x[i] < bound)) pass |= 1u << (q * V + i);
  }
#pragma unroll 1
  while (pass) {
    const int i = __ffs(pass) - 1;
    pass &= pass - 1;
    const int e = (i / V) * stride * V + i % V;
    if (cls + e < 0 || cls + e >= classes) continue;
    const int n = atomicAdd(count, 1);
    if (n < room) list[n] = order_key(to_f(reinterpret_cast<const T*>(at)[e]), cls + e);
  }
}

// Many long rows, read once: a CTA works through its rows alone. They come in chunks by bulk copies
// into a ring of slots, started by a warp of their own as slots fall free, the next row's while this
// one's end is worked out. The first chunk gives a bound (kth_of_groups); after 1, 2, 4, ... chunks
// the k largest of the list stay, and from there on only what exceeds the least of them is listed,
// since of equal logits the first stays: about k a time in a row in no particular order. A row that
// fills the list all the same (a rising one) is read again with the list cut back to the k largest
// after every vector of a thread.
//
// 2048 rows of 128,000 fp32, 64 kept: 0.28 ms, 58 % of the measured copy rate; the rest is listing (a
// warp stops for every vector that holds a candidate) and the rows' ends. Holding each row in a
// cluster's shared memory took 0.93 ms.
constexpr int kTopSlots = 2;
template <typename T, int THREADS, int CTAS>
__global__ void __launch_bounds__(THREADS + 32, CTAS)
top_ring_kernel(const T* logits, int64_t rows, int64_t row_stride, int classes, int k, Scale c,
                double inv_tau, T* values, int32_t* ids, float* lse, int chunks, int vecs,
                int slots) {
  constexpr int V = kVec<T>, kWarps = THREADS / 32, kBatch = 16 / V;
  constexpr int kRoom = THREADS * V + kDistillMaxK;  // a vector of every thread on top of k
  extern __shared__ uint4 s_buf[];                   // `slots` chunks of `vecs` vectors, the list
  __shared__ uint64_t s_kept[kDistillMaxK];
  __shared__ MaxSum s_warp[kWarps];
  __shared__ float s_group[THREADS], s_bound;
  __shared__ int s_count, s_word, s_late;
  __shared__ __align__(8) uint64_t s_full[kTopSlots], s_empty[kTopSlots];
  uint64_t* const list = reinterpret_cast<uint64_t*>(s_buf + slots * vecs);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float ninf = neg_inf();
  const int count = static_cast<int>((rows - blockIdx.x + gridDim.x - 1) / gridDim.x);
  if (tid == 0) {
    s_late = 0;
    for (int i = 0; i < slots; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], kWarps);
    }
  }
  pdl_enter();
  __syncthreads();
  const int64_t step = gridDim.x * row_stride;
  const T* z = logits + blockIdx.x * row_stride;
  int slot = 0;
  auto wait = [&](uint64_t* bar, uint32_t parity, bool rest = false) {
    if (!mbar_wait(bar, parity, rest)) s_late = 1;
  };

  if (warp == kWarps) {  // copies
    uint32_t parity = 1;
    for (int i = 0; i < count; ++i, z += step) {
      const RowShare<T> row = row_share(z, classes, 0, 1);
      const ShareEnds<T> ends = load_ends(row, classes);
      const int b0 = row.cls0 < 0 ? 1 : 0, b1 = row.cls0 + row.v1 * V > classes ? row.v1 - 1 : row.v1;
      for (int j = 0; j < chunks; ++j) {
        const int at = j * vecs, from = max(at, b0), to = min(at + vecs, b1);
        wait(&s_empty[slot], parity, true);
        const int e = ends.at - at * V;
        if (ends.at >= 0 && e >= 0 && e < vecs * V)
          reinterpret_cast<T*>(s_buf + slot * vecs)[e] = ends.x;
        fence_async();  // a later copy into the slot comes after that
        __syncwarp();
        if (lane == 0) {
          const uint32_t bytes = to > from ? 16u * static_cast<uint32_t>(to - from) : 0u;
          mbar_expect(&s_full[slot], bytes);
          if (bytes)
            bulk_load(s_buf + slot * vecs + (from - at), row.first + from * V, bytes, &s_full[slot]);
        }
        if (++slot == slots) slot = 0, parity ^= 1;
      }
    }
    return;
  }

  auto sync = [] { pair_sync<THREADS>(1); };
  uint32_t parity = 0;
  for (int i = 0; i < count; ++i, z += step) {
    const int64_t r = blockIdx.x + static_cast<int64_t>(i) * gridDim.x;
    const RowShare<T> row = row_share(z, classes, 0, 1);
    float bound = ninf;
    bool strict = false;
    if (tid == 0) s_count = 0;
    Running run;
    // a chunk's vectors to the list, and to the sum as well
    auto scan = [&](int j, auto sums) {
      const uint4* buf = s_buf + slot * vecs;
      const int size = min(vecs, row.v1 - j * vecs), cls0 = row.cls0 + j * vecs * V;
      auto several = [&](auto n, int v) {
        constexpr int N = decltype(n)::value;
        uint4 u[N];
        float m[N];
#pragma unroll
        for (int q = 0; q < N; ++q) u[q] = buf[v + q * THREADS];
#pragma unroll
        for (int q = 0; q < N; ++q) m[q] = vec_max(u[q], T{});
        float most = m[0];
#pragma unroll
        for (int q = 1; q < N; ++q) most = max_nan(most, m[q]);
        if (strict ? !(most <= bound) : !(most < bound))
          push<T, N>(buf + v, THREADS, cls0 + v * V, classes, bound, strict, list, kRoom, &s_count);
        if (decltype(sums)::value) {
          float x[N * V];
#pragma unroll
          for (int q = 0; q < N; ++q) {
            float y[V];
            unpack(u[q], y, T{});
#pragma unroll
            for (int p = 0; p < V; ++p) x[q * V + p] = y[p];
          }
          run.add(x, most, c);
        }
      };
      int v = tid;
      for (; v + (kBatch - 1) * THREADS < size; v += kBatch * THREADS) several(Int<kBatch>{}, v);
      for (; v < size; v += THREADS) several(Int<1>{}, v);
    };
    auto sum = [&] {  // the first chunk's vectors to the sum
      const uint4* buf = s_buf + slot * vecs;
      const int size = min(vecs, row.v1);
      int v = tid;
      for (; v + (kBatch - 1) * THREADS < size; v += kBatch * THREADS)
        add_vectors<T, kBatch>(run, buf + v, THREADS, c);
      for (; v < size; v += THREADS) add_vectors<T, 1>(run, buf + v, THREADS, c);
    };
    for (int j = 0; j < chunks; ++j) {
      wait(&s_full[slot], parity);
      if (j == 0) {
        sum();
        bound = kth_of_groups<THREADS>(run.m, k, s_group, &s_bound, sync);
        scan(j, Int<0>{});
      } else {
        scan(j, Int<1>{});
      }
      if (j + 1 < chunks && (j & (j + 1)) == 0) {  // after 1, 2, 4, ... chunks
        sync();
        const int n = s_count;
        sync();  // before the next chunk's are counted
        if (n <= kCounted) {
          sort_kept<THREADS>(list, n, k, s_kept);
          sync();
          bound = key_value(s_kept[k - 1]);
          strict = true;
          for (int q = tid; q < k; q += THREADS) list[q] = s_kept[q];
          if (tid == 0) s_count = k;
          sync();
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_empty[slot]);
      if (++slot == slots) slot = 0, parity ^= 1;
    }
    const MaxSum part = warp_join(run.get(c), c);
    if (lane == 0) s_warp[warp] = part;
    sync();
    int n = s_count;
    if (n > kRoom) {
      // from memory, with the list cut back to the k largest whenever it holds more
      bound = ninf;
      strict = false;
      sync();
      if (tid == 0) s_count = 0;
      sync();
      for (int v0 = 0; v0 < row.v1; v0 += THREADS) {
        const int v = v0 + tid, cls = row.cls0 + v * V;
        if (v < row.v1) {
          uint4 u;
          T* e = reinterpret_cast<T*>(&u);
#pragma unroll
          for (int q = 0; q < V; ++q)
            e[q] = cls + q >= 0 && cls + q < classes ? z[cls + q] : from_f<T>(ninf);
          push<T, 1>(&u, 0, cls, classes, bound, strict, list, kRoom, &s_count);
        }
        sync();
        n = s_count;
        if (n > k) {
          prune<THREADS>(list, n, k, s_kept, &s_word, sync);
          n = k;
          // the least of them
          uint64_t least = ~0ull;
          for (int q = 0; q < k; ++q) least = list[q] < least ? list[q] : least;
          bound = key_value(least);
          strict = true;
          if (tid == 0) s_count = k;
        }
        sync();
      }
    } else if (n > kCounted) {
      prune<THREADS>(list, n, k, s_kept, &s_word, sync);
      n = k;
    }
    sort_kept<THREADS>(list, n, k, s_kept);
    sync();
    for (int q = tid; q < k; q += THREADS) {
      const int cls = key_class(s_kept[q]);
      const bool good = cls >= 0 && cls < classes;  // always, unless a copy was late
      ids[r * k + q] = good ? cls : -1;
      values[r * k + q] = good ? z[cls] : from_f<T>(__int_as_float(0x7fc00000));
    }
    if (warp == 0) {
      const MaxSum all = warp_join(lane < kWarps ? s_warp[lane] : MaxSum{ninf, 0.0f}, c);
      if (lane == 0)
        lse[r] = s_late ? __int_as_float(0x7fc00000)
                        : all.m == ninf ? ninf : static_cast<float>(ln_of(ref_of(all.m, c), inv_tau) + ln_of(all.s));
    }
    sync();
  }
}

// Few long rows: a cluster of CTAs takes one row, each CTA a share of it in shared memory, which
// spreads a row over up to eight SMs. Each finds the k largest of its share; what the cluster's
// first CTA sorts of them is what reaches the largest of the shares' k-th. Bound by latency:
// one row of 100,003 bf16, 50 kept, 19 us.
constexpr int kTopThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kTopThreads)
top_share_kernel(const T* logits, int64_t row_stride, int classes, int k, Scale c, double inv_tau,
                 T* values, int32_t* ids, float* lse) {
  constexpr int V = kVec<T>, kWarps = kTopThreads / 32, kBatch = 16 / V;
  constexpr int kRoom = 8 * kDistillMaxK;
  extern __shared__ uint4 s_buf[];
  __shared__ uint64_t s_list[kRoom], s_kept[kDistillMaxK];
  __shared__ __align__(8) uint64_t s_bar;
  __shared__ __align__(8) MaxSum s_sum;
  __shared__ MaxSum s_warp[kWarps];
  __shared__ float s_group[kTopThreads], s_bound;
  __shared__ int s_count, s_word, s_kept_count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const float ninf = neg_inf();
  auto sync = [] { __syncthreads(); };
  const int64_t r = blockIdx.x / size;
  const T* z = logits + r * row_stride;
  const RowShare<T> share = row_share(z, classes, rank, size);
  const int n = share.v1 - share.v0;
  if (tid == 0) {
    mbar_init(&s_bar, 1);
    s_count = 0;
  }
  pdl_enter();
  if (tid == 0) load_share(share, classes, s_buf, &s_bar);
  if (warp == 1) store_ends(load_ends(share, classes), s_buf);
  __syncthreads();
  const bool late = !mbar_wait(&s_bar, 0);
  Running run;
  int v = tid;
  for (; v + (kBatch - 1) * kTopThreads < n; v += kBatch * kTopThreads)
    add_vectors<T, kBatch>(run, s_buf + v, kTopThreads, c);
  for (; v < n; v += kTopThreads) add_vectors<T, 1>(run, s_buf + v, kTopThreads, c);
  const MaxSum part = warp_join(late ? poison() : run.get(c), c);
  if (lane == 0) s_warp[warp] = part;
  const float bound = kth_of_groups<kTopThreads>(run.m, k, s_group, &s_bound, sync);
  for (v = tid; v < n; v += kTopThreads) {
    const uint4 u = s_buf[v];
    if (!(vec_max(u, T{}) < bound))
      push<T, 1>(s_buf + v, 0, share.cls0 + v * V, classes, bound, false, s_list, kRoom, &s_count);
  }
  if (warp == 0) {
    const MaxSum all = warp_join(lane < kWarps ? s_warp[lane] : MaxSum{ninf, 0.0f}, c);
    if (lane == 0) s_sum = all;
  }
  __syncthreads();
  int found = s_count;
  if (found > kRoom) {
    // many equal logits: the share's k-th largest key by bisection
    uint64_t low = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t at = low | (1ull << bit);
      __syncthreads();
      if (tid == 0) s_word = 0;
      __syncthreads();
      int reach = 0;
      for (v = tid; v < n; v += kTopThreads) {
        float x[V];
        unpack(s_buf[v], x, T{});
#pragma unroll
        for (int q = 0; q < V; ++q) {
          const int cls = share.cls0 + v * V + q;
          reach += cls >= 0 && cls < classes && order_key(x[q], cls) >= at;
        }
      }
      reach = __reduce_add_sync(0xffffffffu, reach);
      if (lane == 0) atomicAdd(&s_word, reach);
      __syncthreads();
      if (s_word >= k) low = at;
    }
    __syncthreads();
    if (tid == 0) s_count = 0;
    __syncthreads();
    for (v = tid; v < n; v += kTopThreads) {
      float x[V];
      unpack(s_buf[v], x, T{});
#pragma unroll
      for (int q = 0; q < V; ++q) {
        const int cls = share.cls0 + v * V + q;
        if (cls >= 0 && cls < classes && order_key(x[q], cls) >= low)
          s_list[atomicAdd(&s_count, 1)] = order_key(x[q], cls);
      }
    }
    __syncthreads();
    found = s_count;
  }
  if (found > kCounted) {
    prune<kTopThreads>(s_list, found, k, s_kept, &s_word, sync);
    found = k;
  }
  sort_kept<kTopThreads>(s_list, found, k, s_kept);
  if (tid == 0) s_kept_count = min(found, k);
  __syncthreads();
  if (size > 1) {
    cluster_sync();  // every CTA's list and sum are there
    if (rank == 0) {
      if (tid == 0) s_count = 0;
      if (warp == 0) {
        uint64_t at = 0, least = 0;
        if (lane < static_cast<int>(size)) {
          at = cluster_load(cluster_addr(&s_sum, lane));
          if (static_cast<int>(cluster_load_u32(cluster_addr(&s_kept_count, lane))) == k)
            least = cluster_load(cluster_addr(&s_kept[k - 1], lane));
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
          const uint64_t o = __shfl_xor_sync(0xffffffffu, least, off);
          least = o > least ? o : least;
        }
        const MaxSum mine = lane < static_cast<int>(size)
                                ? MaxSum{__uint_as_float(static_cast<uint32_t>(at)),
                                         __uint_as_float(static_cast<uint32_t>(at >> 32))}
                                : MaxSum{ninf, 0.0f};
        const MaxSum all = warp_join(mine, c);
        __syncwarp();
        if (lane == 0) {
          s_sum = all;
          s_list[kRoom - 1] = least;  // the shares' lists are shorter than that
        }
      }
      __syncthreads();
      const uint64_t least = s_list[kRoom - 1];
      __syncthreads();
      for (int i = tid; i < static_cast<int>(size) * k; i += kTopThreads) {
        const uint32_t q = i / k;
        if (i % k < static_cast<int>(cluster_load_u32(cluster_addr(&s_kept_count, q)))) {
          const uint64_t key = cluster_load(cluster_addr(&s_kept[i % k], q));
          if (key >= least) s_list[atomicAdd(&s_count, 1)] = key;
        }
      }
      __syncthreads();
      found = s_count;
    }
    cluster_sync();  // the lists are read
    if (rank != 0) return;
    sort_kept<kTopThreads>(s_list, found, k, s_kept);
    __syncthreads();
  }
  for (int q = tid; q < k; q += kTopThreads) {
    const int cls = key_class(s_kept[q]);
    const bool good = cls >= 0 && cls < classes;  // always, unless a copy was late
    ids[r * k + q] = good ? cls : -1;
    values[r * k + q] = good ? z[cls] : from_f<T>(__int_as_float(0x7fc00000));
  }
  if (tid == 0) lse[r] = s_sum.m == ninf ? ninf : static_cast<float>(ln_of(ref_of(s_sum.m, c), inv_tau) + ln_of(s_sum.s));
}

// Keys of 16-bit logits in rows of fewer than 65536 classes fit 32 bits, others take 64.
__device__ __forceinline__ uint32_t short_key(__nv_bfloat16 x, int cls) {
  const uint32_t o = order_bits(to_f(x));
  return (o & 0xffff0000u) | (0xffffu - static_cast<uint32_t>(cls));
}
__device__ __forceinline__ uint32_t short_key(__half x, int cls) {
  uint32_t u = __half_as_ushort(x);
  if ((u & 0x7fffu) == 0) u = 0;  // the zeros are equal
  u = (u & 0x7fffu) > 0x7c00u ? 0xffffu : (u & 0x8000u) ? u ^ 0xffffu : u | 0x8000u;
  return u << 16 | (0xffffu - static_cast<uint32_t>(cls));
}
__device__ __forceinline__ uint64_t short_key(float x, int cls) { return order_key(x, cls); }
__device__ __forceinline__ int short_key_class(uint32_t key) { return 0xffff - (key & 0xffff); }
__device__ __forceinline__ int short_key_class(uint64_t key) { return key_class(key); }
template <typename T>
using ShortKey = decltype(short_key(T{}, 0));

template <typename K>
struct alignas(16) Four {
  K a, b, c, d;
};

struct TopPlan {
  int rows;   // of a tile
  int pitch;  // of a row in a stage where rows are copied one by one, 0: a tile at once
  int stage;  // bytes
  int room;   // candidates of a row, a multiple of four
  int warp;   // bytes: the stages, then the candidates of a pass and their places
};

// The k-th largest of the maxima of the row's G H heaps, -inf if fewer than k are not empty.
template <int G, int H>
__device__ __forceinline__ float kth_of_heaps(const float (&h)[8], int k) {
  int larger[H] = {};
#pragma unroll 4
  for (int from = 0; from < G; ++from)
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const float o = __shfl_sync(0xffffffffu, h[i], from, G);
#pragma unroll
      for (int j = 0; j < H; ++j) larger[j] += o > h[j];
    }
  float least = __int_as_float(0x7f800000);
#pragma unroll
  for (int i = 0; i < H; ++i)
    if (larger[i] < k) least = fminf(least, h[i]);
#pragma unroll
  for (int off = G / 2; off > 0; off >>= 1)
    least = fminf(least, __shfl_xor_sync(0xffffffffu, least, off));
  return least;
}

// Short rows: a warp works alone on tiles of consecutive rows, which come by bulk copies a tile
// ahead; G lanes take a row, up to E classes a lane, in registers. A lane's classes fall into
// groups of four, whose maxima are dealt into heaps, 2 k or more in a row; the k-th largest of the
// heaps' maxima is a bound that at least k logits reach and few more do (about 1.4 k in a row in no
// particular order). Those go to a list in shared memory, where each counts the ones before it.
// Where the list is too short (many equal logits) the warp finds the k largest one after another.
//
// Bound by instruction issue: about 200 a row of 150 fp16 classes with 8 kept, half of them for listing,
// ordering and writing the 8. 1080p x 150 fp16 0.57 ms (19 % of the measured copy rate), 800 x 800 x 512 bf16 with 16
// kept 0.56 ms (20 %); the k largest one after another for all rows took 22.3 and 16.6 ms. One list
// for all rows of a warp, shared out evenly, was 11 % slower.
template <typename T, int G, int E>
__global__ void __launch_bounds__(32 * kTileWarps, 4)
top_tile_kernel(const T* logits, int64_t all_rows, int64_t row_stride, int classes, int k,
                int heaps, TopPlan plan, Scale c, double inv_tau, T* values, int32_t* ids,
                float* lse) {
  constexpr int P = 32 / G, Q = E / 4;
  using Key = ShortKey<T>;
  extern __shared__ uint4 s_buf[];
  __shared__ __align__(8) uint64_t s_bar[kTileWarps][kTileStages];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row_in_pass = lane / G, l = lane % G;
  const float ninf = neg_inf();
  char* const mine = reinterpret_cast<char*>(s_buf) + warp * plan.warp;
  Key* const list = reinterpret_cast<Key*>(mine + kTileStages * plan.stage) + row_in_pass * plan.room;
  uint16_t* const places = reinterpret_cast<uint16_t*>(list - row_in_pass * plan.room + P * plan.room) +
                           row_in_pass * plan.room;
  uint64_t* const bars = s_bar[warp];
  if (lane < kTileStages) mbar_init(&bars[lane], 1);
  __syncwarp();
  pdl_enter();
  const uintptr_t base = reinterpret_cast<uintptr_t>(logits);
  const int64_t stride = row_stride * static_cast<int64_t>(sizeof(T));  // bytes
  const int width = classes * static_cast<int>(sizeof(T));
  const uintptr_t limit = base + (all_rows - 1) * stride + width;
  const int64_t tiles = (all_rows + plan.rows - 1) / plan.rows;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTileWarps;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kTileWarps + warp;
  auto load = [&](int64_t tile, int at) {
    const int64_t r0 = tile * plan.rows, r1 = min(r0 + plan.rows, all_rows);
    char* s = mine + at * plan.stage;
    auto part = [&](int64_t from, int64_t to, int i) {
      return part_of(s + i * plan.pitch, base, base + from * stride, base + (to - 1) * stride + width,
                     limit);
    };
    uint32_t bytes = 0;
    if (plan.pitch == 0) {
      const Part q = part(r0, r1, 0);
      if (lane == 0) {
        mbar_expect(&bars[at], static_cast<uint32_t>(q.e16 - q.b16));
        load_part(q, &bars[at]);
      }
      return;
    }
    for (int64_t r = r0 + lane; r < r1; r += 32) {
      const Part q = part(r, r + 1, static_cast<int>(r - r0));
      bytes += static_cast<uint32_t>(q.e16 - q.b16);
    }
    bytes = __reduce_add_sync(0xffffffffu, bytes);
    if (lane == 0) mbar_expect(&bars[at], bytes);
    __syncwarp();
    for (int64_t r = r0 + lane; r < r1; r += 32)
      load_part(part(r, r + 1, static_cast<int>(r - r0)), &bars[at]);
  };
  if (first < tiles) load(first, 0);
  int at = 0;
  uint32_t parity = 0;
  for (int64_t tile = first; tile < tiles; tile += step) {
    const int next = at + 1 == kTileStages ? 0 : at + 1;
    fence_async();  // what plain loads have put there
    __syncwarp();
    if (tile + step < tiles) load(tile + step, next);
    const bool late = __any_sync(0xffffffffu, !mbar_wait(&bars[at], parity));
    __syncwarp();
    const int64_t r0 = tile * plan.rows;
    const int rows = static_cast<int>(min(static_cast<int64_t>(plan.rows), all_rows - r0));
    const char* s = mine + at * plan.stage;
    const int in0 = static_cast<int>(base + r0 * stride) & 15;
    for (int from = 0; from < rows; from += P) {
      const bool there = from + row_in_pass < rows;
      const int row = there ? from + row_in_pass : 0;
      const T* const z = reinterpret_cast<const T*>(
          s + (plan.pitch ? row * plan.pitch + (static_cast<int>(base + (r0 + row) * stride) & 15)
                          : in0 + row * static_cast<int>(stride)));
      // two neighbouring classes at a time, from the even address at or before the row's first
      const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(z) / sizeof(T)) & 1;
      const T* const zw = z - lead;
      // the row, the maxima of the lane's groups of four, and which of its classes exist
      float x[E], top[Q];
      uint64_t real = 0;
#pragma unroll
      for (int j = 0; j < E; j += 8) {
        top[j / 4] = top[j / 4 + 1] = ninf;
        if ((j + 8) * G <= classes) {  // the row goes on: no test per class
#pragma unroll
          for (int i = j; i < j + 8; i += 2) {
            load_pair(zw + i * G + 2 * l, x[i], x[i + 1]);
            if (i == 0 && l == 0 && lead) x[i] = ninf;
            top[i / 4] = max3_nan(top[i / 4], x[i], x[i + 1]);
          }
          real |= 0xffull << j;
        } else if (j * G < classes + lead) {
#pragma unroll
          for (int i = j; i < j + 8; ++i) {
            const int cls = (i & ~1) * G + 2 * l + (i & 1) - lead;
            x[i] = ninf;
            if (cls >= 0 && cls < classes) {
              x[i] = to_f(z[cls]);
              real |= 1ull << i;
            }
            top[i / 4] = max_nan(top[i / 4], x[i]);
          }
        }
      }
      if (l == 0 && lead) real &= ~1ull;
      float m = top[0];
#pragma unroll
      for (int i = 1; i < Q; ++i) m = max_nan(m, top[i]);
      m = group_max<G>(m);
      const Ref r = ref_of(m, c);
      // the bound; NaN counts as the largest
      float bound;
      {
        float h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = ninf;
#pragma unroll
        for (int i = 0; i < Q; ++i) {
          const float t = top[i] != top[i] ? __int_as_float(0x7f800000) : top[i];
          h[i % 8] = fmaxf(h[i % 8], t);
        }
        if (heaps == 8) {
          bound = kth_of_heaps<G, 8>(h, k);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) h[i] = fmaxf(h[i], h[i + 4]);
          if (heaps == 4) {
            bound = kth_of_heaps<G, 4>(h, k);
          } else {
            h[0] = fmaxf(h[0], h[2]);
            h[1] = fmaxf(h[1], h[3]);
            if (heaps == 2) {
              bound = kth_of_heaps<G, 2>(h, k);
            } else {
              h[0] = fmaxf(h[0], h[1]);
              bound = kth_of_heaps<G, 1>(h, k);
            }
          }
        }
      }
      uint64_t reach = 0;
      float2 sum[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
#pragma unroll
      for (int j = 0; j < E; j += 8) {
        if (j * G < classes + lead) {
          if (r.plain()) {
#pragma unroll
            for (int i = j; i < j + 8; i += 2) {
              const float2 t = exponent2({x[i], x[i + 1]}, r.ms, c);
              sum[i / 2 & 1] = add2(sum[i / 2 & 1], {ex2_approx(t.x), ex2_approx(t.y)});
            }
          } else {
#pragma unroll
            for (int i = j; i < j + 8; ++i) sum[0].x += ex2_approx(exponent(x[i], r, c));
          }
#pragma unroll
          for (int i = j; i < j + 8; ++i)
            if (!(x[i] < bound)) reach |= 1ull << i;
        }
      }
      reach &= real;
      const float2 both = add2(sum[0], sum[1]);
      const float total = group_sum<G>(both.x + both.y);
      if (there && l == 0)
        lse[r0 + row] = late ? __int_as_float(0x7fc00000)
                             : m == ninf ? ninf : static_cast<float>(ln_of(r, inv_tau) + ln_of(total));
      if (!there) reach = 0;
      // the list
      int count = __popcll(reach), before = count;
#pragma unroll
      for (int off = 1; off < G; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, before, off, G);
        if (l >= off) before += o;
      }
      const int found = __shfl_sync(0xffffffffu, before, G - 1, G);
      T* const v_out = values + (r0 + row) * k;
      int32_t* const i_out = ids + (r0 + row) * k;
      if (!__any_sync(0xffffffffu, found > plan.room)) {
        // what a lane found as places, which the row's lanes then share out
        uint16_t* to = places + before - count;
#pragma unroll
        for (int half = 0; half < 64; half += 32) {
          uint32_t bits = static_cast<uint32_t>(reach >> half);
          while (bits) {
            *to++ = static_cast<uint16_t>(l * 64 + half + __ffs(bits) - 1);
            bits &= bits - 1;
          }
        }
        __syncwarp();
        const int quads = (found + 3) / 4;
        for (int i = l; i < 4 * quads; i += G) {
          Key key = 0;
          if (i < found) {
            const int place = places[i], e = place & 63;
            const int cls = (e & ~1) * G + 2 * (place >> 6) + (e & 1) - lead;
            key = short_key(z[cls], cls);
          }
          list[i] = key;
        }
        __syncwarp();
        for (int i = l; i < found; i += G) {
          const Key key = list[i];
          int rank = 0;
          for (int j = 0; j < quads; ++j) {
            const Four<Key> f = reinterpret_cast<const Four<Key>*>(list)[j];
            rank += (f.a > key) + (f.b > key) + (f.c > key) + (f.d > key);
          }
          if (rank < k) {
            const int cls = short_key_class(key);
            v_out[rank] = z[cls];
            i_out[rank] = cls;
          }
        }
        __syncwarp();
      } else {
        Key last = ~Key{0};
        for (int e = 0; e < k; ++e) {
          Key best = 0;
          for (int cls = l; cls < classes; cls += G) {
            const Key key = short_key(z[cls], cls);
            if ((e == 0 || key < last) && key > best) best = key;
          }
#pragma unroll
          for (int off = G / 2; off > 0; off >>= 1) {
            const Key o = __shfl_xor_sync(0xffffffffu, best, off);
            best = o > best ? o : best;
          }
          last = best;
          const int cls = short_key_class(best);
          if (there && l == 0 && cls < classes) {
            v_out[e] = z[cls];
            i_out[e] = cls;
          }
        }
      }
    }
    at = next;
    if (at == 0) parity ^= 1;
  }
}

TopPlan plan_top(const TopLogitsArgs& a, int G, int size, int key, int sms) {
  const int pass = 32 / G;
  const int64_t stride = a.row_stride * size, width = static_cast<int64_t>(a.classes) * size;
  // rows far apart are copied one by one; close ones with what lies between
  const bool apart = stride > width + width / 4 + 32;
  TopPlan t;
  t.pitch = apart ? static_cast<int>((width + 31) & ~int64_t{15}) : 0;
  int64_t rows = kTileBytes / (apart ? t.pitch : stride);
  const int64_t share = (a.rows + sms * 16 - 1) / (sms * 16);
  if (rows > share) rows = share + pass - 1;
  rows = rows / pass * pass;
  if (rows < pass) rows = pass;
  t.rows = static_cast<int>(rows);
  t.stage = apart ? t.rows * t.pitch
                  : static_cast<int>(((rows - 1) * stride + width + 30) & ~int64_t{15});
  t.room = a.k <= 16 ? 64 : 4 * a.k;
  if (t.room > a.classes) t.room = (a.classes + 3) & ~3;
  t.warp = (kTileStages * t.stage + pass * t.room * (key + 2) + 15) & ~15;
  return t;
}

template <typename T, int G, int E>
void launch_top_tiles(const TopLogitsArgs& a, const TopPlan& t, cudaStream_t stream) {
  const int sms = sm_count();
  const double inv = 1.0 / a.temperature;
  const int64_t tiles = (a.rows + t.rows - 1) / t.rows;
  int per_sm = kSharedMost / (kTileWarps * t.warp + 1536);
  per_sm = per_sm < 1 ? 1 : per_sm > 4 ? 4 : per_sm;
  int64_t grid = (tiles + kTileWarps - 1) / kTileWarps;
  if (grid > sms * per_sm) grid = sms * per_sm;
  int heaps = 1;
  while (heaps < 8 && heaps * G < 2 * a.k) heaps *= 2;
  launch_clusters(top_tile_kernel<T, G, E>, static_cast<unsigned>(grid), 1, 32 * kTileWarps,
                  kTileWarps * t.warp, stream, static_cast<const T*>(a.logits), a.rows, a.row_stride, a.classes, a.k, heaps, t,
                  scale_of(a.temperature), inv,
                  static_cast<T*>(a.values), a.ids, a.lse);
}

// Lanes to a row: of those that hold it in registers, make k heaps and fit shared memory with room
// for a second CTA, the cheapest.
template <typename T>
void launch_top_short(const TopLogitsArgs& a, cudaStream_t stream) {
  const int sms = sm_count(), size = sizeof(T), key = size == 4 ? 8 : 4;
  int G = 32;
  TopPlan t = plan_top(a, 32, size, key, sms);
  double least = 1e30;
  for (int g = 1; g <= 32; g *= 2) {
    const TopPlan u = plan_top(a, g, size, key, sms);
    if (a.classes >= 40 * g || a.k > 8 * g || kTileWarps * u.warp > kSharedMost / 2 - 2048) continue;
    const double cost = tile_cost(g, a.classes, u.pitch ? u.pitch : a.row_stride * size, size);
    if (cost < least) least = cost, G = g, t = u;
  }
  if (a.classes >= 1280) return launch_top_tiles<T, 32, 64>(a, t, stream);
  switch (G) {
    case 1: return launch_top_tiles<T, 1, 40>(a, t, stream);
    case 2: return launch_top_tiles<T, 2, 40>(a, t, stream);
    case 4: return launch_top_tiles<T, 4, 40>(a, t, stream);
    case 8: return launch_top_tiles<T, 8, 40>(a, t, stream);
    case 16: return launch_top_tiles<T, 16, 40>(a, t, stream);
    default: return launch_top_tiles<T, 32, 40>(a, t, stream);
  }
}

// Five small CTAs an SM, whose row ends hide behind one another's chunks, at any length: 2048 rows of
// 128,000 bf16 take 232 us, with one CTA of 512 threads and chunks of 50 KB 316; 16,000 rows of 20,000
// bf16 310 and 566.
template <typename T>
void launch_top_ring(const TopLogitsArgs& a, cudaStream_t stream) {
  constexpr int THREADS = 128, CTAS = 5, SLOTS = kTopSlots, EACH = 7;
  const double inv = 1.0 / a.temperature;
  const int all = row_share_vecs(a.classes, kVec<T>, 1), most = EACH * THREADS + 32;
  const int chunks = (all + most - 1) / most, vecs = ((all + chunks - 1) / chunks + 31) & ~31;
  const int64_t fit = static_cast<int64_t>(sm_count()) * CTAS;
  const size_t smem = 16 * static_cast<size_t>(vecs) * SLOTS + 8 * (THREADS * kVec<T> + kDistillMaxK);
  launch_clusters(top_ring_kernel<T, THREADS, CTAS>,
                  static_cast<unsigned>(a.rows < fit ? a.rows : fit), 1, THREADS + 32, smem, stream,
                  static_cast<const T*>(a.logits), a.rows, a.row_stride, a.classes, a.k,
                  scale_of(a.temperature), inv,
                  static_cast<T*>(a.values), a.ids, a.lse, chunks, vecs, SLOTS);
}

template <typename T>
int launch_top_t(const TopLogitsArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return 0;
  const double inv = 1.0 / a.temperature;
  if (a.classes < 2048) {  // 2000 x 100,000 rows bf16 210 us, by the ring 580
    launch_top_short<T>(a, stream);
    return 1;
  }
  const Scale c = scale_of(a.temperature);
  const T* z = static_cast<const T*>(a.logits);
  T* values = static_cast<T*>(a.values);
  if (a.rows < sm_count()) {  // 120 rows of 65,537 fp32: 24 us, by the ring 32
    const unsigned size =
        row_cluster(a.rows, a.classes * static_cast<int64_t>(sizeof(T)), sm_count());
    launch_clusters(top_share_kernel<T>, static_cast<unsigned>(a.rows), size, kTopThreads,
                    16 * row_share_vecs(a.classes, kVec<T>, size), stream, z, a.row_stride,
                    a.classes, a.k, c, inv, values, a.ids, a.lse);
  } else {
    launch_top_ring<T>(a, stream);
  }
  return 1;
}

}  // namespace

int launch_top_logits(const TopLogitsArgs& a, cudaStream_t stream) {
  if (a.dtype == SPLAX_F32) return launch_top_t<float>(a, stream);
  if (a.dtype == SPLAX_BF16) return launch_top_t<__nv_bfloat16>(a, stream);
  return launch_top_t<__half>(a, stream);
}

}  // namespace splax
