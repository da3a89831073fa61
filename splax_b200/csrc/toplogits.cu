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

struct TopPlan {
  int rows;   // of a tile
  int pitch;  // of a row in a stage where rows are copied one by one, 0: a tile at once
  int stage;  // bytes
  int room;   // candidates of a row
  int warp;   // bytes: the stages, then the candidates of a pass
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
template <typename T, int G, int E>
__global__ void __launch_bounds__(32 * kTileWarps, 4)
top_tile_kernel(const T* logits, int64_t all_rows, int64_t row_stride, int classes, int k,
                int heaps, TopPlan plan, float c, float inv_tau, T* values, int32_t* ids,
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
    const bool late = !mbar_wait(&bars[at], parity);
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
      const float2 c2 = splat2(c), n2 = splat2(-r.ms);
#pragma unroll
      for (int j = 0; j < E; j += 8) {
        if (j * G < classes + lead) {
          if (r.plain()) {
#pragma unroll
            for (int i = j; i < j + 8; i += 2) {
              const float2 t = fma2({x[i], x[i + 1]}, c2, n2);
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
                             : m == ninf ? ninf : fmaf(m, inv_tau, logf(total));
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
        Key* to = list + before - count;
        while (reach) {
          const int i = __ffsll(static_cast<long long>(reach)) - 1;
          reach &= reach - 1;
          const int cls = (i & ~1) * G + 2 * l + (i & 1) - lead;
          *to++ = short_key(z[cls], cls);
        }
        __syncwarp();
        for (int i = l; i < found; i += G) {
          const Key key = list[i];
          int rank = 0;
          for (int j = 0; j < found; ++j) rank += list[j] > key;
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

unsigned row_threads(int vecs) { return vecs > 2048 ? 512u : 256u; }

TopPlan plan_top(const TopLogitsArgs& a, int G, int size, int key, int sms) {
  const int pass = 32 / G;
  const int64_t stride = a.row_stride * size, width = static_cast<int64_t>(a.classes) * size;
  // rows far apart are copied one by one; close ones with what lies between
  const bool apart = stride > width + width / 4 + 32;
  TopPlan t;
  t.pitch = apart ? static_cast<int>((width + 31) & ~int64_t{15}) : 0;
  int64_t rows = 3 * 1024 / (apart ? t.pitch : stride);
  const int64_t share = (a.rows + sms * 16 - 1) / (sms * 16);
  if (rows > share) rows = share;
  rows = (rows + pass - 1) / pass * pass;
  if (rows < pass) rows = pass;
  t.rows = static_cast<int>(rows);
  t.stage = apart ? t.rows * t.pitch
                  : static_cast<int>(((rows - 1) * stride + width + 30) & ~int64_t{15});
  t.room = a.k <= 16 ? 64 : 4 * a.k;
  if (t.room > a.classes) t.room = (a.classes + 3) & ~3;
  t.warp = (kTileStages * t.stage + pass * t.room * key + 15) & ~15;
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
                  static_cast<float>(1.4426950408889634 * inv), static_cast<float>(inv),
                  static_cast<T*>(a.values), a.ids, a.lse);
}

// As few lanes to a row as hold it in registers, make k heaps, fit shared memory with room for a
// second CTA and do not meet in the banks more than four at a time.
template <typename T>
void launch_top_short(const TopLogitsArgs& a, cudaStream_t stream) {
  const int sms = sm_count();
  int G = 1;
  TopPlan t;
  for (;; G *= 2) {
    t = plan_top(a, G, sizeof(T), sizeof(T) == 4 ? 8 : 4, sms);
    const int64_t pitch = t.pitch ? t.pitch : a.row_stride * static_cast<int64_t>(sizeof(T));
    if (G == 32 || (a.classes < 40 * G && a.k <= 8 * G &&
                    kTileWarps * t.warp <= kSharedMost / 2 - 2048 &&
                    bank_conflicts(G, pitch, sizeof(T)) <= 4))
      break;
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

template <typename T>
int launch_top_t(const TopLogitsArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return 0;
  const double inv = 1.0 / a.temperature;
  if (a.classes < 2048) {
    launch_top_short<T>(a, stream);
    return 1;
  }
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

}  // namespace

int launch_top_logits(const TopLogitsArgs& a, cudaStream_t stream) {
  if (a.dtype == SPLAX_F32) return launch_top_t<float>(a, stream);
  if (a.dtype == SPLAX_BF16) return launch_top_t<__nv_bfloat16>(a, stream);
  return launch_top_t<__half>(a, stream);
}

}  // namespace splax
