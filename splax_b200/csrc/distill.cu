// Distillation from a teacher's top logits, the student's side: the divergence of its softmax from the
// distribution that the teacher's entries give, and the gradient.
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
// Sums and probabilities are fp32, a row's loss and the sum over rows fp64; the gradient is rounded
// once, to the logits' type, with the cotangent in it (a cotangent other than one multiplies an fp32
// gradient that is there already, distill_scale_kernel, which rounds it again). Maxima propagate NaN, so a NaN logit reaches the row's loss and gradient.
//
// Bound: the logits are read once and the gradient is written once, 2 R C bytes an element and the
// teacher's R k (a value and a class). Three kernels, by the length and the number of the rows:
//   up to 2047 classes    distill_tile_kernel, a warp on tiles of rows in shared memory
//   longer, few rows      distill_share_kernel, a cluster of CTAs on a row
//   longer, many rows     distill_ring_kernel, a CTA on a row in chunks
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
  Scale scale;
  float inv_hi, inv_lo;    // 1 / tau
  float grad_scale;        // tau / denom
  const float* v_loss;
  void* grad;
  double* partials;
  bool unless_one;         // nothing to do where the cotangent is one
  __device__ __forceinline__ bool done() const { return unless_one && *v_loss == 1.0f; }
};

// What the entries of one row say.
struct EntrySums {
  MaxSum z;       // of the student's logits, each class once
  double norm;    // ln p = (value - top) / tau - norm
  float top;      // the largest value, of which differences are taken first; 0 with a log-sum-exp
  float mass;     // sum of p
  float w;        // the row's weight
  int32_t live;   // the row counts, as far as the teacher and its weight say
  int32_t twice;  // some class is named more than once
};
// Of each entry: its class (-1: empty), probability, the teacher's logit and the student's (-inf
// where an earlier entry names the class).
template <int K>
struct Entries {
  EntrySums sum;
  int32_t id[K];
  float p[K], v[K], z[K];
};
// What the student's side adds to it.
struct RowSums {
  Ref r;       // maximum over all classes
  float all;   // sum over all classes against r
  float lsum;  // its log2
  float rho;
  MaxSum o;    // over the classes that no entry names
  int32_t live;
};

// One warp's entries of one row on their way to shared memory: entry lane + 32 j in place j. What
// is loaded stays as it came until it is needed: the first use of a load waits for it.
template <int N>
struct LaneEntries {
  uint32_t id_lo[N], id_hi[N], v[N], z[N];
  float w, lse;
};
__device__ __forceinline__ uint32_t load_raw(const void* p, int dtype, int64_t i) {
  return dtype == SPLAX_F32 ? static_cast<const uint32_t*>(p)[i]
                            : static_cast<const uint16_t*>(p)[i];
}
__device__ __forceinline__ float from_raw(uint32_t u, int dtype) {
  if (dtype == SPLAX_F32) return __uint_as_float(u);
  if (dtype == SPLAX_BF16) return __uint_as_float(u << 16);
  return __half2float(__ushort_as_half(static_cast<unsigned short>(u)));
}
template <int N>
__device__ __forceinline__ void load_teacher(LaneEntries<N>& t, const LossParams& a, int64_t r) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int e = lane + 32 * j;
    if (e >= a.k) break;
    const int64_t at = r * a.k + e;
    t.id_lo[j] = static_cast<const uint32_t*>(a.top_ids)[a.wide_ids ? 2 * at : at];
    if (a.wide_ids) t.id_hi[j] = static_cast<const uint32_t*>(a.top_ids)[2 * at + 1];
    t.v[j] = load_raw(a.top_values, a.value_dtype, at);
  }
  t.w = a.weights ? a.weights[r] : 1.0f;
  t.lse = a.top_lse ? a.top_lse[r] : 0.0f;
}
// The class of the entry in place j, -1 for none.
template <int N>
__device__ __forceinline__ int32_t entry_class(const LaneEntries<N>& t, const LossParams& a,
                                               int j) {
  const bool there = static_cast<int>(threadIdx.x & 31) + 32 * j < a.k;
  const bool in = there && t.id_lo[j] < static_cast<uint32_t>(a.classes) &&
                  (!a.wide_ids || t.id_hi[j] == 0u);
  return in ? static_cast<int32_t>(t.id_lo[j]) : -1;
}
// The student's logits of the entries, asked for once their classes are known.
template <typename T, int N>
__device__ __forceinline__ void load_student(LaneEntries<N>& t, const LossParams& a, int64_t r) {
  const T* z = static_cast<const T*>(a.logits) + r * a.row_stride;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int32_t c = entry_class(t, a, j);
    if (c >= 0) t.z[j] = load_raw(z, sizeof(T) == 4 ? SPLAX_F32 : SPLAX_BF16, c);
  }
}
// Probabilities and sums of one row's entries. Without a log-sum-exp they are renormalised, and
// their mass is one by definition.
template <int N>
__device__ __forceinline__ void put_entries(Entries<32 * N>& s, const LaneEntries<N>& t,
                                            const LossParams& a, int dtype) {
  const int lane = threadIdx.x & 31;
  const float ninf = neg_inf();
  float vmax = ninf, zmax = ninf;
  int32_t id[N];
  float val[N], z[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    id[j] = entry_class(t, a, j);
    val[j] = id[j] < 0 ? ninf : from_raw(t.v[j], a.value_dtype);
    z[j] = id[j] < 0 ? ninf : from_raw(t.z[j], dtype);
    vmax = max_nan(vmax, val[j]);
    zmax = max_nan(zmax, z[j]);
  }
  zmax = warp_max(zmax);
  const Ref r = ref_of(zmax, a.scale);
  float norm = t.lse, mass = 0.0f, sum = 0.0f;
  double norm64 = norm;
  bool live = !(norm == ninf), some = false;
#pragma unroll
  for (int j = 0; j < N; ++j) some = some || id[j] >= 0;
  live = __any_sync(0xffffffffu, some) && live;
  if (!a.top_lse) {
    vmax = warp_max(vmax);
    live = !(vmax == ninf);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (val[j] != ninf) sum += expf((val[j] - vmax) * a.inv_hi);
    sum = warp_sum(sum);
    norm = logf(sum);
    norm64 = ln_of(sum);
    sum = 0.0f;
  }
  bool twice = false;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float x = ninf;
    if (val[j] != ninf)
      x = a.top_lse ? fmaf(val[j], a.inv_lo, fmaf(val[j], a.inv_hi, -norm))
                    : (val[j] - vmax) * a.inv_hi - norm;
    const float p = expf(x);
    mass += p;
    // a class counts once in the student's sum: with the first entry that names it
    const unsigned same = __match_any_sync(0xffffffffu, id[j]);
    bool first = (same & ((1u << lane) - 1u)) == 0u;
#pragma unroll
    for (int i = 0; i < j; ++i)
      for (int l = 0; l < 32; ++l) {
        const int32_t before = __shfl_sync(0xffffffffu, id[i], l);  // by all lanes, always
        first = first && before != id[j];
      }
    twice = twice || (!first && id[j] >= 0);
    if (first) sum += ex2_approx(exponent(z[j], r, a.scale));
    const int e = lane + 32 * j;
    if (e < a.k) {
      s.v[e] = val[j];
      s.p[e] = p;
      s.z[e] = first ? z[j] : ninf;
      s.id[e] = id[j];
    }
  }
  mass = a.top_lse ? warp_sum(mass) : 1.0f;
  sum = warp_sum(sum);
  twice = __any_sync(0xffffffffu, twice);
  if (lane == 0)
    s.sum = {{zmax, sum}, norm64, a.top_lse ? 0.0f : vmax, mass, t.w, live && t.w != 0.0f, twice};
}
// Loss of a row, in 64 bits: a divergence is a small difference of logarithms. The student's are
// taken from the row's maximum, which ln_beside explains; as a difference first, since a product with
// 1 / tau that another is taken from would be fused, and leave its own rounding.
template <int K>
__device__ __forceinline__ double row_loss(const Entries<K>& s, const RowSums& y,
                                           const LossParams& a) {
  const double m = y.r.m, ln_all = ln_beside(y.r, y.r.m, a.inv_tau) + ln_of(y.all);
  double loss = 0.0;
  for (int e = threadIdx.x & 31; e < a.k; e += 32)
    if (s.p[e] != 0.0f) {
      float z = s.z[e];
      if (s.sum.twice)  // the logit stands with the first entry of the class
        for (int j = 0; j < e; ++j)
          if (s.id[j] == s.id[e]) {
            z = s.z[j];
            break;
          }
      const double ln_p = (static_cast<double>(s.v[e]) - s.sum.top) * a.inv_tau - s.sum.norm;
      loss += s.p[e] * (ln_p - ((z - m) * a.inv_tau - ln_all));
    }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, off);
  if (y.rho > 0.0f)
    loss += y.rho * (ln_of(y.rho) - (ln_beside(ref_of(y.o.m, a.scale), y.r.m, a.inv_tau) +
                                     (ln_of(y.o.s) - ln_all)));
  return loss * s.sum.w;
}

// The row's sums from that over O.
__device__ __forceinline__ RowSums row_sums(MaxSum o, const EntrySums& s, const LossParams& a,
                                            bool late) {
  if (late) o = poison();
  const bool some = !(o.m == neg_inf());
  const MaxSum all = join(o, s.z, a.scale);
  return {ref_of(all.m, a.scale), all.s, log2f(all.s),
          a.top_lse && some ? fmaxf(0.0f, 1.0f - s.mass) : 0.0f, o,
          s.live && !(all.m == neg_inf())};
}
// Factor of the gradient over O: ((P + rho) q_O - rho) / (sum over O), with q_O's own exponent.
__device__ __forceinline__ float outside_factor(const RowSums& y, const EntrySums& s,
                                                const LossParams& a, float cot) {
  if (!y.live || y.o.m == neg_inf()) return 0.0f;
  const float qo = ex2_approx(shift(ref_of(y.o.m, a.scale), y.r, a.scale) - y.lsum) * y.o.s;
  return s.w * a.grad_scale * cot * (((s.mass + y.rho) * qo - y.rho) / y.o.s);
}
// Gradients of the classes that the entries name, of those in [c0, c1), by one warp.
template <typename T, int K>
__device__ __forceinline__ void entry_gradients(const Entries<K>& s, const RowSums& y,
                                                const LossParams& a, float cot, T* g, int c0,
                                                int c1) {
  const float gs = s.sum.w * a.grad_scale * cot;
  for (int e = threadIdx.x & 31; e < a.k; e += 32) {
    if (s.id[e] < 0 || s.id[e] < c0 || s.id[e] >= c1) continue;
    float p = s.p[e];
    bool first = true;
    if (s.sum.twice)
      for (int j = 0; j < a.k; ++j)
        if (j != e && s.id[j] == s.id[e]) {
          first = first && j > e;
          p += s.p[j];
        }
    const float q = ex2_approx(exponent(s.z[e], y.r, a.scale) - y.lsum);
    if (first) g[s.id[e]] = from_f<T>(gs * ((s.sum.mass + y.rho) * q - p));
  }
  __syncwarp();
}

// f 2^(x c - ms), in the type's rounding.
template <typename T>
__device__ __forceinline__ uint4 gradient_vector(uint4 u, Scale c, float ms, float2 f) {
  float x[kVec<T>];
  unpack(u, x, T{});
#pragma unroll
  for (int q = 0; q < kVec<T>; q += 2) {
    const float2 t = exponent2({x[q], x[q + 1]}, ms, c);
    const float2 w = mul2({ex2_approx(t.x), ex2_approx(t.y)}, f);
    x[q] = w.x;
    x[q + 1] = w.y;
  }
  return pack(x, T{});
}

// The gradient over O of any row.
template <typename T>
__device__ __forceinline__ uint4 any_gradient_vector(uint4 u, bool live, Ref r, Scale c, float c0) {
  if (!live) return make_uint4(0u, 0u, 0u, 0u);
  if (r.plain()) return gradient_vector<T>(u, c, r.ms, splat2(c0));
  float x[kVec<T>];
  unpack(u, x, T{});
#pragma unroll
  for (int q = 0; q < kVec<T>; ++q) x[q] = c0 * ex2_approx(exponent(x[q], r, c));
  return pack(x, T{});
}
// An aligned vector whose first class is `cls`; of one that reaches over an end of the row, the
// row's elements.
template <typename T>
__device__ __forceinline__ void store_vector(T* to, uint4 u, int cls, int classes) {
  if (cls >= 0 && cls + kVec<T> <= classes) {
    __stcs(reinterpret_cast<uint4*>(to), u);
    return;
  }
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int q = 0; q < kVec<T>; ++q)
    if (cls + q >= 0 && cls + q < classes) to[q] = e[q];
}

// Few long rows: a cluster of CTAs takes one row, each CTA a share of it in shared memory, which
// spreads a row over up to eight SMs. One warp starts the share's bulk copy, one fills the ends of
// the row, one works out the entries (in every CTA, which saves exchanging them); once both are
// there the entries' places in the share are set to -inf, so that the passes over it need no test
// for them. The CTAs exchange a maximum and a sum between the passes. Bound by the latency of
// loads, barriers and the launch: the loss of 33 rows of 65,537 fp32 7.6 us.
constexpr int kShareThreads = 256;
template <typename T, int K>
__global__ void __launch_bounds__(kShareThreads)
distill_share_kernel(LossParams a, float* loss, double loss_scale) {
  constexpr int V = kVec<T>, kWarps = kShareThreads / 32, kBatch = 16 / V;
  extern __shared__ uint4 s_buf[];
  __shared__ Entries<K> s_ent;
  __shared__ __align__(8) uint64_t s_bar;
  __shared__ MaxSum s_warp[kWarps], s_part[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const float ninf = neg_inf();
  const Scale c = a.scale;
  const int64_t r = blockIdx.x / size;
  const T* z = static_cast<const T*>(a.logits) + r * a.row_stride;
  const RowShare<T> share = row_share(z, a.classes, rank, size);
  const int n = share.v1 - share.v0;
  if (tid == 0) mbar_init(&s_bar, 1);
  pdl_enter();
  if (a.done()) return;
  // a CTA of the cluster may only be written to once it runs
  if (size > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  const float cot = a.v_loss ? *a.v_loss : 1.0f;
  if (tid == 0) load_share(share, a.classes, s_buf, &s_bar);
  if (warp == 1) store_ends(load_ends(share, a.classes), s_buf);
  LaneEntries<K / 32> t;
  if (warp == 2) {
    load_teacher(t, a, r);
    load_student<T>(t, a, r);
    put_entries(s_ent, t, a, kDtype<T>);
  }
  __syncthreads();
  const bool late = !mbar_wait(&s_bar, 0);
  if (warp == 2) {
#pragma unroll
    for (int j = 0; j < K / 32; ++j) {
      const int32_t cls = entry_class(t, a, j);
      const int at = cls - share.cls0;
      if (cls >= 0 && at >= 0 && at < n * V) reinterpret_cast<T*>(s_buf)[at] = from_f<T>(ninf);
    }
  }
  __syncthreads();
  Running run;
  int v = tid;
  for (; v + (kBatch - 1) * kShareThreads < n; v += kBatch * kShareThreads)
    add_vectors<T, kBatch>(run, s_buf + v, kShareThreads, c);
  for (; v < n; v += kShareThreads) add_vectors<T, 1>(run, s_buf + v, kShareThreads, c);
  // a late copy poisons the row in every CTA of the cluster: before the sums are joined
  MaxSum o = warp_join(late ? poison() : run.get(c), c);
  if (lane == 0) s_warp[warp] = o;
  __syncthreads();
  // every warp for itself: cheaper than another barrier
  o = warp_join(lane < kWarps ? s_warp[lane] : MaxSum{ninf, 0.0f}, c);
  if (size > 1) {
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (warp == 0 && lane < static_cast<int>(size)) {
      const uint32_t to = cluster_addr(&s_part[rank], lane);
      cluster_store(to, o.m);
      cluster_store(to + 4, o.s);
    }
    cluster_sync();
    o = warp_join(lane < static_cast<int>(size) ? s_part[lane] : MaxSum{ninf, 0.0f}, c);
  }
  const EntrySums& s = s_ent.sum;
  const RowSums y = row_sums(o, s, a, false);
  if (a.grad) {
    const Ref ro = ref_of(o.m, c);
    const float c0 = outside_factor(y, s, a, cot);
    T* g = static_cast<T*>(a.grad) + r * a.classes;
    const bool even = ((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(z)) & 15u) == 0;
    T* out = g + share.cls0;
    for (v = tid; v < n; v += kShareThreads) {
      const uint4 u = any_gradient_vector<T>(s_buf[v], y.live, ro, c, c0);
      const int cls = share.cls0 + v * V;
      if (!even) s_buf[v] = u;
      else store_vector(out + v * V, u, cls, a.classes);
    }
    __syncthreads();
    if (!even) {  // in consecutive elements: the gradient's row is not aligned as the logits'
      const int lo = share.cls0 < 0 ? -share.cls0 : 0, hi = min(n * V, a.classes - share.cls0);
      const T* e = reinterpret_cast<const T*>(s_buf);
      for (int j = lo + tid; j < hi; j += kShareThreads) out[j] = e[j];
      __syncthreads();
    }
    if (warp == 0 && y.live) entry_gradients(s_ent, y, a, cot, g, share.cls0, share.cls0 + n * V);
  }
  if (warp == 2 && rank == 0 && (loss || a.partials)) {
    const double total = y.live ? row_loss(s_ent, y, a) : 0.0;
    if (lane == 0) {
      if (loss) *loss = static_cast<float>(total * loss_scale);  // the only row
      else a.partials[r] = total;
    }
  }
}

// Many long rows: a CTA works through its rows alone. A row comes in chunks by bulk copies into a
// ring of slots, far ahead of its use; the last `keep` chunks of a row stay in their slots for the
// gradient (all of them where the row fits the ring), the others are copied again, from the L2
// cache, since the rows in flight fit it. Each warp that helps has one task and runs as far ahead
// as the slots allow: one starts the copies; one fetches a row's entries, works out their
// probabilities and sets their places in each chunk to -inf as it arrives, so that the passes over
// the chunks need no test for them; one turns the working warps' sums into the row's and, while they
// write the gradient, works out the loss and, a row later, the gradients of the entries.
// HBM-bound: 4000 rows of 128,000 bf16 with gradient 0.40 ms, 78 % of the measured copy rate; the
// same with a cluster per row holding all of it in shared memory took 0.73 ms, and with the rows of six
// CTAs an SM in flight, which do not fit the L2 cache, 0.53. 10,000 rows of 32,000 bf16 0.26 ms
// (76 %); rows of 4 to 16 KB 26 to 68 %, where the work per row (entries, sums, barriers) shows.
// fp32: 4000 rows of 64,000 0.35 ms (90 %), 2000 of 128,000 0.45 (70 %), 1000 of 262,144, of which 148
// do not fit the L2 cache, 0.50 (65 %). With k > 32 the forms of several CTAs an SM spill 132 to 188 bytes.
constexpr int kRingSlots = 3, kRingEntries = 4;
template <typename T, int THREADS, int CTAS, int K>
__global__ void __launch_bounds__(THREADS + 96, CTAS)
distill_ring_kernel(LossParams a, int chunks, int vecs, int slots, int keep) {
  constexpr int V = kVec<T>, kWarps = THREADS / 32;
  constexpr int kBatch = 16 / V;  // vectors a thread works on together
  extern __shared__ uint4 s_buf[];  // `slots` chunks of `vecs` vectors
  __shared__ Entries<K> s_ent[kRingEntries];
  __shared__ MaxSum s_warp[kWarps];
  __shared__ Ref s_ref;    // of the sum over O
  __shared__ float s_c0;   // factor of the gradient over O
  __shared__ int s_live, s_late;
  // a chunk is there, marked, read; a row's entries are there, read
  __shared__ __align__(8) uint64_t s_full[kRingSlots], s_ready[kRingSlots], s_empty[kRingSlots];
  __shared__ __align__(8) uint64_t s_ent_full[kRingEntries], s_ent_empty[kRingEntries];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float ninf = neg_inf();
  const int count = static_cast<int>((a.rows - blockIdx.x + gridDim.x - 1) / gridDim.x);
  const int again = a.grad ? chunks - keep : 0;  // chunks that are copied a second time
  if (tid == 0) {
    s_late = 0;
    for (int i = 0; i < slots; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_ready[i], 1);
      mbar_init(&s_empty[i], kWarps);
    }
    for (int i = 0; i < kRingEntries; ++i) {
      mbar_init(&s_ent_full[i], 1);
      mbar_init(&s_ent_empty[i], 1);
    }
  }
  pdl_enter();
  if (a.done()) return;
  __syncthreads();
  const int64_t step = gridDim.x * a.row_stride;
  const int64_t out_step = static_cast<int64_t>(gridDim.x) * a.classes;
  const T* z = static_cast<const T*>(a.logits) + blockIdx.x * a.row_stride;
  T* g = a.grad ? static_cast<T*>(a.grad) + static_cast<int64_t>(blockIdx.x) * a.classes : nullptr;
  auto lead_of = [](const T* p) {
    return static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
  };
  auto wait = [&](uint64_t* bar, uint32_t parity, bool rest = false) {
    if (!mbar_wait(bar, parity, rest)) s_late = 1;
  };

  if (warp == kWarps) {  // copies
    if (lane != 0) return;
    int slot = 0;
    uint32_t parity = 1;
    for (int i = 0; i < count; ++i, z += step) {
      const int lead = lead_of(z), n = (lead + a.classes + V - 1) / V;
      const int b0 = lead > 0 ? 1 : 0, b1 = (lead + a.classes) % V ? n - 1 : n;
      for (int j = 0; j < chunks + again; ++j) {
        const int at = (j < chunks ? j : j - chunks) * vecs;
        const int from = max(at, b0), to = min(at + vecs, b1);
        wait(&s_empty[slot], parity, true);
        const uint32_t bytes = to > from ? 16u * static_cast<uint32_t>(to - from) : 0u;
        mbar_expect(&s_full[slot], bytes);
        if (bytes)
          bulk_load(s_buf + slot * vecs + (from - at), z - lead + from * V, bytes, &s_full[slot]);
        if (++slot == slots) slot = 0, parity ^= 1;
      }
    }
    return;
  }

  if (warp == kWarps + 1) {  // entries
    LaneEntries<K / 32> now, next;
    int slot = 0, ent = 0;
    uint32_t parity = 0, ent_parity = 1;
    int64_t r = blockIdx.x;
    load_teacher(next, a, r);
    for (int i = 0; i < count; ++i, z += step, r += gridDim.x) {
      now = next;
      load_student<T>(now, a, r);
      const RowShare<T> row = row_share(z, a.classes, 0, 1);
      const ShareEnds<T> ends = load_ends(row, a.classes);
      if (i + 1 < count) load_teacher(next, a, r + gridDim.x);
      wait(&s_ent_empty[ent], ent_parity, true);
      put_entries(s_ent[ent], now, a, kDtype<T>);
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_ent_full[ent]);
      if (++ent == kRingEntries) ent = 0, ent_parity ^= 1;
      for (int j = 0; j < chunks + again; ++j) {
        const int first = (j < chunks ? j : j - chunks) * vecs * V, size = vecs * V;
        T* e = reinterpret_cast<T*>(s_buf + slot * vecs);
        wait(&s_full[slot], parity, true);
        if (ends.at >= first && ends.at < first + size) e[ends.at - first] = ends.x;
        __syncwarp();
#pragma unroll
        for (int q = 0; q < K / 32; ++q) {
          const int32_t c = entry_class(now, a, q);
          const int at = c + row.lead - first;
          if (c >= 0 && at >= 0 && at < size) e[at] = from_f<T>(ninf);
        }
        fence_async();  // a later copy into the slot comes after these stores
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_ready[slot]);
        if (++slot == slots) slot = 0, parity ^= 1;
      }
    }
    return;
  }

  if (warp == kWarps + 2) {  // sums, loss, the entries' gradients
    const float cot = a.v_loss ? *a.v_loss : 1.0f;
    double total = 0.0;
    RowSums y{}, before{};
    int ent = 0, ent_before = 0;
    uint32_t ent_parity = 0;
    T* g_before = g;
    for (int i = 0; i <= count; ++i) {
      if (i < count) wait(&s_ent_full[ent], ent_parity, true);
      pair_sync<THREADS + 32>(1);  // row i is summed, the gradient of row i - 1 written
      if (i < count) {
        const EntrySums& s = s_ent[ent].sum;
        y = row_sums(warp_join(lane < kWarps ? s_warp[lane] : MaxSum{ninf, 0.0f}, a.scale), s, a,
                     s_late);
        if (lane == 0) {
          s_c0 = outside_factor(y, s, a, cot);
          s_ref = ref_of(y.o.m, a.scale);
          s_live = y.live;
        }
        pair_arrive<THREADS + 32>(2);
      }
      if (i > 0) {
        if (before.live) {
          const Entries<K>& s = s_ent[ent_before];
          if (g) entry_gradients(s, before, a, cot, g_before, 0, a.classes);
          if (a.partials) total += row_loss(s, before, a);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_ent_empty[ent_before]);
        g_before += out_step;
      }
      before = y;
      ent_before = ent;
      if (++ent == kRingEntries) ent = 0, ent_parity ^= 1;
    }
    if (lane == 0 && a.partials) a.partials[blockIdx.x] = total;
    return;
  }

  const Scale c = a.scale;
  int slot = 0;
  uint32_t parity = 0;
  auto next_slot = [&] {
    if (++slot == slots) slot = 0, parity ^= 1;
  };
  auto release = [&](int at) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&s_empty[at]);
  };
  for (int i = 0; i < count; ++i, z += step, g += out_step) {
    const int lead = lead_of(z), n = (lead + a.classes + V - 1) / V;
    const int slot0 = slot;
    Running run;
    for (int j = 0; j < chunks; ++j) {
      wait(&s_ready[slot], parity);
      const uint4* buf = s_buf + slot * vecs;
      const int size = min(vecs, n - j * vecs);
      int v = tid;
      for (; v + (kBatch - 1) * THREADS < size; v += kBatch * THREADS)
        add_vectors<T, kBatch>(run, buf + v, THREADS, c);
      for (; v < size; v += THREADS) add_vectors<T, 1>(run, buf + v, THREADS, c);
      if (!a.grad || j < again) release(slot);
      next_slot();
    }
    const MaxSum o = warp_join(run.get(c), c);
    if (lane == 0) s_warp[warp] = o;
    pair_arrive<THREADS + 32>(1);
    pair_sync<THREADS + 32>(2);
    if (!a.grad) continue;
    const Ref ro = s_ref;
    const float c0 = s_c0;
    const bool live = s_live, plain = ro.plain();
    const float2 f2 = splat2(c0);
    const bool even = ((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(z)) & 15u) == 0;
    auto write = [&](uint4* buf, int first) {  // a chunk whose first vector is `first`
      const int size = min(vecs, n - first);
      T* out = g - lead + first * V;
      const int c_first = first * V - lead;
      auto give = [&](uint4 u, int v) {
        if (even) {
          store_vector(out + v * V, u, c_first + v * V, a.classes);
        } else {  // in consecutive elements, by way of the chunk itself
          if (v < size) buf[v] = u;
          __syncwarp();
          const T* e = reinterpret_cast<const T*>(buf);
          const int at = (v - lane) * V, end = min(size * V, at + 32 * V);
          for (int q = at + lane; q < end; q += 32)
            if (c_first + q >= 0 && c_first + q < a.classes) out[q] = e[q];
        }
      };
      int v = tid;
      if (live && plain)
        for (; v + (kBatch - 1) * THREADS < size; v += kBatch * THREADS) {
          uint4 u[kBatch];
#pragma unroll
          for (int q = 0; q < kBatch; ++q)
            u[q] = gradient_vector<T>(buf[v + q * THREADS], c, ro.ms, f2);
#pragma unroll
          for (int q = 0; q < kBatch; ++q) give(u[q], v + q * THREADS);
        }
      // whole warps stay together for the unaligned store
      for (; v < (even ? size : (size + 31) & ~31); v += THREADS)
        give(any_gradient_vector<T>(v < size ? buf[v] : make_uint4(0u, 0u, 0u, 0u), live, ro, c, c0),
             v);
      if (!even) fence_async();
    };
    // the chunks that are still there, then those that are copied again
    int at = slot0 + again;
    while (at >= slots) at -= slots;
    for (int j = again; j < chunks; ++j) {
      write(s_buf + at * vecs, j * vecs);
      release(at);
      if (++at == slots) at = 0;
    }
    for (int j = 0; j < again; ++j) {
      wait(&s_ready[slot], parity);
      write(s_buf + slot * vecs, j * vecs);
      release(slot);
      next_slot();
    }
  }
  pair_arrive<THREADS + 32>(1);
}

// A warp works alone on tiles of consecutive rows, G lanes to a row and up to E classes to a lane,
// held in registers from the first pass over them to the last, so that a logit takes one
// exponential. A tile's logits and the teacher's side of its rows come by bulk copies into a stage
// of shared memory, a tile ahead; the gradient replaces the logits there and leaves by one bulk
// copy, whatever the alignment of the rows. Warps never wait for one another: what time the
// entries of a row take is covered by the other warps of the SM.
//
// Bound by latency: 2.3 of 4 instructions a cycle, 166 a row of 150 fp32 classes, from four warps a
// scheduler. 1080p x 150 fp32 with gradient 0.62 ms (65 % of the measured copy rate), 800 x 800 x
// 513 bf16 0.57 ms (37 %). 128 registers, with up to 60 bytes spilled (184 from 1280 classes on).
// Measured and not kept: a running maximum instead of the classes in registers, which allows fewer
// lanes a row (0.67 ms), groups of four classes instead of eight between tests for the row's end
// (8 to 20 % slower), five CTAs an SM at 96 registers (up to 23 % slower, spills).
// Sizes in bytes. A stage holds the parts in this order, each with room for aligned copies.
struct TilePlan {
  int rows;   // of a tile
  int pitch;  // of a row of logits in a stage where rows are copied one by one, 0: a tile at once
  int values, ids, lse, weights, stage;  // where the parts begin (the logits: 16), and the size
  int warp;                              // all stages of a warp
};

// Bits of -inf. What follows it by up to 128 marks the place of an entry's class: other bits for
// each entry, none of them -inf.
template <typename T>
struct MarkBits;
template <>
struct MarkBits<float> {
  using U = uint32_t;
  static constexpr U kInf = 0xff800000u;
};
template <>
struct MarkBits<__nv_bfloat16> {
  using U = uint16_t;
  static constexpr U kInf = 0xff80u;
};
template <>
struct MarkBits<__half> {
  using U = uint16_t;
  static constexpr U kInf = 0xfc00u;
};

__device__ __forceinline__ void store_pair(float* p, float a, float b) {
  *reinterpret_cast<float2*>(p) = make_float2(a, b);
}
template <typename T>
__device__ __forceinline__ void store_pair(T* p, float a, float b) {
  *reinterpret_cast<uint32_t*>(p) = pack2(a, b, T{});
}

// PAIR: the gradient's rows lie to two elements as the logits' rows do, so a lane takes two
// neighbouring classes at a time, from the even address at or before the row's first.
constexpr int kLaneKept = 4;  // entries of a row that a lane takes: k <= kLaneKept G
template <typename T, int G, int E, bool PAIR>
__global__ void __launch_bounds__(32 * kTileWarps, 4)
distill_tile_kernel(LossParams a, TilePlan plan, float* loss, double loss_scale) {
  constexpr int P = 32 / G, S = PAIR ? 2 : 1;  // rows of a pass, classes a lane takes at a time
  using Mark = typename MarkBits<T>::U;
  extern __shared__ uint4 s_buf[];
  __shared__ __align__(8) uint64_t s_bar[kTileWarps][kTileStages];
  __shared__ double s_total[kTileWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row_in_pass = lane / G, l = lane % G;
  const float ninf = neg_inf();
  const Scale c = a.scale;
  char* const mine = reinterpret_cast<char*>(s_buf) + warp * plan.warp;
  uint64_t* const bars = s_bar[warp];
  if (lane < kTileStages) mbar_init(&bars[lane], 1);
  __syncwarp();
  pdl_enter();
  if (a.done()) return;
  const float cot = a.v_loss ? *a.v_loss : 1.0f;
  const uintptr_t logits = reinterpret_cast<uintptr_t>(a.logits);
  const int64_t stride = a.row_stride * static_cast<int64_t>(sizeof(T));  // bytes
  const int width = a.classes * static_cast<int>(sizeof(T)), k = a.k;
  const int value_size = a.value_dtype == SPLAX_F32 ? 4 : 2, id_size = a.wide_ids ? 8 : 4;
  const int64_t tiles = (a.rows + plan.rows - 1) / plan.rows;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTileWarps;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kTileWarps + warp;

  // A lane per part: logits, values, classes, log-sum-exps, weights, and the gradient, whose place
  // in a stage follows from the address alone. Each keeps the address of its part of the tile
  // after next, and of the present tile the part's address mod 16.
  uintptr_t base = logits;
  int64_t size = stride;  // bytes of a row
  int cut = static_cast<int>(stride - width);  // that the last row of all does not have
  int to = 16;  // so that a gradient of another alignment never overtakes the logits it replaces
  if (lane == 1) base = reinterpret_cast<uintptr_t>(a.top_values), size = k * value_size, to = plan.values;
  if (lane == 2) base = reinterpret_cast<uintptr_t>(a.top_ids), size = k * id_size, to = plan.ids;
  if (lane == 3) base = reinterpret_cast<uintptr_t>(a.top_lse), size = 4, to = plan.lse;
  if (lane == 4) base = reinterpret_cast<uintptr_t>(a.weights), size = 4, to = plan.weights;
  if (lane == 5) base = reinterpret_cast<uintptr_t>(a.grad), size = width;
  if (lane > 0) cut = 0;
  const bool copies = lane < 5 && base != 0 && (lane > 0 || plan.pitch == 0);
  const uintptr_t limit = base + a.rows * size - cut;
  const int64_t advance = step * plan.rows * size;
  const uint32_t tile_bytes = static_cast<uint32_t>(plan.rows * size);
  uintptr_t ahead = base + first * plan.rows * size;  // of the next tile to load
  int low = 0, low_ahead = 0;
  auto load = [&](int64_t tile, int at) {
    char* s = mine + at * plan.stage;
    uint64_t* bar = &bars[at];
    const uintptr_t end = min(ahead + tile_bytes, limit + cut) - cut;
    const Part part = part_of(s + to, base, ahead, end, limit);
    low_ahead = static_cast<int>(ahead) & 15;
    ahead += advance;
    uint32_t bytes = copies ? static_cast<uint32_t>(part.e16 - part.b16) : 0u;
    const int64_t r0 = tile * plan.rows, r1 = min(r0 + plan.rows, a.rows);
    auto row_part = [&](int64_t r) {
      return part_of(s + 16 + (r - r0) * plan.pitch, logits, logits + r * stride,
                     logits + r * stride + width, logits + (a.rows - 1) * stride + width);
    };
    if (plan.pitch)
      for (int64_t r = r0 + lane; r < r1; r += 32) {
        const Part q = row_part(r);
        bytes += static_cast<uint32_t>(q.e16 - q.b16);
      }
    bytes = __reduce_add_sync(0xffffffffu, bytes);
    if (lane == 0) mbar_expect(bar, bytes);
    __syncwarp();
    if (copies) load_part(part, bar);
    if (plan.pitch)
      for (int64_t r = r0 + lane; r < r1; r += 32) load_part(row_part(r), bar);
  };

  double total = 0.0;
  if (first < tiles) load(first, 0);
  int at = 0;
  uint32_t parity = 0;
  for (int64_t tile = first; tile < tiles; tile += step) {
    const int next = at + 1 == kTileStages ? 0 : at + 1;
    // the next stage's last gradient has left it
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
    low = low_ahead;
    if (tile + step < tiles) load(tile + step, next);
    const bool late = __any_sync(0xffffffffu, !mbar_wait(&bars[at], parity));
    __syncwarp();
    const int64_t r0 = tile * plan.rows;
    const int rows = static_cast<int>(min(static_cast<int64_t>(plan.rows), a.rows - r0));
    char* s = mine + at * plan.stage;
    auto part_at = [&](int q) { return __shfl_sync(0xffffffffu, low, q); };
    // where a row of logits begins; its alignment may differ from row to row where they are apart
    const int in0 = 16 + part_at(0), stride32 = static_cast<int>(stride);
    const char* values = s + plan.values + part_at(1);
    const char* ids = s + plan.ids + part_at(2);
    const float* lses = reinterpret_cast<const float*>(s + plan.lse + part_at(3));
    const float* ws = reinterpret_cast<const float*>(s + plan.weights + part_at(4));
    T* const out = reinterpret_cast<T*>(s + part_at(5));

    for (int from = 0; from < rows; from += P) {
      const bool there = from + row_in_pass < rows;
      const int row = there ? from + row_in_pass : 0;
      T* const z = reinterpret_cast<T*>(
          s + (plan.pitch ? 16 + row * plan.pitch +
                                (static_cast<int>(logits + (r0 + row) * stride) & 15)
                          : in0 + row * stride32));
      const int lead = PAIR ? static_cast<int>(reinterpret_cast<uintptr_t>(z) / sizeof(T)) & 1 : 0;
      const float w = there ? (a.weights ? ws[row] : 1.0f) : 0.0f;
      float norm = a.top_lse ? lses[row] : 0.0f;
      double norm64 = norm;  // ln p = (value - v0) / tau - norm64
      float v0 = 0.0f;       // the largest value, of which differences are taken first
      bool live = there && w != 0.0f && !(norm == ninf);
      // the entries' classes and logits, and their marks
      int id[kLaneKept];
      float ze[kLaneKept], p[kLaneKept];  // the student's logit; the teacher's, then the probability
      float m = ninf, vmax = ninf;
#pragma unroll
      for (int q = 0; q < kLaneKept; ++q) {
        id[q] = -1;
        ze[q] = p[q] = ninf;
        if (q * G >= k) continue;
        const int e = q * G + l;
        if (there && e < k) {
          const int i = row * k + e;
          uint32_t cls = reinterpret_cast<const uint32_t*>(ids)[a.wide_ids ? 2 * i : i];
          if (a.wide_ids && reinterpret_cast<const uint32_t*>(ids)[2 * i + 1]) cls = ~0u;
          if (cls < static_cast<uint32_t>(a.classes)) {
            id[q] = static_cast<int>(cls);
            ze[q] = to_f(z[cls]);
            p[q] = value_size == 4
                       ? reinterpret_cast<const float*>(values)[i]
                       : from_raw(reinterpret_cast<const uint16_t*>(values)[i], a.value_dtype);
            m = max_nan(m, ze[q]);
            vmax = max_nan(vmax, p[q]);
          }
        }
      }
      bool some = false;
#pragma unroll
      for (int q = 0; q < kLaneKept; ++q) some = some || id[q] >= 0;
      const unsigned named_in = __ballot_sync(0xffffffffu, some);
      live = live && (named_in >> (lane - l) & (~0u >> (32 - G))) != 0u;
      // another lane's entry may name the same class: its mark comes after this lane's reading
      __syncwarp();
#pragma unroll
      for (int q = 0; q < kLaneKept; ++q)
        if (q * G < k && id[q] >= 0)
          reinterpret_cast<Mark*>(z)[id[q]] = static_cast<Mark>(MarkBits<T>::kInf + 1 + q * G + l);
      if (!a.top_lse) {
        vmax = group_max<G>(vmax);
        live = live && !(vmax == ninf);
        v0 = vmax == ninf ? 0.0f : vmax;
        float sum = 0.0f;
#pragma unroll
        for (int q = 0; q < kLaneKept; ++q)
          if (q * G < k && id[q] >= 0) sum += ex2_approx((p[q] - v0) * c.hi);
        sum = group_sum<G>(sum);
        norm = __log2f(sum);
        norm64 = ln_of(sum);
      }
      __syncwarp();
      // probabilities; the places of the named classes to -inf
      // of this lane's entries; the loss in 64 bits: a divergence is a small difference of logarithms
      float mass = 0.0f;
      double mass64 = 0.0, loss64 = 0.0;
      bool lost = false;
#pragma unroll
      for (int q = 0; q < kLaneKept; ++q) {
        if (q * G < k && id[q] >= 0) {
          Mark* const place = reinterpret_cast<Mark*>(z) + id[q];
          lost = lost || *place != static_cast<Mark>(MarkBits<T>::kInf + 1 + q * G + l);
          *place = MarkBits<T>::kInf;
          const float v = p[q];
          float x = ninf;  // log2 of the probability
          if (v != ninf)
            x = a.top_lse ? fmaf(v, a.inv_lo, fmaf(v, a.inv_hi, -norm)) * kLog2e
                          : (v - vmax) * c.hi - norm;
          p[q] = ex2_approx(x);
          if (p[q] != 0.0f) {
            loss64 += p[q] * ((static_cast<double>(v) - v0) * a.inv_tau - norm64);
            mass64 += p[q];
          }
          mass += p[q];
        } else {
          p[q] = 0.0f;
        }
      }
      const bool twice = __any_sync(0xffffffffu, lost);  // a class is named more than once
      __syncwarp();
      // the classes that no entry names
      T* const zw = z - lead;
      float x[E];
      auto read = [&](float top) {
#pragma unroll
        for (int j = 0; j < E; j += 4 * S) {
          if ((j + 4 * S) * G <= a.classes) {  // the row goes on: no test per class
#pragma unroll
            for (int i = j; i < j + 4 * S; i += S) {
              if constexpr (PAIR) {
                load_pair(zw + i * G + l * S, x[i], x[i + 1]);
                if (i == 0 && l == 0 && lead) x[i] = ninf;
                top = max3_nan(top, x[i], x[i + 1]);
              } else {
                x[i] = to_f(z[i * G + l]);
                top = max_nan(top, x[i]);
              }
            }
          } else if (j * G < a.classes + lead) {
#pragma unroll
            for (int i = j; i < j + 4 * S; i += S) {
              const int cls = i * G + l * S - lead;
              x[i] = ninf;
              if constexpr (PAIR) {
                x[i + 1] = ninf;
                if (cls < a.classes) load_pair(zw + i * G + l * S, x[i], x[i + 1]);
                if (i == 0 && cls < 0) x[i] = ninf;
                if (cls + 1 >= a.classes) x[i + 1] = ninf;
                top = max3_nan(top, x[i], x[i + 1]);
              } else {
                if (cls < a.classes) x[i] = to_f(z[cls]);
                top = max_nan(top, x[i]);
              }
            }
          }
        }
        return group_max<G>(top);
      };
      const Ref r = ref_of(read(m), c);
      live = live && !(r.m == ninf);
      auto powers = [&](Ref from) {
        float2 sum[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
        const bool plain = from.plain();
#pragma unroll
        for (int j = 0; j < E; j += 4 * S) {
          if (j * G < a.classes + lead) {
            if (plain) {
#pragma unroll
              for (int i = j; i < j + 4 * S; i += 2) {
                const float2 t = exponent2({x[i], x[i + 1]}, from.ms, c);
                x[i] = ex2_approx(t.x);
                x[i + 1] = ex2_approx(t.y);
                sum[i / 2 & 1] = add2(sum[i / 2 & 1], {x[i], x[i + 1]});
              }
            } else {
#pragma unroll
              for (int i = j; i < j + 4 * S; ++i) {
                x[i] = ex2_approx(exponent(x[i], from, c));
                sum[0].x += x[i];
              }
            }
          }
        }
        const float2 both = add2(sum[0], sum[1]);
        return both.x + both.y;
      };
      float o = powers(r);
      // a class counts once: with the first entry that names it, which adds the others'
      // probabilities to its own
      unsigned counts = ~0u;
      float named = 0.0f, again[kLaneKept] = {};
      if (twice) {
#pragma unroll
        for (int h = 0; h < kLaneKept; ++h)
          for (int i = 0; i < G; ++i) {
            const int other = __shfl_sync(0xffffffffu, id[h], i, G);
            const float its = __shfl_sync(0xffffffffu, p[h], i, G);
#pragma unroll
            for (int q = 0; q < kLaneKept; ++q)
              if (other == id[q] && (h != q || i != l)) {
                again[q] += its;
                if (h * G + i < q * G + l) counts &= ~(1u << q);
              }
          }
#pragma unroll
        for (int q = 0; q < kLaneKept; ++q) {
          if (id[q] >= 0 && (counts >> q & 1u)) named += ex2_approx(exponent(ze[q], r, c));
        }
      } else {
#pragma unroll
        for (int q = 0; q < kLaneKept; ++q) {
          if (q * G < k && id[q] >= 0) named += ex2_approx(exponent(ze[q], r, c));
        }
      }
      float all, rho = 0.0f, c0, shifted = 0.0f, row_mass = 1.0f;
      Ref ro = r;  // of the sum over O
      if (!a.top_lse) {
        all = group_sum<G>(o + named);
      } else {
        row_mass = group_sum<G>(mass);
        o = group_sum<G>(o);
        all = o + group_sum<G>(named);
        if (__any_sync(0xffffffffu, o < 1e-18f)) {
          // a student that is sure of the entries: O against its own maximum
          ro = ref_of(read(ninf), c);
          o = group_sum<G>(powers(ro));
          shifted = shift(ro, r, c);
        }
        if (!(ro.m == ninf)) rho = fmaxf(0.0f, 1.0f - row_mass);
      }
      if (late) {
        all = __int_as_float(0x7fc00000);
        live = there;
      }
      const float lsum = __log2f(all);
      if (live) {
        // the student's logarithms from the row's maximum, see ln_beside
        const double ln_all = ln_beside(r, r.m, a.inv_tau) + ln_of(all);
        double away = 0.0;
#pragma unroll
        for (int q = 0; q < kLaneKept; ++q)
          if (q * G < k && p[q] != 0.0f) away += p[q] * (static_cast<double>(ze[q]) - r.m);
        loss64 += mass64 * ln_all - away * a.inv_tau;
        if (l == 0 && rho > 0.0f)
          loss64 += rho * (ln_of(__fdividef(rho, o)) - ln_beside(ro, r.m, a.inv_tau) + ln_all);
        total += w * loss64;
      }
      if (a.grad) {
        const float gs = w * a.grad_scale * cot;
        if (!a.top_lse)
          c0 = __fdividef(gs, all);
        else  // ((P + rho) q_O - rho) / (sum over O), with q_O's own exponent
          c0 = ro.m == ninf
                   ? 0.0f
                   : gs * __fdividef((row_mass + rho) * ex2_approx(shifted - lsum) * o - rho, o);
        if (!live) {
          c0 = 0.0f;
#pragma unroll
          for (int i = 0; i < E; ++i) x[i] = 0.0f;
        }
        T* const g = out + row * a.classes;
        T* const gw = g - lead;
        __syncwarp();  // the pass has read its logits
#pragma unroll
        for (int j = 0; j < E; j += 4 * S) {
          if ((j + 4 * S) * G <= a.classes) {
#pragma unroll
            for (int i = j; i < j + 4 * S; i += S) {
              if constexpr (PAIR) {
                const float2 y = mul2({x[i], x[i + 1]}, splat2(c0));
                if (i > 0 || l > 0 || !lead) {
                  if (there) store_pair(gw + i * G + l * S, y.x, y.y);
                } else if (there) {  // a first class at an odd address
                  g[0] = from_f<T>(y.y);
                }
              } else {
                if (there) g[i * G + l] = from_f<T>(c0 * x[i]);
              }
            }
          } else if (j * G < a.classes + lead) {
#pragma unroll
            for (int i = j; i < j + 4 * S; i += S) {
              const int cls = i * G + l * S - lead;
#pragma unroll
              for (int h = 0; h < S; ++h)
                if (there && cls + h < a.classes && (i > 0 || cls + h >= 0))
                  g[cls + h] = from_f<T>(c0 * x[i + h]);
            }
          }
        }
        __syncwarp();
        if (live) {
#pragma unroll
          for (int q = 0; q < kLaneKept; ++q)
            if (q * G < k && id[q] >= 0 && (counts >> q & 1u)) {
              const float e = ex2_approx(exponent(ze[q], r, c) - lsum);
              g[id[q]] = from_f<T>(gs * ((row_mass + rho) * e - (p[q] + again[q])));
            }
        }
      }
      __syncwarp();
    }
    fence_async();  // the gradient is read, and a later tile written, by bulk copies
    __syncwarp();
    if (a.grad) {
      const uintptr_t b = reinterpret_cast<uintptr_t>(a.grad) + r0 * width;
      const uintptr_t e = b + rows * width;
      const uintptr_t b16 = (b + 15) & ~static_cast<uintptr_t>(15);
      const uintptr_t e16 = e & ~static_cast<uintptr_t>(15);
      auto plain = [&](uintptr_t from, uintptr_t end) {
        for (uintptr_t x = from + lane * sizeof(T); x < end; x += 32 * sizeof(T))
          *reinterpret_cast<T*>(x) = *reinterpret_cast<const T*>(
              reinterpret_cast<const char*>(out) + (x - b));
      };
      if (e16 > b16) {
        if (lane == 0)
          bulk_store(reinterpret_cast<void*>(b16), reinterpret_cast<const char*>(out) + (b16 - b),
                     static_cast<uint32_t>(e16 - b16));
        plain(b, b16);
        plain(e16, e);
      } else {
        plain(b, e);
      }
    }
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    at = next;
    if (at == 0) parity ^= 1;
  }
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
  if (lane == 0) s_total[warp] = total;
  __syncthreads();
  if (threadIdx.x == 0 && (a.partials || loss)) {
    total = 0.0;
    for (int i = 0; i < kTileWarps; ++i) total += s_total[i];
    if (loss) *loss = static_cast<float>(total * loss_scale);  // the only CTA
    else a.partials[blockIdx.x] = total;
  }
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

// How tiles of the call's rows lie in shared memory when G lanes take a row.
TilePlan plan_tiles(const DistillArgs& a, int G, int size, int sms) {
  const int pass = 32 / G, vs = a.value_dtype == SPLAX_F32 ? 4 : 2, is = a.wide_ids ? 8 : 4;
  const int64_t stride = a.row_stride * size, width = static_cast<int64_t>(a.classes) * size;
  // rows far apart are copied one by one; close ones with what lies between
  const bool apart = stride > width + width / 4 + 32;
  TilePlan t;
  t.pitch = apart ? static_cast<int>((width + 31) & ~int64_t{15}) : 0;
  const int64_t row = (apart ? t.pitch : stride) + a.k * (vs + is) + 8;
  // two tiles for each of 16 warps an SM, as far as there are rows for every warp
  int64_t rows = kTileBytes / row;
  const int64_t share = (a.rows + sms * 16 - 1) / (sms * 16);
  if (rows > share) rows = share + pass - 1;
  rows = rows / pass * pass;
  if (rows < pass) rows = pass;
  auto room = [](int64_t bytes) { return static_cast<int>((bytes + 30) & ~int64_t{15}); };
  t.rows = static_cast<int>(rows);
  t.values = 16 + (apart ? static_cast<int>(rows) * t.pitch : room((rows - 1) * stride + width));
  t.ids = t.values + room(rows * a.k * vs);
  t.lse = t.ids + room(rows * a.k * is);
  t.weights = t.lse + (a.top_lse ? room(rows * 4) : 0);
  t.stage = t.weights + (a.weights ? room(rows * 4) : 0);
  t.warp = kTileStages * t.stage;
  return t;
}

template <typename T, int G, int E>
int launch_tiles(const DistillArgs& a, const LossParams& p, const TilePlan& t,
                 cudaStream_t stream) {
  const int sms = sm_count(), size = sizeof(T);
  const int64_t tiles = (a.rows + t.rows - 1) / t.rows;
  int per_sm = kSharedMost / (kTileWarps * t.warp + 1536);
  per_sm = per_sm < 1 ? 1 : per_sm > 4 ? 4 : per_sm;
  int64_t grid = (tiles + kTileWarps - 1) / kTileWarps;
  if (grid > sms * per_sm) grid = sms * per_sm;
  const uintptr_t both = reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.grad);
  const bool pair = !a.grad || (both % (2 * size) == 0 && (a.row_stride - a.classes) % 2 == 0);
  launch_clusters(pair ? distill_tile_kernel<T, G, E, true> : distill_tile_kernel<T, G, E, false>,
                  static_cast<unsigned>(grid), 1, 32 * kTileWarps, kTileWarps * t.warp, stream, p,
                  t, grid == 1 ? a.loss : nullptr, a.temperature * a.temperature / a.denom);
  return static_cast<int>(grid);
}

// Lanes to a row: of those that hold it in registers, take its entries and fit the tiles of four
// warps into shared memory with room for a second CTA, the cheapest.
template <typename T>
int launch_short(const DistillArgs& a, const LossParams& p, cudaStream_t stream) {
  const int sms = sm_count(), size = sizeof(T);
  int G = 32;
  TilePlan t = plan_tiles(a, 32, size, sms);
  double least = 1e30;
  for (int g = 1; g <= 32; g *= 2) {
    const TilePlan u = plan_tiles(a, g, size, sms);
    if (a.classes >= 40 * g || a.k > kLaneKept * g || kTileWarps * u.warp > kSharedMost / 2 - 2048)
      continue;
    const double cost = tile_cost(g, a.classes, u.pitch ? u.pitch : a.row_stride * size, size);
    if (cost < least) least = cost, G = g, t = u;
  }
  if (a.classes >= 1280) return launch_tiles<T, 32, 64>(a, p, t, stream);
  switch (G) {
    case 1: return launch_tiles<T, 1, 40>(a, p, t, stream);
    case 2: return launch_tiles<T, 2, 40>(a, p, t, stream);
    case 4: return launch_tiles<T, 4, 40>(a, p, t, stream);
    case 8: return launch_tiles<T, 8, 40>(a, p, t, stream);
    case 16: return launch_tiles<T, 16, 40>(a, p, t, stream);
    default: return launch_tiles<T, 32, 40>(a, p, t, stream);
  }
}

// Chunks of a row, for the threads that work on one: eight vectors a thread (fewer, and the cost of
// passing a chunk on shows: 32 % at four), and slack for a row that is a little longer than a
// power of two.
constexpr int chunk_vecs(int threads) { return 8 * threads + 32; }

template <typename T, int THREADS, int CTAS, int SLOTS>
int launch_ring(const DistillArgs& a, const LossParams& p, cudaStream_t stream) {
  const int all = row_share_vecs(a.classes, kVec<T>, 1);
  const int chunks = (all + chunk_vecs(THREADS) - 1) / chunk_vecs(THREADS);
  const int vecs = ((all + chunks - 1) / chunks + 31) & ~31;
  const int keep = chunks <= SLOTS ? chunks : 1;
  const int64_t fit = static_cast<int64_t>(sm_count()) * CTAS;
  const unsigned grid = static_cast<unsigned>(a.rows < fit ? a.rows : fit);
  launch_clusters(a.k <= 32 ? distill_ring_kernel<T, THREADS, CTAS, 32>
                            : distill_ring_kernel<T, THREADS, CTAS, 128>,
                  grid, 1, THREADS + 96, 16 * vecs * SLOTS, stream, p, chunks, vecs, SLOTS, keep);
  return static_cast<int>(grid);
}

template <typename T>
int launch_distill_t(const DistillArgs& a, cudaStream_t stream) {
  const double inv = 1.0 / a.temperature;
  LossParams p{a.logits,      a.rows,
               a.row_stride,  a.classes,
               a.k,           a.top_values,
               a.top_ids,     a.top_lse,
               a.weights,     a.value_dtype,
               a.wide_ids,    inv,
               scale_of(a.temperature), static_cast<float>(inv),
               static_cast<float>(inv - static_cast<float>(inv)),
               static_cast<float>(a.temperature / a.denom), a.v_loss,
               a.grad,        a.partials,
               a.unless_one};
  const double loss_scale = a.temperature * a.temperature / a.denom;
  int partials = 0, launched = 1;
  if (a.rows == 0) {
    launched = 0;
  } else if (a.classes < 2048) {  // 2000 x 100,000 rows bf16 278 us, by the ring 467
    partials = launch_short<T>(a, p, stream);
  } else if (2 * a.rows < sm_count()) {  // loss, 33 rows of 65,537 fp32 7.8 us, by the ring 10; 120: 14, 10
    const int64_t bytes = a.classes * static_cast<int64_t>(sizeof(T));
    const unsigned size = row_cluster(a.rows, bytes, sm_count());
    const int vecs = row_share_vecs(a.classes, kVec<T>, size);
    partials = static_cast<int>(a.rows);
    launch_clusters(a.k <= 32 ? distill_share_kernel<T, 32> : distill_share_kernel<T, 128>,
                    partials, size, kShareThreads, 16 * vecs, stream, p,
                    partials == 1 ? a.loss : nullptr, loss_scale);
  } else {
    // Rows of one chunk, two in flight in each of five CTAs an SM (with six, at 40
    // registers, 40,000 rows of 8193 bf16 356 us instead of 334, 20,000 of 4000 fp32 166 instead of
    // 159, 100,000 of 2050 fp32 503 instead of 501); rows of which three CTAs' an SM fit
    // the L2 cache for their second reading; longer ones, one an SM. With gradient, bf16, these three
    // in turn: 13,000 classes x 20,000 rows 243, 252, 426 us; 50,000 x 8000 364, 334, 365;
    // 80,000 x 5000 394, 355, 340.
    const int vecs = row_share_vecs(a.classes, kVec<T>, 1);
    if (vecs <= chunk_vecs(128)) partials = launch_ring<T, 128, 5, 2>(a, p, stream);
    else if (vecs <= 4 * chunk_vecs(256)) partials = launch_ring<T, 256, 3, 2>(a, p, stream);
    else partials = launch_ring<T, 512, 1, 3>(a, p, stream);
  }
  if (a.loss && partials != 1) {
    launch_pdl(distill_finish_kernel, 1, 256, 0, stream, a.partials, partials, loss_scale, a.loss);
    ++launched;
  }
  return launched;
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

}  // namespace splax
