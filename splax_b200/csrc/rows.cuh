// Device helpers of the kernels on rows of logits: element types and 16-byte vectors of them,
// bulk copies between global and shared memory, and a cluster's share of one row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/splax_b200.h"
#include "common.cuh"

namespace splax {

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

template <typename T>
constexpr int kDtype = SPLAX_F32;
template <>
constexpr int kDtype<__nv_bfloat16> = SPLAX_BF16;
template <>
constexpr int kDtype<__half> = SPLAX_F16;

// Elements of a 16-byte vector.
template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));

__device__ __forceinline__ void unpack(uint4 u, float (&x)[4], float) {
  x[0] = __uint_as_float(u.x);
  x[1] = __uint_as_float(u.y);
  x[2] = __uint_as_float(u.z);
  x[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack2(uint32_t u, float& a, float& b, __nv_bfloat16) {
  a = __uint_as_float(u << 16);
  b = __uint_as_float(u & 0xffff0000u);
}
__device__ __forceinline__ void unpack2(uint32_t u, float& a, float& b, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
  a = f.x;
  b = f.y;
}
template <typename T>
__device__ __forceinline__ void unpack(uint4 u, float (&x)[8], T t) {
  unpack2(u.x, x[0], x[1], t);
  unpack2(u.y, x[2], x[3], t);
  unpack2(u.z, x[4], x[5], t);
  unpack2(u.w, x[6], x[7], t);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint4 pack(const float (&x)[4], float) {
  return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                    __float_as_uint(x[3]));
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&x)[8], T t) {
  return make_uint4(pack2(x[0], x[1], t), pack2(x[2], x[3], t), pack2(x[4], x[5], t),
                    pack2(x[6], x[7], t));
}

// Maximum that returns NaN if either operand is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float warp_max(float x) {  // NaN if any lane has one
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

// log2(e) / tau in two parts, both positive (so that -inf times either is -inf): with one alone the
// probabilities would be those of a temperature 1e-8 away, which a small divergence shows.
struct Scale {
  float hi, lo;
};
inline Scale scale_of(double temperature) {
  const double c = 1.4426950408889634 / temperature;
  float hi = static_cast<float>(c);
  if (hi >= c) hi = std::nextafterf(hi, 0.0f);
  const float lo = static_cast<float>(c - hi);
  return {hi, lo > 0.0f ? lo : 1.4e-45f};  // which near a temperature of 1e30 may fall below fp32
}

// Sums of powers of two are held against a reference logit m: s = sum 2^(x c - ms), c = log2(e) /
// tau, ms = m c rounded to a whole number, which makes the factor between two references exact. As
// fused multiply-adds, the larger part of c first, the exponent has two roundings of its own size.
// That is a plain reference. Beyond 2^22 ms is no longer within one of m c (at 2^33 it is some
// hundreds off, and the sum overflows), so there, and for an infinite or NaN m, the difference
// x - m is taken first and the sum is sum 2^((x - m) c).
struct Ref {
  float m, ms;
  __device__ __forceinline__ bool plain() const { return fabsf(ms) < 4194304.0f; }
};
__device__ __forceinline__ Ref ref_of(float m, Scale c) { return {m, rintf(m * c.hi)}; }
__device__ __forceinline__ float exponent(float x, Ref r, Scale c) {
  return r.plain() ? fmaf(x, c.lo, fmaf(x, c.hi, -r.ms))
                   : (x - (r.m == neg_inf() ? 0.0f : r.m)) * c.hi;
}
__device__ __forceinline__ float2 exponent2(float2 x, float ms, Scale c) {  // against a plain one
  return fma2(x, splat2(c.lo), fma2(x, splat2(c.hi), splat2(-ms)));
}
// Exponent of the factor that brings a sum against `from` to the larger reference `to`.
__device__ __forceinline__ float shift(Ref from, Ref to, Scale c) {
  float e = from.ms - to.ms;
  if (!(max_nan(fabsf(from.ms), fabsf(to.ms)) < 4194304.0f)) {
    if (to.plain()) e = exponent(from.m, to, c);
    else if (from.plain()) e = -exponent(to.m, from, c);
    else e = (from.m - (to.m == neg_inf() ? 0.0f : to.m)) * c.hi;
  }
  return e;
}
constexpr double kLn2 = 0.693147180559945309;
// ln of 2^ms, in 64 bits.
__device__ __forceinline__ double ln_of(Ref r, double inv_tau) {
  return r.plain() ? kLn2 * r.ms : r.m * inv_tau;
}
// The same less m / tau, m a logit of the row: beside the type's lowest value 64 bits have no room for
// ln of a sum, so large logits are subtracted from one another before anything else is added.
__device__ __forceinline__ double ln_beside(Ref r, float m, double inv_tau) {
  return r.plain() ? kLn2 * r.ms - m * inv_tau : (static_cast<double>(r.m) - m) * inv_tau;
}
// ln s, to the rounding of a number below one.
__device__ __forceinline__ double ln_of(float s) {
  const uint32_t u = __float_as_uint(s);
  if (!(s >= 1.2e-38f && s < 3e38f)) return logf(s);
  return kLn2 * (static_cast<int>(u >> 23) - 127) +
         logf(__uint_as_float((u & 0x7fffffu) | 0x3f800000u));
}

// A maximum and the sum against it; of nothing (-inf, 0).
struct MaxSum {
  float m, s;
};
// In the place of what a late copy should have brought: NaN, which every join hands on.
__device__ __forceinline__ MaxSum poison() {
  return {__int_as_float(0x7fc00000), __int_as_float(0x7fc00000)};
}
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, Scale c) {
  const float m = max_nan(a.m, b.m);
  const Ref r = ref_of(m, c);
  return {m, a.s * ex2_approx(shift(ref_of(a.m, c), r, c)) +
                 b.s * ex2_approx(shift(ref_of(b.m, c), r, c))};
}
__device__ __forceinline__ MaxSum warp_join(MaxSum a, Scale c) {
  const float m = warp_max(a.m);
  return {m, warp_sum(a.s * ex2_approx(shift(ref_of(a.m, c), ref_of(m, c), c)))};
}
// A thread's running maximum and sum, N values at a time. The sum stays against its reference while
// no term exceeds 2^kSlack, so that it is hardly ever rescaled after the first batch: with a
// rescaling for every new maximum some lane of a warp had one in nearly every batch (loss of
// 4000 x 128,000 bf16 246 us). A reference that is not plain has NaN for ms, which
// sends every batch through the test.
struct Running {
  static constexpr float kSlack = 32.0f;
  float m = -INFINITY;
  Ref r{-INFINITY, __builtin_nanf("")};
  float2 s{0.0f, 0.0f};
  __device__ __forceinline__ MaxSum get(Scale c) const {
    return {m, (s.x + s.y) * ex2_approx(shift(r, ref_of(m, c), c))};
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&x)[N], float vm, Scale c) {
    m = max_nan(m, vm);
    if (!(fmaf(vm, c.hi, -r.ms) < kSlack)) {
      const Ref to = ref_of(m, c);
      const float f = ex2_approx(shift(r, to, c));
      s.x *= f;
      s.y *= f;
      r = to;
      if (!to.plain()) {
        r.ms = __builtin_nanf("");
        float one = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) one += ex2_approx(exponent(x[i], r, c));
        s.x += one;
        return;
      }
    }
    float2 sum[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};  // their own sum first: fewer roundings in s
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 t = exponent2({x[i], x[i + 1]}, r.ms, c);
      sum[i / 2 & 1] = add2(sum[i / 2 & 1], {ex2_approx(t.x), ex2_approx(t.y)});
    }
    s = add2(s, add2(sum[0], sum[1]));
  }
};

// Maximum of a 16-byte vector, NaN if it holds one.
__device__ __forceinline__ float vec_max(uint4 u, float) {
  return max_nan(max_nan(__uint_as_float(u.x), __uint_as_float(u.y)),
                 max_nan(__uint_as_float(u.z), __uint_as_float(u.w)));
}
__device__ __forceinline__ float vec_max(uint4 u, __nv_bfloat16) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
  const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
  return max_nan(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float vec_max(uint4 u, __half) {
  const __half2* h = reinterpret_cast<const __half2*>(&u);
  const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
  return max_nan(__low2float(m), __high2float(m));
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint64_t* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void mbar_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Waits for the phase of the given parity; false if the limit ran out, which no copy that was
// issued within bounds can cause (the caller then poisons its results instead of using them).
// `rest`: a warp that runs ahead of the others leaves them its issue slots between tries.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, bool rest = false) {
  for (int i = 0; i < (1 << 22); ++i) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n"
        " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (done) return true;
    if (rest) __nanosleep(64);
  }
  return false;
}
// 16-byte aligned addresses, a multiple of 16 bytes.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}
// The other way; part of the thread's current bulk group.
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst),
               "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}
// Orders this thread's accesses to shared memory before later bulk copies that touch it.
__device__ __forceinline__ void fence_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// The address of this CTA's shared variable in the cluster's CTA of the given rank.
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void cluster_store(uint32_t addr, float x) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(x) : "memory");
}
__device__ __forceinline__ uint64_t cluster_load(uint32_t addr) {
  uint64_t x;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(x) : "r"(addr) : "memory");
  return x;
}

// A barrier of some of a CTA's warps, THREADS threads in all; those that arrive do not wait.
template <int THREADS>
__device__ __forceinline__ void pair_sync(int id) {
  asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
}
template <int THREADS>
__device__ __forceinline__ void pair_arrive(int id) {
  asm volatile("barrier.cta.arrive %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
}
template <typename T, int N>
__device__ __forceinline__ void add_vectors(Running& run, const uint4* at, int stride, Scale c) {
  uint4 u[N];
#pragma unroll
  for (int q = 0; q < N; ++q) u[q] = at[q * stride];
  float x[N * kVec<T>], vm = neg_inf();
#pragma unroll
  for (int q = 0; q < N; ++q) {
    float y[kVec<T>];
    unpack(u[q], y, T{});
    vm = max_nan(vm, vec_max(u[q], T{}));
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) x[q * kVec<T> + i] = y[i];
  }
  run.add(x, vm, c);
}
template <int N>
struct Int {
  static constexpr int value = N;
};

__device__ __forceinline__ uint32_t cluster_load_u32(uint32_t addr) {
  uint32_t x;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(addr) : "memory");
  return x;
}

// One CTA's share of a row: the 16-byte vectors [v0, v1) of the aligned span around it. A vector
// that reaches over either end of the row is filled by plain loads, with -inf in the places that
// are not the row's; the others come by one bulk copy.
template <typename T>
struct RowShare {
  int lead;        // elements of the first vector before the row
  int v0, v1;      // vectors of this CTA
  int cls0;        // class of the first element of vector v0 (negative by `lead` at v0 = 0)
  const T* first;  // address of vector v0
};
template <typename T>
__device__ __forceinline__ RowShare<T> row_share(const T* z, int classes, int rank, int size) {
  RowShare<T> s;
  s.lead = static_cast<int>((reinterpret_cast<uintptr_t>(z) & 15u) / sizeof(T));
  const int all = (s.lead + classes + kVec<T> - 1) / kVec<T>;
  const int per = (all + size - 1) >> (31 - __clz(size));  // size is a power of two
  s.v0 = min(rank * per, all);
  s.v1 = min(s.v0 + per, all);
  s.cls0 = s.v0 * kVec<T> - s.lead;
  s.first = z + s.cls0;
  return s;
}
// Vectors of shared memory that any share takes.
inline int row_share_vecs(int classes, int vec, int size) {
  const int all = (vec - 1 + classes + vec - 1) / vec;
  return (all + size - 1) / size;
}
// One thread: the bulk copy of a share. The shared memory must be free of earlier accesses (a
// barrier, with fence_async by those that made them).
template <typename T>
__device__ __forceinline__ void load_share(const RowShare<T>& s, int classes, uint4* buf,
                                           uint64_t* bar) {
  const int n = s.v1 - s.v0;
  const int b0 = n > 0 && s.cls0 < 0 ? 1 : 0;
  const int b1 = n > 0 && s.cls0 + n * kVec<T> > classes ? n - 1 : n;
  const uint32_t bytes = b1 > b0 ? 16u * static_cast<uint32_t>(b1 - b0) : 0u;
  mbar_expect(bar, bytes);
  if (bytes) bulk_load(buf + b0, s.first + b0 * kVec<T>, bytes, bar);
}
// One warp: the vectors that reach over an end of the row, by plain loads, one element a lane
// (lanes below 2 kVec: the first vector's, then the last's). The store may come later.
template <typename T>
struct ShareEnds {
  int at;  // element of the share, -1 for none
  T x;
};
template <typename T>
__device__ __forceinline__ ShareEnds<T> load_ends(const RowShare<T>& s, int classes) {
  const int lane = threadIdx.x & 31, n = s.v1 - s.v0;
  const bool head = n > 0 && s.cls0 < 0, tail = n > 0 && s.cls0 + n * kVec<T> > classes;
  const bool mine = lane < kVec<T> ? head : lane < 2 * kVec<T> && tail && !(head && n == 1);
  ShareEnds<T> r{-1, from_f<T>(neg_inf())};
  if (mine) {
    r.at = lane < kVec<T> ? lane : (n - 2) * kVec<T> + lane;
    const int c = s.cls0 + r.at;
    if (c >= 0 && c < classes) r.x = s.first[r.at];
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store_ends(const ShareEnds<T>& r, uint4* buf) {
  if (r.at >= 0) reinterpret_cast<T*>(buf)[r.at] = r.x;
}

constexpr int kTileWarps = 4, kTileStages = 2;  // short rows: warps of a CTA, tiles of a warp
constexpr int kSharedMost = 227 * 1024;         // bytes a CTA may have
constexpr int kDynamicMost = 216 * 1024;        // beside what a kernel declares
constexpr int kTileBytes = 6656;

// The bytes [b, e) on their way to `to` + their addresses, which are `to` + 16-byte aligned: a bulk
// copy of the 16-byte pieces [b16, e16) that lie within the whole array [base, limit), plain loads
// of what an end of the array leaves over.
struct Part {
  uintptr_t b, e, b16, e16, to;
};
__device__ __forceinline__ Part part_of(char* dst, uintptr_t base, uintptr_t b, uintptr_t e,
                                        uintptr_t limit) {
  Part p;
  p.b = b;
  p.e = e;
  p.b16 = p.b & ~static_cast<uintptr_t>(15);
  p.e16 = (p.e + 15) & ~static_cast<uintptr_t>(15);
  p.to = reinterpret_cast<uintptr_t>(dst) - p.b16;
  if (p.b16 < base) p.b16 += 16;
  if (p.e16 > limit) p.e16 -= 16;
  if (p.e16 <= p.b16 || p.b16 >= p.e) p.b16 = p.e16 = p.e;  // no such piece
  return p;
}
// By one lane.
__device__ __forceinline__ void load_part(const Part& p, uint64_t* bar) {
  if (p.e16 > p.b16)
    bulk_load(reinterpret_cast<void*>(p.to + p.b16), reinterpret_cast<const void*>(p.b16),
              static_cast<uint32_t>(p.e16 - p.b16), bar);
  auto plain = [&](uintptr_t from, uintptr_t to) {
    for (uintptr_t x = from; x < to; x += 2)
      *reinterpret_cast<uint16_t*>(p.to + x) = *reinterpret_cast<const uint16_t*>(x);
  };
  plain(p.b, p.b16);  // nothing, but for an array that is not aligned
  plain(p.e16, p.e);
}

__device__ __forceinline__ void load_pair(const float* p, float& a, float& b) {
  const float2 v = *reinterpret_cast<const float2*>(p);
  a = v.x;
  b = v.y;
}
template <typename T>
__device__ __forceinline__ void load_pair(const T* p, float& a, float& b) {
  unpack2(*reinterpret_cast<const uint32_t*>(p), a, b, T{});
}

template <int G>
__device__ __forceinline__ float group_max(float x) {
  if constexpr (G == 32) return warp_max(x);
#pragma unroll
  for (int off = G / 2; off > 0; off >>= 1) x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, off));
  return x;
}
template <int G>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int off = G / 2; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

// Order of the kept logits as one 64-bit number: the value (NaN above all, the two zeros alike),
// then the lower class. Never 0.
__device__ __forceinline__ uint32_t order_bits(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  if (v != v) return 0xffffffffu;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(float v, int32_t c) {
  return (static_cast<uint64_t>(order_bits(v)) << 32) | (0xffffffffu - static_cast<uint32_t>(c));
}
__device__ __forceinline__ int32_t key_class(uint64_t key) {
  return static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(key));
}

// Largest number of lanes of a warp that meet in one bank of shared memory when G lanes a row read
// consecutive elements of rows `pitch` bytes apart.
inline int bank_conflicts(int G, int64_t pitch, int bytes) {
  int banks[32] = {}, most = 0;
  for (int i = 0; i < 32; ++i) {
    const int64_t at = (i / G) * pitch + (i % G) * bytes;
    int& n = banks[at / 4 % 32];
    // neighbours in one word are one access
    if (i % G == 0 || at / 4 != (at - bytes) / 4) ++n;
    most = n > most ? n : most;
  }
  return most;
}

// Cycles of an SM per row when G lanes take a row in a pass of a warp: about 900 instructions a pass
// and 12 a class of a lane (counted by the profiler for rows of 21 to 513 classes), at 2.4 a cycle, and
// the shared memory's passes for reading a class and writing it back. So few lanes, which share the
// pass among many rows, unless rows some power of two apart then meet in the banks: 32 fp32
// classes with gradient cost 292 us a million rows with 8 lanes, without conflicts beyond 4.
inline double tile_cost(int G, int classes, int64_t pitch, int bytes) {
  const int each = (classes + G - 1) / G;
  return ((900 + 12 * each) / 2.4 + 2.0 * each * bank_conflicts(G, pitch, bytes)) * G / 32;
}

// Launch with clusters of `size` CTAs, programmatic like launch_pdl.
template <typename... KArgs, typename... Args>
inline void launch_clusters(void (*kernel)(KArgs...), unsigned clusters, unsigned size,
                            unsigned block, size_t smem, cudaStream_t stream, Args... args) {
  // 48 KB, the kernel's own part included, need no asking. The same for every call: one with less
  // must not take it back from a captured launch with more.
  if (smem > 32 * 1024)
    (void)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kDynamicMost);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * size);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = size;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = size > 1 ? 2 : 1;
  (void)cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

// CTAs of one cluster for a long row: while the rows are too few to give every SM a CTA, and in any
// case until the share of a CTA is kShareBytes or less, a row is split further, down to
// kMinShareBytes a CTA, up to eight.
constexpr int64_t kShareBytes = 35 * 1024;
constexpr int64_t kMinShareBytes = 4 * 1024;
inline unsigned row_cluster(int64_t rows, int64_t row_bytes, int sms) {
  unsigned size = 1;
  while (size < 8 && row_bytes > kShareBytes * size) size *= 2;
  while (size < 8 && rows * size < sms && row_bytes >= 2 * kMinShareBytes * size) size *= 2;
  return size;
}
inline int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess)
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

}  // namespace splax
