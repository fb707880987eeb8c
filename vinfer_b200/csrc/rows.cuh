// rows.cuh — reading rows of logits: 16-byte vectors at any element alignment, exponentials in
// base 2, and warp and block helpers shared by the kernels beside the sampler.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include <nvtx3/nvToolsExt.h>

#include "vinfer_sampler.h"

namespace rows {

constexpr unsigned FULL = 0xffffffffu;
constexpr float L2E = 1.4426950408889634f;      // log2(e) rounded to float
constexpr double L2E_D = 1.4426950408889634074;  // log2(e)
constexpr double LN2_D = 0.69314718055994530942;

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

// 2^x by the hardware's approximation (2 ulp; 0 below the normal range)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// two floats in one 64-bit register: sm_100 multiplies and adds them in one instruction
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(uint64_t r, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t ex2_2(uint64_t a) {
  float x, y;
  split(a, x, y);
  return pair(ex2(x), ex2(y));
}

// order-preserving key of a float; -0 folds into +0
__device__ __forceinline__ uint32_t okey(float v) {
  const uint32_t b = __float_as_uint(__fadd_rn(v, 0.0f));
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float from_okey(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// 16 bytes of logits as floats
template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int A = 8;
  static constexpr uint32_t NEG_INF_WORD = 0xff80ff80u;
  static __device__ __forceinline__ void unpack(const uint4& q, float (&f)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  // pairs of floats, in element order
  static __device__ __forceinline__ void pairs(const uint4& q, uint64_t (&f)[4]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  // largest element of U vectors, NaN ignored: packed comparisons, unpacked once
  template <int U>
  static __device__ __forceinline__ float max(const uint4 (&q)[U]) {
    __nv_bfloat162 m[4];
    memcpy(m, &q[0], 16);
#pragma unroll
    for (int u = 1; u < U; ++u) {
      __nv_bfloat162 x[4];
      memcpy(x, &q[u], 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) m[i] = __hmax2(m[i], x[i]);
    }
    const __nv_bfloat162 r = __hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3]));
    return fmaxf(__low2float(r), __high2float(r));
  }
  // largest element, NaN ignored (two packed comparisons a word pair)
  static __device__ __forceinline__ float max(const uint4& q) {
    __nv_bfloat162 a, b, c, d;
    memcpy(&a, &q.x, 4);
    memcpy(&b, &q.y, 4);
    memcpy(&c, &q.z, 4);
    memcpy(&d, &q.w, 4);
    const __nv_bfloat162 m = __hmax2(__hmax2(a, b), __hmax2(c, d));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ float get(const uint4& q, int j) {
    const uint32_t w = j < 4 ? (j < 2 ? q.x : q.y) : (j < 6 ? q.z : q.w);
    return __uint_as_float((j & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ void put(uint4& q, int j, uint32_t bits) {
    const uint32_t keep = (j & 1) ? 0x0000ffffu : 0xffff0000u;
    const uint32_t add = (j & 1) ? bits << 16 : bits & 0xffffu;
    if (j < 2) q.x = (q.x & keep) | add;
    else if (j < 4) q.y = (q.y & keep) | add;
    else if (j < 6) q.z = (q.z & keep) | add;
    else q.w = (q.w & keep) | add;
  }
  static __device__ __forceinline__ uint32_t bits(const __nv_bfloat16* p) {
    return *reinterpret_cast<const unsigned short*>(p);
  }
  static constexpr uint32_t NEG_INF_BITS = 0xff80u;
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) {
    return __bfloat162float(*p);
  }
  static __device__ __forceinline__ __nv_bfloat16 round(float f) { return __float2bfloat16_rn(f); }
  // rounded to nearest even, the gradient's type
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      memcpy(&w[i], &h, 4);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Vec<float> {
  static constexpr int A = 4;
  static constexpr uint32_t NEG_INF_WORD = 0xff800000u;
  static __device__ __forceinline__ void unpack(const uint4& q, float (&f)[4]) {
    f[0] = __uint_as_float(q.x);
    f[1] = __uint_as_float(q.y);
    f[2] = __uint_as_float(q.z);
    f[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ void pairs(const uint4& q, uint64_t (&f)[2]) {
    f[0] = pair(__uint_as_float(q.x), __uint_as_float(q.y));
    f[1] = pair(__uint_as_float(q.z), __uint_as_float(q.w));
  }
  template <int U>
  static __device__ __forceinline__ float max(const uint4 (&q)[U]) {
    float m = max(q[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) m = fmaxf(m, max(q[u]));
    return m;
  }
  static __device__ __forceinline__ float max(const uint4& q) {
    return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)),
                 fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
  }
  static __device__ __forceinline__ float get(const uint4& q, int j) {
    return __uint_as_float(j < 2 ? (j == 0 ? q.x : q.y) : (j == 2 ? q.z : q.w));
  }
  static __device__ __forceinline__ void put(uint4& q, int j, uint32_t bits) {
    if (j == 0) q.x = bits;
    else if (j == 1) q.y = bits;
    else if (j == 2) q.z = bits;
    else q.w = bits;
  }
  static __device__ __forceinline__ uint32_t bits(const float* p) { return __float_as_uint(*p); }
  static constexpr uint32_t NEG_INF_BITS = 0xff800000u;
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ float round(float f) { return f; }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3]));
  }
};

// A row cut into aligned 16-byte vectors: vector v holds elements [v * A - off, v * A - off + A).
// The first and the last one may hold elements outside the row; those are never read.
template <typename T>
struct Row {
  const T* p;  // the row's first element
  int off;     // elements between the aligned address below p and p
  int V;
  int nv;      // vectors that hold an element of the row
  __device__ __forceinline__ Row(const T* p_, int V_) : p(p_), V(V_) {
    off = (int)(((uintptr_t)p & 15) / sizeof(T));
    nv = (V + off + Vec<T>::A - 1) / Vec<T>::A;
  }
  __device__ __forceinline__ bool whole(int v) const {
    const int e = v * Vec<T>::A - off;
    return e >= 0 && e + Vec<T>::A <= V;
  }
  // vector v; elements outside the row read as -inf
  __device__ __forceinline__ uint4 load(int v) const {
    if (whole(v)) {
      uint4 q;
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                   : "l"(p + ((int64_t)v * Vec<T>::A - off)));
      return q;
    }
    return edge(p, V, v * Vec<T>::A - off);
  }
  // The thread's vectors vb + u * NT + threadIdx.x of a round, below v1; -inf behind it. No
  // branches between the loads, so that all are in flight together: rounds inside the row load
  // at constant offsets, the others by predicate, and their ragged ends are read behind them.
  template <int U, int NT>
  __device__ __forceinline__ void load_round(int vb, int v1, uint4 (&q)[U]) const {
    const T* at = p + ((int64_t)(vb + (int)threadIdx.x) * Vec<T>::A - off);
    const int lo = off ? 1 : 0, hi = min(v1, (V + off) / Vec<T>::A);  // whole vectors
    if (vb >= lo && vb + U * NT <= hi) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(q[u].x), "=r"(q[u].y), "=r"(q[u].z), "=r"(q[u].w)
                     : "l"(at + u * NT * Vec<T>::A));
      return;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = vb + u * NT + (int)threadIdx.x;
      const uint32_t n = Vec<T>::NEG_INF_WORD;
      q[u] = make_uint4(n, n, n, n);
      asm volatile(
          "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\t"
          "@p ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n\t}"
          : "+r"(q[u].x), "+r"(q[u].y), "+r"(q[u].z), "+r"(q[u].w)
          : "l"(at + u * NT * Vec<T>::A), "r"((uint32_t)(v >= lo && v < hi)));
    }
    if (vb == 0 && off && threadIdx.x == 0) q[0] = edge(p, V, -off);
    if (hi < v1 && hi >= vb && hi < vb + U * NT && (hi > 0 || !off)) {  // the last, a ragged one
      const int mine = hi - vb - (int)threadIdx.x;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (mine == u * NT) q[u] = edge(p, V, hi * Vec<T>::A - off);
    }
  }
  // the vector whose first element is e0, element by element
  static __device__ __noinline__ uint4 edge(const T* p, int V, int e0) {
    const uint32_t n = Vec<T>::NEG_INF_WORD;
    uint4 q = make_uint4(n, n, n, n);
    for (int j = 0; j < Vec<T>::A; ++j)
      if (e0 + j >= 0 && e0 + j < V) Vec<T>::put(q, j, Vec<T>::bits(p + e0 + j));
    return q;
  }
};

// Streams vectors [v0, v1) of a row through work(q, first vector) in rounds of U a thread, with
// BUFS - 1 rounds in flight while one is worked on. v0 < v1.
template <int U, int NT, int BUFS, typename T, typename F>
__device__ __forceinline__ void stream_rounds(const Row<T>& R, int v0, int v1, F&& work) {
  uint4 q[BUFS][U];
#pragma unroll
  for (int b = 0; b < BUFS - 1; ++b)
    if (v0 + b * NT * U < v1) R.template load_round<U, NT>(v0 + b * NT * U, v1, q[b]);
  for (int v = v0;; v += BUFS * NT * U) {
#pragma unroll
    for (int b = 0; b < BUFS; ++b) {
      const int vb = v + b * NT * U, ahead = vb + (BUFS - 1) * NT * U;
      if (ahead < v1) R.template load_round<U, NT>(ahead, v1, q[(b + BUFS - 1) % BUFS]);
      work(q[b], vb);
      if (vb + NT * U >= v1) return;
    }
  }
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}

// Softmax sums are held as (m, s): s in units of 2^(m * scale), m a logit of those summed, scale =
// log2(e) / temperature rounded to float. m stays a logit, so sums of rows at the type's lowest
// value (a mask) need no exponent beyond the float's range, and the rounding of `scale` only
// stretches distances from m.
//
// A thread's sum while it streams: m is the largest element of its first round, and moves only when a
// later one counts 16 times as much, so that exponents stay small and few rounds rescale: a
// round costs an ex2 an element, and a multiply-add and an addition for each two. The argument
// x * scale - c is rounded once, and what c misses of m * scale (a small d) is put right in the round's
// sum, by 2^-d - 1 taken as a series. From |c| = NEAR_ZERO on, where d is no longer small (2^-3 below
// it), distances from m are formed first: they are exact there, since elements that count are within
// a factor of two of m.
//
// S is float, or double where the sum's rounding decides something: rounds are then added, and the sum
// moved to another m, without loss (a beam step 28.6 -> 29.1 us and 95.7 -> 98.2; with the move out of
// line 30.4 and 100.8, with pairs of floats 31.3 and 102.2).
__device__ __forceinline__ double moved(double s, float from, float to, float scale) {
  return s * exp2(((double)from - (double)to) * (double)scale);
}
__device__ __forceinline__ float moved(float s, float from, float to, float scale) {
  return s * ex2((from - to) * scale);
}
template <typename S>
struct Exps {
  static constexpr float NEAR_ZERO = 4194304.f;  // 2^22
  float m;
  S s;
  float c, fix;  // m * scale rounded, and what that does to a round's sum
  float scale;
  __device__ __forceinline__ explicit Exps(float scale_)
      : m(neg_inf()), s(0), c(0.f), fix(0.f), scale(scale_) {}
  // the thread's vectors q, whose largest element is mx
  template <typename T, int U>
  __device__ __forceinline__ void add(const uint4 (&q)[U], float mx) {
    constexpr int H = Vec<T>::A / 2;
    if ((mx - m) * scale > 4.f) {  // the first round (m is -inf) and seldom again
      if (s != 0) s = moved(s, m, mx, scale);
      m = mx;
      c = m * scale;
      const float y = -fmaf(m, scale, -c) * (float)LN2_D;  // e^y - 1; y^6 / 720 is left out, below 1e-9
      fix = y * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 1.f / 120, 1.f / 24), 1.f / 6), 0.5f), 1.f);
    }
    float sum;
    if (fabsf(c) < NEAR_ZERO) {
      const uint64_t k = pair(scale, scale), d = pair(-c, -c);
      uint64_t all = pair(0.f, 0.f);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint64_t f[H];
        Vec<T>::pairs(q[u], f);
        uint64_t t = ex2_2(fma2(f[0], k, d));
#pragma unroll
        for (int j = 1; j < H; ++j) t = add2(t, ex2_2(fma2(f[j], k, d)));
        all = add2(all, t);
      }
      float a, b;
      split(all, a, b);
      sum = a + b;
      sum = fmaf(sum, fix, sum);
    } else {  // distances first
      sum = 0.f;
#pragma unroll 1
      for (int u = 0; u < U; ++u) {
        uint4 v = q[0];
#pragma unroll
        for (int i = 1; i < U; ++i)
          if (i == u) v = q[i];
        for (int j = 0; j < Vec<T>::A; ++j) sum += ex2((Vec<T>::get(v, j) - m) * scale);
      }
    }
    s += sum;
  }
};

// Joins the sums of a block's threads: every thread gets the block's. Fixed order: the result does
// not depend on timing. `sm`: 2 * NW floats.
template <int NW>
__device__ __forceinline__ void block_join(float& m, float& s, float scale, float* sm) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if (s == 0.f) m = neg_inf();
  const float mw = warp_max(m);
  float sw = s == 0.f ? 0.f : moved(s, m, mw, scale);
#pragma unroll
  for (int o = 16; o; o >>= 1) sw += __shfl_xor_sync(FULL, sw, o);
  if (lane == 0) {
    sm[w] = mw;
    sm[NW + w] = sw;
  }
  __syncthreads();
  float mb = sm[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) mb = fmaxf(mb, sm[i]);
  float sb = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) sb += sm[NW + i] == 0.f ? 0.f : moved(sm[NW + i], sm[i], mb, scale);
  m = mb;
  s = sb;
  __syncthreads();
}
// The same in double, moved once: the block's largest m is found first. `sm`: NW doubles, `mx`: NW floats.
template <int NW>
__device__ __forceinline__ void block_join(float& m, double& s, float scale, double* sm, float* mx) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const float mw = warp_max(s == 0 ? neg_inf() : m);
  if (lane == 0) mx[w] = mw;
  __syncthreads();
  float mb = mx[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) mb = fmaxf(mb, mx[i]);
  const double sw = warp_sum(s == 0 ? 0.0 : moved(s, m, mb, scale));
  if (lane == 0) sm[w] = sw;
  __syncthreads();
  s = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) s += sm[i];
  m = mb;
  __syncthreads();
}

// ---- barriers in shared memory and bulk copies ----
__device__ __forceinline__ void bar_init(uint64_t* b, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(b)),
               "r"(bytes)
               : "memory");
}
// The limit of a wait: tries that may each leave the warp suspended for suspend_ns, and sleep a little
// behind it: a warp that polled would take issue slots from those that compute (512 -> 494 us for the
// distillation step).
struct WaitLimit {
  int32_t tries;
  uint32_t suspend_ns;
};
constexpr WaitLimit WAIT_LIMIT = {1 << 18, 20000};  // 0.1 to 5 s; the waits here last microseconds
// CLUSTER: what other CTAs of the cluster sent is seen behind it.
template <bool CLUSTER>
__device__ __forceinline__ bool bar_try(uint64_t* b, uint32_t parity, uint32_t suspend_ns) {
  uint32_t done;
  if (CLUSTER)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(b)), "r"(parity), "r"(suspend_ns)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(b)), "r"(parity), "r"(suspend_ns)
        : "memory");
  return done;
}
// Waits for the phase of this parity to end; false when the limit is reached, or once another wait of
// the CTA has given up: *dead is then set, and every role leaves. One thread's wait.
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity, volatile int* dead,
                                         WaitLimit limit) {
  for (int i = 0; i < limit.tries; ++i) {
    if (bar_try<false>(b, parity, limit.suspend_ns)) return true;
    if (*dead) return false;
    __nanosleep(100);
  }
  *dead = 1;
  return false;
}
// The same for a whole warp, whose lanes all get the same answer.
template <bool CLUSTER = false>
__device__ __forceinline__ bool warp_wait(uint64_t* b, uint32_t parity, volatile int* dead,
                                          WaitLimit limit) {
  for (int i = 0; i < limit.tries; ++i) {
    if (__all_sync(FULL, bar_try<CLUSTER>(b, parity, limit.suspend_ns))) return true;
    if (__any_sync(FULL, *dead)) return false;
    __nanosleep(100);
  }
  *dead = 1;
  return false;
}
// L2 policy for data that is not needed again
__device__ __forceinline__ uint64_t evict_first() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void store_once(void* dst, const uint4& q, uint64_t policy) {
  asm volatile("st.global.L2::cache_hint.v4.b32 [%0], {%1, %2, %3, %4}, %5;" ::"l"(dst), "r"(q.x),
               "r"(q.y), "r"(q.z), "r"(q.w), "l"(policy)
               : "memory");
}
// bytes: a multiple of 16, both addresses 16-byte aligned; completes on the barrier. `once`: the
// bytes are not read again (policy: evict_first()).
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* b,
                                          bool once, uint64_t policy) {
  if (once)
    asm volatile(
        "cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], "
        "%2, [%3], %4;" ::"r"(smem_addr(dst)),
        "l"(src), "r"(bytes), "r"(smem_addr(b)), "l"(policy)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
            smem_addr(dst)),
        "l"(src), "r"(bytes), "r"(smem_addr(b))
        : "memory");
}

// ---- clusters ----
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
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::
                   : "memory");
}
// Stores 8 bytes in another CTA's shared memory and arrives on its barrier. Both are done before this
// thread's next cluster_sync() is (a copy that completes by itself might land behind it, in a CTA that
// has left without waiting for it).
__device__ __forceinline__ void send(void* dst, uint64_t* bar, uint32_t rank, uint64_t value) {
  uint32_t d, b;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(smem_addr(dst)), "r"(rank));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(smem_addr(bar)), "r"(rank));
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(d), "l"(value) : "memory");
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(b) : "memory");
}

// The dependent kernel may take its place on the SMs now; it still waits for this grid's end.
__device__ __forceinline__ void grid_dependents_may_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void grid_dependency_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// An NVTX range over one entry point's host work.
struct NvtxRange {
  explicit NvtxRange(const char* name) { nvtxRangePushA(name); }
  ~NvtxRange() { nvtxRangePop(); }
  NvtxRange(const NvtxRange&) = delete;
  NvtxRange& operator=(const NvtxRange&) = delete;
};

// Parts of each row for kernels of 4 CTAs an SM that stream parts in rounds of `round` vectors: the
// fewest waves of CTAs times the rounds of one, where beginning and ending a part costs about as
// much as START rounds. Measured (us a beam step): 256 rows of 151,936 bf16 32.3 / 29.7 / 32.3 /
// 31.9 with 1 / 2 / 3 / 4 parts (2 taken), 512 rows of 248,320 float32 107 / 117 / 124 with 1 / 2 / 3
// (1 taken).
inline int plan_parts(int64_t rows, int64_t nv, int round, int limit) {
  constexpr int64_t SLOTS = 148 * 4, START = 2;
  int best = 1;
  int64_t least = INT64_MAX;
  for (int p = 1; p <= limit && (p - 1) * (int64_t)round < nv; ++p) {
    const int64_t cost =
        (rows * p + SLOTS - 1) / SLOTS * ((nv + (int64_t)p * round - 1) / ((int64_t)p * round) + START);
    if (cost < least) {
      least = cost;
      best = p;
    }
  }
  return best;
}

// An error code for the caller; the runtime's own error state is cleared, so that a refused launch
// does not show up in somebody else's check.
inline int result(cudaError_t e) {
  if (e == cudaSuccess) return VINFER_OK;
  (void)cudaGetLastError();
  return VINFER_E_CUDA;
}

// Shared memory above 48 KB has to be asked for (a host-side setting of the kernel on the current
// device, no work on a stream): the most that any launch of KERN takes, once for each device. A call
// that asked for its own need would lower the limit under another thread's launch.
template <auto KERN>
int opt_in(size_t most) {
  static std::atomic<bool> done[64];
  int dev = 0;
  if (result(cudaGetDevice(&dev)) != VINFER_OK || dev < 0 || dev >= 64) return VINFER_E_CUDA;
  if (done[dev].load(std::memory_order_acquire)) return VINFER_OK;
  const int rc =
      result(cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
  if (rc == VINFER_OK) done[dev].store(true, std::memory_order_release);
  return rc;
}

// One launch, of clusters of `cluster` CTAs; `dependent`: may begin while the stream's kernel before
// it drains (that kernel's writes are read behind grid_dependency_wait()).
template <typename... KA, typename... A>
int launch(void (*kern)(KA...), unsigned grid, unsigned block, size_t smem, cudaStream_t st,
           bool dependent, unsigned cluster, A... args) {
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (dependent) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return result(cudaLaunchKernelEx(&cfg, kern, args...));
}

}  // namespace rows
