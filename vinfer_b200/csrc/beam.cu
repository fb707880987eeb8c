// beam.cu — one step of beam search over rows of logits (sm_100a).
//
// A request has W beams; beam w holds the accumulated log-probability b_w and a row x_w of logits.
// Its continuations score  s(w, t) = b_w + x_w[t] - lse(x_w);  the n best over beams and tokens
// are listed (descending score, ties by beam, then token), and the best W of them that do not end
// the sequence are laid into the request's slots.
//
//   * k_beam_rows streams each live row once, cut into parts (one CTA each): the part's softmax sum
//     and its n best logits. Within a beam the scores' order is the logits' order, so no score is
//     needed to list a part exactly. A dead beam (score -inf) costs a CTA that returns at once.
//   * k_beam_pick, one CTA a request, launched as its programmatic dependent: a warp joins each
//     beam's parts (sum and n best), then the beams' lists are ranked by score in double. Two
//     beams' scores closer than NEAR could be ordered by the rounding of their sums, so the sums of
//     such beams (rare) are taken again in double before the order stands.
//
// What bounds it: for many long rows reading the logits once; for fewer, no single unit: a step of 256 rows of
// 151,936 bf16 has 48 % of the issue slots and 53 % of the ex2 unit busy, its 512 parts leave some SMs
// with three CTAs beside others with four, and two rounds in registers do not cover all of a load's
// latency (largest stall); launch and ramp take 3 us and picking 4 more. Measured on one B200, us a step: 32
// requests of 16 beams, 248,320 float32 logits 98.1 (508 MB: 5.2 TB/s, 0.79 of the measured copy
// bandwidth); 64 of 4, 151,936 bf16 29.0 (77.8 MB: 0.41); one of 4 10.0, most of it the two kernels'
// latency. Selecting costs little because it is not sorting: a part of a row finds a bar that n of
// its elements reach from its lanes' maxima, and looks again only at the 16-vector rounds of the
// threads that reach it (keeping the vectors themselves in shared memory cost 3 us more of 32).
#include "rows.cuh"

#include <algorithm>

namespace {

using namespace rows;

constexpr int NT = 256, NW = NT / 32;
constexpr int U = 4;              // 16-byte vectors of a thread and round: 16 KiB a CTA
constexpr int BUFS = 2;           // rounds in registers
constexpr int MAX_PARTS = 64;     // parts of a row
constexpr int MAX_JOIN = 1024;    // entries of a beam's parts together (a warp joins them)
constexpr int MAX_STAGED = 8192;  // entries of a request's parts together (64 KiB staged)
constexpr int PT = 512, PW = PT / 32;  // threads of k_beam_pick
constexpr int MAXN = VINFER_BEAM_MAX_N, MAXW = VINFER_BEAM_MAX_WIDTH;
// Scores of different beams within this distance are compared with sums taken again in double. A streamed
// sum is off, relative to itself and in units of 2^-24, by at most
//   4    ex2 (2^-22, the instruction's bound),
//   5.7  an exponent's argument, rounded once: half a step at 8 to 16 below the thread's reference;
//        farther down a thread has at most 2^10 elements, 2^-6 of its sum,
//   8    the additions within a round (3 + 3 + 1, and the correction); everything behind it is in double,
//   0.5  the correction's own rounding,
// so two sums differ by at most 36.4 of these from what they should. log2(e) as a float stretches all
// exponents alike, by 1.4e-8 of them; a sum's mean exponent is at most its log2(V) = 18, another 2.8. In
// all 2.4e-6. (Rounds added in float, one chain of 61 for a row of 248,320: scores off by 3.7e-6
// either way, seen with 256 tokens raised above a constant rest.)
constexpr double NEAR = 2.5e-6;

static_assert(MAXN <= 128 && MAXW <= 32, "lists fit the picking kernel's shared memory");

typedef unsigned long long u64;

// A candidate of one row: ascending keys are descending logits, equal logits by ascending id.
__device__ __forceinline__ u64 entry(float x, int id) {
  return ((u64)(~okey(x)) << 32) | (uint32_t)id;
}
__device__ __forceinline__ float entry_x(u64 e) { return from_okey(~(uint32_t)(e >> 32)); }
__device__ __forceinline__ int entry_id(u64 e) { return (int)(uint32_t)e; }

struct PartHdr {
  double s;    // softmax sum of the part, (m, s) at scale L2E
  float m;
  int pad;
};

struct RowsP {
  const void* logits;
  int64_t ld;
  int V, n, parts;
  const float* scores;
  PartHdr* hdr;  // [rows, parts]
  u64* list;     // [rows, parts, n], ascending, NONE behind the last
};
constexpr u64 NONE = ~0ull;

constexpr int DCAP = 1024; // delegates: threads' rounds that may hold one of the part's n best
constexpr int LCAP = 1024; // their elements that still may
struct Delegates {         // dynamic shared memory of k_beam_rows
  int v[DCAP];             // the round's first vector of the thread
  float mx[DCAP];          // the largest element
  u64 list[LCAP];
};
struct RowsS {
  u64 best[MAXN];
  double sum[NW];
  float f[NW];
  float kth[NW];
  int cnt, got, nd;
  uint32_t hist[256];
  uint32_t bin, before;
};
__host__ __device__ constexpr int list_cap(int n, int A) { return U * A * n + 2 * n + 64; }

// The n smallest of list[0, L) into best (any order); L > n. Radix select by bytes: keys are
// unique, so it ends with exactly n.
__device__ void select_best(const u64* list, int L, int n, RowsS& S) {
  u64 prefix = 0, mask = 0;
  int want = n;  // rank of the last kept key within the keys that share the prefix
  for (int shift = 56; shift >= 0; shift -= 8) {
    S.hist[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < L; i += NT)
      if ((list[i] & mask) == prefix) atomicAdd(&S.hist[(list[i] >> shift) & 255], 1u);
    __syncthreads();
    if (threadIdx.x < 32) {  // lane l holds bins [8l, 8l + 8)
      uint32_t sum = 0;
      for (int b = 0; b < 8; ++b) sum += S.hist[threadIdx.x * 8 + b];
      uint32_t incl = sum;
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(FULL, incl, o);
        if ((int)threadIdx.x >= o) incl += t;
      }
      uint32_t run = incl - sum;
      if (run < (uint32_t)want && (uint32_t)want <= incl) {
        for (int b = 0; b < 8; ++b) {
          const uint32_t h = S.hist[threadIdx.x * 8 + b];
          if ((uint32_t)want <= run + h) {
            S.bin = threadIdx.x * 8 + b;
            S.before = run;
            break;
          }
          run += h;
        }
      }
    }
    __syncthreads();
    prefix |= (u64)S.bin << shift;
    mask |= (u64)255 << shift;
    want -= (int)S.before;
    __syncthreads();
  }
  if (threadIdx.x == 0) S.got = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < L; i += NT)
    if (list[i] <= prefix) {
      const int at = atomicAdd(&S.got, 1);
      if (at < MAXN) S.best[at] = list[i];
    }
  __syncthreads();
}

// The n-th largest of the block's lane maxima (exact: every lane counts the larger ones).
// -inf when fewer than n lanes hold more than -inf.
__device__ float nth_lane_max(float mx, int n, float* all, float* out) {
  all[threadIdx.x] = mx;
  if (threadIdx.x == 0) *out = neg_inf();
  __syncthreads();
  int larger = 0, equal_before = 0;
  for (int i = 0; i < NT; ++i) {
    larger += all[i] > mx;
    equal_before += all[i] == mx && i < (int)threadIdx.x;
  }
  if (larger + equal_before == n - 1) *out = mx;
  __syncthreads();
  return *out;
}

// A part's n best whatever the data (flat, sorted or clustered rows, few elements): every round
// lists at most (n - 1) * U * A elements above a bar, and the lowest ids of those equal to it.
// Returns the entries of `list`, which holds at most list_cap(n, A).
template <typename T>
__device__ __noinline__ int list_carefully(const T* p, int V, int v0, int v1, int n, u64* list,
                                           RowsS& S) {
  using V8 = Vec<T>;
  constexpr int A = V8::A;
  const Row<T> R(p, V);
  const int cap = list_cap(n, A), tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  float bar = neg_inf();  // n listed elements are >= bar, at lower ids than what follows
  int have = 0;
  for (int vb = v0; vb < v1; vb += NT * U) {
    float mx = neg_inf();
    for (int u = 0; u < U; ++u) {
      const int v = vb + u * NT + tid;
      if (v < v1) mx = fmaxf(mx, V8::max(R.load(v)));
    }
    if (have > n) {
      select_best(list, have, n, S);
      for (int i = tid; i < n; i += NT) list[i] = S.best[i];
      have = n;
    }
    __syncthreads();
    // above the higher of the bar so far and this round's n-th lane maximum lie the elements of
    // fewer than n lanes
    const float nth = nth_lane_max(mx, n, reinterpret_cast<float*>(S.hist), S.f);
    const float lo = fmaxf(bar, nth);
    int eq_room = nth > bar ? n : 0;  // elements equal to the bar count only where this round set it
    if (tid == 0) S.cnt = have;
    __syncthreads();
    for (int u = 0; u < U; ++u) {
      const int v = vb + u * NT + tid;
      const uint32_t ni = V8::NEG_INF_WORD;
      const uint4 r = v < v1 ? R.load(v) : make_uint4(ni, ni, ni, ni);
      const int e0 = v * A - R.off;
      int eq = 0;
      for (int j = 0; j < A; ++j) {
        const float x = V8::get(r, j);
        if (x > lo) {
          const int at = atomicAdd(&S.cnt, 1);
          if (at < cap) list[at] = entry(x, e0 + j);
        }
        eq += x == lo && x > neg_inf();
      }
      if (eq_room > 0) {  // uniform: the lowest ids among the elements equal to the bar
        int incl = eq;
        for (int o = 1; o < 32; o <<= 1) {
          const int t = __shfl_up_sync(FULL, incl, o);
          if (lane >= o) incl += t;
        }
        __syncthreads();
        int* wsum = reinterpret_cast<int*>(S.kth);
        if (lane == 31) wsum[w] = incl;
        __syncthreads();
        int base = incl - eq, total = 0;
        for (int i = 0; i < NW; ++i) {
          if (i < w) base += wsum[i];
          total += wsum[i];
        }
        for (int j = 0; j < A && base < eq_room; ++j) {
          const float x = V8::get(r, j);
          if (x == lo && x > neg_inf()) {
            const int at = atomicAdd(&S.cnt, 1);
            if (at < cap) list[at] = entry(x, e0 + j);
            ++base;
          }
        }
        eq_room -= total;
      }
    }
    __syncthreads();
    have = min(S.cnt, cap);
    bar = lo;
    __syncthreads();
  }
  return have;
}

template <typename T>
__global__ void __launch_bounds__(NT, 4) k_beam_rows(const RowsP P) {
  using V8 = Vec<T>;
  constexpr int A = V8::A;
  extern __shared__ __align__(16) unsigned char dyn[];
  Delegates& D = *reinterpret_cast<Delegates*>(dyn);
  __shared__ RowsS S;
  const uint32_t row = blockIdx.x / (uint32_t)P.parts, part = blockIdx.x - row * P.parts;
  const float b = P.scores[row];
  if (!(b > neg_inf() && b < -neg_inf())) return;  // dead, or refused by k_beam_pick
  const Row<T> R(static_cast<const T*>(P.logits) + (int64_t)row * P.ld, P.V);
  const int v0 = (int)(R.nv * part / P.parts);  // below 2^18 * 64
  const int v1 = (int)(R.nv * (part + 1) / P.parts);
  const int n = P.n, tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  if (tid == 0) {
    S.nd = 0;
    S.cnt = 0;
  }

  // The bar: a logit that at least n lanes' maxima, so at least n elements, reach: the smallest of
  // the warps' k-th largest lane maxima (8k >= n). A thread's round below it holds none of the n
  // best; the others (about 3n in the first round) are noted as delegates. The warps raise it as
  // their maxima rise; a warp that still sees an older, lower one notes a few more.
  Exps<double> sum(L2E);
  float seen = neg_inf();  // this lane's largest element so far
  const int k = (n + NW - 1) / NW;
  volatile float* kth = S.kth;
  float bar = neg_inf();
  int round = 0;
  auto work = [&](const uint4 (&q)[U], int vb) {
    const float mx = V8::max(q);
    seen = fmaxf(seen, mx);
    if ((round & (round + 1)) == 0) {  // rounds 0, 1, 3, 7, ...
      uint32_t key = okey(seen), top = 0;
      for (int i = k; i > 0; --i) {
        top = __reduce_max_sync(FULL, key);
        const unsigned who = __ballot_sync(FULL, key == top);
        if (lane == __ffs(who) - 1) key = 0;
      }
      if (lane == 0) kth[w] = from_okey(top);
      if (round == 0) __syncthreads();
      bar = kth[0];
#pragma unroll
      for (int i = 1; i < NW; ++i) bar = fminf(bar, kth[i]);
    }
    ++round;
    if (mx >= bar) {
      const int at = atomicAdd(&S.nd, 1);
      if (at < DCAP) {
        D.v[at] = vb + tid;
        D.mx[at] = mx;
      }
    }
    sum.add<T>(q, mx);
  };
  stream_rounds<U, NT, BUFS>(R, v0, v1, work);
  grid_dependents_may_start();
  __syncthreads();

  // the delegates' elements that reach the final bar: their vectors are read again, from L2
  bar = S.kth[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) bar = fminf(bar, S.kth[i]);
  bool careful = !(bar > neg_inf()) || S.nd > DCAP;
  if (!careful) {
    for (int i = tid; i < S.nd * U; i += NT) {
      const int v = D.v[i / U] + i % U * NT;
      if (D.mx[i / U] < bar || v >= v1) continue;
      const uint4 q = R.load(v);
      if (V8::max(q) < bar) continue;
      for (int j = 0; j < A; ++j) {
        const float f = V8::get(q, j);
        if (f >= bar) {
          const int at = atomicAdd(&S.cnt, 1);
          if (at < LCAP) D.list[at] = entry(f, v * A - R.off + j);
        }
      }
    }
    __syncthreads();
    careful = S.cnt > LCAP;
  }
  const u64* src = D.list;
  u64* all = reinterpret_cast<u64*>(dyn);
  int have = S.cnt;
  __syncthreads();
  if (careful) {
    have = list_carefully<T>(R.p, P.V, v0, v1, n, all, S);
    src = all;
  }
  // the part's n best, in order, and its sum
  if (have > 384 && have > n) {
    select_best(src, have, n, S);
    src = S.best;
    have = n;
  }
  const int64_t at = (int64_t)blockIdx.x;
  u64* out = P.list + at * n;
  for (int i = tid; i < have; i += NT) {
    const u64 e = src[i];
    int rank = 0;
    for (int j = 0; j < have; ++j) rank += src[j] < e;
    if (rank < n) out[rank] = e;
  }
  for (int i = have + tid; i < n; i += NT) out[i] = NONE;
  block_join<NW>(sum.m, sum.s, L2E, S.sum, S.f);
  if (tid == 0) P.hdr[at] = PartHdr{sum.s, sum.m, 0};
}

struct PickP {
  RowsP r;
  int W, n_eos;
  const int* eos;
  float* out_scores;
  int* out_beams;
  int* out_tokens;
  float* next_scores;
  int* parents;
  int* next_tokens;
  int* status;
};

// 8 bytes from global to shared memory, without waiting; all of a thread's: copies_async_wait.
__device__ __forceinline__ void copy_async8(u64* dst, const u64* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_async_wait() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}

struct PickS {
  double m[MAXW], lns[MAXW];  // log-sum of each beam's row: m + lns
  double sum[MAXW];           // lns = log(sum)
  float b[MAXW];              // beam scores
  int cnt[MAXW];              // entries of each beam's list
  int head[MAXN];             // ranked candidates: beam << 16 | place in its list
  int eos[VINFER_BEAM_MAX_EOS];
  uint32_t flags;             // beams whose sums are taken again
  double red[PW];
  int sel[MAXW];              // continuing candidates: their ranks
};

template <typename T>
__device__ void row_sum_double(const RowsP& P, int row, double top, double* red, double* m_out,
                               double* lns_out) {
  // strided by element and from the row's largest one, so equal rows get equal sums whatever their
  // alignment and parts
  const T* x = static_cast<const T*>(P.logits) + (int64_t)row * P.ld;
  double s = 0;
  for (int i = threadIdx.x; i < P.V; i += PT) s += exp((double)Vec<T>::load(x + i) - top);
  __syncthreads();
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0;
  for (int i = 0; i < PW; ++i) s += red[i];
  __syncthreads();
  if (threadIdx.x == 0) {
    *m_out = top;
    *lns_out = log(s);
  }
}

// One CTA a request. Dynamic shared memory: the staged entries of its parts [W, parts, n], the
// beams' lists [W, n], their scores [W, n] and the same as integers of that order [W, n].
template <typename T>
__global__ void __launch_bounds__(PT, 1) k_beam_pick(const PickP Q) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ PickS S;
  const RowsP& P = Q.r;
  const int W = Q.W, n = P.n, per = P.parts * n;
  const int req = blockIdx.x, tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  u64* staged = reinterpret_cast<u64*>(dyn);
  u64* lists = staged + W * per;
  double* sc = reinterpret_cast<double*>(lists + W * n);
  long long* order = reinterpret_cast<long long*>(sc + W * n);
  if (tid == 0) S.flags = 0;
  if (tid < W) S.b[tid] = P.scores[(int64_t)req * W + tid];
  if (tid < Q.n_eos) S.eos[tid] = Q.eos[tid];
  grid_dependency_wait();

  const u64* E = P.list + (int64_t)req * W * per;
  for (int i = tid; i < W * per; i += PT) copy_async8(staged + i, E + i);  // dead beams': whatever is there
  for (int beam = w; beam < W; beam += PW) {
    const PartHdr* H = P.hdr + ((int64_t)req * W + beam) * P.parts;
    float m = neg_inf(), m2 = neg_inf();  // MAX_PARTS is two a lane
    double s0 = 0, s1 = 0;
    if (lane < P.parts) {
      m = H[lane].m;
      s0 = H[lane].s;
    }
    if (lane + 32 < P.parts) {
      m2 = H[lane + 32].m;
      s1 = H[lane + 32].s;
    }
    const float top = warp_max(fmaxf(m, m2));
    double s = 0;
    if (s0 != 0) s += s0 * exp2(((double)m - (double)top) * (double)L2E);
    if (s1 != 0) s += s1 * exp2(((double)m2 - (double)top) * (double)L2E);
    s = warp_sum(s);
    if (lane == 0) {
      S.m[beam] = top;
      S.sum[beam] = s;
      S.lns[beam] = log(s);
    }
  }
  copies_async_wait();
  __syncthreads();

  for (int beam = w; beam < W; beam += PW) {
    const float b = S.b[beam];
    const double s = S.sum[beam];
    int cnt = 0;
    unsigned bad = 0;
    if (!(b > neg_inf() && b < -neg_inf())) {
      if (b != neg_inf()) bad = VINFER_ST_BAD_SCORE;
    } else if (!(s > 0 && s < (double)FLT_MAX)) {
      bad = VINFER_ST_NONFINITE;  // a NaN or +inf, or every logit -inf
    } else {
      // n best of the parts' lists, which are sorted: with parts * (d + 1) >= n the largest of the
      // parts' entries at depth d bounds the n-th best from below, and with as many parts as
      // entries the n-th best of their first ones. What reaches it is ranked by counting.
      u64* mine = staged + beam * per;
      const int d = (n + P.parts - 1) / P.parts - 1;
      const u64 h0 = lane < P.parts ? mine[lane * n + d] : 0;
      const u64 h1 = lane + 32 < P.parts ? mine[(lane + 32) * n + d] : 0;
      u64 bound = h0 > h1 ? h0 : h1;
      if (d == 0 && P.parts > n) {
        const uint32_t k0 = (uint32_t)(h0 >> 32), k1 = (uint32_t)(h1 >> 32);  // by their logits
        int r0 = 0, r1 = 0;
#pragma unroll 8
        for (int o = 0; o < P.parts; ++o) {
          const uint32_t k = (uint32_t)(mine[o * n] >> 32);
          r0 += k < k0 || (k == k0 && o < lane);
          r1 += k < k1 || (k == k1 && o < lane + 32);
        }
        bound = 0;
        if (lane < P.parts && r0 == n - 1) bound = h0 | 0xffffffffu;
        if (lane + 32 < P.parts && r1 == n - 1) bound = h1 | 0xffffffffu;
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        const u64 other = __shfl_xor_sync(FULL, bound, o);
        bound = other > bound ? other : bound;
      }
      int alive = 0;
      for (int i0 = 0; i0 < per; i0 += 128) {
        u64 e[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int i = i0 + x * 32 + lane;
          e[x] = i < per ? mine[i] : NONE;
        }
        __syncwarp();  // all have read; places are behind what is read next
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const bool keep = e[x] <= bound && e[x] != NONE;
          const unsigned who = __ballot_sync(FULL, keep);
          if (keep) mine[alive + __popc(who & ((1u << lane) - 1))] = e[x];
          alive += __popc(who);
        }
        __syncwarp();
      }
      __syncwarp();
      for (int i = lane; i < alive; i += 32) {
        const u64 e = mine[i];
        int rank = 0;
        for (int j = 0; j < alive; ++j) rank += mine[j] < e;
        if (rank < n) lists[beam * n + rank] = e;
      }
      cnt = min(alive, n);
    }
    if (lane == 0) {
      if (bad && Q.status) atomicOr(Q.status, (int)bad);
      S.cnt[beam] = cnt;
    }
  }
  __syncthreads();

  auto score = [&](int beam, int j) {
    return (double)S.b[beam] +
           (((double)entry_x(lists[beam * n + j]) - S.m[beam]) - S.lns[beam]);
  };
  const int top_step = 1 << (31 - __clz(n));
  for (int pass = 0; pass < 2; ++pass) {
    for (int i = tid; i < W * n; i += PT) {
      const int beam = i / n, j = i - beam * n;
      sc[i] = j < S.cnt[beam] ? score(beam, j) : -HUGE_VAL;
      const long long bits = __double_as_longlong(sc[i] + 0.0);  // -0 and 0 are one score
      order[i] = bits ^ (long long)((unsigned long long)(bits >> 63) >> 1);
    }
    __syncthreads();
    // A candidate's place: its place in its own list and, by bisection, how many of every other
    // list are better (higher, or equal from an earlier beam). Its neighbours there show scores
    // that are too close to order. Four lists at a time, so that their steps overlap; scores as
    // integers of the same order, lists padded to n.
    for (int i = tid; i < W * n; i += PT) {
      const int bi = i / n, ji = i - bi * n;
      if (ji >= S.cnt[bi]) continue;
      const long long mine = order[i];
      const double my = sc[i];
      int rank = ji;
      uint32_t close = 0;
      for (int k0 = 0; k0 < W && rank < n; k0 += 4) {
        int lo[4] = {0, 0, 0, 0};
        for (int step = top_step; step; step >>= 1) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            // no branches: the loads of the four are in flight together
            const int k = k0 + x, at = lo[x] + step - 1;
            const long long o = order[min(k, W - 1) * n + min(at, n - 1)];
            lo[x] += at < n && o >= mine + (k < bi ? 0 : 1) ? step : 0;
          }
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int k = k0 + x;
          const double* o = sc + min(k, W - 1) * n;
          const double up = o[max(lo[x] - 1, 0)], down = o[min(lo[x], n - 1)];
          const bool near = (lo[x] > 0 && up - my <= NEAR) || (lo[x] < n && my - down <= NEAR);
          if (k < W && k != bi) {
            rank += lo[x];
            close |= near ? 1u << k : 0u;
          }
        }
      }
      if (rank < n) {
        S.head[rank] = bi << 16 | ji;
        if (close && pass == 0) atomicOr(&S.flags, close | 1u << bi);
      }
    }
    __syncthreads();
    const uint32_t flags = S.flags;
    if (pass == 1 || flags == 0) break;
    for (int beam = 0; beam < W; ++beam)
      if (flags >> beam & 1)
        row_sum_double<T>(P, req * W + beam, entry_x(lists[beam * n]), S.red, &S.m[beam],
                          &S.lns[beam]);
    __syncthreads();
  }

  // the list of candidates
  int have = 0;  // candidates there are
  for (int k = 0; k < W; ++k) have += S.cnt[k];
  have = min(have, n);
  for (int i = tid; i < n; i += PT) {
    const int64_t o = (int64_t)req * n + i;
    if (i < have) {
      const int beam = S.head[i] >> 16, j = S.head[i] & 0xffff;
      Q.out_scores[o] = (float)sc[beam * n + j];
      Q.out_beams[o] = beam;
      Q.out_tokens[o] = entry_id(lists[beam * n + j]);
    } else {
      Q.out_scores[o] = neg_inf();
      Q.out_beams[o] = -1;
      Q.out_tokens[o] = -1;
    }
  }
  // the beams that go on: the first W candidates whose token is no stop id
  if (w == PW - 1 && Q.parents) {  // beside the warps that write the list
    int nsel = 0;
    for (int i0 = 0; i0 < have && nsel < W; i0 += 32) {
      const int i = i0 + lane;
      bool on = i < have;
      if (on) {
        const int id = entry_id(lists[(S.head[i] >> 16) * n + (S.head[i] & 0xffff)]);
        for (int e = 0; e < Q.n_eos; ++e) on = on && id != S.eos[e];
      }
      const unsigned m = __ballot_sync(FULL, on);
      const int at = nsel + __popc(m & ((1u << lane) - 1));
      if (on && at < W) S.sel[at] = i;
      nsel = min(W, nsel + __popc(m));
    }
    __syncwarp();
    // lane i: the i-th of them. The best child of a beam keeps the beam's slot (its state stays
    // where it is), the others take the slots without a child in turn.
    const bool on = lane < nsel;
    const int cand = on ? S.head[S.sel[lane]] : 0;
    const int beam = on ? cand >> 16 : MAXW + lane;
    const unsigned same = __match_any_sync(FULL, beam);
    const bool stays = on && (__ffs(same) - 1) == lane;
    const unsigned taken = __reduce_or_sync(FULL, stays ? 1u << beam : 0u);
    const unsigned late = __ballot_sync(FULL, on && !stays);
    int slot = beam;
    const unsigned open = ~taken & (W == 32 ? FULL : (1u << W) - 1);
    if (on && !stays) {
      unsigned f = open;
      for (int k = __popc(late & ((1u << lane) - 1)); k > 0; --k) f &= f - 1;
      slot = __ffs(f) - 1;
    }
    const unsigned filled = __reduce_or_sync(FULL, on ? 1u << slot : 0u);
    if (on) {
      const int64_t o = (int64_t)req * W + slot;
      Q.next_scores[o] = (float)sc[beam * n + (cand & 0xffff)];
      Q.parents[o] = req * W + beam;
      Q.next_tokens[o] = entry_id(lists[beam * n + (cand & 0xffff)]);
    }
    if (lane < W && !(filled >> lane & 1)) {
      const int64_t o = (int64_t)req * W + lane;
      Q.next_scores[o] = neg_inf();
      Q.parents[o] = req * W + lane;
      Q.next_tokens[o] = -1;
    }
  }
}

// Parts of a row, no more entries than a warp joins or a request stages.
int beam_parts(int64_t rows_, int W, int64_t vocab, int dtype, int n) {
  const int64_t A = dtype == VINFER_DTYPE_BF16 ? 8 : 4;
  const int limit = std::min(MAX_PARTS, std::min(MAX_JOIN / n, MAX_STAGED / (W * n)));
  return plan_parts(rows_, (vocab + A - 1) / A, NT * U, limit);
}

size_t pick_smem(int W, int n, int parts) {
  return (size_t)W * n * (8 * (size_t)parts + 8 + 8 + 8);
}
// the most of both kernels: the longest lists, and MAX_STAGED entries beside lists of all beams
constexpr size_t ROWS_SMEM = std::max(sizeof(Delegates), (size_t)list_cap(MAXN, 8) * 8);
constexpr size_t PICK_SMEM = 8 * (size_t)MAX_STAGED + (size_t)MAXW * MAXN * 24;
static_assert(MAX_STAGED >= MAXW * MAXN && PICK_SMEM <= 220 * 1024, "every request fits an SM");

bool beam_shape_ok(int64_t requests, int32_t beams, int64_t vocab, int32_t dtype, int32_t n) {
  return requests >= 1 && beams >= 1 && beams <= MAXW && vocab >= 1 && vocab <= VINFER_MAX_VOCAB &&
         n >= 1 && n <= MAXN && requests <= VINFER_MAX_BATCH && requests * beams <= VINFER_MAX_BATCH &&
         (dtype == VINFER_DTYPE_F32 || dtype == VINFER_DTYPE_BF16);
}

template <typename T>
int launch_beam(const PickP& Q, int64_t requests, cudaStream_t st) {
  const int64_t rows_ = requests * Q.W;
  const size_t sm_rows = std::max(sizeof(Delegates), (size_t)list_cap(Q.r.n, Vec<T>::A) * 8);
  const size_t sm_pick = pick_smem(Q.W, Q.r.n, Q.r.parts);
  if (opt_in<k_beam_rows<T>>(ROWS_SMEM) != VINFER_OK || opt_in<k_beam_pick<T>>(PICK_SMEM) != VINFER_OK)
    return VINFER_E_CUDA;
  const int rc = launch(k_beam_rows<T>, (unsigned)(rows_ * Q.r.parts), NT, sm_rows, st, false, 1, Q.r);
  if (rc != VINFER_OK) return rc;
  return launch(k_beam_pick<T>, (unsigned)requests, PT, sm_pick, st, true, 1, Q);
}

}  // namespace

extern "C" {

size_t vinfer_beam_workspace_bytes(int64_t requests, int32_t beams, int64_t vocab, int32_t dtype,
                                   int32_t n) {
  if (!beam_shape_ok(requests, beams, vocab, dtype, n)) return 0;
  const int64_t rows_ = requests * beams;
  return (size_t)rows_ * beam_parts(rows_, beams, vocab, dtype, n) * (sizeof(PartHdr) + 8 * (size_t)n);
}

int vinfer_beam_select(const VinferBeamArgs* a, void* workspace, size_t workspace_bytes,
                       void* stream) {
  NvtxRange nvtx_range("vinfer_beam_select");
  if (!a || !a->logits || !a->scores || !a->out_scores || !a->out_beams || !a->out_tokens)
    return VINFER_E_ARG;
  if (a->dtype != VINFER_DTYPE_F32 && a->dtype != VINFER_DTYPE_BF16) return VINFER_E_ARG;
  if (a->requests < 1 || a->beams < 1 || a->vocab < 1 || a->ld < a->vocab || a->n < 1)
    return VINFER_E_ARG;
  if (a->n_eos < 0 || (a->n_eos > 0 && !a->eos)) return VINFER_E_ARG;
  if (!a->next_scores != !a->parents || !a->parents != !a->next_tokens) return VINFER_E_ARG;
  if (((uintptr_t)a->logits) % (a->dtype == VINFER_DTYPE_BF16 ? 2 : 4)) return VINFER_E_ARG;
  if (a->n_eos > VINFER_BEAM_MAX_EOS ||
      !beam_shape_ok(a->requests, a->beams, a->vocab, a->dtype, a->n))
    return VINFER_E_LIMIT;
  if (!workspace || ((uintptr_t)workspace) % 16) return VINFER_E_ARG;
  if (workspace_bytes <
      vinfer_beam_workspace_bytes(a->requests, a->beams, a->vocab, a->dtype, a->n))
    return VINFER_E_LIMIT;
  const int64_t rows_ = a->requests * a->beams;
  PickP Q = {};
  Q.r.logits = a->logits;
  Q.r.ld = a->ld;
  Q.r.V = (int)a->vocab;
  Q.r.n = a->n;
  Q.r.parts = beam_parts(rows_, a->beams, a->vocab, a->dtype, a->n);
  Q.r.scores = a->scores;
  Q.r.hdr = static_cast<PartHdr*>(workspace);
  Q.r.list = reinterpret_cast<u64*>(static_cast<unsigned char*>(workspace) +
                                    (size_t)rows_ * Q.r.parts * sizeof(PartHdr));
  Q.W = a->beams;
  Q.n_eos = a->n_eos;
  Q.eos = a->eos;
  Q.out_scores = a->out_scores;
  Q.out_beams = a->out_beams;
  Q.out_tokens = a->out_tokens;
  Q.next_scores = a->next_scores;
  Q.parents = a->parents;
  Q.next_tokens = a->next_tokens;
  Q.status = a->status;
  cudaStream_t st = (cudaStream_t)stream;
  return a->dtype == VINFER_DTYPE_BF16 ? launch_beam<__nv_bfloat16>(Q, a->requests, st)
                                       : launch_beam<float>(Q, a->requests, st);
}

}  // extern "C"
