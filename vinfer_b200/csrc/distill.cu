// distill.cu — distillation from a teacher's top log-probabilities, loss and gradient (sm_100a).
//
// A row of student logits x[V], temperature T, z = x / T, q = softmax(z); the teacher's list
// (id_j, l_j), j < k, with p_j = exp(l_j), renormalised to one without the tail, or as they are
// with it (the rest of the mass, p_t = 1 - sum p, is then matched with the student's mass outside
// the list, q_t):
//   loss = sum_j p_j (ln p_j - ln q_{id_j})  [ + p_t (ln p_t - ln q_t) ]
//   T dloss/dx_i = M q_i - (p_j summed over entries that list i)   inside the list
//                = q_i (M - p_t / q_t)                              outside it
// where M = sum p + p_t is the target's mass. Ids below 0 are empty entries.
//
//   * k_distill_rows streams each row once, cut into parts for small batches: the online softmax
//     sum over the elements OUTSIDE the list (a listed element is set to -inf in the registers
//     that hold it), so that q_t is summed, not left over from a difference.
//   * k_distill_finish, one warp a row: joins the parts and the list's k terms in double.
//   * k_distill_grad reads the row again and writes the gradient, one exponential an element; the
//     listed elements are stored behind it.
//   * k_distill_step does all of it for long rows, which it reads from HBM once (below).
//
// What bounds them: HBM, then the exponentials' instructions. Measured on one B200, in us, with the share
// of the measured copy bandwidth: losses of 1,024 rows of 151,936 bf16 58.8 (0.81); of 256 rows 27; the
// gradient alone of 1,024 rows 104 (6.0 TB/s, 0.91); loss and gradient in one call of 4,096 rows of
// 151,936 bf16, 512 of them masked, 487 (0.73) against 591 by the three kernels, of 512 rows of 248,320
// float32 with lists of 128 233 (0.67) against 307.
#include "rows.cuh"

#include <algorithm>
#include <atomic>

namespace {

using namespace rows;

constexpr int NT = 256, NW = NT / 32;
constexpr int RU = 4;           // 16-byte vectors of a thread and round while summing: 16 KiB a CTA
constexpr int BUFS = 2;         // rounds in registers
constexpr int U = 8;            // vectors of a thread and round while writing the gradient
constexpr int MAX_PARTS = 64;
constexpr int MAXK = VINFER_DISTILL_MAX_K;
static_assert(MAXK <= NT && MAXK <= 128, "one thread an entry; four entries a lane");

struct Part {
  float m, s;  // softmax sum outside the list, (m, s)
};
struct Stat {
  float m, coef;  // an element outside the list has dloss/dz = coef * 2^((x - m) * scale)
};

struct DistP {
  const void* logits;
  int64_t ld, rows;
  int V, k, parts;
  int tail;
  float scale;       // log2(e) / T rounded to float
  double scale_d;
  float inv_t;
  const int* ids;
  const float* lp;
  const float* weights;
  Part* part;        // [rows, parts]
  float* loss;
  Stat* stat;        // [rows], null: loss only
  float* listg;      // [rows, k]: dloss/dz of the listed elements
  int* status;
  const float* grad_out;
  int64_t go_stride;
  void* grad;
  int64_t ldg;
  WaitLimit limit;   // of the waits of k_distill_step
};

// The word of marks that has the bit of vector v, where rounds are of U vectors for each of N threads
// and a warp's U words of a round lie side by side.
template <int N, int U>
__device__ __forceinline__ uint32_t* mark_word(uint4* marks, int v) {
  const int c = v / (N * U), u = v % (N * U) / N, w = v % N / 32;
  return reinterpret_cast<uint32_t*>(marks) + (c * (N / 32) + w) * U + u;
}
// A warp's words of round c; whether any has a bit.
template <int N, int U>
__device__ __forceinline__ bool marks_of(const uint4* marks, int c, int w, uint32_t (&word)[U]) {
  const uint32_t* at = reinterpret_cast<const uint32_t*>(marks) + (c * (N / 32) + w) * U;
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (U % 4 == 0 && i % 4 == 0) {
      const uint4 m = *reinterpret_cast<const uint4*>(at + i);
      word[i] = m.x;
      word[i + 1] = m.y;
      word[i + 2] = m.z;
      word[i + 3] = m.w;
    } else if (U % 4 != 0) {
      word[i] = at[i];
    }
    any |= word[i];
  }
  return any != 0;
}
template <int N, int U>
__device__ __forceinline__ bool has_marks(const uint4* marks, int c, int w) {
  uint32_t word[U];
  return marks_of<N, U>(marks, c, w, word);
}

// Which elements of vector v are among the n places `at` (a place: element counted from the first
// vector, -1: none): one bit each. The whole warp calls it with the same v.
template <int A>
__device__ __forceinline__ uint32_t listed_in(const int* at, int n, int v) {
  uint32_t bits = 0;
  for (int j = threadIdx.x & 31; j < n; j += 32)
    if (at[j] >= 0 && at[j] / A == v) bits |= 1u << (at[j] & (A - 1));
  return __reduce_or_sync(FULL, bits);
}

// The warp's vectors with their listed elements taken out: lane l holds vector v0 + l as q, `word` has
// the bit of each that holds one.
template <typename T>
__device__ __forceinline__ uint4 take_out(uint4 q, uint32_t word, const int* at, int n, int v0) {
  for (; word; word &= word - 1) {
    const int l = __ffs(word) - 1;
    const uint32_t bits = listed_in<Vec<T>::A>(at, n, v0 + l);
    if ((threadIdx.x & 31) == l) {
#pragma unroll
      for (int j = 0; j < Vec<T>::A; ++j)
        if (bits >> j & 1) Vec<T>::put(q, j, Vec<T>::NEG_INF_BITS);
    }
  }
  return q;
}

// Stores the gradients of the listed elements of the warp's vectors, each by the lane that has just
// stored its vector. `first`: where the element counted as place 0 goes.
template <typename T>
__device__ __noinline__ void store_listed(T* first, uint32_t word, const int* at,
                                          const float* listg, int n, int v0) {
  constexpr int A = Vec<T>::A;
  for (; word; word &= word - 1) {
    const int l = __ffs(word) - 1;
    for (int j0 = 0; j0 < n; j0 += 32) {
      const int mine = j0 + (threadIdx.x & 31) < n ? at[j0 + (threadIdx.x & 31)] : -1;
      unsigned who = __ballot_sync(FULL, mine >= 0 && mine / A == v0 + l);
      for (; who; who &= who - 1) {
        const int j = j0 + __ffs(who) - 1;
        if ((threadIdx.x & 31) == l) first[at[j]] = Vec<T>::round(listg[j]);
      }
    }
  }
}

// Stores the elements of one vector that lie in [0, V): the vector's first is element e0.
template <typename T>
__device__ __noinline__ void store_ragged(T* out, uint4 q, int e0, int V) {
  for (int j = 0; j < Vec<T>::A; ++j)
    if (e0 + j >= 0 && e0 + j < V) out[e0 + j] = Vec<T>::round(Vec<T>::get(q, j));
}

// Dynamic shared memory: one bit for each vector of the part's rounds, set where it holds a listed
// element.
template <typename T>
__global__ void __launch_bounds__(NT, 4) k_distill_rows(const DistP P) {
  using VT = Vec<T>;
  constexpr int A = VT::A;
  extern __shared__ uint4 marked[];  // a warp's RU words of a round side by side
  __shared__ float sm[2 * NW];
  __shared__ int hit[MAXK];
  __shared__ int hits;
  const uint32_t row = blockIdx.x / (uint32_t)P.parts, part = blockIdx.x - row * P.parts;
  const int tid = threadIdx.x;
  if (P.weights && P.weights[row] == 0.f) return;
  const Row<T> R(static_cast<const T*>(P.logits) + row * P.ld, P.V);
  const int v0 = (int)(R.nv * part / P.parts);  // below 2^18 * 64
  const int v1 = (int)(R.nv * (part + 1) / P.parts);
  const int id = tid < P.k ? P.ids[row * P.k + tid] : -1;
  for (int i = tid; i < (v1 - v0 + NT * RU - 1) / (NT * RU) * NW * RU; i += NT)
    reinterpret_cast<uint32_t*>(marked)[i] = 0;
  if (tid == 0) hits = 0;
  __syncthreads();
  {
    const int e = id + R.off - v0 * A;  // the part's elements, counted from its first vector
    if (id >= 0 && id < P.V && e >= 0 && e < (v1 - v0) * A) {
      hit[atomicAdd(&hits, 1)] = e;
      atomicOr(mark_word<NT, RU>(marked, e / A), 1u << (e / A & 31));
    }
  }
  __syncthreads();
  Exps<float> sum(P.scale);
  stream_rounds<RU, NT, BUFS>(R, v0, v1, [&](uint4 (&q)[RU], int vb) {
    uint32_t word[RU];
    if (marks_of<NT, RU>(marked, (vb - v0) / (NT * RU), tid / 32, word)) {
#pragma unroll
      for (int u = 0; u < RU; ++u)
        if (word[u])
          q[u] = take_out<T>(q[u], word[u], hit, hits, vb - v0 + u * NT + (tid & ~31));
    }
    sum.add<T>(q, VT::max(q));
  });
  grid_dependents_may_start();
  block_join<NW>(sum.m, sum.s, P.scale, sm);
  if (tid == 0) P.part[blockIdx.x] = Part{sum.m, sum.s};
}

// A row's list as one warp works on it, four entries a lane.
struct ListS {
  double e[MAXK];     // 2^((z - top) * scale): all that takes exponentials is ready before the sum is
  double p[MAXK];     // masses as listed
  double psum[MAXK];  // ... summed over the entries of the same id
  float z[MAXK];      // listed logits
  float l[MAXK];      // log-probabilities
  int id[MAXK];       // -1: empty
  double mass;        // sum of p
  double esum;        // sum of e, each id once
  float top;          // largest z
  int distinct;       // ids
  bool bad;           // an id or a log-probability out of range
};

// What depends on the list alone, and its logits.
template <typename T>
__device__ __forceinline__ void list_begin(const DistP& P, int64_t row, ListS& L) {
  const int lane = threadIdx.x & 31;
  const T* x = static_cast<const T*>(P.logits) + row * P.ld;
  int id[4];
  float z[4];
  bool bad = false;
  double mass = 0;
  float top = neg_inf();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = lane + 32 * i;
    id[i] = -1;
    z[i] = neg_inf();
    if (j < P.k) {
      id[i] = P.ids[row * P.k + j];
      float l = P.lp[row * P.k + j];
      if (id[i] < 0) {
        id[i] = -1;
        l = neg_inf();
      }
      const bool off = id[i] >= P.V || !(l < -neg_inf());
      bad = bad || off;
      if (id[i] >= 0 && !off) z[i] = Vec<T>::load(x + id[i]);
      const double p = id[i] >= 0 ? exp((double)l) : 0.0;
      L.id[j] = id[i];
      L.l[j] = l;
      L.z[j] = z[i];
      L.p[j] = p;
      mass += p;
      if (z[i] > top || z[i] != z[i]) top = z[i];
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float t = __shfl_xor_sync(FULL, top, o);
    if (t > top || t != t) top = t;
  }
  __syncwarp();
  double psum[4] = {0, 0, 0, 0};
  bool lead[4] = {id[0] >= 0, id[1] >= 0, id[2] >= 0, id[3] >= 0};
  for (int o = 0; o < P.k; ++o) {
    const int other = L.id[o];
    const double po = L.p[o];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (other == id[i] && other >= 0) {
        psum[i] += po;
        if (o < lane + 32 * i) lead[i] = false;
      }
  }
  int distinct = 0;
  double esum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = lane + 32 * i;
    if (j < P.k) {
      const double e =
          z[i] == neg_inf() ? 0.0 : exp2(((double)z[i] - (double)top) * P.scale_d);
      L.e[j] = e;
      L.psum[j] = psum[i];
      if (lead[i]) {
        esum += e;
        ++distinct;
      }
    }
  }
  mass = warp_sum(mass);
  esum = warp_sum(esum);
  distinct = (int)__reduce_add_sync(FULL, (unsigned)distinct);
  bad = __any_sync(FULL, bad);
  if (lane == 0) {
    L.mass = mass;
    L.esum = esum;
    L.top = top;
    L.distinct = distinct;
    L.bad = bad;
  }
  __syncwarp();
}

// The row solved, in distances from its largest logit `ref`, whatever its magnitude.
struct Solved {
  double ref;
  double total;        // sum of 2^((x - ref) * scale) over the row
  double listed;       // 2^((top - ref) * scale) / total: q of a listed element is e * listed
  double rest;         // share of what is outside the list
  double mass;         // the target's mass M
  double pt;           // its tail
  double norm;         // a listed mass is p * norm
  bool bad;
};

// From the list and the sum outside it, (m, r) with r in units of 2^(m * scale). This is what the
// gradient waits for: two exponentials and a division.
__device__ __forceinline__ Solved list_solve(const DistP& P, const ListS& L, float m, double r) {
  const float top = L.top;
  Solved S;
  S.bad = L.bad;
  S.ref = r != 0 && m > top ? m : top;  // a NaN top stays
  const double ft = exp2(((double)top - S.ref) * P.scale_d);
  const double fr = r == 0 ? 0.0 : r * exp2(((double)m - S.ref) * P.scale_d);
  S.total = (L.esum == 0 ? 0.0 : L.esum * ft) + fr;
  if (S.ref != S.ref || S.ref == (double)neg_inf()) S.total = (double)__int_as_float(0x7fffffff);
  const double inv = 1.0 / S.total;
  S.listed = L.esum == 0 ? 0.0 : ft * inv;
  S.rest = fr * inv;
  S.mass = L.mass;
  S.pt = 0;
  S.norm = 1;
  if (P.tail) {
    S.pt = L.distinct < P.V ? fmax(0.0, 1.0 - S.mass) : 0.0;
  } else if (S.mass > 0) {
    S.norm = 1.0 / S.mass;
    S.mass = 1.0;
  }
  S.mass += S.pt;
  return S;
}
__device__ __forceinline__ bool lost(const Solved& S) {
  return S.bad || !(S.total < (double)-neg_inf());
}

// The gradient's terms, times f: of the listed elements, and of those outside.
__device__ __forceinline__ Stat list_grads(const DistP& P, const ListS& L, const Solved& S, float m,
                                           double r, float f, float* listg) {
  const float nan = __int_as_float(0x7fffffff);
  for (int j = threadIdx.x & 31; j < P.k; j += 32)
    listg[j] = lost(S)       ? nan
               : L.id[j] < 0 ? 0.f
                             : f * (float)(S.mass * (L.e[j] * S.listed) - L.psum[j] * S.norm);
  if (lost(S)) return Stat{nan, nan};
  if (r == 0) return Stat{0.f, 0.f};
  return Stat{m, f * (float)((S.mass * S.rest - S.pt) / r)};
}

// The row's loss, to be weighted before it is rounded.
__device__ __forceinline__ double list_loss(const DistP& P, const ListS& L, const Solved& S) {
  const int lane = threadIdx.x & 31;
  if (lost(S)) {
    if (lane == 0 && P.status)
      atomicOr(P.status, (int)(S.bad ? VINFER_ST_BAD_LIST : VINFER_ST_NONFINITE));
    return (double)__int_as_float(0x7fffffff);
  }
  const double lse = log(S.total), lnorm = S.norm == 1 ? 0.0 : -log(S.norm);
  const double unit = P.scale_d * LN2_D;
  double loss = 0;
  for (int j = lane; j < P.k; j += 32)
    if (L.p[j] > 0)
      loss += L.p[j] * S.norm *
              (((double)L.l[j] - lnorm) - (((double)L.z[j] - S.ref) * unit - lse));
  loss = warp_sum(loss);
  if (S.pt > 0) loss += S.pt * (log(S.pt) - log(S.rest));
  return loss;
}

constexpr int FW = 4;  // rows of a finishing CTA, one a warp

template <typename T>
__global__ void __launch_bounds__(FW * 32) k_distill_finish(const DistP P) {
  __shared__ ListS lists[FW];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * FW + w;
  const bool there = row < P.rows;
  const float weight = there && P.weights ? P.weights[row] : 1.f;
  const bool live = there && weight != 0.f;
  ListS& L = lists[w];
  if (live) list_begin<T>(P, row, L);
  grid_dependency_wait();
  if (!there) return;
  if (!live) {
    if (lane == 0) P.loss[row] = 0.f;
    return;
  }
  float m = neg_inf();
  for (int p = lane; p < P.parts; p += 32) {
    const Part h = P.part[row * P.parts + p];
    if (h.s != 0.f) m = fmaxf(m, h.m);
  }
  m = warp_max(m);
  double r = 0;
  for (int p = lane; p < P.parts; p += 32) {
    const Part h = P.part[row * P.parts + p];
    if (h.s != 0.f) r += (double)h.s * exp2(((double)h.m - (double)m) * (double)P.scale);
  }
  r = warp_sum(r);
  const Solved S = list_solve(P, L, m, r);
  if (P.stat) {
    const Stat st = list_grads(P, L, S, m, r, 1.f, P.listg + row * P.k);
    if (lane == 0) P.stat[row] = st;
  }
  const double loss = list_loss(P, L, S);
  if (lane == 0) P.loss[row] = (float)(loss * weight);
}

// CTAs an SM, us with 2 / 3 / 4 / 5: 256 rows of 151,936 bf16 28.0 / 28.0 / 28.9 / 28.4, 1,024 rows 104.4 / 104.5
// / 104.9 / 106.1, 64 rows of 40,001 float32 7.6 / 7.8 / 7.0 / 7.2.
template <typename T>
__global__ void __launch_bounds__(NT, 3) k_distill_grad(const DistP P) {
  using VT = Vec<T>;
  constexpr int A = VT::A;
  const uint32_t row = blockIdx.x / (uint32_t)P.parts, part = blockIdx.x - row * P.parts;
  const int tid = threadIdx.x;
  const Row<T> R(static_cast<const T*>(P.logits) + row * P.ld, P.V);
  T* out = static_cast<T*>(P.grad) + row * P.ldg;
  const bool aligned = (int)(((uintptr_t)out & 15) / sizeof(T)) == R.off;
  const int v0 = (int)(R.nv * part / P.parts);  // below 2^18 * 64
  const int v1 = (int)(R.nv * (part + 1) / P.parts);
  const float weight = P.weights ? P.weights[row] : 1.f;
  grid_dependency_wait();
  const float f =
      weight == 0.f ? 0.f : weight * P.inv_t * (P.grad_out ? P.grad_out[row * P.go_stride] : 1.f);
  Stat st = {0.f, 0.f};
  if (f != 0.f) st = P.stat[row];
  const float coef = f * st.coef;
  const uint64_t neg_m = pair(-st.m, -st.m), scale = pair(P.scale, P.scale);
  const uint64_t coef2 = pair(coef, coef);
  for (int vb = v0; vb < v1; vb += NT * U) {
    uint4 q[U];
    if (f != 0.f) R.template load_round<U, NT>(vb, v1, q);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = vb + u * NT + tid;
      if (v < v1) {
        float g[A];
        if (f != 0.f) {
          uint64_t h[A / 2];
          VT::pairs(q[u], h);
#pragma unroll
          for (int j = 0; j < A / 2; ++j)
            split(mul2(ex2_2(mul2(add2(h[j], neg_m), scale)), coef2), g[2 * j], g[2 * j + 1]);
        } else {
#pragma unroll
          for (int j = 0; j < A; ++j) g[j] = 0.f;
        }
        const int64_t e0 = (int64_t)v * A - R.off;
        if (aligned && R.whole(v)) *reinterpret_cast<uint4*>(out + e0) = VT::pack(g);
        else store_ragged(out, VT::pack(g), (int)e0, P.V);
      }
    }
  }
  if (f == 0.f) return;
  __syncthreads();  // the listed elements over what was just stored
  if (tid < P.k) {
    const int id = P.ids[row * P.k + tid];
    const int e = id + R.off;
    if (id >= 0 && id < P.V && e >= v0 * A && e < v1 * A)
      out[id] = VT::round(f * P.listg[row * P.k + tid]);
  }
}

// ---- loss and gradient in one pass ------------------------------------------------------------
// A cluster of CTAs takes a row at a time, each CTA a slice of it. In each CTA a producer thread
// streams the slice into a ring of chunks by bulk copies; CW warps sum the chunks, releasing
// each until the ring can hold the rest of the slice, and write the gradient once the row is
// solved: first of the chunks the ring still holds, then of the others, which the producer brings
// once more, from L2 (policies keep nothing else there: without them half of these bytes came from
// HBM again). HBM sees every row read once and written once. Two warps solve rows in turn: each
// prepares its row's list ahead, joins the CTA's sum with the other CTAs' (each sends its own to
// all), and hands out the gradient's terms. Two CTAs an SM, so that one streams while the other
// solves.
//
// Measured for 4,096 rows of 151,936 bf16 (512 masked): 487 us (4.8 TB/s). The same kernel without any
// arithmetic took 452 where it took 494, so it is the pipeline of copies that bounds it: nine of a
// row's thirteen chunks cross from L2 twice, in a mix of reads and writes that a plain streaming kernel
// takes at 6.0 TB/s. 512 rows of 248,320 float32 are eight turns of the 71 clusters of four that run at
// once, the last a fifth full. Also against those 494: one CTA an SM with a ring twice as large 545; a
// row whole in the shared memory of four CTAs, the next one summed before it is written, 894 (what
// a slice waits for, the solution and the copies, takes longer than the slice); chunks of 8
// vectors a thread 569; three or four CTAs an SM 606 (their slices no longer stay in L2).
constexpr int STEP_CTAS = 2;              // CTAs of an SM
constexpr int CW = 12, CT = CW * 32;      // warps and threads that sum and write
constexpr int CU = 4;                     // vectors a thread takes of a chunk
constexpr int CV = CT * CU;               // vectors of a chunk: 24 KiB
constexpr int SLOTS = 4;                  // chunks of the ring
constexpr int SLICE = 13;                 // chunks of a slice at most
constexpr int MAXC = 4;                   // CTAs of a cluster
constexpr int LW = 2;                     // warps that solve, and rows under way
constexpr int STEP_T = CT + 32 + LW * 32;

// What belongs to one row under way. Buffer j serves the live rows i with i % LW == j. It is safe
// to refill: a CTA sends its sum of row i + 2 after its gradient of row i + 1, which needs every
// CTA's sum of row i + 1, taken there after row i was solved and written.
static_assert(LW == 2, "a buffer's last reader is done two rows later");
struct StepRow {
  uint64_t list_full, list_empty;  // marks and places are set; ... and no longer needed
  uint64_t summed;                 // the CTA's warps have left their sums
  uint64_t joined;                 // every CTA's sum has arrived
  uint64_t solved;                 // m, coef and listg are set
  uint64_t part[MAXC];             // the CTAs' sums (m, s)
  float part_m[CW], part_s[CW];    // this CTA's warps'
  float m, coef;
  float listg[MAXK];
  int at[MAXK];                    // places of the listed elements in the slice, -1: not in it
  uint4 marks[SLICE * CW * CU / 4]; // a bit for each vector that holds one: a warp's CU of a chunk
  ListS list;
};
constexpr int ROWQ = 4;            // rows handed out ahead, the next two of them before they are loaded
struct StepS {
  uint64_t full[SLOTS], empty[SLOTS];
  uint64_t row_full[ROWQ], row_empty[ROWQ];
  int64_t next_row[ROWQ];          // -1: no more
  float next_weight[ROWQ];
  StepRow row[LW];
  int dead;
};

// The rows of a cluster, as every CTA's producer walks them: the live rows (weight not 0) are dealt
// out in turn, and so are the others, so that every cluster gets as many of each.
struct RowWalk {
  const float* weights;
  int64_t rows, base;    // the 32 rows under the lanes
  float w, ahead;        // this lane's weight, and that of the next 32
  unsigned mine;         // rows of the 32 that are the cluster's and still to come
  uint32_t live, dead;   // live and other rows before base, modulo the clusters
  int me, all;
  __device__ __forceinline__ RowWalk(const DistP& P, int cluster, int clusters)
      : weights(P.weights), rows(P.rows), base(-32), w(0), ahead(0), mine(0), live(0), dead(0),
        me(cluster), all(clusters) {
    ahead = at(0);
  }
  __device__ __forceinline__ float at(int64_t b) const {
    const int64_t r = b + (threadIdx.x & 31);
    return r < rows ? (weights ? weights[r] : 1.f) : 0.f;
  }
  // The next row and its weight; false behind the last. The whole warp calls it.
  __device__ __forceinline__ bool next(int64_t& row, float& weight) {
    while (!mine) {
      base += 32;
      if (base >= rows) return false;
      w = ahead;
      ahead = at(base + 32);
      const int lane = threadIdx.x & 31;
      const bool there = base + lane < rows, l = there && w != 0.f, d = there && w == 0.f;
      const unsigned lm = __ballot_sync(FULL, l), dm = __ballot_sync(FULL, d);
      const unsigned below = (1u << lane) - 1;
      const uint32_t turn = l ? live + __popc(lm & below) : dead + __popc(dm & below);
      mine = __ballot_sync(FULL, there && (int)(turn % all) == me);
      live = (live + __popc(lm)) % all;
      dead = (dead + __popc(dm)) % all;
    }
    const int l = __ffs(mine) - 1;
    mine &= mine - 1;
    row = base + l;
    weight = __shfl_sync(FULL, w, l);
    return true;
  }
};

// The warp is done with a chunk of the ring: what it read and wrote there comes before the copy that
// refills it. Copies go through another proxy than loads and stores, so the arrival alone does not
// order them: a warp's loads still in flight (waiting behind stores, say) would see the next chunk
// (without the fence about one step in eight over 512 rows of 248,320 float32 had 64 wrong
// elements). It costs nothing that shows: 497 us against 494 for 4,096 rows of 151,936 bf16, 227
// against 229 for those 512 float32 rows.
__device__ __forceinline__ void release_chunk(uint64_t* empty) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if ((threadIdx.x & 31) == 0) bar_arrive(empty);
}

// What a warp needs of a chunk besides its place in the ring; the calls below are rare, and out of line
// so that the streaming loops keep their registers.
template <typename T>
struct Chunk {
  const T* p;      // the row
  int V, off, v;   // its length, its offset from an aligned address, the chunk's first vector
  int v0, v1;      // the slice
};

// Makes the warp's vectors of a chunk in the ring what the loops take them for: the row's ragged ends
// filled from memory, -inf behind the slice and, with `marks`, in the place of listed elements.
template <typename T>
__device__ __noinline__ void mend_chunk(uint4* chunk, Chunk<T> K, const uint4* marks,
                                        const int* at, int n) {
  constexpr int A = Vec<T>::A;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int lo = K.off ? 1 : 0, hi = min(K.v1, (K.V + K.off) / A);
  for (int u = 0; u < CU; ++u) {
    const int x = K.v + u * CT + tid;
    if (x < lo || x >= hi)
      chunk[u * CT + tid] = Row<T>::edge(K.p, x < K.v1 ? K.V : 0, x * A - K.off);
  }
  __syncwarp();
  if (marks) {
    const int c = (K.v - K.v0) / CV;
    const uint32_t* words = reinterpret_cast<const uint32_t*>(marks) + (c * CW + w) * CU;
    for (int u = 0; u < CU; ++u)
      for (uint32_t word = words[u]; word; word &= word - 1) {
        const int l = __ffs(word) - 1;
        const uint32_t bits = listed_in<A>(at, n, c * CV + u * CT + w * 32 + l);
        if (lane == l) {
          uint4 q = chunk[u * CT + tid];
          for (int j = 0; j < A; ++j)
            if (bits >> j & 1) Vec<T>::put(q, j, Vec<T>::NEG_INF_BITS);
          chunk[u * CT + tid] = q;
        }
      }
  }
  __syncwarp();
}

// The gradient of a chunk that cannot be stored by whole vectors.
template <typename T>
__device__ __noinline__ void put_chunk(const uint4* chunk, Chunk<T> K, T* out, float m, float scale,
                                       float coef) {
  constexpr int A = Vec<T>::A;
  for (int u = 0; u < CU; ++u) {
    const int x = K.v + u * CT + (int)threadIdx.x;
    if (x >= K.v1) continue;
    const uint4 q = chunk[u * CT + threadIdx.x];
    for (int j = 0; j < A; ++j) {
      const int e = x * A - K.off + j;
      if (e >= 0 && e < K.V)
        out[e] = Vec<T>::round(coef * ex2((Vec<T>::get(q, j) - m) * scale));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(STEP_T, STEP_CTAS) k_distill_step(const __grid_constant__ DistP P) {
  using VT = Vec<T>;
  constexpr int A = VT::A;
  extern __shared__ __align__(128) unsigned char dyn[];
  uint4* ring = reinterpret_cast<uint4*>(dyn);
  StepS& S = *reinterpret_cast<StepS*>(dyn + (size_t)SLOTS * CV * 16);
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int size = (int)cluster_size(), rank = (int)cluster_rank();
  if (tid == 0) {
    for (int i = 0; i < SLOTS; ++i) {
      bar_init(&S.full[i], 1);
      bar_init(&S.empty[i], CW);
    }
    for (int i = 0; i < ROWQ; ++i) {
      bar_init(&S.row_full[i], 1);
      bar_init(&S.row_empty[i], CW + LW);
    }
    for (int i = 0; i < LW; ++i) {
      bar_init(&S.row[i].list_full, 1);
      bar_init(&S.row[i].list_empty, CW);
      bar_init(&S.row[i].summed, CW);
      bar_init(&S.row[i].joined, size);
      bar_init(&S.row[i].solved, 1);
    }
    S.dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int j = w; j < LW; j += STEP_T / 32) {
    for (int i = lane; i < MAXK; i += 32) S.row[j].at[i] = -1;
    for (int i = lane; i < SLICE * CW * CU / 4; i += 32)
      S.row[j].marks[i] = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  if (size > 1) cluster_sync();  // every CTA's barriers are ready for the others' sums
  volatile int* dead = &S.dead;
  const uint64_t once = evict_first();
  // a warp's next row and its weight; false behind the last
  uint32_t taken = 0;
  auto next_row = [&](int64_t& row, float& weight) {
    const int i = taken % ROWQ;
    if (!warp_wait(&S.row_full[i], (taken / ROWQ) & 1, dead, P.limit)) return false;
    row = S.next_row[i];
    weight = S.next_weight[i];
    __syncwarp();
    if (lane == 0) bar_arrive(&S.row_empty[i]);
    ++taken;
    return row >= 0;
  };
  int64_t row;
  float weight;
  uint32_t it = 0;  // chunks so far

  if (w == CW) {  // ---- the producer
    RowWalk walk(P, blockIdx.x / size, gridDim.x / size);
    uint32_t handed = 0;  // rows so far
    int ok = 1;
    auto hand = [&](int64_t& r, float& wt) {
      if (!walk.next(r, wt)) r = -1;
      if (lane == 0) {
        const int i = handed % ROWQ;
        if (handed >= ROWQ)
          ok = bar_wait(&S.row_empty[i], (handed / ROWQ - 1) & 1, dead, P.limit);
        if (ok) {
          S.next_row[i] = r;
          S.next_weight[i] = wt;
          bar_arrive(&S.row_full[i]);
        }
      }
      ++handed;
      ok = __shfl_sync(FULL, ok, 0);
    };
    int64_t row1 = -1, row2 = -1;
    float weight1 = 0.f, weight2 = 0.f;
    hand(row, weight);
    if (ok && row >= 0) hand(row1, weight1);
    for (; ok && row >= 0; row = row1, weight = weight1, row1 = row2, weight1 = weight2) {
      row2 = -1;
      if (row1 >= 0) hand(row2, weight2);
      if (!ok) break;
      if (weight == 0.f) continue;
      if (lane == 0) {
        const Row<T> R(static_cast<const T*>(P.logits) + row * P.ld, P.V);
        const int v0 = R.nv * rank / size, v1 = R.nv * (rank + 1) / size;
        const int lo = max(v0, R.off ? 1 : 0), hi = min(v1, (R.V + R.off) / A);  // whole vectors
        const int C = (v1 - v0 + CV - 1) / CV, again = max(C - SLOTS, 0);
        for (int c = 0; c < C + again; ++c, ++it) {
          const int slot = it % SLOTS, v = v0 + (c < C ? c : c - C) * CV;
          if (it >= SLOTS && !(ok = bar_wait(&S.empty[slot], (it / SLOTS - 1) & 1, dead, P.limit)))
            break;
          const int a = max(v, lo), b = min(v + CV, hi);
          if (b > a) {
            bar_expect(&S.full[slot], (uint32_t)(b - a) * 16);
            bulk_load(ring + (size_t)slot * CV + (a - v), R.p + ((int64_t)a * A - R.off),
                      (uint32_t)(b - a) * 16, &S.full[slot], c >= again, once);
          } else {
            bar_arrive(&S.full[slot]);
          }
        }
      }
      ok = __shfl_sync(FULL, ok, 0);
    }
  } else if (w > CW) {  // ---- the lists' warps
    const int mine = w - CW - 1;
    StepRow& B = S.row[mine];
    uint32_t live = 0;
    while (next_row(row, weight)) {
      if (weight == 0.f) {
        if (mine == 0 && rank == 0 && lane == 0) P.loss[row] = 0.f;
        continue;
      }
      const uint32_t use = live / LW;
      if ((int)(live++ % LW) != mine) continue;
      const Row<T> R(static_cast<const T*>(P.logits) + row * P.ld, P.V);
      const int v0 = R.nv * rank / size, v1 = R.nv * (rank + 1) / size;
      list_begin<T>(P, row, B.list);
      if (use > 0 && !warp_wait(&B.list_empty, (use - 1) & 1, dead, P.limit)) break;
      for (int j = lane; j < P.k; j += 32)
        if (B.at[j] >= 0) *mark_word<CT, CU>(B.marks, B.at[j] / A) = 0;
      __syncwarp();
      for (int j = lane; j < P.k; j += 32) {
        const int id = B.list.id[j], at = id + R.off - v0 * A;
        const bool in = id >= 0 && id < P.V && at >= 0 && at < (v1 - v0) * A;
        B.at[j] = in ? at : -1;
        if (in) atomicOr(mark_word<CT, CU>(B.marks, at / A), 1u << (at / A & 31));
      }
      __syncwarp();
      if (lane == 0) bar_arrive(&B.list_full);
      if (!warp_wait(&B.summed, use & 1, dead, P.limit)) break;
      // this CTA's sum to all, and all joined: in a fixed order, the same in every CTA
      float pm = lane < CW ? B.part_m[lane] : neg_inf(), ps = lane < CW ? B.part_s[lane] : 0.f;
      float m = warp_max(pm);
      float s = ps == 0.f ? 0.f : ps * exp2f((pm - m) * P.scale);
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(FULL, s, o);
      double r = s;
      if (size > 1) {
        if (lane < size)
          send(&B.part[rank], &B.joined, lane,
               (uint64_t)__float_as_uint(s) << 32 | __float_as_uint(m));
        __syncwarp();
        if (!warp_wait<true>(&B.joined, use & 1, dead, P.limit)) break;
        const uint64_t got = lane < size ? B.part[lane] : 0;
        pm = __uint_as_float((uint32_t)got);
        ps = __uint_as_float((uint32_t)(got >> 32));
        if (ps == 0.f) pm = neg_inf();
        m = warp_max(pm);
        r = warp_sum(ps == 0.f ? 0.0 : (double)ps * (double)exp2f((pm - m) * P.scale));
      }
      const Solved sol = list_solve(P, B.list, m, r);
      const Stat st = list_grads(P, B.list, sol, m, r, weight * P.inv_t, B.listg);
      if (lane == 0) {
        B.m = st.m;
        B.coef = st.coef;
      }
      __syncwarp();
      if (lane == 0) bar_arrive(&B.solved);
      const double loss = list_loss(P, B.list, sol);
      if (rank == 0 && lane == 0) P.loss[row] = (float)(loss * weight);
      __syncwarp();
    }
  } else {  // ---- the warps that sum and write
    const uint64_t scale2 = pair(P.scale, P.scale);
    uint32_t live = 0;  // rows so far
    bool ok = true;
    while (ok && next_row(row, weight)) {
      T* out = static_cast<T*>(P.grad) + row * P.ldg;
      if (weight == 0.f) {
        const int a = (int)((int64_t)P.V * rank / size), b = (int)((int64_t)P.V * (rank + 1) / size);
        const int head = min(b, a + (int)((16 - ((uintptr_t)(out + a) & 15)) % 16 / sizeof(T)));
        const int body = head + (b - head) / A * A;
        for (int e = a + tid; e < head; e += CT) out[e] = VT::round(0.f);
        for (int e = head + tid * A; e < body; e += CT * A)
          store_once(out + e, make_uint4(0, 0, 0, 0), once);
        for (int e = body + tid; e < b; e += CT) out[e] = VT::round(0.f);
        continue;
      }
      const Row<T> R(static_cast<const T*>(P.logits) + row * P.ld, P.V);
      const bool aligned = (int)(((uintptr_t)out & 15) / sizeof(T)) == R.off;
      const int v0 = R.nv * rank / size, v1 = R.nv * (rank + 1) / size;
      const int lo = R.off ? 1 : 0, end = min(v1, (R.V + R.off) / A);
      const int C = (v1 - v0 + CV - 1) / CV, again = max(C - SLOTS, 0);
      StepRow& B = S.row[live % LW];
      const uint32_t use = live++ / LW;
      if (!(ok = warp_wait(&B.list_full, use & 1, dead, P.limit))) break;
      Exps<float> sum(P.scale);
      for (int c = 0; c < C; ++c, ++it) {
        if (!(ok = warp_wait(&S.full[it % SLOTS], (it / SLOTS) & 1, dead, P.limit))) break;
        const int v = v0 + c * CV;
        uint4* chunk = ring + (size_t)(it % SLOTS) * CV;
        if (!(v >= lo && v + CV <= end) || has_marks<CT, CU>(B.marks, c, w))
          mend_chunk<T>(chunk, Chunk<T>{R.p, R.V, R.off, v, v0, v1}, B.marks, B.at, P.k);
        uint4 q[CU];
#pragma unroll
        for (int u = 0; u < CU; ++u) q[u] = chunk[u * CT + tid];
        if (c < again) release_chunk(&S.empty[it % SLOTS]);  // not held for the gradient
        sum.add<T>(q, VT::max(q));
      }
      if (!ok) break;
      float m = sum.m;
      const float s = sum.s;
      if (s == 0.f) m = neg_inf();
      const float mw = warp_max(m);
      float sw = s == 0.f ? 0.f : s * ex2((m - mw) * P.scale);
#pragma unroll
      for (int o = 16; o; o >>= 1) sw += __shfl_xor_sync(FULL, sw, o);
      if (lane == 0) {
        B.part_m[w] = mw;
        B.part_s[w] = sw;
        bar_arrive(&B.summed);
      }
      __syncwarp();
      if (!(ok = warp_wait(&B.solved, use & 1, dead, P.limit))) break;
      const uint64_t neg_m = pair(-B.m, -B.m), coef = pair(B.coef, B.coef);
      // the chunks the ring still holds, in order, then the others once more
      const int held = C - again;
      const uint32_t n0 = it - held;
      for (int k = 0; k < C; ++k) {
        const int c = k < held ? again + k : k - held;
        const uint32_t n = n0 + k;
        if (k >= held && !(ok = warp_wait(&S.full[n % SLOTS], (n / SLOTS) & 1, dead, P.limit)))
          break;
        const int v = v0 + c * CV;
        uint4* chunk = ring + (size_t)(n % SLOTS) * CV;
        const bool inside = v >= lo && v + CV <= end;
        if (inside && aligned) {
          uint4 q[CU];
#pragma unroll
          for (int u = 0; u < CU; ++u) q[u] = chunk[u * CT + tid];
          release_chunk(&S.empty[n % SLOTS]);
          T* to = out + ((int64_t)(v + tid) * A - R.off);
#pragma unroll
          for (int u = 0; u < CU; ++u) {
            uint64_t h[A / 2];
            float g[A];
            VT::pairs(q[u], h);
#pragma unroll
            for (int j = 0; j < A / 2; ++j)
              split(mul2(ex2_2(mul2(add2(h[j], neg_m), scale2)), coef), g[2 * j], g[2 * j + 1]);
            store_once(to + u * CT * A, VT::pack(g), once);
          }
        } else {
          const Chunk<T> K = {R.p, R.V, R.off, v, v0, v1};
          if (k >= held && !inside) mend_chunk<T>(chunk, K, nullptr, nullptr, 0);
          put_chunk<T>(chunk, K, out, B.m, P.scale, B.coef);
          release_chunk(&S.empty[n % SLOTS]);
        }
        if (has_marks<CT, CU>(B.marks, c, w)) {
          const uint32_t* words = reinterpret_cast<const uint32_t*>(B.marks) + (c * CW + w) * CU;
          for (int u = 0; u < CU; ++u)
            store_listed(out + ((int64_t)v0 * A - R.off), words[u], B.at, B.listg, P.k,
                         c * CV + u * CT + w * 32);
        }
      }
      if (!ok) break;
      it += again;
      __syncwarp();
      if (lane == 0) bar_arrive(&B.list_empty);
    }
  }
  __syncthreads();
  if (*dead) {  // a wait has given up, whichever and however late
    if (tid == 0 && P.status) atomicOr(P.status, (int)VINFER_ST_INTERNAL);
    if (w == CW && lane == 0)  // no copy of this CTA may land behind its end
      for (uint32_t k = it > SLOTS ? it - SLOTS : 0; k < it; ++k) {
        int none = 0;
        bar_wait(&S.full[k % SLOTS], (k / SLOTS) & 1, &none, WAIT_LIMIT);
      }
    __syncwarp();
  }
  if (size > 1) cluster_sync();  // no sum is sent to a CTA that has left
}

int distill_parts(int64_t rows_, int64_t vocab, int dtype) {
  const int64_t A = dtype == VINFER_DTYPE_BF16 ? 8 : 4;
  return plan_parts(rows_, (vocab + A - 1) / A, NT * RU, MAX_PARTS);
}

int check(const VinferDistillArgs* a) {
  if (!a || !a->logits || !a->ids || !a->logprobs) return VINFER_E_ARG;
  if (a->dtype != VINFER_DTYPE_F32 && a->dtype != VINFER_DTYPE_BF16) return VINFER_E_ARG;
  if (a->rows < 1 || a->vocab < 1 || a->ld < a->vocab || a->k < 1) return VINFER_E_ARG;
  if (!(a->temperature >= 1e-37f) || !(a->temperature <= 1e37f)) return VINFER_E_ARG;
  if (((uintptr_t)a->logits) % (a->dtype == VINFER_DTYPE_BF16 ? 2 : 4)) return VINFER_E_ARG;
  if (a->vocab > VINFER_MAX_VOCAB || a->rows > VINFER_DISTILL_MAX_ROWS || a->k > MAXK)
    return VINFER_E_LIMIT;
  return VINFER_OK;
}

DistP params(const VinferDistillArgs* a) {
  DistP P = {};
  P.logits = a->logits;
  P.ld = a->ld;
  P.rows = a->rows;
  P.V = (int)a->vocab;
  P.k = a->k;
  P.parts = distill_parts(a->rows, a->vocab, a->dtype);
  P.tail = a->tail != 0;
  P.scale_d = L2E_D / (double)a->temperature;
  P.scale = (float)P.scale_d;
  P.inv_t = 1.f / a->temperature;
  P.ids = a->ids;
  P.lp = a->logprobs;
  P.weights = a->weights;
  P.status = a->status;
  P.limit = WAIT_LIMIT;
  return P;
}

template <typename T>
int launch_loss(const DistP& P, cudaStream_t st) {
  const int part_vecs = (P.V / Vec<T>::A + 2 + P.parts - 1) / P.parts + 1;
  const size_t smem = (size_t)(part_vecs + NT * RU - 1) / (NT * RU) * (NT * RU / 8);
  const int rc = launch(k_distill_rows<T>, (unsigned)(P.rows * P.parts), NT, smem, st, false, 1, P);
  if (rc != VINFER_OK) return rc;
  return launch(k_distill_finish<T>, (unsigned)((P.rows + FW - 1) / FW), FW * 32, 0, st, true, 1, P);
}

// The gradient's parts need no joining: many, of two vectors a thread at least (256 rows of 151,936
// bf16: 27.6 us with 5 parts, 30.1 with 2).
template <typename T>
int launch_grad(DistP P, cudaStream_t st, bool dependent) {
  const int64_t nv = (P.V + Vec<T>::A - 1) / Vec<T>::A;
  P.parts = (int)std::max<int64_t>(
      1, std::min<int64_t>((148 * 8 + P.rows - 1) / P.rows, (nv + 2 * NT - 1) / (2 * NT)));
  return launch(k_distill_grad<T>, (unsigned)(P.rows * P.parts), NT, 0, st, dependent, 1, P);
}

// The CTAs a row is cut into, a power of two. A single CTA is launched without a cluster dimension and
// uses nothing of one.
static_assert((VINFER_MAX_VOCAB + 6) / 4 <= MAXC * SLICE * CV, "every row fits a cluster");
int step_cluster(int64_t V, int A) {
  const int64_t nv = (V + 2 * A - 2) / A;  // at any alignment
  int c = 1;
  while ((nv + c - 1) / c > SLICE * CV) c *= 2;
  return c;
}

constexpr size_t STEP_SMEM = (size_t)SLOTS * CV * 16 + sizeof(StepS);
static_assert(STEP_CTAS * (STEP_SMEM + 1024) <= 228 * 1024, "STEP_CTAS fit an SM");

// Clusters of c CTAs that fit the current device at once (a property of the device: asked once).
template <typename T>
int step_clusters(int c, int* clusters) {
  static std::atomic<int> known[64][MAXC + 1];
  int dev = 0;
  if (result(cudaGetDevice(&dev)) != VINFER_OK || dev < 0 || dev >= 64) return VINFER_E_CUDA;
  *clusters = known[dev][c].load();
  if (*clusters > 0) return VINFER_OK;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(148 * STEP_CTAS / c * c);
  cfg.blockDim = dim3(STEP_T);
  cfg.dynamicSmemBytes = STEP_SMEM;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (c == 1) {
    *clusters = 148 * STEP_CTAS;
    return VINFER_OK;
  }
  const int rc = result(cudaOccupancyMaxActiveClusters(clusters, k_distill_step<T>, &cfg));
  if (rc != VINFER_OK || *clusters < 1) return VINFER_E_CUDA;
  known[dev][c].store(*clusters);
  return VINFER_OK;
}

template <typename T>
int launch_step(const DistP& P, cudaStream_t st) {
  const int c = step_cluster(P.V, Vec<T>::A);
  if (opt_in<k_distill_step<T>>(STEP_SMEM) != VINFER_OK) return VINFER_E_CUDA;
  int clusters = 0;
  if (step_clusters<T>(c, &clusters) != VINFER_OK) return VINFER_E_CUDA;
  return launch(k_distill_step<T>, (unsigned)(std::min<int64_t>(P.rows, clusters) * c), STEP_T,
                STEP_SMEM, st, false, (unsigned)c, P);
}

// One pass where rows are long and there are enough of them to fill the clusters; otherwise the three
// kernels, whose second read of short rows comes from L2 anyway. Measured (us, one pass against
// three kernels, rows of 151,936 bf16): 31.2 / 24.4 at 32 rows, 33.5 / 43.4 at 148, 169 / 219 at
// 1,200; 1,200 rows of 65,536 bf16 103 / 100, of 33,000 bf16 80 / 67, of 33,000 float32 86 / 104. Rows
// that clusters take: 248,320 float32 (four CTAs, 71 clusters) 51.2 / 57.7 at 96, 78.7 / 80.2 at 148 (a
// third turn), 223 / 292 at 600; 120,007 float32 (two) 31.2 / 36.2 at 96; 262,144 bf16 (two) 39.8 / 40.6
// at 96, 67.2 / 66.2 at 200, 151 / 165 at 600.
bool step_in_one(const DistP& P, int dtype) {
  const bool bf = dtype == VINFER_DTYPE_BF16;
  const int64_t bytes = (int64_t)P.V * (bf ? 2 : 4);
  return P.rows >= 96 && bytes >= (bf ? 160 << 10 : 96 << 10);
}

size_t align_up(size_t n) { return (n + 255) / 256 * 256; }

bool grad_ok(const VinferDistillArgs* a, const void* grad, int64_t ld_grad) {
  return grad && ld_grad >= a->vocab && ((uintptr_t)grad) % (a->dtype == VINFER_DTYPE_BF16 ? 2 : 4) == 0;
}

}  // namespace

extern "C" {

size_t vinfer_distill_workspace_bytes(int64_t rows_, int64_t vocab, int32_t dtype, int32_t k) {
  if (rows_ < 1 || rows_ > VINFER_DISTILL_MAX_ROWS || vocab < 1 || vocab > VINFER_MAX_VOCAB ||
      k < 1 || k > MAXK || (dtype != VINFER_DTYPE_F32 && dtype != VINFER_DTYPE_BF16))
    return 0;
  return align_up((size_t)rows_ * distill_parts(rows_, vocab, dtype) * sizeof(Part)) +
         align_up((size_t)rows_ * sizeof(Stat)) + (size_t)rows_ * k * sizeof(float);
}

int vinfer_distill_loss(const VinferDistillArgs* a, float* loss, float* row_stats,
                        float* list_grads, void* workspace, size_t workspace_bytes,
                        void* stream) {
  NvtxRange nvtx_range("vinfer_distill_loss");
  const int rc = check(a);
  if (rc != VINFER_OK) return rc;
  if (!loss || !row_stats != !list_grads || !workspace) return VINFER_E_ARG;
  if (((uintptr_t)workspace) % 16 || ((uintptr_t)row_stats) % 8) return VINFER_E_ARG;
  if (workspace_bytes < vinfer_distill_workspace_bytes(a->rows, a->vocab, a->dtype, a->k))
    return VINFER_E_LIMIT;
  DistP P = params(a);
  P.part = static_cast<Part*>(workspace);
  P.loss = loss;
  P.stat = reinterpret_cast<Stat*>(row_stats);
  P.listg = list_grads;
  cudaStream_t st = (cudaStream_t)stream;
  return a->dtype == VINFER_DTYPE_BF16 ? launch_loss<__nv_bfloat16>(P, st)
                                       : launch_loss<float>(P, st);
}

int vinfer_distill_grad(const VinferDistillArgs* a, const float* row_stats,
                        const float* list_grads, const float* grad_out, int64_t grad_out_stride,
                        void* grad, int64_t ld_grad, void* stream) {
  NvtxRange nvtx_range("vinfer_distill_grad");
  const int rc = check(a);
  if (rc != VINFER_OK) return rc;
  if (!row_stats || !list_grads || grad_out_stride < 0 || !grad_ok(a, grad, ld_grad))
    return VINFER_E_ARG;
  if (((uintptr_t)row_stats) % 8) return VINFER_E_ARG;
  DistP P = params(a);
  P.stat = reinterpret_cast<Stat*>(const_cast<float*>(row_stats));
  P.listg = const_cast<float*>(list_grads);
  P.grad_out = grad_out;
  P.go_stride = grad_out_stride;
  P.grad = grad;
  P.ldg = ld_grad;
  cudaStream_t st = (cudaStream_t)stream;
  return a->dtype == VINFER_DTYPE_BF16 ? launch_grad<__nv_bfloat16>(P, st, false)
                                       : launch_grad<float>(P, st, false);
}

int vinfer_distill_step(const VinferDistillArgs* a, float* loss, void* grad, int64_t ld_grad,
                        void* workspace, size_t workspace_bytes, void* stream) {
  return vinfer_distill_step_within(a, loss, grad, ld_grad, workspace, workspace_bytes, -1, stream);
}

int vinfer_distill_step_within(const VinferDistillArgs* a, float* loss, void* grad, int64_t ld_grad,
                               void* workspace, size_t workspace_bytes, int64_t wait_ns,
                               void* stream) {
  NvtxRange nvtx_range("vinfer_distill_step");
  int rc = check(a);
  if (rc != VINFER_OK) return rc;
  if (!loss || !grad_ok(a, grad, ld_grad) || !workspace) return VINFER_E_ARG;
  if (((uintptr_t)workspace) % 16) return VINFER_E_ARG;
  if (workspace_bytes < vinfer_distill_workspace_bytes(a->rows, a->vocab, a->dtype, a->k))
    return VINFER_E_LIMIT;
  DistP P = params(a);
  if (wait_ns >= 0) {  // at least one try; at most the usual number
    P.limit.suspend_ns = (uint32_t)std::min<int64_t>(wait_ns, WAIT_LIMIT.suspend_ns);
    P.limit.tries = (int32_t)std::min<int64_t>(
        std::max<int64_t>(wait_ns / WAIT_LIMIT.suspend_ns, 1), WAIT_LIMIT.tries);
  }
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  P.part = reinterpret_cast<Part*>(ws);
  ws += align_up((size_t)P.rows * P.parts * sizeof(Part));
  P.stat = reinterpret_cast<Stat*>(ws);
  ws += align_up((size_t)P.rows * sizeof(Stat));
  P.listg = reinterpret_cast<float*>(ws);
  P.loss = loss;
  P.grad = grad;
  P.ldg = ld_grad;
  cudaStream_t st = (cudaStream_t)stream;
  if (step_in_one(P, a->dtype))
    return a->dtype == VINFER_DTYPE_BF16 ? launch_step<__nv_bfloat16>(P, st)
                                         : launch_step<float>(P, st);
  if (a->dtype == VINFER_DTYPE_BF16) {
    rc = launch_loss<__nv_bfloat16>(P, st);
    return rc != VINFER_OK ? rc : launch_grad<__nv_bfloat16>(P, st, true);
  }
  rc = launch_loss<float>(P, st);
  return rc != VINFER_OK ? rc : launch_grad<float>(P, st, true);
}

}  // extern "C"
