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
#include "rows.cuh"

#include <algorithm>

namespace {

using namespace rows;

constexpr int NT = 256, NW = NT / 32;
constexpr int U = 8;            // 16-byte vectors a thread holds: 32 KiB a CTA and round
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
  void* grad;
  int64_t ldg;
};

// Which elements of vector v are among the n places `at` (a place: element counted from the first
// vector, -1: none): one bit each. The whole warp calls it with the same v.
template <int A>
__device__ __forceinline__ uint32_t listed_in(const int* at, int n, int v) {
  uint32_t bits = 0;
  for (int j = threadIdx.x & 31; j < n; j += 32)
    if (at[j] >= 0 && at[j] / A == v) bits |= 1u << (at[j] & (A - 1));
  return __reduce_or_sync(FULL, bits);
}

// Takes the listed elements out of the warp's vectors: lane l holds vector v0 + l, `word` has the
// bit of each that holds one.
template <typename T>
__device__ __forceinline__ void take_out(uint4& q, uint32_t word, const int* at, int n, int v0) {
  for (; word; word &= word - 1) {
    const int l = __ffs(word) - 1;
    const uint32_t bits = listed_in<Vec<T>::A>(at, n, v0 + l);
    if ((threadIdx.x & 31) == l) {
#pragma unroll
      for (int j = 0; j < Vec<T>::A; ++j)
        if (bits >> j & 1) Vec<T>::put(q, j, Vec<T>::NEG_INF_BITS);
    }
  }
}

// Dynamic shared memory: one bit for each vector of the part's rounds, set where it holds a listed
// element.
template <typename T>
__global__ void __launch_bounds__(NT, 4) k_distill_rows(const DistP P) {
  using VT = Vec<T>;
  constexpr int A = VT::A;
  extern __shared__ uint32_t marked[];
  __shared__ float sm[2 * NW];
  __shared__ int hit[MAXK];
  __shared__ int hits;
  const int64_t row = blockIdx.x / P.parts;
  const int part = (int)(blockIdx.x - row * P.parts), tid = threadIdx.x;
  if (P.weights && P.weights[row] == 0.f) return;
  const Row<T> R(static_cast<const T*>(P.logits) + row * P.ld, P.V);
  const int v0 = (int)((int64_t)R.nv * part / P.parts);
  const int v1 = (int)((int64_t)R.nv * (part + 1) / P.parts);
  const int id = tid < P.k ? P.ids[row * P.k + tid] : -1;
  for (int i = tid; i < (v1 - v0 + NT * U - 1) / (NT * U) * (NT * U / 32); i += NT) marked[i] = 0;
  if (tid == 0) hits = 0;
  __syncthreads();
  {
    const int e = id + R.off - v0 * A;  // the part's elements, counted from its first vector
    if (id >= 0 && id < P.V && e >= 0 && e < (v1 - v0) * A) {
      hit[atomicAdd(&hits, 1)] = e;
      atomicOr(&marked[e / A / 32], 1u << (e / A & 31));
    }
  }
  __syncthreads();
  float m = neg_inf(), s = 0.f;
  for (int vb = v0; vb < v1; vb += NT * U) {
    uint4 q[U];
    R.template load_round<U, NT>(vb, v1, q);
#pragma unroll
    for (int u = 0; u < U; ++u) {  // a warp's 32 vectors are one word (and zeros behind the part)
      const int first = vb - v0 + u * NT + (tid & ~31);
      if (const uint32_t word = marked[first / 32]) take_out<T>(q[u], word, hit, hits, first);
    }
    add_exps<T>(q, VT::max(q), P.scale, m, s);
  }
  block_join<NW>(m, s, P.scale, sm);
  if (tid == 0) P.part[blockIdx.x] = Part{m, s};
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

__device__ __forceinline__ float list_loss(const DistP& P, const ListS& L, const Solved& S) {
  const int lane = threadIdx.x & 31;
  if (lost(S)) {
    if (lane == 0 && P.status)
      atomicOr(P.status, (int)(S.bad ? VINFER_ST_BAD_LIST : VINFER_ST_NONFINITE));
    return __int_as_float(0x7fffffff);
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
  return (float)loss;
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
  const float loss = list_loss(P, L, S);
  if (lane == 0) P.loss[row] = loss * weight;
}

template <typename T>
__global__ void __launch_bounds__(NT, 4) k_distill_grad(const DistP P) {
  using VT = Vec<T>;
  constexpr int A = VT::A;
  const int64_t row = blockIdx.x / P.parts;
  const int part = (int)(blockIdx.x - row * P.parts), tid = threadIdx.x;
  const Row<T> R(static_cast<const T*>(P.logits) + row * P.ld, P.V);
  T* out = static_cast<T*>(P.grad) + row * P.ldg;
  const bool aligned = (int)(((uintptr_t)out & 15) / sizeof(T)) == R.off;
  const int v0 = (int)((int64_t)R.nv * part / P.parts);
  const int v1 = (int)((int64_t)R.nv * (part + 1) / P.parts);
  const float weight = P.weights ? P.weights[row] : 1.f;
  grid_dependency_wait();
  const float f =
      weight == 0.f ? 0.f : weight * P.inv_t * (P.grad_out ? P.grad_out[row] : 1.f);
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
        if (aligned && R.whole(v)) {
          *reinterpret_cast<uint4*>(out + e0) = VT::pack(g);
        } else {
#pragma unroll
          for (int j = 0; j < A; ++j)
            if (e0 + j >= 0 && e0 + j < P.V) out[e0 + j] = VT::round(g[j]);
        }
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
// One persistent CTA an SM takes whole rows. A producer thread streams a row's chunks into a ring of
// shared memory by bulk copies; CW warps sum them, releasing each chunk until the ring can hold the
// rest of the row; the list's warp solves the row; the CW warps then write the gradient of the
// chunks the ring still holds, and of the others, which the producer brings once more (from L2:
// every SM re-reads what it read some microseconds before). HBM sees each row read once and written
// once. While a row is solved and written, the producer fills the ring with the next row, and
// the list's warp prepares the next list.
constexpr int CW = 16, CT = CW * 32;      // warps and threads that sum and write
constexpr int CU = 4;                     // vectors a thread takes of a chunk
constexpr int CV = CT * CU;               // vectors of a chunk: 32 KiB
constexpr int SLOTS = 6;                  // chunks of the ring
constexpr int STEP_CTAS = 1;              // CTAs of an SM
constexpr int ROWQ = 4;                   // rows handed out ahead of the warps
constexpr int STEP_T = CT + 64;           // and a warp each for the producer and the lists

struct StepRow {  // what the warps need to write a row
  float m, coef;
};
struct StepS {
  uint64_t full[SLOTS], empty[SLOTS];
  uint64_t row_full[ROWQ], row_empty[ROWQ];
  uint64_t list_full[2], list_empty[2];  // lists and marks of this row and the next
  uint64_t summed, solved;
  int row[ROWQ];
  float part_m[CW], part_s[CW];
  StepRow out;
  float listg[2][MAXK];
  int at[2][MAXK];                       // places of the listed elements, -1: empty
  ListS list;
  int dead;
};
__host__ __device__ inline int step_chunks(int V, int A) { return (V + A - 1 + A - 1 + CV * A - 1) / (CV * A); }

template <typename T>
__global__ void __launch_bounds__(STEP_T, STEP_CTAS) k_distill_step(const DistP P, int* next_row) {
  using VT = Vec<T>;
  constexpr int A = VT::A;
  extern __shared__ __align__(128) unsigned char dyn[];
  uint4* ring = reinterpret_cast<uint4*>(dyn);
  StepS& S = *reinterpret_cast<StepS*>(dyn + (size_t)SLOTS * CV * 16);
  uint32_t* marks = reinterpret_cast<uint32_t*>(&S + 1);  // [2][chunks * CV / 32]
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int words = step_chunks(P.V, A) * (CV / 32);
  if (tid == 0) {
    for (int i = 0; i < SLOTS; ++i) {
      bar_init(&S.full[i], 1);
      bar_init(&S.empty[i], CW);
    }
    for (int i = 0; i < ROWQ; ++i) {
      bar_init(&S.row_full[i], 1);
      bar_init(&S.row_empty[i], CW + 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(&S.list_full[i], 1);
      bar_init(&S.list_empty[i], CW);
    }
    bar_init(&S.summed, CW);
    bar_init(&S.solved, 1);
    S.dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = tid; i < 2 * words; i += STEP_T) marks[i] = 0;
  for (int i = tid; i < 2 * MAXK; i += STEP_T) (&S.at[0][0])[i] = -1;
  __syncthreads();
  volatile int* dead = &S.dead;

  if (w == CW) {  // ---- the producer
    if (lane == 0) {
      uint32_t it = 0;  // chunks so far
      int row = blockIdx.x;
      for (uint32_t i = 0;; ++i) {
        const int qi = i % ROWQ;
        if (i >= ROWQ && !bar_wait(&S.row_empty[qi], (i / ROWQ - 1) & 1, dead)) break;
        S.row[qi] = row < P.rows ? row : -1;
        bar_arrive(&S.row_full[qi]);
        if (row >= P.rows) break;
        if (!P.weights || P.weights[row] != 0.f) {
          const Row<T> R(static_cast<const T*>(P.logits) + (int64_t)row * P.ld, P.V);
          const int C = (R.nv + CV - 1) / CV, again = C > SLOTS ? C - SLOTS : 0;
          const int lo = R.off ? 1 : 0, hi = (R.V + R.off) / A;  // whole vectors
          bool ok = true;
          for (int c = 0; c < C + again && ok; ++c, ++it) {
            const int slot = it % SLOTS, chunk = c < C ? c : c - C;
            if (it >= SLOTS) ok = bar_wait(&S.empty[slot], (it / SLOTS - 1) & 1, dead);
            if (!ok) break;
            const int a = max(chunk * CV, lo), b = min((chunk + 1) * CV, hi);
            if (b > a) {
              bar_expect(&S.full[slot], (uint32_t)(b - a) * 16);
              bulk_load(ring + (size_t)slot * CV + (a - chunk * CV),
                        R.p + ((int64_t)a * A - R.off), (uint32_t)(b - a) * 16, &S.full[slot]);
            } else {
              bar_arrive(&S.full[slot]);
            }
          }
          if (!ok) break;
        }
        row = gridDim.x + atomicAdd(next_row, 1);
      }
      // no copy of this CTA may land behind its end
      if (*dead)
        for (uint32_t k = it > SLOTS ? it - SLOTS : 0; k < it; ++k) {
          int none = 0;
          bar_wait(&S.full[k % SLOTS], (k / SLOTS) & 1, &none);
        }
    }
    return;
  }

  if (w == CW + 1) {  // ---- the list's warp
    uint32_t live = 0;
    for (uint32_t i = 0;; ++i) {
      if (!bar_wait(&S.row_full[i % ROWQ], (i / ROWQ) & 1, dead)) break;
      const int row = S.row[i % ROWQ];
      __syncwarp();
      if (lane == 0) bar_arrive(&S.row_empty[i % ROWQ]);
      if (row < 0) break;
      const float weight = P.weights ? P.weights[row] : 1.f;
      if (weight == 0.f) {
        if (lane == 0) P.loss[row] = 0.f;
        continue;
      }
      const int b = live & 1;
      list_begin<T>(P, row, S.list);
      if (live >= 2 && !bar_wait(&S.list_empty[b], (live / 2 - 1) & 1, dead)) break;
      const int off = (int)(((uintptr_t)(static_cast<const T*>(P.logits) + (int64_t)row * P.ld) & 15) /
                            sizeof(T));
      uint32_t* mk = marks + b * words;
      for (int j = lane; j < P.k; j += 32)
        if (S.at[b][j] >= 0) mk[S.at[b][j] / A / 32] = 0;
      __syncwarp();
      for (int j = lane; j < P.k; j += 32) {
        const int id = S.list.id[j];
        const int at = id >= 0 && id < P.V ? id + off : -1;
        S.at[b][j] = at;
        if (at >= 0) atomicOr(&mk[at / A / 32], 1u << (at / A & 31));
      }
      __syncwarp();
      if (lane == 0) bar_arrive(&S.list_full[b]);
      if (!bar_wait(&S.summed, live & 1, dead)) break;
      // the warps' sums, joined in a fixed order
      const float pm = lane < CW ? S.part_m[lane] : neg_inf(), ps = lane < CW ? S.part_s[lane] : 0.f;
      const float m = warp_max(pm);
      const double r =
          warp_sum(ps == 0.f ? 0.0 : (double)ps * (double)exp2f((pm - m) * P.scale));
      const Solved sol = list_solve(P, S.list, m, r);
      const Stat st = list_grads(P, S.list, sol, m, r, weight * P.inv_t, S.listg[b]);
      if (lane == 0) S.out = StepRow{st.m, st.coef};
      __syncwarp();
      if (lane == 0) bar_arrive(&S.solved);
      const float loss = list_loss(P, S.list, sol);
      if (lane == 0) P.loss[row] = loss * weight;
      __syncwarp();
      ++live;
    }
    if (lane == 0 && *dead && P.status) atomicOr(P.status, (int)VINFER_ST_INTERNAL);
    return;
  }

  // ---- the warps that sum and write
  uint32_t it = 0, live = 0;  // chunks and rows so far
  const uint64_t scale2 = pair(P.scale, P.scale);
  for (uint32_t i = 0;; ++i) {
    if (!bar_wait(&S.row_full[i % ROWQ], (i / ROWQ) & 1, dead)) break;
    const int row = S.row[i % ROWQ];
    __syncwarp();
    if (lane == 0) bar_arrive(&S.row_empty[i % ROWQ]);
    if (row < 0) break;
    const Row<T> R(static_cast<const T*>(P.logits) + (int64_t)row * P.ld, P.V);
    T* out = static_cast<T*>(P.grad) + (int64_t)row * P.ldg;
    const bool aligned = (int)(((uintptr_t)out & 15) / sizeof(T)) == R.off;
    const int C = (R.nv + CV - 1) / CV, again = C > SLOTS ? C - SLOTS : 0;
    const int lo = R.off ? 1 : 0, hi = (R.V + R.off) / A;

    // the thread's vectors of a chunk: in the ring, at the row's ragged ends from memory
    auto take = [&](int chunk, uint32_t n, uint4 (&q)[CU]) {
      const uint4* src = ring + (size_t)(n % SLOTS) * CV + tid;
#pragma unroll
      for (int u = 0; u < CU; ++u) q[u] = src[u * CT];
      const int v0 = chunk * CV;
      if (v0 < lo || v0 + CV > hi) {
#pragma unroll
        for (int u = 0; u < CU; ++u) {
          const int v = v0 + u * CT + tid;
          const uint32_t ni = VT::NEG_INF_WORD;
          if (v >= R.nv) q[u] = make_uint4(ni, ni, ni, ni);
          else if (v < lo || v >= hi) q[u] = R.edge(R.p, R.V, v * A - R.off);
        }
      }
    };
    auto put = [&](int v, const float (&g)[A]) {
      const int64_t e0 = (int64_t)v * A - R.off;
      if (aligned && v >= lo && v < hi) {
        *reinterpret_cast<uint4*>(out + e0) = VT::pack(g);
      } else {
#pragma unroll
        for (int j = 0; j < A; ++j)
          if (e0 + j >= 0 && e0 + j < P.V) out[e0 + j] = VT::round(g[j]);
      }
    };

    if (P.weights && P.weights[row] == 0.f) {
      float g[A];
#pragma unroll
      for (int j = 0; j < A; ++j) g[j] = 0.f;
      for (int v = tid; v < R.nv; v += CT) put(v, g);
      continue;
    }
    const int b = live & 1;
    const uint32_t* mk = marks + b * words;
    if (!bar_wait(&S.list_full[b], (live / 2) & 1, dead)) break;
    float m = neg_inf(), s = 0.f;
    bool ok = true;
    for (int c = 0; c < C; ++c, ++it) {
      if (!(ok = bar_wait(&S.full[it % SLOTS], (it / SLOTS) & 1, dead))) break;
      uint4 q[CU];
      take(c, it, q);
      if (c < C - SLOTS) {  // not held for the gradient
        __syncwarp();
        if (lane == 0) bar_arrive(&S.empty[it % SLOTS]);
      }
#pragma unroll
      for (int u = 0; u < CU; ++u) {
        const int first = c * CV + u * CT + w * 32;
        if (const uint32_t word = mk[first / 32]) take_out<T>(q[u], word, S.at[b], P.k, first);
      }
      add_exps<T>(q, VT::max(q), P.scale, m, s);
    }
    if (!ok) break;
    if (s == 0.f) m = neg_inf();
    const float mw = warp_max(m);
    float sw = s == 0.f ? 0.f : s * ex2((m - mw) * P.scale);
#pragma unroll
    for (int o = 16; o; o >>= 1) sw += __shfl_xor_sync(FULL, sw, o);
    if (lane == 0) {
      S.part_m[w] = mw;
      S.part_s[w] = sw;
      bar_arrive(&S.summed);
    }
    __syncwarp();
    if (!bar_wait(&S.solved, live & 1, dead)) break;
    const StepRow o = S.out;
    const uint64_t neg_m = pair(-o.m, -o.m), coef = pair(o.coef, o.coef);
    // chunks the ring still holds, in order, then the others once more
    const int held = C - again;
    for (int k = 0; k < C; ++k) {
      const int c = k < held ? again + k : k - held;
      const uint32_t n = k < held ? it - held + k : it + (k - held);
      if (k >= held && !(ok = bar_wait(&S.full[n % SLOTS], (n / SLOTS) & 1, dead))) break;
      uint4 q[CU];
      take(c, n, q);
      __syncwarp();
      if (lane == 0) bar_arrive(&S.empty[n % SLOTS]);
#pragma unroll
      for (int u = 0; u < CU; ++u) {
        const int first = c * CV + u * CT + w * 32, v = first + lane;
        uint64_t h[A / 2];
        float g[A];
        VT::pairs(q[u], h);
#pragma unroll
        for (int j = 0; j < A / 2; ++j)
          split(mul2(ex2_2(mul2(add2(h[j], neg_m), scale2)), coef), g[2 * j], g[2 * j + 1]);
        for (uint32_t word = mk[first / 32]; word; word &= word - 1) {  // listed elements
          const int l = __ffs(word) - 1;
          for (int j0 = 0; j0 < P.k; j0 += 32) {
            const int at = j0 + lane < P.k ? S.at[b][j0 + lane] : -1;
            unsigned who = __ballot_sync(FULL, at >= 0 && at / A == first + l);
            for (; who; who &= who - 1) {
              const int j = j0 + __ffs(who) - 1;
              const int e = S.at[b][j] & (A - 1);
              if (lane == l) {
#pragma unroll
                for (int a = 0; a < A; ++a)
                  if (a == e) g[a] = S.listg[b][j];
              }
            }
          }
        }
        if (v < R.nv) put(v, g);
      }
    }
    if (!ok) break;
    it += again;
    __syncwarp();
    if (lane == 0) bar_arrive(&S.list_empty[b]);
    ++live;
  }
}

// Parts of a row: enough CTAs to fill the 148 SMs several times over, at least two vectors a
// thread in each.
int distill_parts(int64_t rows_, int64_t vocab, int dtype) {
  const int64_t A = dtype == VINFER_DTYPE_BF16 ? 8 : 4;
  const int64_t nv = (vocab + A - 1) / A;
  int64_t p = (148 * 8 + rows_ - 1) / rows_;
  p = std::min<int64_t>(p, (nv + 2 * NT - 1) / (2 * NT));
  return (int)std::max<int64_t>(1, std::min<int64_t>(p, MAX_PARTS));
}

// Rows taken whole by one CTA each, where there are enough and they are long.
bool step_in_one(const DistP& P, int dtype) {
  const int64_t bytes = (int64_t)P.V * (dtype == VINFER_DTYPE_BF16 ? 2 : 4);
  return P.rows >= 2 * 148 * STEP_CTAS && bytes >= (64 << 10);
}

int check(const VinferDistillArgs* a) {
  if (!a || !a->logits || !a->ids || !a->logprobs) return VINFER_E_ARG;
  if (a->dtype != VINFER_DTYPE_F32 && a->dtype != VINFER_DTYPE_BF16) return VINFER_E_ARG;
  if (a->rows < 1 || a->vocab < 1 || a->ld < a->vocab || a->k < 1) return VINFER_E_ARG;
  if (!(a->temperature > 0.f) || !(a->temperature < INFINITY)) return VINFER_E_ARG;
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
  return P;
}

template <typename T>
int launch_loss(const DistP& P, cudaStream_t st) {
  const int part_vecs = (P.V / Vec<T>::A + 2 + P.parts - 1) / P.parts + 1;
  const size_t smem = (size_t)(part_vecs + NT * U - 1) / (NT * U) * (NT * U / 8);
  const int rc = launch(k_distill_rows<T>, (unsigned)(P.rows * P.parts), NT, smem, st, false, P);
  if (rc != VINFER_OK) return rc;
  return launch(k_distill_finish<T>, (unsigned)((P.rows + FW - 1) / FW), FW * 32, 0, st, true, P);
}

template <typename T>
int launch_grad(const DistP& P, cudaStream_t st, bool dependent) {
  return launch(k_distill_grad<T>, (unsigned)(P.rows * P.parts), NT, 0, st, dependent, P);
}

size_t step_smem(int V, int A) {
  return (size_t)SLOTS * CV * 16 + sizeof(StepS) + 2 * (size_t)step_chunks(V, A) * (CV / 8);
}

template <typename T>
int launch_step(const DistP& P, int* next_row, cudaStream_t st) {
  const size_t smem = step_smem(P.V, Vec<T>::A);
  if (opt_in(k_distill_step<T>, smem) != VINFER_OK) return VINFER_E_CUDA;
  if (result(cudaMemsetAsync(next_row, 0, sizeof(int), st)) != VINFER_OK) return VINFER_E_CUDA;
  return launch(k_distill_step<T>, (unsigned)std::min<int64_t>(P.rows, 148 * STEP_CTAS), STEP_T, smem, st, false,
                P, next_row);
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
                        const float* list_grads, const float* grad_out, void* grad,
                        int64_t ld_grad, void* stream) {
  NvtxRange nvtx_range("vinfer_distill_grad");
  const int rc = check(a);
  if (rc != VINFER_OK) return rc;
  if (!row_stats || !list_grads || !grad_ok(a, grad, ld_grad)) return VINFER_E_ARG;
  if (((uintptr_t)row_stats) % 8) return VINFER_E_ARG;
  DistP P = params(a);
  P.stat = reinterpret_cast<Stat*>(const_cast<float*>(row_stats));
  P.listg = const_cast<float*>(list_grads);
  P.grad_out = grad_out;
  P.grad = grad;
  P.ldg = ld_grad;
  cudaStream_t st = (cudaStream_t)stream;
  return a->dtype == VINFER_DTYPE_BF16 ? launch_grad<__nv_bfloat16>(P, st, false)
                                       : launch_grad<float>(P, st, false);
}

int vinfer_distill_step(const VinferDistillArgs* a, float* loss, void* grad, int64_t ld_grad,
                        void* workspace, size_t workspace_bytes, void* stream) {
  NvtxRange nvtx_range("vinfer_distill_step");
  int rc = check(a);
  if (rc != VINFER_OK) return rc;
  if (!loss || !grad_ok(a, grad, ld_grad) || !workspace) return VINFER_E_ARG;
  if (((uintptr_t)workspace) % 16) return VINFER_E_ARG;
  if (workspace_bytes < vinfer_distill_workspace_bytes(a->rows, a->vocab, a->dtype, a->k))
    return VINFER_E_LIMIT;
  DistP P = params(a);
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
    return a->dtype == VINFER_DTYPE_BF16 ? launch_step<__nv_bfloat16>(P, (int*)workspace, st)
                                         : launch_step<float>(P, (int*)workspace, st);
  if (a->dtype == VINFER_DTYPE_BF16) {
    rc = launch_loss<__nv_bfloat16>(P, st);
    return rc != VINFER_OK ? rc : launch_grad<__nv_bfloat16>(P, st, true);
  }
  rc = launch_loss<float>(P, st);
  return rc != VINFER_OK ? rc : launch_grad<float>(P, st, true);
}

}  // extern "C"
