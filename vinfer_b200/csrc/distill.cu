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

// Vector v of the part with its listed elements taken out.
template <typename T>
__device__ __noinline__ uint4 without(uint4 q, int v, const int* hit, int hits) {
  for (int h = 0; h < hits; ++h)
    if (hit[h] / Vec<T>::A == v) Vec<T>::put(q, hit[h] & (Vec<T>::A - 1), Vec<T>::NEG_INF_BITS);
  return q;
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
      const uint32_t word = marked[(vb - v0 + u * NT) / 32 + tid / 32];
      if (word && word >> (tid & 31) & 1) q[u] = without<T>(q[u], vb - v0 + u * NT + tid, hit, hits);
    }
    add_exps<T>(q, VT::max(q), P.scale, m, s);
  }
  block_join<NW>(m, s, P.scale, sm);
  if (tid == 0) P.part[blockIdx.x] = Part{m, s};
}

// A row's list as one warp works on it, four entries a lane.
struct ListS {
  double z[MAXK];     // listed logits; behind the join distances from the row's largest, in log2
  double p[MAXK];     // masses as listed
  double psum[MAXK];  // ... summed over the entries of the same id
  float l[MAXK];      // log-probabilities
  int id[MAXK];       // -1: empty
  bool lead[MAXK];    // the first entry of its id
  double mass;        // sum of p
  double top;         // largest z
  int distinct;       // ids
  bool bad;           // an id or a log-probability out of range
};

// What depends on the list alone, and its logits.
template <typename T>
__device__ __forceinline__ void list_begin(const DistP& P, int64_t row, ListS& L) {
  const int lane = threadIdx.x & 31;
  const T* x = static_cast<const T*>(P.logits) + row * P.ld;
  int id[4];
  bool bad = false;
  double mass = 0, top = (double)neg_inf();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = lane + 32 * i;
    id[i] = -1;
    if (j < P.k) {
      id[i] = P.ids[row * P.k + j];
      float l = P.lp[row * P.k + j];
      if (id[i] < 0) {
        id[i] = -1;
        l = neg_inf();
      }
      const bool off = id[i] >= P.V || !(l < -neg_inf());
      bad = bad || off;
      const double z = id[i] >= 0 && !off ? (double)Vec<T>::load(x + id[i]) : (double)neg_inf();
      const double p = id[i] >= 0 ? exp((double)l) : 0.0;
      L.id[j] = id[i];
      L.l[j] = l;
      L.z[j] = z;
      L.p[j] = p;
      mass += p;
      if (z > top || z != z) top = z;
    }
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
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = lane + 32 * i;
    if (j < P.k) {
      L.psum[j] = psum[i];
      L.lead[j] = lead[i];
      distinct += lead[i];
    }
  }
  mass = warp_sum(mass);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const double t = __shfl_xor_sync(FULL, top, o);
    if (t > top || t != t) top = t;
  }
  distinct = (int)__reduce_add_sync(FULL, (unsigned)distinct);
  bad = __any_sync(FULL, bad);
  if (lane == 0) {
    L.mass = mass;
    L.top = top;
    L.distinct = distinct;
    L.bad = bad;
  }
  __syncwarp();
}

// The row's loss and gradient terms from the list and the sum outside it, (m, r) with r in units of
// 2^(m * scale). listg[j]: dloss/dz of the j-th listed element.
__device__ __forceinline__ float list_finish(const DistP& P, ListS& L, float m, double r,
                                             Stat* stat, float* listg) {
  const int lane = threadIdx.x & 31;
  const float nan = __int_as_float(0x7fffffff);
  if (L.bad) {
    if (lane == 0 && P.status) atomicOr(P.status, (int)VINFER_ST_BAD_LIST);
    if (listg)
      for (int j = lane; j < P.k; j += 32) listg[j] = nan;
    if (stat) *stat = Stat{nan, nan};
    return nan;
  }
  // all in distances from the row's largest logit, whatever its magnitude, and in log2
  const double inf = (double)-neg_inf();
  double ref = L.top;
  if (r != 0 && !(ref != ref) && (double)m > ref) ref = m;
  double total = 0;
  for (int j = lane; j < P.k; j += 32) {
    L.z[j] = (L.z[j] - ref) * P.scale_d;
    if (L.lead[j]) total += exp2(L.z[j]);
  }
  const double rest = r == 0 ? -inf : ((double)m - ref) * P.scale_d + log2(r);
  total = warp_sum(total) + (r == 0 ? 0.0 : exp2(rest));
  const double lse = log2(total);
  if (lane == 0 && P.status && !(fabs(lse) < inf)) atomicOr(P.status, (int)VINFER_ST_NONFINITE);
  // the target's masses
  double mass = L.mass, pt = 0, norm = 1, lnorm = 0;
  if (P.tail) {
    pt = L.distinct < P.V ? fmax(0.0, 1.0 - mass) : 0.0;
  } else if (mass > 0) {
    norm = 1.0 / mass;
    lnorm = log(mass);
    mass = 1.0;
  }
  const double M = mass + pt;
  double loss = 0;
  for (int j = lane; j < P.k; j += 32) {
    const double z = L.z[j] - lse, p = L.p[j];
    if (p > 0) loss += p * norm * (((double)L.l[j] - lnorm) - z * LN2_D);
    if (listg) listg[j] = L.id[j] >= 0 ? (float)(M * exp2(z) - L.psum[j] * norm) : 0.f;
  }
  loss = warp_sum(loss);
  if (pt > 0) loss += pt * (log(pt) - (rest - lse) * LN2_D);
  if (lse != lse) loss = lse;
  if (stat) {
    Stat t = {0.f, 0.f};
    if (r != 0) t = Stat{m, (float)((M * exp2(rest - lse) - pt) / r)};
    if (lse != lse) t = Stat{nan, nan};
    *stat = t;
  }
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
  Stat st;
  const float loss = list_finish(P, L, m, r, P.stat ? &st : nullptr,
                                 P.stat ? P.listg + row * P.k : nullptr);
  if (lane == 0) {
    P.loss[row] = loss * weight;
    if (P.stat) P.stat[row] = st;
  }
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

// Parts of a row: enough CTAs to fill the 148 SMs several times over, at least two vectors a
// thread in each.
int distill_parts(int64_t rows_, int64_t vocab, int dtype) {
  const int64_t A = dtype == VINFER_DTYPE_BF16 ? 8 : 4;
  const int64_t nv = (vocab + A - 1) / A;
  int64_t p = (148 * 8 + rows_ - 1) / rows_;
  p = std::min<int64_t>(p, (nv + 2 * NT - 1) / (2 * NT));
  return (int)std::max<int64_t>(1, std::min<int64_t>(p, MAX_PARTS));
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
  if (a->dtype == VINFER_DTYPE_BF16) {
    rc = launch_loss<__nv_bfloat16>(P, st);
    return rc != VINFER_OK ? rc : launch_grad<__nv_bfloat16>(P, st, true);
  }
  rc = launch_loss<float>(P, st);
  return rc != VINFER_OK ? rc : launch_grad<float>(P, st, true);
}

}  // extern "C"
