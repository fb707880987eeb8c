// states.cu — decode states follow the beams: slot s takes the state of slot parents[s] (sm_100a).
//
// A state is a tensor with a slot dimension (token counts, recurrent and convolution states,
// key/value caches); the host describes it as runs of contiguous bytes under up to four outer
// dimensions. One launch copies the moved slots of up to MAX_STATES tensors.
//
// In place, a slot may only take the state of a slot that keeps its own (parents[parents[s]] ==
// parents[s], as vinfer_beam_select lays beams out): sources are then never written, so the copies
// need no order and no second buffer. Into another buffer any slot may take any slot's state.
//
// Copies are bound by HBM: each distinct source is read from HBM once (its copies run close enough
// together to find it in L2) and each moved slot written once. Slots that stay cost nothing but
// a look at their parent. Measured on one B200: 64 slots with 16 tensors [8, 1024, 128] bf16 of ragged
// lengths, half of them moved, 187 us (1.14 GB: 6.1 TB/s, 0.93 of the measured copy bandwidth); 32
// slots with six [32, 128, 128] float32 states and their convolution states 68 us (0.91); three
// small arrays 3.0 us.
#include "rows.cuh"

#include <algorithm>

namespace {

using namespace rows;

constexpr int NT = 256;
constexpr int CTAS = 3;         // CTAs of an SM: 48 KiB of copies in flight (2 / 3 / 4 / 5 CTAs: 225 / 187 /
                                // 196 / 204 us for 64 slots of 16 tensors [8, 1024, 128] bf16, half moved)
constexpr int UV = 4;           // vectors a thread copies per item, all loads before the stores
constexpr int MAX_STATES = 64;  // tensors of one launch (they travel as kernel parameters)
constexpr int OUTER = VINFER_STATE_MAX_OUTER;

struct Desc {
  const unsigned char* src;
  unsigned char* dst;
  int64_t src_slot, dst_slot;   // byte strides of the slot dimension
  int64_t src_st[OUTER], dst_st[OUTER];
  uint32_t size[OUTER];         // outer dimensions, the last n_outer places
  uint32_t run_vecs;            // vectors of a run
  uint32_t vecs;                // vectors of one slot: outer sizes x run_vecs
  uint32_t chunks;              // items of one moved slot
  uint32_t unit_vecs;           // vectors of one position of the run, 0: lengths do not cut it
  int32_t len_max;              // positions along the length dimension
  int32_t len_outer;            // the outer dimension that lengths cut, -1: none
  int32_t n_outer;
  int32_t vec;                  // bytes of a vector: 16, 8, 4, 2 or 1
};

struct StatesP {
  Desc d[MAX_STATES];
  int n;
  int slots, in_place;
  const int* parents;
  const int* lengths;
  int* status;
};

// One item: NT * UV vectors of slot `from` to slot `to`, counted over the live part of its runs (`rv`
// vectors each). 32-bit index arithmetic; an item within one run, the usual one, is placed once and
// copied at constant offsets (placing every vector kept 62 % of the issue slots busy).
template <typename VT>
__device__ __forceinline__ void copy_item(const Desc& D, int from, int to, uint32_t chunk,
                                          uint32_t rv, uint32_t vecs, int len) {
  constexpr uint32_t SPAN = NT * UV;
  const unsigned char* src = D.src + (int64_t)from * D.src_slot;
  unsigned char* dst = D.dst + (int64_t)to * D.dst_slot;
  const uint32_t i0 = chunk * SPAN;
  const uint32_t o0 = D.n_outer ? i0 / rv : 0, r0 = i0 - o0 * rv;
  // the outer dimensions' offsets of run o; false where lengths cut it off
  auto place = [&](uint32_t o, int64_t& so, int64_t& po) {
    bool live = true;
    for (int k = OUTER - 1; k >= OUTER - D.n_outer; --k) {
      uint32_t x = o;
      if (k > OUTER - D.n_outer) {
        o /= D.size[k];
        x -= o * D.size[k];
      }
      so += x * D.src_st[k];
      po += x * D.dst_st[k];
      if (k == D.len_outer) live = live && (int)x < len;
    }
    return live;
  };
  if (r0 + SPAN <= rv && i0 + SPAN <= vecs) {
    int64_t so = 0, po = 0;
    if (!place(o0, so, po)) return;
    const VT* from_v = reinterpret_cast<const VT*>(src + so) + r0 + threadIdx.x;
    VT* to_v = reinterpret_cast<VT*>(dst + po) + r0 + threadIdx.x;
    VT v[UV];
#pragma unroll
    for (int u = 0; u < UV; ++u) v[u] = from_v[u * NT];
#pragma unroll
    for (int u = 0; u < UV; ++u) to_v[u * NT] = v[u];
    return;
  }
  VT v[UV];
  int64_t at[UV];
#pragma unroll
  for (int u = 0; u < UV; ++u) {
    const uint32_t step = u * NT + threadIdx.x;
    uint32_t r = r0 + step, o = o0;
    if (r >= rv && D.n_outer) {
      const uint32_t q = rv >= SPAN ? 1 : r / rv;
      o += q;
      r -= q * rv;
    }
    int64_t so = (int64_t)r * sizeof(VT), po = so;
    const bool live = i0 + step < vecs && place(o, so, po);
    at[u] = live ? po : -1;
    if (live) v[u] = *reinterpret_cast<const VT*>(src + so);
  }
#pragma unroll
  for (int u = 0; u < UV; ++u)
    if (at[u] >= 0) *reinterpret_cast<VT*>(dst + at[u]) = v[u];
}

// Dynamic shared memory: for every slot a packed move (source << 16 | slot) and the items of the
// moves before it.
__global__ void __launch_bounds__(NT, CTAS) k_reorder(const __grid_constant__ StatesP P) {
  extern __shared__ uint32_t moves[];
  uint32_t* before = moves + P.slots;  // [M + 1]
  __shared__ int wcnt[NT / 32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  uint32_t M = 0;  // the slots that move, ascending: every CTA makes the same list
  for (int s0 = 0; s0 < P.slots; s0 += NT) {
    const int s = s0 + threadIdx.x;
    bool move = false;
    int p = 0;
    if (s < P.slots) {
      p = P.parents[s];
      const bool ok = p >= 0 && p < P.slots && (!P.in_place || p == s || P.parents[p] == p);
      if (!ok && P.status && blockIdx.x == 0) atomicOr(P.status, (int)VINFER_ST_BAD_PARENT);
      move = ok && (!P.in_place || p != s);
    }
    const unsigned m = __ballot_sync(FULL, move);
    if (lane == 0) wcnt[w] = __popc(m);
    __syncthreads();
    uint32_t at = M + __popc(m & ((1u << lane) - 1));
    for (int i = 0; i < NT / 32; ++i) {
      if (i < w) at += wcnt[i];
      M += wcnt[i];
    }
    if (move) moves[at] = (uint32_t)p << 16 | (uint32_t)s;
    __syncthreads();
  }
  // items: whole states chunk by chunk with the moves of a chunk side by side; states cut by lengths
  // move by move, the live part alone; tensor after tensor
  auto live_vecs = [&](const Desc& D, uint32_t mv) {  // of one run
    return (uint32_t)min(max(P.lengths[mv & 0xffff], 0), D.len_max) * D.unit_vecs;
  };
  uint32_t g = blockIdx.x, unit = 0, run = 0, vecs = 0;  // of the tensor that `before` counts
  for (int t = 0; t < P.n; ++t) {
    const Desc& D = P.d[t];
    const bool cut = D.unit_vecs != 0;
    if (cut && (D.unit_vecs != unit || D.run_vecs != run || D.vecs != vecs)) {
      unit = D.unit_vecs;
      run = D.run_vecs;
      vecs = D.vecs;
      uint32_t sum = 0;
      for (uint32_t i0 = 0; i0 < M; i0 += NT) {
        const uint32_t i = i0 + threadIdx.x;
        const uint32_t mine =
            i < M ? (vecs / run * live_vecs(D, moves[i]) + NT * UV - 1) / (NT * UV) : 0;
        uint32_t incl = mine;
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t up = __shfl_up_sync(FULL, incl, o);
          if (lane >= o) incl += up;
        }
        __syncthreads();  // wcnt and `before` were read by all
        if (lane == 31) wcnt[w] = incl;
        __syncthreads();
        uint32_t at = sum + incl - mine;
        for (int k = 0; k < NT / 32; ++k) {
          if (k < w) at += wcnt[k];
          sum += wcnt[k];
        }
        if (i < M) before[i] = at;
      }
      if (threadIdx.x == 0) before[M] = sum;
      __syncthreads();
    }
    const uint32_t items = cut ? before[M] : D.chunks * M;
    for (; g < items; g += gridDim.x) {
      uint32_t chunk, i;
      if (cut) {  // the last move that begins at or before g
        uint32_t lo = 0, hi = M;
        while (hi - lo > 1) {
          const uint32_t mid = (lo + hi) / 2;
          if (before[mid] <= g) lo = mid;
          else hi = mid;
        }
        i = lo;
        chunk = g - before[i];
      } else {
        chunk = g / M;
        i = g - chunk * M;
      }
      const uint32_t mv = moves[i];
      const int from = mv >> 16, to = mv & 0xffff;
      const int len = D.len_outer >= 0 ? min(max(P.lengths[to], 0), D.len_max) : 0;
      const uint32_t rv = cut ? live_vecs(D, mv) : D.run_vecs;
      const uint32_t n = cut ? D.vecs / D.run_vecs * rv : D.vecs;
      switch (D.vec) {
        case 16: copy_item<uint4>(D, from, to, chunk, rv, n, len); break;
        case 8: copy_item<uint2>(D, from, to, chunk, rv, n, len); break;
        case 4: copy_item<uint32_t>(D, from, to, chunk, rv, n, len); break;
        case 2: copy_item<uint16_t>(D, from, to, chunk, rv, n, len); break;
        default: copy_item<uint8_t>(D, from, to, chunk, rv, n, len); break;
      }
    }
    g -= items;
  }
}

// A state as the kernel takes it.
int describe(const VinferState& s, int64_t slots, Desc* out) {
  Desc& D = *out;
  D = Desc{};
  D.src = static_cast<const unsigned char*>(s.src);
  D.dst = static_cast<unsigned char*>(s.dst);
  D.src_slot = s.src_slot_stride;
  D.dst_slot = s.dst_slot_stride;
  D.n_outer = s.n_outer;
  D.len_outer = -1;
  uint64_t bits = (uint64_t)(uintptr_t)s.src | (uint64_t)(uintptr_t)s.dst |
                  (uint64_t)s.src_slot_stride | (uint64_t)s.dst_slot_stride |
                  (uint64_t)s.run_bytes | (uint64_t)s.len_unit_bytes | 16;
  int64_t len_max = s.len_unit_bytes ? s.run_bytes / s.len_unit_bytes : 0;
  int64_t outer = 1;
  for (int j = 0; j < s.n_outer; ++j) {
    const int k = OUTER - s.n_outer + j;
    if (s.outer_size[j] > (int64_t)INT32_MAX / outer) return VINFER_E_LIMIT;
    D.size[k] = (uint32_t)s.outer_size[j];
    D.src_st[k] = s.src_outer_stride[j];
    D.dst_st[k] = s.dst_outer_stride[j];
    if (j == s.len_outer) {
      D.len_outer = k;
      len_max = s.outer_size[j];
    }
    bits |= (uint64_t)D.src_st[k] | (uint64_t)D.dst_st[k];
    outer *= s.outer_size[j];
  }
  D.vec = (int)(bits & (~bits + 1));  // the lowest set bit divides every address and size
  const int64_t run_vecs = s.run_bytes / D.vec;
  if (run_vecs > (int64_t)INT32_MAX / outer) return VINFER_E_LIMIT;
  D.run_vecs = (uint32_t)run_vecs;
  D.vecs = (uint32_t)(outer * run_vecs);
  D.unit_vecs = (uint32_t)(s.len_unit_bytes / D.vec);
  D.len_max = (int32_t)len_max;
  D.chunks = (D.vecs + (uint32_t)(NT * UV) - 1) / (uint32_t)(NT * UV);
  if ((int64_t)D.chunks * slots > (int64_t)INT32_MAX) return VINFER_E_LIMIT;
  return VINFER_OK;
}

}  // namespace

extern "C" int vinfer_reorder_states(const VinferState* states, int32_t n_states,
                                     const int32_t* parents, int64_t slots,
                                     const int32_t* lengths, int32_t* status, void* stream) {
  NvtxRange nvtx_range("vinfer_reorder_states");
  if (!states || n_states < 1 || !parents || slots < 1) return VINFER_E_ARG;
  if (slots > VINFER_STATE_MAX_SLOTS) return VINFER_E_LIMIT;
  const bool in_place = states[0].src == states[0].dst;
  for (int i = 0; i < n_states; ++i) {
    const VinferState& s = states[i];
    if (!s.src || !s.dst || s.run_bytes < 1 || s.n_outer < 0 || s.n_outer > OUTER) return VINFER_E_ARG;
    if ((s.src == s.dst) != in_place || s.len_outer < -1 || s.len_outer >= s.n_outer) return VINFER_E_ARG;
    if (s.len_unit_bytes < 0 || (s.len_unit_bytes > 0 && (s.run_bytes % s.len_unit_bytes || s.len_outer >= 0)))
      return VINFER_E_ARG;
    if ((s.len_unit_bytes > 0 || s.len_outer >= 0) && !lengths) return VINFER_E_ARG;
    if (in_place && s.src_slot_stride != s.dst_slot_stride) return VINFER_E_ARG;
    for (int k = 0; k < s.n_outer; ++k)
      if (s.outer_size[k] < 1 || (in_place && s.src_outer_stride[k] != s.dst_outer_stride[k]))
        return VINFER_E_ARG;
  }
  Desc d;
  for (int i = 0; i < n_states; ++i) {  // nothing is copied unless everything can be
    const int rc = describe(states[i], slots, &d);
    if (rc != VINFER_OK) return rc;
  }
  for (int i0 = 0; i0 < n_states; i0 += MAX_STATES) {
    StatesP P = {};
    P.n = std::min(MAX_STATES, n_states - i0);
    P.slots = (int)slots;
    P.in_place = in_place;
    P.parents = parents;
    P.lengths = lengths;
    P.status = status;
    int64_t chunks = 0;
    for (int i = 0; i < P.n; ++i) {
      describe(states[i0 + i], slots, &P.d[i]);
      chunks += P.d[i].chunks;
    }
    // every slot may move: no more CTAs than items, at most what is resident
    const int64_t grid = std::min<int64_t>(148 * CTAS, chunks * slots);
    const size_t smem = (size_t)slots * 8 + 4;
    if (opt_in<k_reorder>(VINFER_STATE_MAX_SLOTS * 8 + 4) != VINFER_OK) return VINFER_E_CUDA;
    const int rc = launch(k_reorder, (unsigned)grid, NT, smem, (cudaStream_t)stream, false, 1, P);
    if (rc != VINFER_OK) return rc;
  }
  return VINFER_OK;
}
