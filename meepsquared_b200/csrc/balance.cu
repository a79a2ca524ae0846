// The load-balancing loss of a router over one layer or many, the tokens each expert got, and the gradient of the
// router logits.
//
// Over the N unmasked tokens of all layers, with p the softmax of a token's E logits and S its top_k experts:
//   counts_le = tokens of layer l with e in S,  f_e = sum_l counts_le / N,  m_e = sum p_e / N
//   loss = E sum_e f_e m_e,   dx_te = g E / N p_te (f_e - sum_j p_tj f_j)
// The selection carries no gradient. A constant added to every f_e drops out of dx, so the kernels use f_e less its
// mean: near balance the differences are small against f itself and would lose their bits.
//
// Bound by memory: the logits are read once a direction and the gradient written once. A token is a group of 1 to 32
// lanes, each with consecutive experts in registers; the selection takes the largest remaining (logit, lower index
// first) top_k times, by one unsigned maximum over keys that hold both. The probabilities' sums stay in registers
// over a group's tokens, are joined per CTA, and the CTAs' sums by a second kernel in a fixed order; the counts are
// whole numbers, so that the order of their additions does not matter.
#include "common.cuh"
#include "host.hpp"

namespace meep2b {
namespace balance {

constexpr int THREADS = 256;
constexpr int MAX_LAYERS = 128;
constexpr int MAX_EXPERTS = 1024;
constexpr int MAX_CTAS = 592;

struct Layers {
  const void* logits[MAX_LAYERS];
  void* other[MAX_LAYERS];  // forward: the chosen experts (int64), or null; backward: the gradients
};

struct Params {
  int layers, experts, top_k;
  int64_t tokens;
  const uint8_t* mask;   // per token, or null
  int64_t* counts;       // (layers, experts)
  float* partial;        // (CTAs, experts)
  int32_t* live;         // (CTAs): unmasked tokens seen
  const float* coef;     // backward: E / N (f_e - mean f)
  const float* upstream;
};

__device__ __forceinline__ float value_of(const float* p) { return *p; }
__device__ __forceinline__ float value_of(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// Consecutive experts of a row as float32; -inf past the last. VEC: the row and the run are whole 16-byte pieces.
template <typename T, int PER, bool VEC>
__device__ __forceinline__ void load_row(const T* row, int e0, int experts, float (&v)[PER]) {
  constexpr int N = 16 / sizeof(T);
  if constexpr (VEC && PER >= N) {
#pragma unroll
    for (int i = 0; i < PER; i += N) {
      if (e0 + i < experts) {
        const uint4 w = *reinterpret_cast<const uint4*>(row + e0 + i);
        if constexpr (sizeof(T) == 2) {
          v[i] = bf16_lo(w.x), v[i + 1] = bf16_hi(w.x), v[i + 2] = bf16_lo(w.y), v[i + 3] = bf16_hi(w.y);
          v[i + 4] = bf16_lo(w.z), v[i + 5] = bf16_hi(w.z), v[i + 6] = bf16_lo(w.w), v[i + 7] = bf16_hi(w.w);
        } else {
          v[i] = __uint_as_float(w.x), v[i + 1] = __uint_as_float(w.y);
          v[i + 2] = __uint_as_float(w.z), v[i + 3] = __uint_as_float(w.w);
        }
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[i + j] = -INFINITY;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = e0 + i < experts ? value_of(row + e0 + i) : -INFINITY;
  }
}

template <typename T, int PER, bool VEC>
__device__ __forceinline__ void store_row(T* row, int e0, int experts, const float (&v)[PER]) {
  constexpr int N = 16 / sizeof(T);
  if constexpr (VEC && PER >= N) {
#pragma unroll
    for (int i = 0; i < PER; i += N) {
      if (e0 + i < experts) {
        if constexpr (sizeof(T) == 2)
          *reinterpret_cast<uint4*>(row + e0 + i) =
              make_uint4(pack_bf16x2(v[i], v[i + 1]), pack_bf16x2(v[i + 2], v[i + 3]),
                         pack_bf16x2(v[i + 4], v[i + 5]), pack_bf16x2(v[i + 6], v[i + 7]));
        else
          *reinterpret_cast<float4*>(row + e0 + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (e0 + i < experts) {
        if constexpr (sizeof(T) == 2) row[e0 + i] = __float2bfloat16_rn(v[i]);
        else row[e0 + i] = v[i];
      }
    }
  }
}

template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int off = G / 2; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int off = G / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// v becomes the softmax of the group's logits (float32).
template <int G, int PER>
__device__ __forceinline__ void softmax(float (&v)[PER]) {
  float top = v[0];
#pragma unroll
  for (int i = 1; i < PER; ++i) top = fmaxf(top, v[i]);
  top = group_max<G>(top);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    v[i] = expf(v[i] - top);
    sum += v[i];
  }
  const float inv = 1.0f / group_sum<G>(sum);
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] *= inv;
}

// An order of float32 values as unsigned numbers (NaN as torch sorts it: above everything; the zeros equal), from 1.
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0xfffeffffu;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

template <typename T, int G, int PER, bool VEC>
__global__ void __launch_bounds__(THREADS) forward(const __grid_constant__ Layers L, const Params p) {
  extern __shared__ float shared[];
  int* hist = reinterpret_cast<int*>(shared);  // experts, of the layer in hand
  const int lane = threadIdx.x & (G - 1);
  constexpr int GROUPS = THREADS / G;
  const int group = threadIdx.x / G;
  const int e0 = lane * PER;
  float mass[PER] = {};
  int live = 0;
  const int64_t rounds = (p.tokens + GROUPS - 1) / GROUPS;  // of a layer, a token a group
  const int64_t all = rounds * p.layers;
  const int64_t r0 = all * blockIdx.x / gridDim.x, r1 = all * (blockIdx.x + 1) / gridDim.x;
  int64_t r = r0;
  while (r < r1) {
    const int layer = static_cast<int>(r / rounds);
    const int64_t end = min(r1, (layer + 1) * rounds);
    const T* logits = static_cast<const T*>(L.logits[layer]);
    const int64_t* ids = static_cast<const int64_t*>(L.other[layer]);
    for (int e = threadIdx.x; e < p.experts; e += THREADS) hist[e] = 0;
    __syncthreads();
    for (; r < end; ++r) {
      const int64_t t = (r - layer * rounds) * GROUPS + group;
      const bool on = t < p.tokens && (p.mask == nullptr || p.mask[t] != 0);
      float v[PER];
      if (on) {
        load_row<T, PER, VEC>(logits + t * p.experts, e0, p.experts, v);
      } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = 0.f;
      }
      if (ids != nullptr) {
        if (on) {
          for (int j = lane; j < p.top_k; j += G) {
            const int64_t e = ids[t * p.top_k + j];
            if (e >= 0 && e < p.experts) atomicAdd(&hist[e], 1);
          }
        }
      } else if constexpr (sizeof(T) == 2) {
        // a bf16 logit has 16 bits: above the 16 bits of its index, one 32-bit key for both
        uint32_t key[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i)
          key[i] = e0 + i < p.experts ? (ordered(v[i]) & 0xffff0000u) | (0xffffu - (e0 + i)) : 0u;
        uint32_t below = 0xffffffffu;
        for (int j = 0; j < p.top_k; ++j) {
          uint32_t best = 0;
#pragma unroll
          for (int i = 0; i < PER; ++i) best = max(best, key[i] < below ? key[i] : 0u);
#pragma unroll
          for (int off = G / 2; off > 0; off >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, off));
          below = best;
          if (on && lane == (j & (G - 1))) atomicAdd(&hist[0xffffu - (best & 0xffffu)], 1);
        }
      } else {
        uint64_t below = ~uint64_t(0);
        uint64_t key[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i)
          key[i] = e0 + i < p.experts ? (static_cast<uint64_t>(ordered(v[i])) << 16) | (0xffffu - (e0 + i)) : 0u;
        for (int j = 0; j < p.top_k; ++j) {
          uint64_t best = 0;
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const uint64_t k = key[i] < below ? key[i] : 0u;
            best = k > best ? k : best;
          }
#pragma unroll
          for (int off = G / 2; off > 0; off >>= 1) {
            const uint64_t o = __shfl_xor_sync(0xffffffffu, best, off);
            best = o > best ? o : best;
          }
          below = best;
          if (on && lane == (j & (G - 1))) atomicAdd(&hist[0xffffu - static_cast<uint32_t>(best & 0xffffu)], 1);
        }
      }
      softmax<G, PER>(v);
      if (on) {
#pragma unroll
        for (int i = 0; i < PER; ++i) mass[i] += v[i];
        live += lane == 0;
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.experts; e += THREADS)
      if (hist[e]) atomicAdd(reinterpret_cast<unsigned long long*>(p.counts + static_cast<int64_t>(layer) * p.experts + e),
                             static_cast<unsigned long long>(hist[e]));
    __syncthreads();
  }
  // the CTA's sums: a round of groups after another, in order
  __shared__ int seen;
  if (threadIdx.x == 0) seen = 0;
  __syncthreads();
  if (live) atomicAdd(&seen, live);
  for (int i = 0; i < PER; ++i)
    if (e0 + i < p.experts) shared[group * p.experts + e0 + i] = mass[i];
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += THREADS) {
    float t = 0.f;
    for (int g = 0; g < GROUPS; ++g) t += shared[g * p.experts + e];
    p.partial[static_cast<int64_t>(blockIdx.x) * p.experts + e] = t;
  }
  if (threadIdx.x == 0) p.live[blockIdx.x] = seen;
}

// The loss, and the gradient's coefficients, from the CTAs' sums (joined in order, in float64). One CTA: 32 experts at
// a time, 32 threads an expert.
__global__ void __launch_bounds__(1024) join(const Params p, int ctas, float* __restrict__ loss, float* __restrict__ coef) {
  __shared__ double sums[32][33];
  __shared__ double mass[MAX_EXPERTS];
  __shared__ double reduce[3][32];
  __shared__ double totals[3];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  for (int eb = 0; eb < p.experts; eb += 32) {
    const int e = eb + x;
    double m = 0.0;
    if (e < p.experts) {
#pragma unroll 8
      for (int b = y; b < ctas; b += 32) m += p.partial[static_cast<int64_t>(b) * p.experts + e];
    }
    sums[y][x] = m;
    __syncthreads();
    if (y == 0 && e < p.experts) {
      for (int i = 1; i < 32; ++i) m += sums[i][x];
      mass[e] = m;
    }
    __syncthreads();
  }
  const int e = threadIdx.x;
  double count = 0.0, live = 0.0;
  for (int b = threadIdx.x; b < ctas; b += 1024) live += p.live[b];
  if (e < p.experts) {
#pragma unroll 8
    for (int l = 0; l < p.layers; ++l) count += static_cast<double>(p.counts[static_cast<int64_t>(l) * p.experts + e]);
  }
  double v[3] = {e < p.experts ? mass[e] * count : 0.0, count, live};
#pragma unroll
  for (int k = 0; k < 3; ++k) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
    if (x == 0) reduce[k][y] = v[k];
  }
  __syncthreads();
  if (y == 0) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      double t = reduce[k][x];
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) t += __shfl_xor_sync(0xffffffffu, t, off);
      if (x == 0) totals[k] = t;
    }
  }
  __syncthreads();
  const double n = totals[2] > 0.0 ? totals[2] : 1.0;
  if (threadIdx.x == 0) *loss = static_cast<float>(p.experts * totals[0] / (n * n));
  if (e < p.experts) coef[e] = static_cast<float>(p.experts / (n * n) * (count - totals[1] / p.experts));
}

template <typename T, int G, int PER, bool VEC>
__global__ void __launch_bounds__(THREADS) backward(const __grid_constant__ Layers L, const Params p) {
  const int lane = threadIdx.x & (G - 1);
  constexpr int GROUPS = THREADS / G;
  const int group = threadIdx.x / G;
  const int e0 = lane * PER;
  const float g = *p.upstream;
  float coef[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) coef[i] = e0 + i < p.experts ? p.coef[e0 + i] : 0.f;
  const int64_t rounds = (p.tokens + GROUPS - 1) / GROUPS;
  const int64_t all = rounds * p.layers;
  for (int64_t r = blockIdx.x; r < all; r += gridDim.x) {
    const int layer = static_cast<int>(r / rounds);
    const int64_t t = (r - layer * rounds) * GROUPS + group;
    const bool inside = t < p.tokens;
    const bool on = inside && (p.mask == nullptr || p.mask[t] != 0);
    float v[PER];
    if (on) {
      load_row<T, PER, VEC>(static_cast<const T*>(L.logits[layer]) + t * p.experts, e0, p.experts, v);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) v[i] = 0.f;
    }
    softmax<G, PER>(v);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) dot = fmaf(v[i], coef[i], dot);
    dot = group_sum<G>(dot);
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = on ? g * (v[i] * (coef[i] - dot)) : 0.f;
    if (inside) store_row<T, PER, VEC>(static_cast<T*>(L.other[layer]) + t * p.experts, e0, p.experts, v);
  }
}

template <typename T, int G, int PER, bool VEC>
static int launch(const Layers& L, const Params& p, bool back, int* ctas, cudaStream_t s) {
  constexpr int GROUPS = THREADS / G;
  const int64_t all = (p.tokens + GROUPS - 1) / GROUPS * p.layers;
  if (back) {
    const int64_t n = all < 148 * 8 ? all : 148 * 8;
    backward<T, G, PER, VEC><<<static_cast<unsigned>(n), THREADS, 0, s>>>(L, p);
  } else {
    *ctas = static_cast<int>(all < MAX_CTAS ? all : MAX_CTAS);
    // at most 32 KB: 8 groups of 1024 experts
    forward<T, G, PER, VEC><<<*ctas, THREADS, static_cast<size_t>(GROUPS) * p.experts * sizeof(float), s>>>(L, p);
  }
  return launch_status();
}

// The group of lanes for a row of experts: eight experts a lane where that fills no more than a warp, fewer for the
// smallest rows (a lane takes a whole row of up to 8), up to 32 beyond 256 experts.
template <typename T>
static int launch_size(const Layers& L, const Params& p, bool back, bool vec, int* ctas, cudaStream_t s) {
#define MEEP2B_ROW(G, PER) \
  return vec ? launch<T, G, PER, true>(L, p, back, ctas, s) : launch<T, G, PER, false>(L, p, back, ctas, s)
  if (p.experts <= 8) MEEP2B_ROW(1, 8);
  if (p.experts <= 16) MEEP2B_ROW(2, 8);
  if (p.experts <= 32) MEEP2B_ROW(4, 8);
  if (p.experts <= 64) MEEP2B_ROW(8, 8);
  if (p.experts <= 128) MEEP2B_ROW(16, 8);
  if (p.experts <= 256) MEEP2B_ROW(32, 8);
  if (p.experts <= 512) MEEP2B_ROW(32, 16);
  MEEP2B_ROW(32, 32);
#undef MEEP2B_ROW
}

}  // namespace balance
}  // namespace meep2b

using namespace meep2b;

namespace {

int balance_params(const meep2b_balance* a, const void* const* second, bool back, balance::Layers* L,
                   balance::Params* p, bool* vec) {
  if (a == nullptr || a->logits == nullptr || a->layers < 1 || a->tokens < 0 || a->experts < 1) return MEEP2B_ERR_SHAPE;
  if (a->layers > balance::MAX_LAYERS || a->experts > balance::MAX_EXPERTS) return MEEP2B_ERR_UNSUPPORTED;
  if (a->top_k < 1 || a->top_k > a->experts) return MEEP2B_ERR_SHAPE;
  if (a->dtype != MEEP2B_BF16 && a->dtype != MEEP2B_F32) return MEEP2B_ERR_DTYPE;
  if (a->coef == nullptr) return MEEP2B_ERR_SHAPE;
  *vec = a->experts % (a->dtype == MEEP2B_BF16 ? 8 : 4) == 0;
  for (int i = 0; i < a->layers; ++i) {
    L->logits[i] = a->logits[i];
    L->other[i] = second == nullptr ? nullptr : const_cast<void*>(second[i]);
    *vec = *vec && aligned16(L->logits[i]) && (!back || aligned16(L->other[i]));
  }
  *p = balance::Params{};
  p->layers = a->layers, p->experts = a->experts, p->top_k = a->top_k, p->tokens = a->tokens;
  p->mask = a->mask, p->coef = a->coef;
  return MEEP2B_OK;
}

}  // namespace

extern "C" {

size_t meep2b_balance_workspace_bytes(int32_t experts) {
  return static_cast<size_t>(balance::MAX_CTAS) * (static_cast<size_t>(experts) * sizeof(float) + sizeof(int32_t));
}

int meep2b_balance_loss(const meep2b_balance* a, void* stream) {
  balance::Layers L;
  balance::Params p;
  bool vec;
  MEEP2B_TRY(balance_params(a, reinterpret_cast<const void* const*>(a ? a->index : nullptr), false, &L, &p, &vec));
  if (a->counts == nullptr || a->loss == nullptr || a->workspace == nullptr) return MEEP2B_ERR_SHAPE;
  cudaStream_t s = as_stream(stream);
  MEEP2B_TRY(bind_stream_device(s));
  p.counts = a->counts;
  p.partial = static_cast<float*>(a->workspace);
  p.live = reinterpret_cast<int32_t*>(p.partial + static_cast<int64_t>(balance::MAX_CTAS) * a->experts);
  if (cudaMemsetAsync(a->counts, 0, static_cast<size_t>(a->layers) * a->experts * sizeof(int64_t), s) != cudaSuccess) {
    cudaGetLastError();
    return MEEP2B_ERR_LAUNCH;
  }
  int ctas = 0;
  if (a->tokens > 0)
    MEEP2B_TRY(a->dtype == MEEP2B_BF16 ? balance::launch_size<__nv_bfloat16>(L, p, false, vec, &ctas, s)
                                       : balance::launch_size<float>(L, p, false, vec, &ctas, s));
  balance::join<<<1, 1024, 0, s>>>(p, ctas, a->loss, a->coef);
  return launch_status();
}

int meep2b_balance_loss_backward(const meep2b_balance* a, void* stream) {
  balance::Layers L;
  balance::Params p;
  bool vec;
  MEEP2B_TRY(balance_params(a, reinterpret_cast<const void* const*>(a ? a->grads : nullptr), true, &L, &p, &vec));
  if (a->grads == nullptr || a->upstream == nullptr) return MEEP2B_ERR_SHAPE;
  cudaStream_t s = as_stream(stream);
  MEEP2B_TRY(bind_stream_device(s));
  if (a->tokens == 0) return MEEP2B_OK;
  p.upstream = a->upstream;
  return a->dtype == MEEP2B_BF16 ? balance::launch_size<__nv_bfloat16>(L, p, true, vec, nullptr, s)
                                 : balance::launch_size<float>(L, p, true, vec, nullptr, s);
}

}  // extern "C"
