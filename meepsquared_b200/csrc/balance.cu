// The load-balancing loss of a router over one layer or many, the tokens each expert got, and the gradient of the
// router logits.
//
// Over the N unmasked tokens of all layers, with p the softmax of a token's E logits and S its top_k experts:
//   counts_le = tokens of layer l with e in S,  f_e = sum_l counts_le / N,  m_e = sum p_e / N
//   loss = E sum_e f_e m_e,   dx_te = g E / N p_te (f_e - sum_j p_tj f_j)
// The selection carries no gradient. A constant added to every f_e drops out of dx, so the kernels use f_e less its
// mean: near balance the differences are small against f itself and would lose their bits.
//
// Bound by memory where there are many tokens: the logits are read once a direction and the gradient written once. A
// token is a group of 1 to 32 lanes; a lane holds up to 32 experts as pieces of 8 (16 bytes of bf16), piece j of lane i
// being the row's piece j G + i, so that a group's loads are whole lines. Few lanes a token keep the exchanges between
// lanes (the largest logit, the sums, the choice) small against the arithmetic on what a lane holds.
//
// The choice, up to 8 of bf16 logits: each piece's 8 (logit, index) keys are sorted by a network in registers, and
// sorted lists are joined by taking the larger of a[i] and b[7 - i] and sorting what comes out (bitonic), within a lane
// and then between lanes: about 60 instructions a token at 128 experts, where top_k rounds of a maximum over all keys
// took 140. More than 8, or float32 logits (64-bit keys), take the rounds.
//
// 24 layers of 16,384 x 128 (8 chosen), kernels alone: bf16 logits, own choice 78 us (1.3 TB/s), choice given 47, backward
// 44 (4.6 TB/s); float32 logits 227, 61 and 66. The top_k rounds took 174 us in bf16. What bounds the forward pass is
// latency: at 128 registers a thread there are 3.5 warps a scheduler and 0.59 instructions issued a cycle; the integer
// pipe (minima and maxima) is the busiest, 64% in bf16 and 79% in float32, whose 64-bit keys also spill.
//
// The probabilities' sums stay in float32 registers over up to 256 of a group's tokens (equal probabilities, one after
// another, would be off by 9e-5 of their sum after 7,000) and are joined per CTA in 64 bits; the CTAs' sums are added as
// 64-bit whole numbers of 2^-36, whose order does not matter, with what a sum has below that in units of 2^-90 beside
// it (sums under 2^-12, for the most), so that experts with hardly any probability keep theirs. The last CTA to finish
// works out the loss and the gradient's coefficients.
#include "common.cuh"
#include "host.hpp"

namespace meep2b {
namespace balance {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_LAYERS = 128;
constexpr int MAX_EXPERTS = 1024;
constexpr int CTAS_PER_SM = 2;
constexpr double kUnit = 68719476736.0;  // 2^36: sums of up to 2^28 probabilities fit 64 bits
constexpr double kFine = 18014398509481984.0;  // 2^54 to a unit: less than one of each of up to 2^9 CTAs fits 64 bits
constexpr int MOST_CTAS = 512;
constexpr int FLUSH = 256;  // tokens whose probabilities a lane sums up before they are joined into its CTA's
constexpr int64_t kMostTokens = int64_t(1) << 27;

struct Layers {
  const void* logits[MAX_LAYERS];
  void* other[MAX_LAYERS];  // forward: the chosen experts (int64), or null; backward: the gradients
};

struct Params {
  int layers, experts, top_k;
  int64_t tokens;
  const uint8_t* mask;              // per token, or null
  unsigned long long* counts;       // (layers, experts), zero at the start
  unsigned long long* mass;         // (2, experts): in units of 2^-36, and what is below them in units of 2^-90; then the
                                    // unmasked tokens, the CTAs done, whether a sum was not finite (zero at the start)
  float* loss;
  float* coef;                      // E / N^2 (c_e - mean c)
  const float* upstream;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// A lane's experts of a row, PER of them, -inf past the last: bf16 in pairs, or float32. VEC: rows are whole 16-byte
// pieces.
template <typename T, int PER>
struct Row;

template <int PER>
struct Row<__nv_bfloat16, PER> {
  uint32_t w[PER / 2];
  template <int G, bool VEC>
  __device__ __forceinline__ void load(const __nv_bfloat16* row, int lane, int experts) {
#pragma unroll
    for (int j = 0; j < PER / 8; ++j) {
      const int e = (j * G + lane) * 8;
      if (VEC) {
        uint4 q = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
        if (e < experts) q = *reinterpret_cast<const uint4*>(row + e);
        w[4 * j] = q.x, w[4 * j + 1] = q.y, w[4 * j + 2] = q.z, w[4 * j + 3] = q.w;
      } else {
        const unsigned short* r = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t lo = e + 2 * i < experts ? r[e + 2 * i] : 0xff80u;
          const uint32_t hi = e + 2 * i + 1 < experts ? r[e + 2 * i + 1] : 0xff80u;
          w[4 * j + i] = lo | (hi << 16);
        }
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ float value(int i) const { return i & 1 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]); }
  __device__ __forceinline__ float largest() const {
    __nv_bfloat162 m = *reinterpret_cast<const __nv_bfloat162*>(&w[0]);
#pragma unroll
    for (int i = 1; i < PER / 2; ++i) m = __hmax2(m, *reinterpret_cast<const __nv_bfloat162*>(&w[i]));
    return fmaxf(__low2float(m), __high2float(m));
  }
};

template <int PER>
struct Row<float, PER> {
  float w[PER];
  template <int G, bool VEC>
  __device__ __forceinline__ void load(const float* row, int lane, int experts) {
#pragma unroll
    for (int j = 0; j < PER / 8; ++j) {
      const int e = (j * G + lane) * 8;
#pragma unroll
      for (int h = 0; h < 8; h += 4) {
        if (VEC) {
          float4 q = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
          if (e + h < experts) q = *reinterpret_cast<const float4*>(row + e + h);
          w[8 * j + h] = q.x, w[8 * j + h + 1] = q.y, w[8 * j + h + 2] = q.z, w[8 * j + h + 3] = q.w;
        } else {
#pragma unroll
          for (int i = h; i < h + 4; ++i) w[8 * j + i] = e + i < experts ? row[e + i] : -INFINITY;
        }
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < PER; ++i) w[i] = 0.f;
  }
  __device__ __forceinline__ float value(int i) const { return w[i]; }
  __device__ __forceinline__ float largest() const {
    float m = w[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) m = fmaxf(m, w[i]);
    return m;
  }
};

template <int G, bool VEC, int PER>
__device__ __forceinline__ void store_row(__nv_bfloat16* row, int lane, int experts, const float (&v)[PER]) {
#pragma unroll
  for (int j = 0; j < PER / 8; ++j) {
    const int e = (j * G + lane) * 8;
    const float* x = v + 8 * j;
    if (VEC) {
      if (e < experts)
        *reinterpret_cast<uint4*>(row + e) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                                        pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e + i < experts) row[e + i] = __float2bfloat16_rn(x[i]);
    }
  }
}

template <int G, bool VEC, int PER>
__device__ __forceinline__ void store_row(float* row, int lane, int experts, const float (&v)[PER]) {
#pragma unroll
  for (int j = 0; j < PER / 8; ++j) {
    const int e = (j * G + lane) * 8;
    const float* x = v + 8 * j;
#pragma unroll
    for (int h = 0; h < 8; h += 4) {
      if (VEC) {
        if (e + h < experts) *reinterpret_cast<float4*>(row + e + h) = make_float4(x[h], x[h + 1], x[h + 2], x[h + 3]);
      } else {
#pragma unroll
        for (int i = h; i < h + 4; ++i)
          if (e + i < experts) row[e + i] = x[i];
      }
    }
  }
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int off = G / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// v: 2^((x - max) log2 e) of the lane's experts; returns 1 over the group's sum of them (float32). The difference is
// taken first: x log2 e - max log2 e in one fused step overflows where a row's largest logit is the type's lowest value
// (a row whose mask leaves nothing), and is off by more than the exponent's range from 1e10 on.
template <int G, int PER, typename R>
__device__ __forceinline__ float softmax(const R& row, float (&v)[PER]) {
  float top = row.largest();
#pragma unroll
  for (int off = G / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    v[i] = exp2_fast((row.value(i) - top) * kLog2e);
    sum += v[i];
  }
  return 1.0f / group_sum<G>(sum);
}

// Sorting 8 keys, largest first (Batcher's odd-even merge, 19 exchanges).
__device__ __forceinline__ void swap_if(uint32_t& a, uint32_t& b) {
  const uint32_t hi = max(a, b), lo = min(a, b);
  a = hi, b = lo;
}
__device__ __forceinline__ void sort8(uint32_t (&k)[8]) {
  swap_if(k[0], k[1]), swap_if(k[2], k[3]), swap_if(k[4], k[5]), swap_if(k[6], k[7]);
  swap_if(k[0], k[2]), swap_if(k[1], k[3]), swap_if(k[4], k[6]), swap_if(k[5], k[7]);
  swap_if(k[1], k[2]), swap_if(k[5], k[6]);
  swap_if(k[0], k[4]), swap_if(k[1], k[5]), swap_if(k[2], k[6]), swap_if(k[3], k[7]);
  swap_if(k[2], k[4]), swap_if(k[3], k[5]);
  swap_if(k[1], k[2]), swap_if(k[3], k[4]), swap_if(k[5], k[6]);
}
// The 8 largest of two sorted lists, sorted, into a.
__device__ __forceinline__ void join8(uint32_t (&a)[8], const uint32_t (&b)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = max(a[i], b[7 - i]);
#pragma unroll
  for (int i = 0; i < 4; ++i) swap_if(a[i], a[i + 4]);
#pragma unroll
  for (int i = 0; i < 8; i += 4) swap_if(a[i], a[i + 2]), swap_if(a[i + 1], a[i + 3]);
#pragma unroll
  for (int i = 0; i < 8; i += 2) swap_if(a[i], a[i + 1]);
}

// Two bf16 as 16-bit numbers in their order (both zeros alike, NaN above everything).
__device__ __forceinline__ uint32_t ordered2(uint32_t w) {
  const __nv_bfloat162 zero = __halves2bfloat162(__ushort_as_bfloat16(0), __ushort_as_bfloat16(0));
  const __nv_bfloat162 x = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&w), zero);  // -0 + 0 = 0
  const uint32_t b = *reinterpret_cast<const uint32_t*>(&x);
  return b ^ (((b >> 15) & 0x00010001u) * 0x7fffu | 0x80008000u);
}
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Experts of the logits' choice counted in hist: keys hold the logit's order above 0xffff less the expert.
template <int G, int PER>
__device__ __forceinline__ void choose(const Row<__nv_bfloat16, PER>& row, int lane, int top_k, bool on, int* hist) {
  auto keys = [&](int j, uint32_t (&k)[8]) {
    const uint32_t low = 0xffffu - (j * G + lane) * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t o = ordered2(row.w[4 * j + i]);
      k[2 * i] = (o << 16) | (low - 2 * i);
      k[2 * i + 1] = (o & 0xffff0000u) | (low - 2 * i - 1);
    }
  };
  if (top_k <= 8) {
    uint32_t best[8];
    keys(0, best);
    sort8(best);
#pragma unroll
    for (int j = 1; j < PER / 8; ++j) {
      uint32_t more[8];
      keys(j, more);
      sort8(more);
      join8(best, more);
    }
#pragma unroll
    for (int off = 1; off < G; off <<= 1) {
      uint32_t other[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) other[i] = __shfl_xor_sync(0xffffffffu, best[i], off);
      join8(best, other);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (on && i < top_k && lane == i % G) atomicAdd(&hist[0xffffu - (best[i] & 0xffffu)], 1);
    return;
  }
  uint32_t below = 0xffffffffu;
  uint32_t key[PER];
#pragma unroll
  for (int j = 0; j < PER / 8; ++j) {
    uint32_t k[8];
    keys(j, k);
#pragma unroll
    for (int i = 0; i < 8; ++i) key[8 * j + i] = k[i];
  }
  for (int r = 0; r < top_k; ++r) {
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) best = max(best, key[i] < below || r == 0 ? key[i] : 0u);
#pragma unroll
    for (int off = G / 2; off > 0; off >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, off));
    below = best;
    if (on && lane == (r & (G - 1))) atomicAdd(&hist[0xffffu - (best & 0xffffu)], 1);
  }
}

template <int G, int PER>
__device__ __forceinline__ void choose(const Row<float, PER>& row, int lane, int top_k, bool on, int* hist) {
  uint32_t order[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) order[i] = ordered(row.w[i]);
  auto key = [&](int i) {
    return (static_cast<uint64_t>(order[i]) << 16) | (0xffffu - ((i / 8 * G + lane) * 8 + i % 8));
  };
  uint64_t below = ~uint64_t(0);
  for (int r = 0; r < top_k; ++r) {
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint64_t k = key(i);
      if (k < below && k > best) best = k;
    }
#pragma unroll
    for (int off = G / 2; off > 0; off >>= 1) {
      const uint64_t o = __shfl_xor_sync(0xffffffffu, best, off);
      best = o > best ? o : best;
    }
    below = best;
    if (on && lane == (r & (G - 1))) atomicAdd(&hist[0xffffu - static_cast<uint32_t>(best & 0xffffu)], 1);
  }
}

template <typename T, int G, int PER, bool VEC>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM) forward(const __grid_constant__ Layers L, const Params p) {
  extern __shared__ __align__(8) float shared[];  // WARPS * experts, then `experts` double
  __shared__ int seen;
  __shared__ bool last;
  __shared__ double reduce[2][WARPS];
  int* hist = reinterpret_cast<int*>(shared);  // experts, of the layer in hand
  double* held = reinterpret_cast<double*>(shared + WARPS * p.experts);  // the CTA's sums of probabilities
  for (int e = threadIdx.x; e < p.experts; e += THREADS) held[e] = 0.0;
  const int lane = threadIdx.x & (G - 1), warp = threadIdx.x >> 5;
  constexpr int GROUPS = THREADS / G;
  const int group = threadIdx.x / G;
  float mass[PER] = {};
  int live = 0;
  if (threadIdx.x == 0) seen = 0;
  const int64_t rounds = (p.tokens + GROUPS - 1) / GROUPS;  // of a layer, a token a group
  const int64_t all = rounds * p.layers;
  const int64_t r0 = all * blockIdx.x / gridDim.x, r1 = all * (blockIdx.x + 1) / gridDim.x;
  // the sums of probabilities in registers joined into the CTA's: the groups of a warp, then the warps, in order
  auto join_mass = [&]() {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
#pragma unroll
      for (int off = G; off < 32; off <<= 1) mass[i] += __shfl_xor_sync(0xffffffffu, mass[i], off);
      const int e = (i / 8 * G + lane) * 8 + i % 8;
      if ((threadIdx.x & 31) < G && e < p.experts) shared[warp * p.experts + e] = mass[i];
      mass[i] = 0.f;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.experts; e += THREADS) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) t += shared[w * p.experts + e];
      held[e] += static_cast<double>(t);
    }
    __syncthreads();
  };
  int64_t r = r0, flush = r0 + FLUSH;
  while (r < r1) {
    const int layer = static_cast<int>(r / rounds);
    const int64_t end = min(min(r1, (layer + 1) * rounds), flush);
    const T* logits = static_cast<const T*>(L.logits[layer]);
    const int64_t* ids = static_cast<const int64_t*>(L.other[layer]);
    for (int e = threadIdx.x; e < p.experts; e += THREADS) hist[e] = 0;
    __syncthreads();
    for (; r < end; ++r) {
      const int64_t t = (r - layer * rounds) * GROUPS + group;
      const bool on = t < p.tokens && (p.mask == nullptr || p.mask[t] != 0);
      Row<T, PER> row;
      if (on) row.template load<G, VEC>(logits + t * p.experts, lane, p.experts);
      else row.zero();
      if (ids != nullptr) {
        if (on) {
          for (int j = lane; j < p.top_k; j += G) {
            const int64_t e = ids[t * p.top_k + j];
            if (e >= 0 && e < p.experts) atomicAdd(&hist[e], 1);
          }
        }
      } else {
        choose<G, PER>(row, lane, p.top_k, on, hist);
      }
      float v[PER];
      const float inv = softmax<G, PER>(row, v);
      if (on) {
#pragma unroll
        for (int i = 0; i < PER; ++i) mass[i] = fmaf(v[i], inv, mass[i]);
        live += lane == 0;
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.experts; e += THREADS)
      if (hist[e]) atomicAdd(p.counts + static_cast<int64_t>(layer) * p.experts + e, static_cast<unsigned long long>(hist[e]));
    __syncthreads();
    if (r == flush && r < r1) join_mass(), flush += FLUSH;
  }
  if (live) atomicAdd(&seen, live);
  join_mass();
  for (int e = threadIdx.x; e < p.experts; e += THREADS) {  // (this thread's own of held)
    const double units = held[e] * kUnit, whole = floor(units);
    if (units < 1.8e19) {
      atomicAdd(p.mass + e, static_cast<unsigned long long>(whole));
      if (units != whole) atomicAdd(p.mass + p.experts + e, __double2ull_rn((units - whole) * kFine));
    } else {
      atomicExch(p.mass + 2 * p.experts + 2, 1ull);
    }
  }
  unsigned long long* const said = p.mass + 2 * p.experts;  // the unmasked tokens, the CTAs done, a sum not finite
  if (threadIdx.x == 0) atomicAdd(said, static_cast<unsigned long long>(seen));
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(said + 1, 1ull) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double* chosen = reinterpret_cast<double*>(shared);
  double both = 0.0, total = 0.0;
  for (int e = threadIdx.x; e < p.experts; e += THREADS) {
    unsigned long long c = 0;
#pragma unroll 8
    for (int l = 0; l < p.layers; ++l) c += __ldcg(p.counts + static_cast<int64_t>(l) * p.experts + e);
    chosen[e] = static_cast<double>(c);
    total += chosen[e];
    both += chosen[e] * (static_cast<double>(__ldcg(p.mass + e)) +
                         static_cast<double>(__ldcg(p.mass + p.experts + e)) / kFine);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    both += __shfl_xor_sync(0xffffffffu, both, off);
    total += __shfl_xor_sync(0xffffffffu, total, off);
  }
  if ((threadIdx.x & 31) == 0) reduce[0][warp] = both, reduce[1][warp] = total;
  __syncthreads();
  both = total = 0.0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) both += reduce[0][w], total += reduce[1][w];
  const double n = static_cast<double>(max(1ull, __ldcg(said)));
  if (threadIdx.x == 0)
    *p.loss = __ldcg(said + 2) ? __int_as_float(0x7fc00000) : static_cast<float>(p.experts * both / (kUnit * n * n));
  for (int e = threadIdx.x; e < p.experts; e += THREADS)
    p.coef[e] = static_cast<float>(p.experts / (n * n) * (chosen[e] - total / p.experts));
}

template <typename T, int G, int PER, bool VEC>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM) backward(const __grid_constant__ Layers L, const Params p) {
  const int lane = threadIdx.x & (G - 1);
  constexpr int GROUPS = THREADS / G;
  const int group = threadIdx.x / G;
  const float g = *p.upstream;
  float coef[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = (i / 8 * G + lane) * 8 + i % 8;
    coef[i] = e < p.experts ? p.coef[e] : 0.f;
  }
  const int64_t rounds = (p.tokens + GROUPS - 1) / GROUPS;
  const int64_t all = rounds * p.layers;
  for (int64_t r = blockIdx.x; r < all; r += gridDim.x) {
    const int layer = static_cast<int>(r / rounds);
    const int64_t t = (r - layer * rounds) * GROUPS + group;
    const bool inside = t < p.tokens;
    const bool on = inside && (p.mask == nullptr || p.mask[t] != 0);
    Row<T, PER> row;
    if (on) row.template load<G, VEC>(static_cast<const T*>(L.logits[layer]) + t * p.experts, lane, p.experts);
    else row.zero();
    float v[PER];
    const float inv = softmax<G, PER>(row, v);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) dot = fmaf(v[i], coef[i], dot);
    dot = group_sum<G>(dot) * inv;
    const float scale = g * inv;
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = on ? scale * v[i] * (coef[i] - dot) : 0.f;
    if (inside) store_row<G, VEC>(static_cast<T*>(L.other[layer]) + t * p.experts, lane, p.experts, v);
  }
}

template <typename T, int G, int PER, bool VEC>
static int launch(const Layers& L, const Params& p, bool back, int sms, cudaStream_t s) {
  constexpr int GROUPS = THREADS / G;
  const int64_t all = (p.tokens + GROUPS - 1) / GROUPS * p.layers;
  const int64_t most = static_cast<int64_t>(sms) * CTAS_PER_SM < MOST_CTAS ? sms * CTAS_PER_SM : MOST_CTAS;
  const unsigned n = static_cast<unsigned>(all < 1 ? 1 : (all < most ? all : most));
  if (back) backward<T, G, PER, VEC><<<n, THREADS, 0, s>>>(L, p);
  else forward<T, G, PER, VEC><<<n, THREADS, (WARPS * sizeof(float) + sizeof(double)) * p.experts, s>>>(L, p);
  return launch_status();
}

// The lanes for a row: 32 experts a lane where there are as many, so that 4 lanes hold 128 experts.
template <typename T>
static int launch_size(const Layers& L, const Params& p, bool back, bool vec, int sms, cudaStream_t s) {
#define MEEP2B_ROW(G, PER) \
  return vec ? launch<T, G, PER, true>(L, p, back, sms, s) : launch<T, G, PER, false>(L, p, back, sms, s)
  if (p.experts <= 8) MEEP2B_ROW(1, 8);
  if (p.experts <= 16) MEEP2B_ROW(1, 16);
  if (p.experts <= 32) MEEP2B_ROW(1, 32);
  if (p.experts <= 64) MEEP2B_ROW(2, 32);
  if (p.experts <= 128) MEEP2B_ROW(4, 32);
  if (p.experts <= 256) MEEP2B_ROW(8, 32);
  if (p.experts <= 512) MEEP2B_ROW(16, 32);
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
  if (a->layers > balance::MAX_LAYERS || a->experts > balance::MAX_EXPERTS ||
      a->tokens > balance::kMostTokens / a->layers)
    return MEEP2B_ERR_SHAPE;
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
  p->mask = a->mask;
  return MEEP2B_OK;
}

}  // namespace

extern "C" {

size_t meep2b_balance_workspace_bytes(int32_t experts) {
  return (2 * static_cast<size_t>(experts) + 3) * sizeof(unsigned long long);
}

int meep2b_balance_loss(const meep2b_balance* a, void* stream) {
  balance::Layers L;
  balance::Params p;
  bool vec;
  MEEP2B_TRY(balance_params(a, reinterpret_cast<const void* const*>(a ? a->index : nullptr), false, &L, &p, &vec));
  if (a->counts == nullptr || a->loss == nullptr || a->workspace == nullptr) return MEEP2B_ERR_SHAPE;
  cudaStream_t s = as_stream(stream);
  MEEP2B_TRY(bind_stream_device(s));
  int sms = 0;
  MEEP2B_TRY(device_sms(&sms));
  p.counts = reinterpret_cast<unsigned long long*>(a->counts);
  p.mass = static_cast<unsigned long long*>(a->workspace);
  p.loss = a->loss, p.coef = a->coef;
  if (cudaMemsetAsync(a->counts, 0, static_cast<size_t>(a->layers) * a->experts * sizeof(int64_t), s) != cudaSuccess ||
      cudaMemsetAsync(a->workspace, 0, meep2b_balance_workspace_bytes(a->experts), s) != cudaSuccess) {
    cudaGetLastError();
    return MEEP2B_ERR_LAUNCH;
  }
  return a->dtype == MEEP2B_BF16 ? balance::launch_size<__nv_bfloat16>(L, p, false, vec, sms, s)
                                 : balance::launch_size<float>(L, p, false, vec, sms, s);
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
  int sms = 0;
  MEEP2B_TRY(device_sms(&sms));
  p.upstream = a->upstream, p.coef = a->coef;
  return a->dtype == MEEP2B_BF16 ? balance::launch_size<__nv_bfloat16>(L, p, true, vec, sms, s)
                                 : balance::launch_size<float>(L, p, true, vec, sms, s);
}

}  // extern "C"
