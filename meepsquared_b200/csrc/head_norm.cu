// RMS norm of every query and key head and the rotation by position, in one pass, and the gradients.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  y = R(pos) (n w)
// R turns the pairs (i, i + half) of the first 2 half dimensions by the position's angles and leaves the others.
// Backward, from x (r is computed again) and dy:
//   u = R^T dy,  dw = sum over rows of u n,  v = u w,  dx = r (v - n mean(v n))
//
// Bound by memory: x in and y out (forward), x and dy in and dx out (backward), once each. A head is read by a group
// of 2 to 32 lanes, each with two 16-byte chunks that turn against each other (i and i + half), so that the rotation
// needs no exchange between lanes and the norm three or four shuffles. A group takes several heads of one token in a
// row, which keeps the token's cosines and sines and the head weight in registers. A CTA works on queries or on keys
// alone, in proportion to their heads. The weights' gradients are summed in registers, joined per CTA, and the CTAs'
// sums by a second kernel in a fixed order.
#include "common.cuh"
#include "host.hpp"

namespace meep2b {
namespace head_norm {

constexpr int THREADS = 256;
constexpr int MAX_PARTIALS = 1184;  // CTAs of the backward pass that may leave sums: eight per SM

struct Side {  // the queries or the keys
  const void* x;
  int64_t sb, st, sh;  // elements between batches, tokens and heads
  int heads;
  const void* weight;
  void* y;             // forward: y; backward: dx (contiguous)
  const void* dy;
  int64_t db, dt, dh;
};

struct Params {
  Side side[2];
  int64_t tokens;      // batch * length
  int length, dim, half, span;  // span: heads a group takes in a row
  const void* cos;
  const void* sin;
  int64_t ld_cos, ld_sin, angles;
  const int64_t* positions;
  float eps;
  int q_blocks;
  float* partial;      // (CTAs, dim)
};

template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(const void* p, float (&v)[8]) {
    const uint4 w = *static_cast<const uint4*>(p);
    v[0] = bf16_lo(w.x), v[1] = bf16_hi(w.x), v[2] = bf16_lo(w.y), v[3] = bf16_hi(w.y);
    v[4] = bf16_lo(w.z), v[5] = bf16_hi(w.z), v[6] = bf16_lo(w.w), v[7] = bf16_hi(w.w);
  }
  static __device__ __forceinline__ void store(void* p, const float (&v)[8]) {
    *static_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                         pack_bf16x2(v[6], v[7]));
  }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void load(const void* p, float (&v)[4]) {
    const float4 w = *static_cast<const float4*>(p);
    v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
  }
  static __device__ __forceinline__ void store(void* p, const float (&v)[4]) {
    *static_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};

// N values of a cosine or sine row; the rows may start anywhere.
template <typename A, int N>
__device__ __forceinline__ void load_angles(const void* base, int64_t at, float (&v)[N]) {
  const A* p = static_cast<const A*>(base) + at;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if constexpr (sizeof(A) == 4) v[j] = p[j];
    else v[j] = __bfloat162float(p[j]);
  }
}

// T: the heads' type; A: the angles'; G: lanes a head; BACKWARD; DW: the weights' gradients too.
template <typename T, typename A, int G, bool BACKWARD, bool DW>
__global__ void __launch_bounds__(THREADS) norm_rotate(const Params p) {
  constexpr int N = Vec<T>::N;
  const int kind = blockIdx.x >= p.q_blocks;
  const Side& s = p.side[kind];
  const int blocks = kind ? gridDim.x - p.q_blocks : p.q_blocks;
  const int block = kind ? blockIdx.x - p.q_blocks : blockIdx.x;
  const int lane = threadIdx.x & (G - 1), group = threadIdx.x / G;
  constexpr int GROUPS = THREADS / G;
  // this lane's two chunks: a rotated pair (slot, slot + half), or two of the chunks that stay
  const int turned = p.half / N;
  const bool here = lane < p.dim / (2 * N), turns = lane < turned;
  const int c0 = turns ? lane : 2 * turned + 2 * (lane - turned), c1 = turns ? lane + turned : c0 + 1;
  const int o0 = c0 * N, o1 = c1 * N;
  float w0[N] = {}, w1[N] = {}, dw0[N] = {}, dw1[N] = {};
  if (here) {
    Vec<T>::load(static_cast<const T*>(s.weight) + o0, w0);
    Vec<T>::load(static_cast<const T*>(s.weight) + o1, w1);
  }
  const int spans = (s.heads + p.span - 1) / p.span;
  const int64_t items = p.tokens * spans;
  const float inv_dim = 1.0f / static_cast<float>(p.dim);
  const int64_t stride = static_cast<int64_t>(blocks) * GROUPS;
  // every group of a warp makes the same number of rounds, so that the shuffles below have all their lanes
  const int64_t first = static_cast<int64_t>(block) * GROUPS + group;
  const int64_t warp_first = static_cast<int64_t>(block) * GROUPS + (threadIdx.x & ~31) / G;
  for (int64_t base = warp_first, item = first; base < items; base += stride, item += stride) {
    const bool live = item < items;
    const int64_t t = live ? item / spans : 0;
    const int h0 = live ? static_cast<int>(item - t * spans) * p.span : 0;
    const int64_t b = t / p.length;
    const int l = static_cast<int>(t - b * p.length);
    float cs[N], sn[N];
#pragma unroll
    for (int j = 0; j < N; ++j) cs[j] = 1.f, sn[j] = 0.f;
    if (live && turns) {
      const int64_t pos = p.positions ? p.positions[t] : l;
      if (pos >= 0 && pos < p.angles) {
        load_angles<A, N>(p.cos, pos * p.ld_cos + o0, cs);
        load_angles<A, N>(p.sin, pos * p.ld_sin + o0, sn);
      } else {  // a position without angles
#pragma unroll
        for (int j = 0; j < N; ++j) cs[j] = sn[j] = __int_as_float(0x7fc00000);
      }
    }
    const T* x = static_cast<const T*>(s.x) + b * s.sb + l * s.st;
    const T* dy = BACKWARD ? static_cast<const T*>(s.dy) + b * s.db + l * s.dt : nullptr;
    T* y = static_cast<T*>(s.y) + t * s.heads * p.dim;
#pragma unroll 2
    for (int i = 0; i < p.span; ++i) {
      const int h = h0 + i;
      const bool on = live && here && h < s.heads;
      float a[N] = {}, c[N] = {};
      if (on) {
        Vec<T>::load(x + h * s.sh + o0, a);
        Vec<T>::load(x + h * s.sh + o1, c);
      }
      float u0[N] = {}, u1[N] = {};
      if (BACKWARD && on) {
        Vec<T>::load(dy + h * s.dh + o0, u0);
        Vec<T>::load(dy + h * s.dh + o1, u1);
      }
      float sq = 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j) sq = fmaf(a[j], a[j], fmaf(c[j], c[j], sq));
#pragma unroll
      for (int off = G / 2; off > 0; off >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, off);
      const float r = rsqrtf(fmaf(sq, inv_dim, p.eps));
      if (!BACKWARD) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float e = a[j] * r * w0[j], f = c[j] * r * w1[j];
          a[j] = turns ? e * cs[j] - f * sn[j] : e;
          c[j] = turns ? f * cs[j] + e * sn[j] : f;
        }
      } else {
        float mean = 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          a[j] *= r, c[j] *= r;
          const float e = turns ? u0[j] * cs[j] + u1[j] * sn[j] : u0[j];
          const float f = turns ? u1[j] * cs[j] - u0[j] * sn[j] : u1[j];
          if (DW) dw0[j] = fmaf(e, a[j], dw0[j]), dw1[j] = fmaf(f, c[j], dw1[j]);
          u0[j] = e * w0[j], u1[j] = f * w1[j];
          mean = fmaf(u0[j], a[j], fmaf(u1[j], c[j], mean));
        }
#pragma unroll
        for (int off = G / 2; off > 0; off >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, off);
        mean *= inv_dim;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          a[j] = r * (u0[j] - a[j] * mean);
          c[j] = r * (u1[j] - c[j] * mean);
        }
      }
      if (on) {
        Vec<T>::store(y + h * p.dim + o0, a);
        Vec<T>::store(y + h * p.dim + o1, c);
      }
    }
  }
  if (DW) {  // the CTA's sum, group after group
    extern __shared__ float sums[];  // (GROUPS, dim)
    if (here) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        sums[group * p.dim + o0 + j] = dw0[j];
        sums[group * p.dim + o1 + j] = dw1[j];
      }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < p.dim; d += THREADS) {
      float t = 0.f;
      for (int g = 0; g < GROUPS; ++g) t += sums[g * p.dim + d];
      p.partial[static_cast<int64_t>(blockIdx.x) * p.dim + d] = t;
    }
  }
}

// The CTAs' sums of one side's weight gradient joined in order: blockIdx.y the side, 32 dimensions a CTA, 32 threads
// a dimension.
template <typename T>
__global__ void __launch_bounds__(1024) join_weight(const float* __restrict__ partial, int q_blocks, int blocks, int dim,
                                                   T* __restrict__ dq, T* __restrict__ dk) {
  __shared__ float sums[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + x;
  const int b0 = blockIdx.y ? q_blocks : 0, b1 = blockIdx.y ? blocks : q_blocks;
  float t = 0.f;
  if (d < dim)
    for (int b = b0 + y; b < b1; b += 32) t += partial[static_cast<int64_t>(b) * dim + d];
  sums[y][x] = t;
  __syncthreads();
  if (y == 0 && d < dim) {
    float all = 0.f;
    for (int i = 0; i < 32; ++i) all += sums[i][x];
    T* to = blockIdx.y ? dk : dq;
    if constexpr (sizeof(T) == 2) to[d] = __float2bfloat16_rn(all);
    else to[d] = all;
  }
}

template <typename T, typename A, bool BACKWARD, bool DW>
static void launch(const Params& p, int blocks, cudaStream_t s) {
  const int slots = p.dim / (2 * Vec<T>::N);  // lanes a head needs
#define MEEP2B_HEADS(G)                                                                                      \
  norm_rotate<T, A, G, BACKWARD, DW>                                                                          \
      <<<blocks, THREADS, DW ? static_cast<size_t>(THREADS / G) * p.dim * sizeof(float) : 0, s>>>(p)
  if (slots <= 2) MEEP2B_HEADS(2);
  else if (slots <= 4) MEEP2B_HEADS(4);
  else if (slots <= 8) MEEP2B_HEADS(8);
  else if (slots <= 16) MEEP2B_HEADS(16);
  else MEEP2B_HEADS(32);
#undef MEEP2B_HEADS
}

template <bool BACKWARD, bool DW>
static void launch_types(const Params& p, int dtype, int angle_dtype, int blocks, cudaStream_t s) {
  if (dtype == MEEP2B_BF16) {
    if (angle_dtype == MEEP2B_BF16) launch<__nv_bfloat16, __nv_bfloat16, BACKWARD, DW>(p, blocks, s);
    else launch<__nv_bfloat16, float, BACKWARD, DW>(p, blocks, s);
  } else {
    if (angle_dtype == MEEP2B_BF16) launch<float, __nv_bfloat16, BACKWARD, DW>(p, blocks, s);
    else launch<float, float, BACKWARD, DW>(p, blocks, s);
  }
}

// How the heads of a token are taken: up to 8 in a row, fewer while that leaves groups without work. blocks: enough
// CTAs for every item, or what the SMs hold at once.
static int shape(Params& p, int lanes, int sms, int most_blocks) {
  const int groups = THREADS / lanes;
  const int64_t heads = p.side[0].heads + p.side[1].heads;
  const int64_t wanted = static_cast<int64_t>(sms) * 8 * groups;  // groups that keep the memory busy
  p.span = 8;
  while (p.span > 1 && p.tokens * heads / p.span < wanted) p.span /= 2;
  int64_t items = 0, q_items = 0;
  for (int i = 0; i < 2; ++i) {
    const int64_t n = p.tokens * ((p.side[i].heads + p.span - 1) / p.span);
    items += n;
    if (i == 0) q_items = n;
  }
  int64_t blocks = (q_items + groups - 1) / groups + (items - q_items + groups - 1) / groups;
  if (blocks <= most_blocks) {
    p.q_blocks = static_cast<int>((q_items + groups - 1) / groups);
    return static_cast<int>(blocks);
  }
  blocks = most_blocks;
  int q = static_cast<int>(blocks * q_items / items);
  q = q < 1 ? 1 : (q > blocks - 1 ? static_cast<int>(blocks) - 1 : q);
  p.q_blocks = q;
  return static_cast<int>(blocks);
}

static int lanes_of(int dim, int dtype) {
  const int slots = dim / (dtype == MEEP2B_BF16 ? 16 : 8);
  int g = 2;
  while (g < slots) g *= 2;
  return g;
}

}  // namespace head_norm
}  // namespace meep2b

using namespace meep2b;

namespace {

int head_norm_params(const meep2b_head_norm* a, bool backward, head_norm::Params* out) {
  if (a == nullptr || a->batch < 0 || a->length < 0 || a->q_heads < 1 || a->kv_heads < 1) return MEEP2B_ERR_SHAPE;
  if (a->dtype != MEEP2B_BF16 && a->dtype != MEEP2B_F32) return MEEP2B_ERR_DTYPE;
  if (a->angle_dtype != MEEP2B_BF16 && a->angle_dtype != MEEP2B_F32) return MEEP2B_ERR_DTYPE;
  if (a->dim < 16 || a->dim > 256 || a->dim % 16 || a->half < 0 || a->half % 8 || 2 * a->half > a->dim)
    return MEEP2B_ERR_SHAPE;
  if (a->positions == nullptr && a->half > 0 && a->angles < a->length) return MEEP2B_ERR_SHAPE;
  if (a->length > INT32_MAX) return MEEP2B_ERR_SHAPE;
  const int64_t vec = a->dtype == MEEP2B_BF16 ? 8 : 4;
  for (int i = 0; i < 3; ++i) {
    if (a->q_stride[i] % vec || a->k_stride[i] % vec) return MEEP2B_ERR_ALIGN;
    if (backward && (a->dq_out_stride[i] % vec || a->dk_out_stride[i] % vec)) return MEEP2B_ERR_ALIGN;
  }
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->q_weight) || !aligned16(a->k_weight) ||
      !aligned16(a->q_out) || !aligned16(a->k_out) || (backward && (!aligned16(a->dq_out) || !aligned16(a->dk_out))))
    return MEEP2B_ERR_ALIGN;
  head_norm::Params p = {};
  p.side[0] = {a->q, a->q_stride[0], a->q_stride[1], a->q_stride[2], a->q_heads, a->q_weight, a->q_out,
               a->dq_out, a->dq_out_stride[0], a->dq_out_stride[1], a->dq_out_stride[2]};
  p.side[1] = {a->k, a->k_stride[0], a->k_stride[1], a->k_stride[2], a->kv_heads, a->k_weight, a->k_out,
               a->dk_out, a->dk_out_stride[0], a->dk_out_stride[1], a->dk_out_stride[2]};
  p.tokens = a->batch * a->length, p.length = static_cast<int>(a->length);
  p.dim = a->dim, p.half = a->half;
  p.cos = a->cos, p.sin = a->sin, p.ld_cos = a->ld_cos, p.ld_sin = a->ld_sin, p.angles = a->angles;
  p.positions = a->positions, p.eps = a->eps;
  *out = p;
  return MEEP2B_OK;
}

}  // namespace

extern "C" {

int meep2b_head_norm_partials(void) { return head_norm::MAX_PARTIALS; }

int meep2b_head_norm_rotate(const meep2b_head_norm* a, void* stream) {
  head_norm::Params p;
  MEEP2B_TRY(head_norm_params(a, false, &p));
  cudaStream_t s = as_stream(stream);
  MEEP2B_TRY(bind_stream_device(s));
  if (p.tokens == 0) return MEEP2B_OK;
  const int blocks = head_norm::shape(p, head_norm::lanes_of(p.dim, a->dtype), 148, 148 * 8);
  head_norm::launch_types<false, false>(p, a->dtype, a->angle_dtype, blocks, s);
  return launch_status();
}

int meep2b_head_norm_rotate_backward(const meep2b_head_norm* a, void* stream) {
  head_norm::Params p;
  MEEP2B_TRY(head_norm_params(a, true, &p));
  const bool dw = a->dq_weight != nullptr;
  if (dw && (a->dk_weight == nullptr || a->partial == nullptr)) return MEEP2B_ERR_SHAPE;
  cudaStream_t s = as_stream(stream);
  MEEP2B_TRY(bind_stream_device(s));
  p.partial = a->partial;
  int blocks = 0;
  if (p.tokens > 0) {
    blocks = head_norm::shape(p, head_norm::lanes_of(p.dim, a->dtype), 148, head_norm::MAX_PARTIALS);
    if (dw) head_norm::launch_types<true, true>(p, a->dtype, a->angle_dtype, blocks, s);
    else head_norm::launch_types<true, false>(p, a->dtype, a->angle_dtype, blocks, s);
    MEEP2B_TRY(launch_status());
  }
  if (dw) {
    const dim3 grid((p.dim + 31) / 32, 2);
    if (a->dtype == MEEP2B_BF16)
      head_norm::join_weight<<<grid, 1024, 0, s>>>(p.partial, p.q_blocks, blocks, p.dim,
                                                   static_cast<__nv_bfloat16*>(a->dq_weight),
                                                   static_cast<__nv_bfloat16*>(a->dk_weight));
    else
      head_norm::join_weight<<<grid, 1024, 0, s>>>(p.partial, p.q_blocks, blocks, p.dim,
                                                   static_cast<float*>(a->dq_weight), static_cast<float*>(a->dk_weight));
    MEEP2B_TRY(launch_status());
  }
  return MEEP2B_OK;
}

}  // extern "C"
