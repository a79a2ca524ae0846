// RMS norm of every query and key head and the rotation by position, in one pass, and the gradients.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  y = R(pos) (n w)
// R turns the pairs (i, i + half) of the first 2 half dimensions by the position's angles and leaves the others.
// Backward, from x (r is computed again) and dy:
//   u = R^T dy,  dw = sum over rows of u n,  v = u w,  dx = r (v - n mean(v n))
//
// Bound by memory: x in and y out (forward), x and dy in and dx out (backward), once each. A head is read by a group
// of 1 to 32 lanes, each with two 16-byte chunks that turn against each other (i and i + half), so that the rotation
// needs no exchange between lanes and the norm three or four shuffles. A group takes several heads of one token in a
// row, which keeps the token's cosines and sines and the head weight in registers. A thread's heads come through a ring
// of its own in shared memory by 16-byte asynchronous copies, a few heads ahead: enough in flight for HBM without
// holding registers, and with no barrier. A CTA works on queries or on keys alone. The forward pass has a group for
// every run of heads; the backward pass with the weights' gradients has as many CTAs as the SMs hold, in proportion
// to the queries' and the keys' heads: their sums stay in registers, are joined per CTA, and the CTAs' sums by a
// second kernel in a fixed order. 4 x 4,096 tokens, 32 + 4 heads of 128 in bf16: forward 50 us (6.0 TB/s, 92% of the
// measured copy rate), backward with the weights' gradients 79 us (5.7 TB/s) and 4 us; with the loads through
// registers, two heads ahead, 56 and 115 us. Float32 norm weights beside bf16 heads are read as they are (16 registers
// a thread instead of 8, no spills): the same times within 1%.
#include "common.cuh"
#include "host.hpp"

namespace meep2b {
namespace head_norm {

constexpr int THREADS = 256;
constexpr int MAX_PARTIALS = 512;  // CTAs of the backward pass that may leave sums

struct Side {  // the queries or the keys
  const void* x;
  int64_t sb, st, sh;  // elements between batches, tokens and heads
  int heads;
  const void* weight;
  void* y;             // forward: y; backward: dx (contiguous)
  const void* dy;
  int64_t db, dt, dh;
  int span;            // heads a group takes in a row
};

struct Params {
  Side side[2];
  int64_t tokens;      // batch * length
  int length, dim, half;
  int angle_vec;       // cosine and sine rows start on 16 bytes
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
  static __device__ __forceinline__ void unpack(uint4 w, float (&v)[8]) {
    v[0] = bf16_lo(w.x), v[1] = bf16_hi(w.x), v[2] = bf16_lo(w.y), v[3] = bf16_hi(w.y);
    v[4] = bf16_lo(w.z), v[5] = bf16_hi(w.z), v[6] = bf16_lo(w.w), v[7] = bf16_hi(w.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                      pack_bf16x2(v[6], v[7]));
  }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(uint4 w, float (&v)[4]) {
    v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};

// N values of a cosine or sine row, which may start anywhere unless vec.
template <typename A, int N>
__device__ __forceinline__ void load_angles(const void* base, int64_t at, bool vec, float (&v)[N]) {
  const A* p = static_cast<const A*>(base) + at;
  if constexpr (sizeof(A) == 4) {
    if (vec) {
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        const float4 q = __ldg(reinterpret_cast<const float4*>(p + j));
        v[j] = q.x, v[j + 1] = q.y, v[j + 2] = q.z, v[j + 3] = q.w;
      }
      return;
    }
  } else if constexpr (N == 8) {
    if (vec) {
      Vec<__nv_bfloat16>::unpack(__ldg(reinterpret_cast<const uint4*>(p)), v);
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if constexpr (sizeof(A) == 4) v[j] = p[j];
    else v[j] = __bfloat162float(p[j]);
  }
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Heads a thread's copies run ahead: 8 KB of shared memory a CTA each forward, 16 KB backward (x and dy).
template <bool BACKWARD>
struct Ring {
  static constexpr int CHUNKS = BACKWARD ? 4 : 2;
  static constexpr int DEPTH = BACKWARD ? 3 : 4;
  static constexpr int BYTES = DEPTH * CHUNKS * THREADS * 16;
};

// A chunk's norm weights as they are stored (half the registers in bf16), widened at each use.
template <typename W, int N>
struct Weights {
  static constexpr int WORDS = N / Vec<W>::N;
  uint4 w[WORDS];
  __device__ __forceinline__ void load(const void* base, int at) {
    const uint4* from = reinterpret_cast<const uint4*>(static_cast<const W*>(base) + at);
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = from[i];
  }
  __device__ __forceinline__ void unpack(float (&v)[N]) const {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      float part[Vec<W>::N];
      Vec<W>::unpack(w[i], part);
#pragma unroll
      for (int j = 0; j < Vec<W>::N; ++j) v[i * Vec<W>::N + j] = part[j];
    }
  }
};

// T: the heads' type; W: the norm weights' (T or float); A: the angles'; G: lanes a head; BACKWARD; DW: the weights'
// gradients too.
template <typename T, typename W, typename A, int G, bool BACKWARD, bool DW>
__global__ void __launch_bounds__(THREADS, BACKWARD ? 2 : 3) norm_rotate(const Params p) {
  constexpr int N = Vec<T>::N;
  using R = Ring<BACKWARD>;
  extern __shared__ __align__(16) uint8_t ring[];
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
  float dw0[N] = {}, dw1[N] = {};
  Weights<W, N> wr0 = {}, wr1 = {};
  if (here) wr0.load(s.weight, o0), wr1.load(s.weight, o1);
  // items fit 31 bits (the entry point's limit on tokens x heads), and a stride more 32
  const int span = s.span;
  const uint32_t spans = (s.heads + span - 1) / span;
  const uint32_t items = static_cast<uint32_t>(p.tokens) * spans;
  const float inv_dim = 1.0f / static_cast<float>(p.dim);
  const uint32_t stride = static_cast<uint32_t>(blocks) * GROUPS;
  // every group of a warp makes the same number of rounds, so that the shuffles below have all their lanes
  const uint32_t first = static_cast<uint32_t>(block) * GROUPS + group;
  const uint32_t warp_first = static_cast<uint32_t>(block) * GROUPS + (threadIdx.x & ~31) / G;
  const int rounds = warp_first < items ? static_cast<int>((items - 1 - warp_first) / stride) + 1 : 0;
  const int steps = rounds * span;

  // the copies' side: step after step, a head each
  uint32_t c_item = first;
  int c_head = 0, c_left = 0, c_slot = 0;
  const T *c_x = nullptr, *c_dy = nullptr;
  const uint32_t mine = smem_u32(ring) + threadIdx.x * 16u;
  auto copy_next = [&]() {
    if (c_left == 0) {  // the next item
      const bool live = c_item < items;
      const uint32_t t = live ? c_item / spans : 0;
      const uint32_t b = t / static_cast<uint32_t>(p.length), l = t - b * static_cast<uint32_t>(p.length);
      c_head = live ? static_cast<int>(c_item - t * spans) * span : s.heads;
      c_x = static_cast<const T*>(s.x) + b * s.sb + l * s.st + c_head * s.sh;
      if (BACKWARD) c_dy = static_cast<const T*>(s.dy) + b * s.db + l * s.dt + c_head * s.dh;
      c_left = span;
      c_item += stride;
    }
    if (here && c_head < s.heads) {
      const uint32_t at = mine + c_slot * (R::CHUNKS * THREADS * 16u);
      copy16(at, c_x + o0);
      copy16(at + THREADS * 16u, c_x + o1);
      if (BACKWARD) {
        copy16(at + 2 * THREADS * 16u, c_dy + o0);
        copy16(at + 3 * THREADS * 16u, c_dy + o1);
      }
    }
    ++c_head, --c_left;
    c_x += s.sh;
    if (BACKWARD) c_dy += s.dh;
    c_slot = c_slot + 1 == R::DEPTH ? 0 : c_slot + 1;
  };
#pragma unroll
  for (int i = 0; i < R::DEPTH - 1; ++i) {
    if (i < steps) copy_next();
    copies_commit();
  }

  float cs[N], sn[N];
  T* y = nullptr;
  uint32_t item = first;
  int head = 0, left = 0, slot = 0;
  for (int step = 0; step < steps; ++step) {
    if (left == 0) {  // the next item: its angles
      const bool live = item < items;
      const uint32_t t = live ? item / spans : 0;
      head = live ? static_cast<int>(item - t * spans) * span : s.heads;
      y = static_cast<T*>(s.y) + (static_cast<int64_t>(t) * s.heads + head) * p.dim;
#pragma unroll
      for (int j = 0; j < N; ++j) cs[j] = 1.f, sn[j] = 0.f;
      if (live && turns) {
        const int64_t pos = p.positions ? p.positions[t] : t % static_cast<uint32_t>(p.length);
        if (pos >= 0 && pos < p.angles) {
          load_angles<A, N>(p.cos, pos * p.ld_cos + o0, p.angle_vec, cs);
          load_angles<A, N>(p.sin, pos * p.ld_sin + o0, p.angle_vec, sn);
        } else {  // a position without angles
#pragma unroll
          for (int j = 0; j < N; ++j) cs[j] = sn[j] = __int_as_float(0x7fc00000);
        }
      }
      left = span;
      item += stride;
    }
    if (step + R::DEPTH - 1 < steps) copy_next();
    copies_commit();
    copies_wait<R::DEPTH - 1>();
    const bool on = here && head < s.heads;
    uint4 rx0 = make_uint4(0, 0, 0, 0), rx1 = rx0, rd0 = rx0, rd1 = rx0;
    if (on) {
      const uint4* at = reinterpret_cast<const uint4*>(ring) + slot * (R::CHUNKS * THREADS) + threadIdx.x;
      rx0 = at[0], rx1 = at[THREADS];
      if (BACKWARD) rd0 = at[2 * THREADS], rd1 = at[3 * THREADS];
    }
    float a[N], c[N], w0[N], w1[N];
    Vec<T>::unpack(rx0, a), Vec<T>::unpack(rx1, c);
    float sq = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) sq = fmaf(a[j], a[j], fmaf(c[j], c[j], sq));
#pragma unroll
    for (int off = G / 2; off > 0; off >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, off);
    const float r = rsqrtf(fmaf(sq, inv_dim, p.eps));
    wr0.unpack(w0), wr1.unpack(w1);
    if (!BACKWARD) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float e = a[j] * r * w0[j], f = c[j] * r * w1[j];
        a[j] = turns ? e * cs[j] - f * sn[j] : e;
        c[j] = turns ? f * cs[j] + e * sn[j] : f;
      }
    } else {
      float u0[N], u1[N];
      Vec<T>::unpack(rd0, u0), Vec<T>::unpack(rd1, u1);
      float mean = 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        a[j] *= r, c[j] *= r;
        const float e = turns ? u0[j] * cs[j] + u1[j] * sn[j] : u0[j];
        const float f = turns ? u1[j] * cs[j] - u0[j] * sn[j] : u1[j];
        if (DW) {
          if (on) dw0[j] = fmaf(e, a[j], dw0[j]), dw1[j] = fmaf(f, c[j], dw1[j]);
        }
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
      *reinterpret_cast<uint4*>(y + o0) = Vec<T>::pack(a);
      *reinterpret_cast<uint4*>(y + o1) = Vec<T>::pack(c);
    }
    ++head, --left;
    y += p.dim;
    slot = slot + 1 == R::DEPTH ? 0 : slot + 1;
  }
  if (DW) {  // the CTA's sum, group after group
    float* sums = reinterpret_cast<float*>(ring);  // (GROUPS, dim): at most 16 KB
    copies_wait<0>();
    __syncthreads();
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
#pragma unroll 8
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
#pragma unroll 8
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

template <typename T, typename W, typename A, bool BACKWARD, bool DW>
static void launch(const Params& p, unsigned blocks, cudaStream_t s) {
  const int slots = p.dim / (2 * Vec<T>::N);  // lanes a head needs
#define MEEP2B_HEADS(G)                                                                                      \
  norm_rotate<T, W, A, G, BACKWARD, DW><<<blocks, THREADS, Ring<BACKWARD>::BYTES, s>>>(p)
  if (slots <= 1) MEEP2B_HEADS(1);
  else if (slots <= 2) MEEP2B_HEADS(2);
  else if (slots <= 4) MEEP2B_HEADS(4);
  else if (slots <= 8) MEEP2B_HEADS(8);
  else if (slots <= 16) MEEP2B_HEADS(16);
  else MEEP2B_HEADS(32);
#undef MEEP2B_HEADS
}

template <typename T, typename W, bool BACKWARD, bool DW>
static void launch_angles(const Params& p, int angle_dtype, unsigned blocks, cudaStream_t s) {
  if (angle_dtype == MEEP2B_BF16) launch<T, W, __nv_bfloat16, BACKWARD, DW>(p, blocks, s);
  else launch<T, W, float, BACKWARD, DW>(p, blocks, s);
}

template <bool BACKWARD, bool DW>
static void launch_types(const Params& p, const meep2b_head_norm* a, unsigned blocks, cudaStream_t s) {
  if (a->dtype == MEEP2B_F32) launch_angles<float, float, BACKWARD, DW>(p, a->angle_dtype, blocks, s);
  else if (a->weight_f32) launch_angles<__nv_bfloat16, float, BACKWARD, DW>(p, a->angle_dtype, blocks, s);
  else launch_angles<__nv_bfloat16, __nv_bfloat16, BACKWARD, DW>(p, a->angle_dtype, blocks, s);
}

// How the heads of a token are taken: up to 8 in a row, fewer while that leaves groups without work, in runs of about
// one length. Returns the CTAs: one for every GROUPS items, or `most` of them in proportion to the queries' and the
// keys' heads.
static int64_t shape(Params& p, int lanes, int sms, int64_t most) {
  const int groups = THREADS / lanes;
  const int64_t heads = p.side[0].heads + p.side[1].heads;
  const int64_t wanted = static_cast<int64_t>(sms) * 3 * groups;  // groups the SMs hold at once
  int span = 8;
  while (span > 1 && p.tokens * heads / span < wanted) span /= 2;
  int64_t blocks[2];
  for (int i = 0; i < 2; ++i) {
    const int runs = (p.side[i].heads + span - 1) / span;
    p.side[i].span = (p.side[i].heads + runs - 1) / runs;
    const int64_t items = p.tokens * ((p.side[i].heads + p.side[i].span - 1) / p.side[i].span);
    blocks[i] = (items + groups - 1) / groups;
  }
  if (blocks[0] + blocks[1] > most) {
    blocks[0] = most * p.side[0].heads / heads;
    blocks[0] = blocks[0] < 1 ? 1 : (blocks[0] > most - 1 ? most - 1 : blocks[0]);
    blocks[1] = most - blocks[0];
  }
  p.q_blocks = static_cast<int>(blocks[0]);
  return blocks[0] + blocks[1];
}

static int lanes_of(int dim, int dtype) {
  const int slots = dim / (dtype == MEEP2B_BF16 ? 16 : 8);
  int g = 1;
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
               a->dq_out, a->dq_out_stride[0], a->dq_out_stride[1], a->dq_out_stride[2], 1};
  p.side[1] = {a->k, a->k_stride[0], a->k_stride[1], a->k_stride[2], a->kv_heads, a->k_weight, a->k_out,
               a->dk_out, a->dk_out_stride[0], a->dk_out_stride[1], a->dk_out_stride[2], 1};
  p.tokens = a->batch * a->length, p.length = static_cast<int>(a->length);
  p.dim = a->dim, p.half = a->half;
  p.cos = a->cos, p.sin = a->sin, p.ld_cos = a->ld_cos, p.ld_sin = a->ld_sin, p.angles = a->angles;
  p.positions = a->positions, p.eps = a->eps;
  const int64_t angle_vec = a->angle_dtype == MEEP2B_BF16 ? 8 : 4;
  p.angle_vec = aligned16(a->cos) && aligned16(a->sin) && a->ld_cos % angle_vec == 0 && a->ld_sin % angle_vec == 0;
  if (a->batch > INT32_MAX || p.tokens > (INT32_MAX >> 1) / (a->q_heads + a->kv_heads)) return MEEP2B_ERR_SHAPE;
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
  int sms = 0;
  MEEP2B_TRY(device_sms(&sms));
  const int64_t blocks = head_norm::shape(p, head_norm::lanes_of(p.dim, a->dtype), sms, INT32_MAX);
  head_norm::launch_types<false, false>(p, a, static_cast<unsigned>(blocks), s);
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
    int sms = 0;
    MEEP2B_TRY(device_sms(&sms));
    const int64_t most = !dw ? INT32_MAX : (2 * sms < head_norm::MAX_PARTIALS ? 2 * sms : head_norm::MAX_PARTIALS);
    blocks = static_cast<int>(head_norm::shape(p, head_norm::lanes_of(p.dim, a->dtype), sms, most));
    if (dw) head_norm::launch_types<true, true>(p, a, blocks, s);
    else head_norm::launch_types<true, false>(p, a, blocks, s);
    MEEP2B_TRY(launch_status());
  }
  if (dw) {
    const dim3 grid((p.dim + 31) / 32, 2);
    if (a->dtype == MEEP2B_BF16 && !a->weight_f32)
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
