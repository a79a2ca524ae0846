// The language-model loss of hidden states against a large vocabulary, without the logits: softmax cross entropy of
// l_tv = <h_t, W_v> against one target per row, its gradient of the hidden states and of the head.
//
// With the target's own logit as each row's reference, q_tv = exp(l_tv - l_t,y) and Z_t = 1 + sum_{v != y} q_tv:
//   loss_t  = log Z_t
//   dh_t    = g_t ((sum_{v != y} q_tv W_v) / Z_t - (1 - 1/Z_t) W_y)
//   dW_v    = sum_t g_t (q_tv / Z_t - [v = y_t]) h_t
// The reference is known before the products (one dot product per row), so that a tile of q is final when it leaves
// its accumulator: no running maximum, no rescaling of what was summed before, and dh needs one pass over the
// vocabulary (the logits' product and the product with W), not a second one for the normaliser. bf16 has float32's
// exponents, so q may lie anywhere within 2^+-96 of the target without losing bits. A 32-column piece of a row whose
// sum leaves that window is summed against its own maximum instead (its logarithm is what is kept, as a negative
// number), and the row tiles that hold such rows have their q and their dh product computed again with the row's
// log-sum as the reference, by launches that return at once where there are none.
//
// Only rows with a target are computed: they are copied to the front of a buffer first (the scan and the gather
// below), which also keeps what stands in ignored rows, infinities and NaN included, out of every sum.
//
// The products are one persistent tcgen05 kernel on CTA pairs (M = 256, N = 256, K = 64 a stage, both operands by
// TMA, two accumulators in tensor memory), or on single CTAs for few rows, with a mode for each epilogue:
//   kStats    the row sums of a 256-column tile (its two halves), nothing else
//   kProbs    the same, and q as bf16 into the vocabulary piece's buffer
//   kReprobs  q alone, for the row tiles to be computed again
//   kGrad     g (q / Z - [v = y]) as bf16 into the piece's buffer (the head's gradient, and dh beside it)
//   kAcc      dh's product: piece x W, float32, stored by the first piece and added (TMA reduction) by the others
//   kWeight   dW's product: piece^T x h, bf16
//
// Bound by the tensor pipe where hidden and rows are large (alone, at 2,048 tokens x 32,768: 84-88% active for the
// products over the logits, 82% for dW's and 77% for dh's, whose 64 units leave some of 74 pairs idle; 16,384 tokens x
// 131,072 at hidden 2048, loss and dh: 13.2-14.3 ms, 1.23-1.34 PFLOP/s at the power cap), by the epilogue's exponentials
// below hidden 512 or so (8,192 tokens x 50,000 at hidden 64: 174 us), and by reading the head for few rows (37 tokens x
// 131,072: 118 us for 537 MB, the L2 cache flushed before each call).
//
// q and g (p - [v = y]) are rounded to bf16 because both operands of the second products have one type, and the head's
// is bf16. dh hardly notices (2e-4 of its norm, against 1.66e-3 for its own rounding): its largest term by far, the
// target's, is kept apart in float32. dW's terms are all rounded before they are summed over the tokens: 1.9e-3 of its
// norm instead of 1.6e-3 (up to 2.4e-3 where few tokens share a target), and 1.5e-4 too long along itself (targets of little probability, whose 1 - p rounds to 1).
//
// The tensor cores cut every step's sum off toward zero. Over the 256 steps of a logit of 4,096 products that made the
// mean loss 1.1e-6 of itself too small; so beyond 2,048 products a logit's sum is taken from tensor memory every 2,048
// and joined in the epilogue's registers (DEEP), with ordinary float32 additions (the loss is then 5e-7 too small at 4,096
// products, 2.5e-7 at 2,048). dh's product sums a whole piece of the vocabulary in tensor memory: measured along itself
// it is 2e-6 (4,093 tokens x 131,072) and 1.4e-5 (trained head, 32,003 at hidden 4096) too short, far below its rounding.
#include <atomic>

#include "common.cuh"
#include "host.hpp"

namespace meep2b {
namespace vocab {

constexpr int TILE = 256;   // rows and columns of a unit (a CTA pair)
constexpr int BK = 64;
constexpr int OPERAND_BYTES = 128 * BK * 2;  // 128 rows or columns of an operand, one stage
constexpr int RING_BYTES = 192 * 1024;

// A unit is 256 rows on a CTA pair, each CTA with its 128 rows and half of the 256 columns; or (SOLO) 128 rows on one
// CTA with all 256 columns, which loads half as much again for each product. Single CTAs are taken where a pair's
// last 128 rows would be empty and are a good part of all (few_rows: an odd number of 128-row tiles, up to five; of all
// tokens, since the host does not know how many have a target). Loss alone at hidden 2048, the L2 cache flushed, us with
// single CTAs / with pairs, by the vocabulary:
//            37 tokens   300 tokens   513-640 tokens
//    16,384   38 / 34      49 / 45       60 / 54
//    32,768   46 / 50      66 / 69       87 / 85
//   131,072  118 / 120    176 / 197   255-290 / 270-320
// and with the gradient at 131,072: 223 / 236, 383 / 427, 565 / 575. Pairs win where the vocabulary is short of units.
inline bool few_rows(int64_t tokens) {
  const int64_t tiles = (tokens + 127) / 128;
  return tiles % 2 == 1 && tiles <= 5;
}
template <bool SOLO>
struct Shape {
  static constexpr int ROWS = SOLO ? 128 : 256;
  static constexpr int B_BYTES = SOLO ? 2 * OPERAND_BYTES : OPERAND_BYTES;
  static constexpr int STAGE_BYTES = OPERAND_BYTES + B_BYTES;
  static constexpr int STAGES = RING_BYTES / STAGE_BYTES;  // 4 or 6
};
constexpr int EPI_WARP0 = 4;
constexpr int STG_BYTES = 32768;  // the epilogue warps' tiles on their way out
constexpr int OFF_STG = RING_BYTES;
constexpr int OFF_BAR = OFF_STG + STG_BYTES;
constexpr int NUM_BARS = 2 * 6 + 5;
constexpr int OFF_TMEM = OFF_BAR + NUM_BARS * 8;
constexpr int SMEM_BYTES = OFF_TMEM + 16 + 1024;
constexpr uint32_t TMEM_COLS = 512;
constexpr int DEEP_BLOCKS = 32;  // k-blocks (2,048 products) that a logit is summed over in tensor memory
constexpr int GROUP = 8;  // row tiles that share a column tile before the next column tile is taken
static_assert(SMEM_BYTES <= 232448, "shared memory plan exceeds 227 KB");

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kWindow = 7.9228162514264338e28f;  // 2^96

enum Mode { kStats, kProbs, kReprobs, kGrad, kAcc, kWeight };

// Epilogue warps, in groups of 8 (four quarters of the rows, which a warp may read of tensor memory, by two halves of
// the columns). Over the logits every element costs an exponential, and one group, each of whose warps waits for the
// unit, loads, computes and stores in turn, left the exponentials' unit idle more than half of the time: two groups
// take every other unit each (5,200 cycles a unit with one, the exponentials alone are 2,048, the product's time at
// hidden 256). The other modes have time enough with one, and DEEP needs its registers.
template <int MODE, bool DEEP>
struct Epi {
  static constexpr int GROUPS = MODE == kAcc || MODE == kWeight || DEEP ? 1 : 2;
  static constexpr int THREADS = 32 * (EPI_WARP0 + 8 * GROUPS);
};
constexpr int SLOTS = 2;  // row sums kept for a column tile, one for every half

// ints of `state`
enum { kLive = 0, kRedo = 1, kDone = 2, kParts = 3, kStateInts = 8 };  // (kParts: planes that kAcc wrote)

struct Rows {  // per live row, float32
  float* ref;    // the reference of q, in units of log 2 (after a recomputation: the row's log-sum)
  float* logit;  // the target's logit
  float* lse;    // log2 of the sum of 2^(logit / log 2) over the vocabulary
  float* scale;  // what q is multiplied by to be the probability: 2^(ref - lse)
  float* miss;   // 1 - the target's probability
};

struct Params {
  int32_t* state;
  const int32_t* flags;    // row tiles to compute again
  const int32_t* target;   // per live row (-1 past the last)
  const int32_t* source;   // the live row's token
  Rows rows;
  float* part;             // (SLOTS * column tiles of the vocabulary) x rows_pad: the row sums
  int64_t rows_pad;
  const float* upstream;   // one value, or one per token
  int per_token, mean;     // how g follows from it
  int vocab, hidden;
  int v0, piece_tiles;     // the piece: its first column and its column tiles
  int k_total;             // depth of the product, in elements (kAcc: the piece's columns; kWeight: live rows)
  int planes, depth;       // kAcc: the most parts the depth may be split into, each summed in a plane of its own, and
                           // a whole piece's depth, which decides how many are used
  int first;               // kAcc: the first piece (stores)
  bool solo;               // see Shape
};

// Into how many parts the depth k of a product of `units` tiles is split on `pairs` CTA pairs: the number whose last
// round of units leaves the least idle, against the plane that each part costs (written, and read at the end: 8 bytes a
// value at 6.5 TB/s, where a round of 74 units of depth k takes k 6.5 ns).
__host__ __device__ inline int depth_parts(int units, int pairs, int most, int k) {
  int best = 1;
  float best_cost = 1e30f;
  for (int s = 1; s <= most; ++s) {
    const float cost = static_cast<float>((units * s + pairs - 1) / pairs) / s + 12.5f * units * s / k;
    if (cost < best_cost) best_cost = cost, best = s;
  }
  return best;
}

struct Units {
  int mt, nt, parts, total, kblocks;

  __device__ void decode(int u, int& m, int& n, int& part) const {
    const int per = mt * nt;
    part = u / per;
    int r = u - part * per;
    const int group = r / (GROUP * nt);
    const int rows = min(GROUP, mt - group * GROUP);
    r -= group * GROUP * nt;
    n = r / rows;
    m = group * GROUP + (r - n * rows);
  }
  __device__ int k_begin(int part) const { return static_cast<int>(static_cast<int64_t>(kblocks) * part / parts); }
};

template <int MODE, bool SOLO>
__device__ __forceinline__ Units units_of(const Params& p, int pairs) {
  Units w;
  const int live = p.state[kLive];
  const int row_tiles = (live + Shape<SOLO>::ROWS - 1) / Shape<SOLO>::ROWS;
  if (MODE == kWeight) {
    w.mt = p.piece_tiles, w.nt = (p.hidden + TILE - 1) / TILE, w.parts = 1;
    w.kblocks = (live + BK - 1) / BK;
  } else if (MODE == kAcc) {
    w.mt = row_tiles, w.nt = (p.hidden + TILE - 1) / TILE;
    w.parts = depth_parts(w.mt * w.nt, pairs, p.planes, p.depth);
    w.kblocks = (p.k_total + BK - 1) / BK;
  } else {
    w.mt = row_tiles, w.nt = p.piece_tiles, w.parts = 1;
    w.kblocks = (p.hidden + BK - 1) / BK;
  }
  w.total = w.mt * w.nt * w.parts;
  return w;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The kernels of a call are launched as programmatic dependents of one another: the next one's CTAs may take their
// places (and set up barriers and tensor memory) while this one runs out, and wait here, before they touch any memory,
// until all of this one's work is done and visible.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void tma_add_2d(const CUtensorMap* map, uint32_t src, int32_t c0, int32_t c1) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(c0), "r"(c1)
               : "memory");
}

// The row `lane` of a tile of 32 rows x 32 bf16 (64-byte swizzle), or of 32 rows x 32 float32 (128-byte swizzle).
__device__ __forceinline__ void stage_bf16(uint32_t tile, int lane, const uint32_t (&w)[16]) {
  const uint32_t r = tile + static_cast<uint32_t>(lane) * 64u;
  const uint32_t sw = (static_cast<uint32_t>(lane) >> 1) & 3u;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(r + ((static_cast<uint32_t>(j) ^ sw) << 4)),
                 "r"(w[4 * j]), "r"(w[4 * j + 1]), "r"(w[4 * j + 2]), "r"(w[4 * j + 3])
                 : "memory");
}

__device__ __forceinline__ void stage_f32(uint32_t tile, int lane, const float (&v)[32]) {
  const uint32_t r = tile + static_cast<uint32_t>(lane) * 128u;
  const uint32_t sw = static_cast<uint32_t>(lane) & 7u;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(r + ((static_cast<uint32_t>(j) ^ sw) << 4)),
                 "r"(__float_as_uint(v[4 * j])), "r"(__float_as_uint(v[4 * j + 1])),
                 "r"(__float_as_uint(v[4 * j + 2])), "r"(__float_as_uint(v[4 * j + 3]))
                 : "memory");
}

// g of a live row: the loss's upstream gradient over the reduction.
__device__ __forceinline__ float row_upstream(const float* upstream, int per_token, int mean, int token, int live) {
  const float g = upstream[per_token ? token : 0];
  return mean ? g / static_cast<float>(max(live, 1)) : g;
}

// The gradient of the target's own logit, g (p - 1).
__device__ __forceinline__ float target_gradient(float miss, float g) { return __fmul_rn(-miss, g); }

// 32 columns of the warp's rows of an accumulator, on their way (load) and there (the registers named, so that they are
// read only afterwards).
__device__ __forceinline__ void tmem_load32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// What an epilogue thread knows of its row of a unit before the unit's sums arrive.
struct RowIn {
  float ref = 0.f, g = 0.f, miss = 0.f;
  int target = -1;
};

template <int MODE>
__device__ __forceinline__ RowIn row_in(const Params& p, int row, int live) {
  RowIn r;
  if (MODE == kAcc || MODE == kWeight || row >= live) return r;
  r.target = p.target[row];
  r.ref = MODE == kGrad ? p.rows.lse[row] : p.rows.ref[row];
  if (MODE == kGrad) {
    r.g = row_upstream(p.upstream, p.per_token, p.mean, p.source[row], live);
    r.miss = p.rows.miss[row];
  }
  return r;
}

// The sums over the vocabulary of one row of a unit: what lies within the window, and log2 of what lies above it,
// against the reference.
struct RowSums {
  float sum = 0.f, far = -INFINITY;
};

// 32 columns of a unit from column `col` of the product, a lane a row (the first is row0): to q, to g (q - [v = y]), or
// as they are, into shared memory and from there out by TMA; and the row's sums.
template <int MODE, int TILES>
__device__ __forceinline__ void columns32(const Params& p, const CUtensorMap* out, const RowIn& in, RowSums& sums,
                                          float (&v)[32], int c, int col, int part, bool empty, int row0, int live,
                                          int lane, uint32_t stg) {
  constexpr bool LOGITS = MODE == kStats || MODE == kProbs || MODE == kReprobs || MODE == kGrad;
  const int row = row0 + lane;  // of the live rows (kWeight: of the piece's columns)
  const int vcol = p.v0 + col;  // LOGITS: of the vocabulary
  const bool own = in.target >= vcol && in.target < vcol + 32;
  if (LOGITS) {
    if (vcol + 32 > p.vocab || own) {  // past the end, or the target's own
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (vcol + j >= p.vocab || vcol + j == in.target) v[j] = -INFINITY;
    }
    float e[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) e[j] = exp2_fast(fmaf(v[j], kLog2e, -in.ref));
    if (MODE == kStats || MODE == kProbs) {
      float s[4] = {e[0], e[1], e[2], e[3]};
#pragma unroll
      for (int j = 4; j < 32; ++j) s[j & 3] += e[j];
      const float all = (s[0] + s[1]) + (s[2] + s[3]);
      if (all < kWindow || row >= live) {
        sums.sum += all;
      } else {  // against the columns' own maximum (a NaN stays one)
        float top = v[0];
#pragma unroll
        for (int j = 1; j < 32; ++j) top = fmaxf(top, v[j]);
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) t += exp2_fast((v[j] - top) * kLog2e);
        const float here = fmaf(top, kLog2e, -in.ref) + log2f(t);
        const float hi = fmaxf(sums.far, here), lo = fminf(sums.far, here);
        sums.far = here != here ? here : (sums.far != sums.far ? sums.far : hi + log2f(1.0f + exp2f(lo - hi)));
      }
    }
    if (MODE == kStats) return;
    if (MODE == kGrad) {  // (rows past the last live one are zero: the head's gradient sums over them)
#pragma unroll
      for (int j = 0; j < 32; ++j) e[j] = row < live ? e[j] * in.g : 0.f;
      if (own) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (vcol + j == in.target) e[j] = target_gradient(in.miss, in.g);
      }
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = e[j];
  } else if (empty) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = 0.f;
  }
  if (MODE == kAcc) {
    if (lane == 0) bulk_wait_read<0>();  // the tile's last store has read it
    __syncwarp();
    stage_f32(stg, lane, v);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0 && col < p.hidden) {
      const int at = part * static_cast<int>(p.rows_pad) + row0;
      if (p.first)
        tma_store_2d(out, stg, col, at);
      else
        tma_add_2d(out, stg, col, at);
      bulk_commit();
    }
  } else {
    uint32_t w[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
    // two tiles a warp of one group, one of two
    const uint32_t tile = stg + (TILES == 2 ? (c & 1) * 2048u : 0u);
    if (lane == 0) bulk_wait_read<TILES - 1>();
    __syncwarp();
    stage_bf16(tile, lane, w);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (LOGITS || (col < p.hidden && p.v0 + row0 < p.vocab)) tma_store_2d(out, tile, col, LOGITS ? row0 : p.v0 + row0);
      bulk_commit();
    }
  }
}

// A row's sums over half a unit's columns, kept for the join: what lies above the window as minus its log2 against the
// reference (over 90, so never near zero).
__device__ __forceinline__ void keep_sums(const Params& p, const RowSums& s, int n, int half, int row) {
  float kept = s.sum;
  if (s.far != -INFINITY) kept = s.far != s.far ? s.far : -(s.far + log2f(1.0f + s.sum * exp2f(-s.far)));
  p.part[static_cast<int64_t>(SLOTS * (p.v0 / TILE + n) + half) * p.rows_pad + row] = kept;
}

template <int MODE, bool REDO, bool DEEP, bool SOLO>
__global__ void __launch_bounds__((Epi<MODE, DEEP>::THREADS), 1)
    vocab_product(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap ta32,
                  const __grid_constant__ CUtensorMap tb, const __grid_constant__ CUtensorMap tout, const Params p) {
  constexpr bool A_MN = MODE == kWeight;
  constexpr bool B_MN = MODE == kWeight || MODE == kAcc;
  using E = Epi<MODE, DEEP>;
  using S = Shape<SOLO>;
  constexpr int STAGES = S::STAGES;
  if (REDO) {
    let_next_start();
    wait_for_last();
    if (p.state[kRedo] == 0) return;
  }
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = SOLO ? 0 : cluster_rank();
  const int pair_id = SOLO ? static_cast<int>(blockIdx.x) : static_cast<int>(cluster_id_x());
  const int pairs = SOLO ? static_cast<int>(gridDim.x) : static_cast<int>(num_clusters_x());
  auto sync_unit = [&]() {  // the CTAs that share a unit
    if (SOLO) __syncthreads();
    else cluster_sync();
  };

  const uint32_t bar0 = sbase + OFF_BAR;
  auto bar_full = [&](int s) { return bar0 + 8u * s; };
  auto bar_empty = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto bar_tfull = [&](int b) { return bar0 + 8u * (2 * STAGES + b); };
  auto bar_tempty = [&](int b) { return bar0 + 8u * (2 * STAGES + 2 + b); };
  const uint32_t bar_drain = bar0 + 8u * (2 * STAGES + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + OFF_TMEM);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_tfull(b), 1);
      mbar_init(bar_tempty(b), SOLO ? 8 : 16);  // eight epilogue warps of each CTA
    }
    mbar_init(bar_drain, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    if (SOLO) {
      tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
      tmem_relinquish();
    } else {
      tmem_alloc_pair(smem_u32(tmem_slot), TMEM_COLS);
      tmem_relinquish_pair();
    }
  }
  tc_fence_before();
  sync_unit();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (!REDO) {
    let_next_start();
    wait_for_last();
  }
  const Units w = units_of<MODE, SOLO>(p, pairs);
  const int live = p.state[kLive];
  if (MODE == kAcc && blockIdx.x == 0 && threadIdx.x == 0) p.state[kParts] = w.parts;

  // DEEP: the epilogue's warpgroups take 208 registers a thread, the first one keeps 88: 384 x 168 in all, what the
  // kernel is launched with (checked there)
  if (warp < EPI_WARP0) {
    if (DEEP) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0 && lane == 0) {  // ------------------------------------------------------- TMA producer (each CTA)
      tma_prefetch_desc(&ta);
      tma_prefetch_desc(&tb);
      int stage = 0;
      uint32_t phase = 0;
      uint32_t last_parity[STAGES];
      bool issued[STAGES];
      for (int s = 0; s < STAGES; ++s) issued[s] = false, last_parity[s] = 0;
      bool ok = true;
      for (int u = pair_id; u < w.total && ok; u += pairs) {
        int m, n, part;
        w.decode(u, m, n, part);
        if (REDO && p.flags[m * S::ROWS / TILE] == 0) continue;
        const int a0 = m * S::ROWS + 128 * static_cast<int>(rank), b0 = n * TILE + 128 * static_cast<int>(rank);
        const int k1 = w.k_begin(part + 1);
        // of a row tile that is not full only the runs of 32 rows that hold live ones are loaded; what stands in the
        // others' places meets nothing but its own rows of the accumulator
        const int have = A_MN ? TILE : live - m * S::ROWS;
        const int runs0 = min(4, max(0, (have + 31) / 32)), runs1 = SOLO ? 0 : min(4, max(0, (have - 128 + 31) / 32));
        const int runs = rank == 0 ? runs0 : runs1;
        const uint32_t bytes = 2 * OPERAND_BYTES + static_cast<uint32_t>(runs0 + runs1) * (OPERAND_BYTES / 4);
        for (int kb = w.k_begin(part); kb < k1; ++kb) {
          if (!mbar_wait(bar_empty(stage), phase ^ 1)) { ok = false; break; }
          const uint32_t fb = SOLO ? bar_full(stage) : map_to_rank(bar_full(stage), 0);
          const uint32_t a_dst = sbase + stage * S::STAGE_BYTES, b_dst = a_dst + OPERAND_BYTES;
          const int k0 = kb * BK;
          auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
            if (SOLO) tma_load_2d(dst, map, fb, x, y);
            else tma_load_2d_pair(dst, map, fb, x, y);
          };
          if (rank == 0) mbar_arrive_expect_tx(bar_full(stage), bytes);
          if (A_MN) {
            load(a_dst, &ta, a0, k0);
            load(a_dst + 8192, &ta, a0 + 64, k0);
          } else if (runs == 4) {
            load(a_dst, &ta, k0, a0);
          } else {
            for (int i = 0; i < runs; ++i) load(a_dst + i * (OPERAND_BYTES / 4), &ta32, k0, a0 + 32 * i);
          }
#pragma unroll
          for (int i = 0; i < S::B_BYTES / OPERAND_BYTES; ++i) {
            const uint32_t dst = b_dst + i * OPERAND_BYTES;
            const int at = b0 + 128 * i;
            if (B_MN) {
              const int kr = MODE == kAcc ? p.v0 + k0 : k0;
              load(dst, &tb, at, kr);
              load(dst + 8192, &tb, at + 64, kr);
            } else {
              load(dst, &tb, k0, p.v0 + at);
            }
          }
          issued[stage] = true;
          last_parity[stage] = phase;
          if (++stage == STAGES) stage = 0, phase ^= 1;
        }
      }
      if (!ok && rank == 0)
        for (int s = 0; s < STAGES; ++s)
          if (issued[s]) mbar_wait_drain(bar_full(s), last_parity[s]);
    } else if (warp == 1 && lane == 0 && rank == 0) {  // ------------------------------------ MMA issuer (the leader)
      constexpr uint32_t IDESC = idesc_bf16(S::ROWS, TILE, A_MN, B_MN);
      auto mma = [&](uint32_t d, uint64_t a, uint64_t b, uint32_t add) {
        if (SOLO) mma_bf16(d, a, b, IDESC, add);
        else mma_bf16_pair(d, a, b, IDESC, add);
      };
      auto commit = [&](uint32_t bar) {
        if (SOLO) mma_commit(bar);
        else mma_commit_pair(bar);
      };
      const uint64_t a_desc0 = A_MN ? smem_desc(sbase, 8192, 1024, 2) : smem_desc(sbase, 16, 1024, 2);
      const uint64_t b_desc0 = B_MN ? smem_desc(sbase + OPERAND_BYTES, 8192, 1024, 2)
                                    : smem_desc(sbase + OPERAND_BYTES, 16, 1024, 2);
      constexpr uint32_t A_KK = A_MN ? 2048 / 16 : 32 / 16, B_KK = B_MN ? 2048 / 16 : 32 / 16;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      int it = 0;
      for (int u = pair_id; u < w.total && ok; u += pairs) {
        int m, n, part;
        w.decode(u, m, n, part);
        if (REDO && p.flags[m * S::ROWS / TILE] == 0) continue;
        const int passes = DEEP ? (w.kblocks + DEEP_BLOCKS - 1) / DEEP_BLOCKS : 1;
        for (int pass = 0; pass < passes && ok; ++pass) {
          const int ab = it & 1;
          const uint32_t freed = ((it >> 1) & 1) ^ 1;
          if (!(SOLO ? mbar_wait(bar_tempty(ab), freed) : mbar_wait_cluster(bar_tempty(ab), freed))) { ok = false; break; }
          tc_fence_after();
          const uint32_t d = tmem_base + ab * TILE;
          const int k0 = DEEP ? w.kblocks * pass / passes : w.k_begin(part);
          const int k1 = DEEP ? w.kblocks * (pass + 1) / passes : w.k_begin(part + 1);
          for (int kb = k0; kb < k1; ++kb) {
            if (!mbar_wait(bar_full(stage), phase)) { ok = false; break; }
            tc_fence_after();
            const uint64_t a_st = a_desc0 + static_cast<uint32_t>(stage) * (S::STAGE_BYTES / 16);
            const uint64_t b_st = b_desc0 + static_cast<uint32_t>(stage) * (S::STAGE_BYTES / 16);
            mma(d, a_st, b_st, kb != k0);
#pragma unroll
            for (int kk = 1; kk < BK / 16; ++kk) mma(d, a_st + A_KK * kk, b_st + B_KK * kk, 1);
            commit(bar_empty(stage));
            if (++stage == STAGES) stage = 0, phase ^= 1;
          }
          if (!ok) break;
          commit(bar_tfull(ab));
          ++it;
        }
      }
      if (!ok) {
        commit(bar_drain);
        mbar_wait_drain(bar_drain, 0);
      }
    }
  } else {  // ------------------------------------------------------------------------------- epilogue (each CTA)
    if (DEEP) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int q = warp & 3, half = ((warp - EPI_WARP0) >> 2) & 1, group = (warp - EPI_WARP0) >> 3;
    const uint32_t stg = sbase + OFF_STG + static_cast<uint32_t>(warp - EPI_WARP0) * (STG_BYTES / (8 * E::GROUPS));
    auto release = [&](uint32_t bar) {  // the warp is done with an accumulator: one arrival for its 32 lanes
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (SOLO) mbar_arrive(bar);
        else mbar_arrive_remote(bar, 0);
      }
    };
    // the next unit, and what is known of this thread's row in it, are looked up a unit ahead
    const int row_in_tile = 128 * static_cast<int>(rank) + 32 * q;
    // (computing again, units without a flag are passed over, and the groups alternate over what remains)
    const int first = REDO ? pair_id : pair_id + group * pairs, step = REDO ? pairs : E::GROUPS * pairs;
    int it = REDO ? 0 : group, m = 0, n = 0, part = 0;
    RowIn next;
    if (first < w.total) {
      w.decode(first, m, n, part);
      next = row_in<MODE>(p, m * S::ROWS + row_in_tile + lane, live);
    }
    for (int u = first; u < w.total; u += step) {
      const int row0 = m * S::ROWS + row_in_tile, c_first = n * TILE + half * 128, tile_n = n, tile_m = m, my_part = part;
      const RowIn in = next;
      if (u + step < w.total) {
        w.decode(u + step, m, n, part);
        next = row_in<MODE>(p, m * S::ROWS + row_in_tile + lane, live);
      }
      if (REDO) {
        if (p.flags[tile_m * S::ROWS / TILE] == 0) continue;
        if (E::GROUPS == 2 && (it & 1) != group) {
          ++it;
          continue;
        }
      }
      // a warp without live rows has nothing to write (kGrad: but zeros, to the end of the last k-block of 64 rows)
      const bool idle = MODE == kWeight ? false : MODE == kGrad ? row0 >= (live + BK - 1) / BK * BK : row0 >= live;
      const bool empty = w.k_begin(my_part) == w.k_begin(my_part + 1);
      const int passes = DEEP ? (w.kblocks + DEEP_BLOCKS - 1) / DEEP_BLOCKS : 1;
      float held[DEEP ? 4 : 1][32];
#pragma unroll
      for (int c = 0; c < (DEEP ? 128 : 0); ++c) held[c / 32][c % 32] = 0.f;
      RowSums sums;
      bool ok = true;
      for (int pass = 0; pass < passes; ++pass, it += REDO ? 1 : E::GROUPS) {
        const int ab = it & 1;
        ok = mbar_wait(bar_tfull(ab), (it >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t acc = tmem_base + ab * TILE + half * 128 + (static_cast<uint32_t>(32 * q) << 16);
        if (idle) {
          release(bar_tempty(ab));
          continue;
        }
        if (DEEP) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            float v[16];
            tmem_ld16(acc + 16 * c, v);
#pragma unroll
            for (int j = 0; j < 16; ++j) held[DEEP ? c / 2 : 0][16 * (c % 2) + j] += v[j];
          }
          release(bar_tempty(ab));
        } else {
          // the next 32 columns are on their way while these are worked on, where registers allow (one group)
          constexpr int BUFFERS = E::GROUPS == 1 ? 2 : 1;
          uint32_t r[BUFFERS][32];
          tmem_load32(acc, r[0]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (BUFFERS == 1 && c > 0) tmem_load32(acc + 32 * c, r[0]);
            tmem_loaded(r[c % BUFFERS]);
            if (BUFFERS == 2 && c < 3) tmem_load32(acc + 32 * (c + 1), r[(c + 1) % BUFFERS]);
            if (c == 3) release(bar_tempty(ab));  // the whole accumulator has been read
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[c % BUFFERS][j]);
            columns32<MODE, E::GROUPS == 1 ? 2 : 1>(p, &tout, in, sums, v, c, c_first + 32 * c, my_part, empty, row0, live,
                                                   lane, stg);
          }
        }
      }
      if (!ok) break;
      if (idle) continue;
      if (DEEP) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          columns32<MODE, E::GROUPS == 1 ? 2 : 1>(p, &tout, in, sums, held[DEEP ? c : 0], c, c_first + 32 * c, my_part,
                                                  empty, row0, live, lane, stg);
      }
      if (MODE == kStats || MODE == kProbs) keep_sums(p, sums, tile_n, half, row0 + lane);
    }
    if (lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  sync_unit();
  if (warp == 1) {
    tc_fence_after();
    if (SOLO) tmem_dealloc(tmem_base, TMEM_COLS);
    else tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------------------------------- rows

// How many of a CTA's threads' earlier threads' tokens have a target, and the CTA's total (in *total): each thread
// gives its own number. words: one int a warp.
template <int WARPS>
__device__ __forceinline__ int scan_before(int mine, int* words, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += v;
  }
  if (lane == 31) words[warp] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const int v = words[w];
    if (w < warp) before += v;
    all += v;
  }
  *total = all;
  return before + incl - mine;
}

// The tokens with a target, in order: source (live row -> token), slot (token -> live row, or -1), their number; the
// losses of the ignored tokens (zero) and the state words of this call. One CTA, each thread a run of tokens: the
// ids are 8 bytes a token and the block's scan is one, so 16,384 tokens take a few microseconds.
__global__ void __launch_bounds__(1024) vocab_scan(const int64_t* __restrict__ targets, int64_t tokens,
                                                  int64_t ignore, int32_t* __restrict__ source,
                                                  int32_t* __restrict__ slot, int32_t* __restrict__ state,
                                                  int32_t* __restrict__ flags, int row_tiles,
                                                  float* __restrict__ token_loss) {
  __shared__ int words[32];
  let_next_start();
  const int64_t per = (tokens + 1023) / 1024;
  const int64_t t0 = min(tokens, per * threadIdx.x), t1 = min(tokens, t0 + per);
  int mine = 0;
  for (int64_t t = t0; t < t1; ++t) mine += targets[t] != ignore;
  int total;
  int at = scan_before<32>(mine, words, &total);
  for (int64_t t = t0; t < t1; ++t) {
    const bool is = targets[t] != ignore;
    slot[t] = is ? at : -1;
    if (is) source[at++] = static_cast<int32_t>(t);
    if (!is && token_loss != nullptr) token_loss[t] = 0.f;
  }
  for (int i = threadIdx.x; i < row_tiles; i += 1024) flags[i] = 0;
  if (threadIdx.x < kStateInts) state[threadIdx.x] = threadIdx.x == kLive ? total : 0;
}

// Each live row copied to the front of `compact`, its target and its target's logit (a float32 dot product): a warp
// per row. The rows from the last live one to the end of its 256-row tile are zero (the head's gradient sums over
// them). A target outside the vocabulary makes the row's reference, and with it its loss and its gradient, NaN.
// SCAN: without vocab_scan, whose work each CTA then does for itself, the first one writing it down: a launch less,
// which counts where there are few tokens (up to kScanned: 32 KB of ids a CTA, from L2).
constexpr int kScanned = 4096;
template <bool SCAN>
__global__ void __launch_bounds__(256) vocab_gather(const __nv_bfloat16* __restrict__ hidden, int64_t ld_hidden,
                                                   const __nv_bfloat16* __restrict__ weight, int64_t ld_weight,
                                                   const int64_t* __restrict__ targets, int tokens, int64_t ignore,
                                                   int vocab, int width, int32_t* __restrict__ state,
                                                   int32_t* __restrict__ flags, int row_tiles,
                                                   int32_t* __restrict__ source, int32_t* __restrict__ slot,
                                                   float* __restrict__ token_loss,
                                                   __nv_bfloat16* __restrict__ compact, int32_t* __restrict__ target,
                                                   Rows rows) {
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
  int live, from = 0;
  let_next_start();
  wait_for_last();
  if (SCAN) {
    __shared__ int words[8], mine_rows[8];
    const int per = (tokens + 255) / 256;
    const int t0 = min(tokens, per * static_cast<int>(threadIdx.x)), t1 = min(tokens, t0 + per);
    int mine = 0;
    uint32_t has = 0;  // per <= 16
    for (int t = t0; t < t1; ++t) {
      const bool is = targets[t] != ignore;
      has |= static_cast<uint32_t>(is) << (t - t0);
      mine += is;
    }
    int at = scan_before<8>(mine, words, &live);
    const bool writes = blockIdx.x == 0;
    for (int t = t0; t < t1; ++t) {
      const bool is = (has >> (t - t0)) & 1u;
      if (is && at / 8 == static_cast<int>(blockIdx.x)) mine_rows[at % 8] = t;
      if (writes) {
        slot[t] = is ? at : -1;
        if (is) source[at] = t;
        if (!is && token_loss != nullptr) token_loss[t] = 0.f;
      }
      at += is;
    }
    if (writes) {
      if (threadIdx.x < row_tiles) flags[threadIdx.x] = 0;
      if (threadIdx.x < kStateInts) state[threadIdx.x] = threadIdx.x == kLive ? live : 0;
    }
    __syncthreads();
    if (row < live) from = mine_rows[threadIdx.x >> 5];
  } else {
    live = state[kLive];
    if (row < live) from = source[row];
  }
  if (row >= (live + TILE - 1) / TILE * TILE) return;
  uint4* to = reinterpret_cast<uint4*>(compact + static_cast<int64_t>(row) * width);
  const int vecs = width / 8;
  if (row >= live) {
    for (int i = lane; i < vecs; i += 32) to[i] = make_uint4(0, 0, 0, 0);
    if (lane == 0) {
      target[row] = -1;
      rows.ref[row] = 0.f, rows.logit[row] = 0.f, rows.lse[row] = 0.f, rows.scale[row] = 0.f, rows.miss[row] = 0.f;
    }
    return;
  }
  const int64_t t = from;
  const int64_t y = targets[t];
  const bool inside = y >= 0 && y < vocab;
  const uint4* h = reinterpret_cast<const uint4*>(hidden + t * ld_hidden);
  const uint4* wr = reinterpret_cast<const uint4*>(weight + (inside ? y : 0) * ld_weight);
  float dot = 0.f;
#pragma unroll 4
  for (int i = lane; i < vecs; i += 32) {
    const uint4 a = h[i], b = wr[i];
    to[i] = a;
    dot = fmaf(bf16_lo(a.x), bf16_lo(b.x), dot), dot = fmaf(bf16_hi(a.x), bf16_hi(b.x), dot);
    dot = fmaf(bf16_lo(a.y), bf16_lo(b.y), dot), dot = fmaf(bf16_hi(a.y), bf16_hi(b.y), dot);
    dot = fmaf(bf16_lo(a.z), bf16_lo(b.z), dot), dot = fmaf(bf16_hi(a.z), bf16_hi(b.z), dot);
    dot = fmaf(bf16_lo(a.w), bf16_lo(b.w), dot), dot = fmaf(bf16_hi(a.w), bf16_hi(b.w), dot);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
  if (lane == 0) {
    if (!inside) dot = __int_as_float(0x7fc00000);
    target[row] = inside ? static_cast<int32_t>(y) : -1;
    rows.logit[row] = dot;
    rows.ref[row] = dot * kLog2e;
  }
}

// Each live row's sums over the vocabulary's tiles joined in order, its loss, and the mean or the sum over the rows
// (by the last CTA to finish, in order). 32 rows a CTA, 32 threads a row.
__global__ void __launch_bounds__(1024) vocab_join(const float* __restrict__ part, int slots, int64_t rows_pad,
                                                  int32_t* __restrict__ state, int32_t* __restrict__ flags,
                                                  const int32_t* __restrict__ source, Rows rows,
                                                  float* __restrict__ token_loss, float* __restrict__ row_loss,
                                                  float* __restrict__ loss, int mean) {
  __shared__ float sums[32][33], fars[32][33];
  __shared__ double reduce[32];
  __shared__ bool last;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  let_next_start();
  wait_for_last();
  const int live = state[kLive];
  {
    const int row = blockIdx.x * 32 + x;
    float sum = 0.f, far = -INFINITY;
    for (int s0 = y; row < live && s0 < slots; s0 += 32 * 16) {
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int s = s0 + 32 * i;
        v[i] = s < slots ? part[static_cast<int64_t>(s) * rows_pad + row] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (v[i] < 0.f) {
          const float hi = fmaxf(far, -v[i]), lo = fminf(far, -v[i]);
          far = hi + log2f(1.0f + exp2f(lo - hi));
        } else {
          sum += v[i];  // (a NaN stays one)
        }
      }
    }
    sums[x][y] = sum, fars[x][y] = far;
  }
  __syncthreads();
  const int row = blockIdx.x * 32 + y;  // from here a warp a row
  if (row < live) {
    float sum = sums[y][x], far = fars[y][x];
    const bool any = __any_sync(0xffffffffu, far != -INFINITY);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, off);
      if (any) {
        const float f = __shfl_xor_sync(0xffffffffu, far, off);
        const float hi = fmaxf(far, f), lo = fminf(far, f);
        if (hi != -INFINITY) far = hi + log2f(1.0f + exp2f(lo - hi));
      }
    }
    if (x == 0) {
      // the reference was rounded to a multiple of log 2: what the rounding took is put back
      const float ref = rows.ref[row], logit = rows.logit[row];
      const float off = fmaf(logit, kLog2e, -ref);
      float value;
      if (!any) {
        sum *= exp2f(-off);
        const float z = 1.0f + sum;
        value = log1pf(sum);
        rows.lse[row] = fmaf(logit, kLog2e, log2f(z));
        rows.scale[row] = exp2f(-off) / z;
        rows.miss[row] = sum / z;
      } else {
        const float more = far + log2f(1.0f + (1.0f + sum) * exp2f(-far)) - off;
        value = more * kLn2;
        const float lse = fmaf(logit, kLog2e, more);
        rows.lse[row] = lse;
        rows.ref[row] = lse;
        rows.scale[row] = 1.0f;
        rows.miss[row] = 1.0f - exp2f(-more);
        flags[row / TILE] = 1;
        state[kRedo] = 1;
      }
      if (token_loss != nullptr) token_loss[source[row]] = value;
      else row_loss[row] = value;
    }
  }
  if (token_loss != nullptr) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(&state[kDone], 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double total = 0.0;
  for (int i = threadIdx.x; i < live; i += 1024) total += static_cast<double>(__ldcg(row_loss + i));
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
  if (x == 0) reduce[y] = total;
  __syncthreads();
  if (y == 0) {
    total = reduce[x];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
    if (x == 0) *loss = static_cast<float>(mean ? total / max(live, 1) : total);
  }
}

// dh of every token from its row's planes, zero for ignored tokens. From the forward pass's q: g (scale sum_planes -
// miss W_y). From the product over g (p - [v = y]) in bf16 (`rounded`): the sum, and what the rounding of the target's
// value took times W_y, which is the largest rounding of a row by far. A warp per 256 columns of a token, so that few
// tokens fill the GPU too.
__global__ void __launch_bounds__(256) vocab_finish(const float* __restrict__ acc, int64_t rows_pad, int width, int64_t tokens,
                                                   const int32_t* __restrict__ state, const int32_t* __restrict__ slot,
                                                   const int32_t* __restrict__ target, Rows rows,
                                                   const __nv_bfloat16* __restrict__ weight, int64_t ld_weight,
                                                   const float* __restrict__ upstream, int per_token, int mean,
                                                   bool rounded, __nv_bfloat16* __restrict__ d_hidden) {
  wait_for_last();
  const int lane = threadIdx.x & 31;
  const int chunks = (width + 255) / 256;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int64_t t = unit / chunks;
  const int i = static_cast<int>(unit - t * chunks) * 32 + lane;  // of the row's pieces of 8 columns
  if (t >= tokens || 8 * i >= width) return;
  uint4* to = reinterpret_cast<uint4*>(d_hidden + t * width);
  const int row = slot[t];
  if (row < 0) {
    to[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  const int live = state[kLive];
  const int parts = state[kParts];
  const float g = row_upstream(upstream, per_token, mean, static_cast<int>(t), live);
  const float own = target_gradient(rows.miss[row], g);
  // scale and g apart: a row whose Z is near 2^96 times a small g is below float32's normal numbers
  const float scale = rounded ? 1.f : rows.scale[row], a = rounded ? 1.f : g;
  const float b = rounded ? own - bf16_round(own) : own;
  const int y = target[row];
  const uint4* wr = reinterpret_cast<const uint4*>(weight + static_cast<int64_t>(y < 0 ? 0 : y) * ld_weight);
  const uint4 k = wr[i];
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < parts; s0 += 4) {
    float4 u[4], w[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      u[s] = w[s] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s0 + s < parts) {
        const float4* from = reinterpret_cast<const float4*>(acc + ((s0 + s) * rows_pad + row) * width) + 2 * i;
        u[s] = __ldcs(from), w[s] = __ldcs(from + 1);
      }
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      v[0] += u[s].x, v[1] += u[s].y, v[2] += u[s].z, v[3] += u[s].w;
      v[4] += w[s].x, v[5] += w[s].y, v[6] += w[s].z, v[7] += w[s].w;
    }
  }
  v[0] = a * (scale * v[0]) + b * bf16_lo(k.x), v[1] = a * (scale * v[1]) + b * bf16_hi(k.x);
  v[2] = a * (scale * v[2]) + b * bf16_lo(k.y), v[3] = a * (scale * v[3]) + b * bf16_hi(k.y);
  v[4] = a * (scale * v[4]) + b * bf16_lo(k.z), v[5] = a * (scale * v[5]) + b * bf16_hi(k.z);
  v[6] = a * (scale * v[6]) + b * bf16_lo(k.w), v[7] = a * (scale * v[7]) + b * bf16_hi(k.w);
  to[i] = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                     pack_bf16x2(v[6], v[7]));
}

// `after`: as a programmatic dependent of the launch before it on the stream (one of this call's, which all wait).
template <typename... P>
static int launch_in(unsigned cluster, bool after, void (*kern)(P...), unsigned grid, unsigned threads, size_t smem,
                     cudaStream_t s, P... args) {
  cudaLaunchAttribute attr[2] = {};
  int n = 0;
  if (after) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster, attr[n].val.clusterDim.y = 1, attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid), config.blockDim = dim3(threads), config.dynamicSmemBytes = smem, config.stream = s;
  config.attrs = attr, config.numAttrs = n;
  if (cudaLaunchKernelEx(&config, kern, args...) != cudaSuccess) return cudaGetLastError(), MEEP2B_ERR_LAUNCH;
  return MEEP2B_OK;
}

template <typename... P>
static int launch_chained(bool after, void (*kern)(P...), unsigned grid, unsigned threads, size_t smem, cudaStream_t s,
                          P... args) {
  return launch_in<P...>(1, after, kern, grid, threads, smem, s, args...);
}

template <int MODE, bool REDO, bool DEEP, bool SOLO>
static int launch_product(const CUtensorMap& a, const CUtensorMap& a32, const CUtensorMap& b, const CUtensorMap& out,
                          const Params& p, int pairs, cudaStream_t s, bool after) {
  auto kern = vocab_product<MODE, REDO, DEEP, SOLO>;
  // per device (a function's attributes are set on the current one); threads may call at once, each then configures
  static std::atomic<uint64_t> configured{0};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return cudaGetLastError(), MEEP2B_ERR_LAUNCH;
  if (device >= 64 || !((configured.load(std::memory_order_acquire) >> device) & 1)) {
    // DEEP's register split adds up to 168 a thread at launch: with fewer the increase would never be granted
    cudaFuncAttributes attr;
    if (cudaFuncGetAttributes(&attr, kern) != cudaSuccess || (DEEP && attr.numRegs != 168) ||
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess) {
      cudaGetLastError();
      return MEEP2B_ERR_LAUNCH;
    }
    if (device < 64) configured.fetch_or(uint64_t(1) << device, std::memory_order_release);
  }
  return launch_in(SOLO ? 1 : 2, after, kern, 2u * pairs, Epi<MODE, DEEP>::THREADS, SMEM_BYTES, s, a, a32, b, out, p);
}

template <int MODE, bool REDO>
static int launch(const CUtensorMap& a, const CUtensorMap& a32, const CUtensorMap& b, const CUtensorMap& out,
                  const Params& p, int pairs, cudaStream_t s, bool after = true) {
  constexpr bool LOGITS = MODE != kAcc && MODE != kWeight;
  const bool deep = p.hidden > DEEP_BLOCKS * BK;
  if constexpr (MODE != kWeight) {
    if (p.solo) {
      if constexpr (LOGITS) {
        if (deep) return launch_product<MODE, REDO, true, true>(a, a32, b, out, p, pairs, s, after);
      }
      return launch_product<MODE, REDO, false, true>(a, a32, b, out, p, pairs, s, after);
    }
  }
  if constexpr (LOGITS) {
    if (deep) return launch_product<MODE, REDO, true, false>(a, a32, b, out, p, pairs, s, after);
  }
  return launch_product<MODE, REDO, false, false>(a, a32, b, out, p, pairs, s, after);
}

static int map_bf16(CUtensorMap* map, const void* base, int64_t inner, int64_t rows, int64_t ld, uint32_t box_inner,
                    uint32_t box_rows, CUtensorMapSwizzle swizzle) {
  const uint64_t dims[2] = {static_cast<uint64_t>(inner), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(ld) * 2};
  const uint32_t box[2] = {box_inner, box_rows};
  return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, swizzle);
}

}  // namespace vocab
}  // namespace meep2b

using namespace meep2b;

namespace {

constexpr int64_t kPieceBytes = int64_t(1) << 30;  // a piece's buffer; see meep2b_linear_ce_plan
constexpr int64_t kPlaneBytes = int64_t(1) << 29;
constexpr int kMostPlanes = 16;

int pairs_of_device(int* pairs) {
  int sms = 0;
  MEEP2B_TRY(device_sms(&sms));
  *pairs = sms / 2 > 0 ? sms / 2 : 1;
  return MEEP2B_OK;
}

int check_linear_ce(const meep2b_linear_ce* a, bool forward) {
  if (a == nullptr || a->tokens < 0 || a->hidden_size < 1 || a->vocab < 1) return MEEP2B_ERR_SHAPE;
  if (a->tokens > (1 << 24) || a->vocab > (1 << 24) || a->hidden_size > (1 << 20)) return MEEP2B_ERR_SHAPE;
  if ((a->tokens / 256 + 1) * (a->vocab / 256 + 1) > (1 << 28)) return MEEP2B_ERR_SHAPE;  // units are counted in 32 bits
  if (a->hidden_size % 8 || a->ld_weight % 8 || a->ld_weight < a->hidden_size || !aligned16(a->weight))
    return MEEP2B_ERR_ALIGN;
  if (forward && (a->ld_hidden % 8 || !aligned16(a->hidden))) return MEEP2B_ERR_ALIGN;
  if (a->reduction < 0 || a->reduction > 2) return MEEP2B_ERR_UNSUPPORTED;
  if (a->rows_pad != (a->tokens + 255) / 256 * 256 || a->piece_cols % vocab::TILE || a->planes < 0)
    return MEEP2B_ERR_SHAPE;
  return MEEP2B_OK;
}

vocab::Rows rows_of(const meep2b_linear_ce* a) {
  float* f = a->row_values;
  const int64_t n = a->rows_pad;
  return vocab::Rows{f, f + n, f + 2 * n, f + 3 * n, f + 4 * n};
}

vocab::Params params_of(const meep2b_linear_ce* a) {
  vocab::Params p = {};
  p.state = a->state, p.flags = a->flags, p.target = a->target, p.source = a->source, p.rows = rows_of(a);
  p.part = a->part, p.rows_pad = a->rows_pad, p.upstream = a->upstream;
  p.per_token = a->reduction == MEEP2B_REDUCE_NONE, p.mean = a->reduction == MEEP2B_REDUCE_MEAN;
  p.vocab = static_cast<int>(a->vocab), p.hidden = static_cast<int>(a->hidden_size), p.planes = a->planes;
  p.solo = vocab::few_rows(a->tokens);
  p.depth = static_cast<int>(a->piece_cols > 0 && a->piece_cols < a->vocab ? a->piece_cols : a->vocab);
  return p;
}

struct CeMaps {
  CUtensorMap rows, rows32, rows_mn, head, head_mn, piece, piece32, piece_mn, piece_out, acc, d_weight;
};

int maps_of(const meep2b_linear_ce* a, CeMaps* m, bool acc, bool d_weight) {
  using vocab::map_bf16;
  const int64_t H = a->hidden_size;
  MEEP2B_TRY(map_bf16(&m->rows, a->compact, H, a->rows_pad, H, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B));
  MEEP2B_TRY(map_bf16(&m->rows32, a->compact, H, a->rows_pad, H, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B));
  MEEP2B_TRY(map_bf16(&m->head, a->weight, H, a->vocab, a->ld_weight, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B));
  if (a->piece != nullptr) {
    MEEP2B_TRY(map_bf16(&m->piece, a->piece, a->piece_cols, a->rows_pad, a->piece_cols, 64, 128,
                        CU_TENSOR_MAP_SWIZZLE_128B));
    MEEP2B_TRY(map_bf16(&m->piece32, a->piece, a->piece_cols, a->rows_pad, a->piece_cols, 64, 32,
                        CU_TENSOR_MAP_SWIZZLE_128B));
    MEEP2B_TRY(map_bf16(&m->piece_out, a->piece, a->piece_cols, a->rows_pad, a->piece_cols, 32, 32,
                        CU_TENSOR_MAP_SWIZZLE_64B));
  } else {
    m->piece_out = m->rows;  // not used
  }
  if (acc) {
    MEEP2B_TRY(map_bf16(&m->head_mn, a->weight, H, a->vocab, a->ld_weight, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B));
    const uint64_t dims[2] = {static_cast<uint64_t>(H), static_cast<uint64_t>(a->planes * a->rows_pad)};
    const uint64_t strides[1] = {static_cast<uint64_t>(H) * 4};
    const uint32_t box[2] = {32, 32};
    MEEP2B_TRY(encode_tiled(&m->acc, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, a->acc, dims, strides, box,
                            CU_TENSOR_MAP_SWIZZLE_128B));
  }
  if (d_weight) {
    MEEP2B_TRY(map_bf16(&m->rows_mn, a->compact, H, a->rows_pad, H, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B));
    MEEP2B_TRY(map_bf16(&m->piece_mn, a->piece, a->piece_cols, a->rows_pad, a->piece_cols, 64, 64,
                        CU_TENSOR_MAP_SWIZZLE_128B));
    MEEP2B_TRY(map_bf16(&m->d_weight, a->d_weight, H, a->vocab, H, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B));
  }
  return MEEP2B_OK;
}

// The vocabulary's pieces: first column, column tiles and depth of each.
template <typename F>
int each_piece(const meep2b_linear_ce* a, vocab::Params p, F f) {
  const int64_t cols = a->piece_cols > 0 ? a->piece_cols : (a->vocab + 255) / 256 * 256;
  for (int64_t v0 = 0; v0 < a->vocab; v0 += cols) {
    const int64_t width = a->vocab - v0 < cols ? a->vocab - v0 : cols;
    p.v0 = static_cast<int>(v0);
    p.piece_tiles = static_cast<int>((width + vocab::TILE - 1) / vocab::TILE);
    p.k_total = static_cast<int>(width);
    p.first = v0 == 0;
    MEEP2B_TRY(f(p));
  }
  return MEEP2B_OK;
}

}  // namespace

extern "C" {

int meep2b_linear_ce_plan(int64_t tokens, int64_t hidden_size, int64_t vocab, int64_t* rows_pad, int64_t* piece_cols,
                          int32_t* planes) {
  if (tokens < 0 || hidden_size < 1 || vocab < 1 || tokens > (1 << 24) || vocab > (1 << 24) || hidden_size > (1 << 20))
    return MEEP2B_ERR_SHAPE;
  *rows_pad = (tokens + 255) / 256 * 256;
  const int64_t rows = *rows_pad > 0 ? *rows_pad : 256;
  const int64_t tiles = (vocab + 255) / 256;
  int64_t most = kPieceBytes / (rows * 2 * 256);
  most = most < 1 ? 1 : most;
  const int64_t pieces = (tiles + most - 1) / most;
  *piece_cols = (tiles + pieces - 1) / pieces * 256;
  int64_t p = kPlaneBytes / (rows * hidden_size * 4);
  p = p < 1 ? 1 : (p > kMostPlanes ? kMostPlanes : p);
  *planes = static_cast<int32_t>(p);
  return MEEP2B_OK;
}

int meep2b_linear_ce_forward(const meep2b_linear_ce* a, void* stream) {
  MEEP2B_TRY(check_linear_ce(a, true));
  if (a->loss == nullptr || a->state == nullptr || a->part == nullptr) return MEEP2B_ERR_SHAPE;
  cudaStream_t s = as_stream(stream);
  MEEP2B_TRY(bind_stream_device(s));
  const bool per_token = a->reduction == MEEP2B_REDUCE_NONE;
  const bool grad = a->acc != nullptr;
  if (grad && (a->piece == nullptr || a->planes < 1)) return MEEP2B_ERR_SHAPE;
  const vocab::Rows rows = rows_of(a);
  const int row_tiles = static_cast<int>(a->rows_pad / vocab::TILE);
  const bool small = a->tokens > 0 && a->tokens <= vocab::kScanned;
  if (!small)
    MEEP2B_TRY(vocab::launch_chained(false, vocab::vocab_scan, 1, 1024, 0, s, a->targets, a->tokens, a->ignore_index,
                                     a->source, a->slot, a->state, a->flags, row_tiles,
                                     per_token ? a->loss : static_cast<float*>(nullptr)));
  const int slots = vocab::SLOTS * static_cast<int>((a->vocab + vocab::TILE - 1) / vocab::TILE);
  int pairs = 0;
  MEEP2B_TRY(pairs_of_device(&pairs));
  CeMaps m;
  if (a->tokens > 0) {
    MEEP2B_TRY(maps_of(a, &m, grad, false));
    MEEP2B_TRY(vocab::launch_chained(
        !small, small ? vocab::vocab_gather<true> : vocab::vocab_gather<false>, static_cast<unsigned>(a->rows_pad / 8),
        256, 0, s, static_cast<const __nv_bfloat16*>(a->hidden), a->ld_hidden,
        static_cast<const __nv_bfloat16*>(a->weight), a->ld_weight, a->targets, static_cast<int>(a->tokens),
        a->ignore_index, static_cast<int>(a->vocab), static_cast<int>(a->hidden_size), a->state, a->flags, row_tiles,
        a->source, a->slot, per_token ? a->loss : static_cast<float*>(nullptr),
        static_cast<__nv_bfloat16*>(a->compact), a->target, rows));
    MEEP2B_TRY(each_piece(a, params_of(a), [&](const vocab::Params& p) -> int {
      if (!grad) return vocab::launch<vocab::kStats, false>(m.rows, m.rows32, m.head, m.piece_out, p, pairs, s);
      MEEP2B_TRY((vocab::launch<vocab::kProbs, false>(m.rows, m.rows32, m.head, m.piece_out, p, pairs, s)));
      return vocab::launch<vocab::kAcc, false>(m.piece, m.piece32, m.head_mn, m.acc, p, pairs, s);
    }));
  }
  const unsigned join = static_cast<unsigned>(a->tokens > 0 ? (a->tokens + 31) / 32 : 1);
  MEEP2B_TRY(vocab::launch_chained(
      true, vocab::vocab_join, join, 1024, 0, s, static_cast<const float*>(a->part), slots, a->rows_pad, a->state,
      a->flags, static_cast<const int32_t*>(a->source), rows, per_token ? a->loss : static_cast<float*>(nullptr),
      a->row_loss, a->loss, static_cast<int>(a->reduction == MEEP2B_REDUCE_MEAN)));
  if (grad && a->tokens > 0) {
    MEEP2B_TRY(each_piece(a, params_of(a), [&](const vocab::Params& p) -> int {
      MEEP2B_TRY((vocab::launch<vocab::kReprobs, true>(m.rows, m.rows32, m.head, m.piece_out, p, pairs, s)));
      return vocab::launch<vocab::kAcc, true>(m.piece, m.piece32, m.head_mn, m.acc, p, pairs, s);
    }));
  }
  return MEEP2B_OK;
}

int meep2b_linear_ce_backward(const meep2b_linear_ce* a, void* stream) {
  MEEP2B_TRY(check_linear_ce(a, false));
  if (a->upstream == nullptr || (a->d_hidden == nullptr && a->d_weight == nullptr)) return MEEP2B_ERR_SHAPE;
  if (a->d_hidden != nullptr && (a->acc == nullptr || a->planes < 1)) return MEEP2B_ERR_SHAPE;
  if ((a->d_hidden && !aligned16(a->d_hidden)) || (a->d_weight && !aligned16(a->d_weight))) return MEEP2B_ERR_ALIGN;
  cudaStream_t s = as_stream(stream);
  MEEP2B_TRY(bind_stream_device(s));
  int pairs = 0;
  MEEP2B_TRY(pairs_of_device(&pairs));
  const bool recompute = a->compact != nullptr;  // else the forward pass left dh's planes
  if (recompute ? a->piece == nullptr || a->piece_cols < vocab::TILE : a->d_weight != nullptr) return MEEP2B_ERR_SHAPE;
  if (a->d_weight != nullptr && a->tokens == 0) {
    const cudaError_t e = cudaMemsetAsync(a->d_weight, 0, static_cast<size_t>(a->vocab) * a->hidden_size * 2, s);
    return e == cudaSuccess ? MEEP2B_OK : (cudaGetLastError(), MEEP2B_ERR_LAUNCH);
  }
  bool after = false;
  if (recompute && a->tokens > 0) {
    CeMaps m;
    MEEP2B_TRY(maps_of(a, &m, a->d_hidden != nullptr, a->d_weight != nullptr));
    MEEP2B_TRY(each_piece(a, params_of(a), [&](const vocab::Params& p) -> int {
      MEEP2B_TRY((vocab::launch<vocab::kGrad, false>(m.rows, m.rows32, m.head, m.piece_out, p, pairs, s, after)));
      after = true;
      if (a->d_hidden != nullptr)
        MEEP2B_TRY((vocab::launch<vocab::kAcc, false>(m.piece, m.piece32, m.head_mn, m.acc, p, pairs, s)));
      if (a->d_weight == nullptr) return MEEP2B_OK;
      return vocab::launch<vocab::kWeight, false>(m.piece_mn, m.piece_mn, m.rows_mn, m.d_weight, p, pairs, s);
    }));
  }
  if (a->d_hidden != nullptr && a->tokens > 0) {
    const vocab::Params p = params_of(a);
    const int64_t warps = a->tokens * ((a->hidden_size + 255) / 256);
    MEEP2B_TRY(vocab::launch_chained(
        after, vocab::vocab_finish, static_cast<unsigned>((warps + 7) / 8), 256, 0, s, static_cast<const float*>(a->acc),
        a->rows_pad, static_cast<int>(a->hidden_size), a->tokens, static_cast<const int32_t*>(a->state),
        static_cast<const int32_t*>(a->slot), static_cast<const int32_t*>(a->target), p.rows,
        static_cast<const __nv_bfloat16*>(a->weight), a->ld_weight, a->upstream, p.per_token, p.mean, recompute,
        static_cast<__nv_bfloat16*>(a->d_hidden)));
  }
  return MEEP2B_OK;
}

}  // extern "C"
