// The head's losses for training: the vocabulary projection, its softmax, a loss against labels or against a teacher's
// highest logits, and the gradients of the rows and of the weight, without fp32 logits in memory: a piece of the rows at a time
// holds one 16-bit value per logit, 1 GiB at most.
//
//   z_n = W x_n / T            q_n = softmax(z_n)
//   label t:                   loss_n = -log q_nt                                           (T = 1, one entry, p = 1)
//   teacher entries (t_k, l_k): p = softmax(l / T) over the entries that are there (l > -inf),
//                              loss_n = T^2 sum_k p_k (log p_k - log q_n,t_k)
//   g_nv = row_n (q_nv - sum over k with t_k = v of p_k)          dx = f g W,  dW = f g^T x
// row_n f is the upstream gradient of a row's loss; f is what all rows share: T, the upstream gradient of the scalar loss, 1 /
// rows for a mean, and of row losses the largest upstream gradient, which row_n is a share of (1 where there are none).
//
// A row that is nearly certain of its label has a loss and a label gradient that are differences of nearly equal numbers in
// these forms (lse - z, q - 1).  They are taken from what is small instead: the label t (of a teacher: its highest entry)
// stays out of the sums, O = log of the sum of exp z_v over the other v, d = O - z_t, and
//   -log q_t = log(1 + e^d),   1 - q_t = e^d / (1 + e^d),   log q_k = z_k - z_t - log(1 + e^d),
//   g_t = row (sum of the p_k of other columns - (1 - q_t)),
// so that both keep their relative precision down to the smallest losses.
//
// Passes over a piece of the rows (all of them while 2 rows x vocabulary bytes fit kPieceBytes):
//   plan     numbers the rows that have a label; rows without one take no part in any product (compact_kernel copies the
//            others together, or does nothing where every row takes part), so what they hold, NaN included, reaches nothing
//   stats    z on the tensor cores; the epilogue leaves, per 128 columns, each row's maximum and sum of exponentials, and for
//            gradients the exponentials themselves in fp16, relative to that maximum (error 2^-11 of each, where a bf16
//            value would add 2^-8 to the one rounding that g needs as a tensor-core operand)
//   finish   per row: O from the tiles' statistics, the labels' logits as fp32 dot products of their own, the loss, and
//            the exponentials times their tile's factor in place, now g in bf16; the labels' entries from fp32
//   products dx and dW, in one launch; f is applied to their fp32 sums.  Inside g it would be rounded with it, and the many
//            labels with 1 - q_t near 1 would all be off by the rounding of 1 / rows (or of a common row_n), up to 2^-8 with
//            one sign: dx and dW of 777 x 50277 x 1544 by 2.6e-3 in the norm so, 1.9e-3 as it is (rounding the exact
//            gradients gives 1.7e-3)
// so a step costs three products of 2 rows x vocabulary x channels, not the four of recomputing z for the backward pass,
// and the weight is read twice.  The price is that gradients are made with the loss, before the upstream gradient is known:
// scale_kernel applies it afterwards (it leaves at once where the gradient is one).
//
// The reference fuses the same cross entropy at csrc/sm90/head/l2wrap_ce/pretrain_bf16_forward.cu:282-286 around library
// products and kept logits; it has no distillation.

#include <cfloat>

#include "head_loss.cuh"

namespace frwkv {
namespace head {
namespace {

using bf16 = __nv_bfloat16;
using IO = Io16<bf16>;

constexpr long long kPieceBytes = 1ll << 30;   // exponentials of one piece
constexpr long long kStatsBytes = 1ll << 28;   // statistics of one piece
constexpr int kMaxTop = 512;
// What truncation takes from the logits of random rows, per channel of an accumulator (2.8e-7 of the logit at 256 channels, 5.2e-7
// at 512, 1.0e-6 at 1024): the scale that turns logits into exponents gives it back.  It lies between what exact sums lose,
// nothing, and what rows lose whose large products come first, 1.1e-8 per channel, so it lowers the largest error and puts it
// at 1.06e-6 of a logit where nothing was lost; an accumulator takes kPartChannels at most, whatever the width.  The mean loss
// of 2048 x 65536 x 1024 to 4096 is off by 1e-7 of itself, without it by 6e-7.
constexpr double kTruncation = 1.03e-9;
constexpr int kFinishThreads = 256;
// Copied by the plan, a launch less, while a warp has two rows at most: steps of 1 x 50277 x 1544 155 us so and 164 with the
// launch, of 40 x 32000 x 768 61 and 62, but of 64 x 50277 x 1544 164 and 161.
constexpr int kFewRows = 64;

// Rows of labels that a warp each finishes rather than a CTA.  A step of 256 channels, by warps / by CTAs in us:
//   vocabulary  300: 29 / 33 at 70 rows, 37 / 43 at 1000, 43 / 66 at 4000      (40 rows, which CTAs share: 26 / 30)
//              4090: 35 / 37 at 70 rows, 49 / 49 at 1000, 77 / 95 at 4000      (40 rows: 33 / 35)
//              6000: 61 / 55 at 1100 rows, 74 / 74 at 2000, 93 / 108 at 4000
//              8190: 72 / 64 at 1100 rows, 86 / 84 at 2000, 109 / 122 at 4000  (40 rows: 37 / 35)
//             12000: 84 / 72 at 1100 rows, 104 / 98 at 2000, 156 / 164 at 4000
// A teacher's row is a CTA's always: its entries are what it waits for, and eight warps gather them at once.
constexpr bool short_rows(long long ldg, int rows) {
  return rows > kFewRows && (ldg <= 4096 || (ldg <= 8192 && rows >= 2048));
}

struct Labels {
  const void* index;        // [rows][top] int32 or int64
  bool wide;                // int64
  const float* teacher;     // [rows][top] logits, or null: one label per row
  long long ignore_index;   // labels only
  int top;
  float inv_temperature, temperature;
  __device__ long long at(long long i) const {
    return wide ? static_cast<const long long*>(index)[i] : (long long)static_cast<const int*>(index)[i];
  }
};

// ---- plan: which rows take part --------------------------------------------------------------------------------------
// highest[row] = the first of the teacher's highest entries for this row, -1 where it has none; a warp per row
__global__ __launch_bounds__(256) void teacher_rows_kernel(Labels labels, int* __restrict__ highest, int rows) {
  chain_begin();
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= rows) return;
  float most = -INFINITY;
  int which = -1;
  for (int k = lane; k < labels.top; k += 32) {
    const float t = labels.teacher[(long long)row * labels.top + k];
    if (!(t == -INFINITY) && (which < 0 || t > most)) {  // a NaN is an entry too: its row becomes NaN
      most = t;
      which = k;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t = __shfl_xor_sync(0xffffffffu, most, o);
    const int w = __shfl_xor_sync(0xffffffffu, which, o);
    if (w >= 0 && (which < 0 || t > most || (t == most && w < which))) {
      most = t;
      which = w;
    }
  }
  if (lane == 0) highest[row] = which;
}

// Copies the rows that take part together; the others get a zero loss and a zero gradient.  The rows behind the last, up
// to the next multiple of 64, become zeros: they meet zeros of g in a block of the contraction over rows.  Where every row
// takes part there is nothing to do, unless rows that are not whole 128-byte lines apart are copied to lines of their own
// (`always`): TMA reads such rows more slowly (a step of 544 x 50277 x 1544 311 us on x as it is, 300 on the copy).
struct CompactArgs {
  const uint4* x;
  const int* position;
  uint4* x_compact;
  uint4* grad_x;
  float* row_losses;
  int rows, pieces, pitch;  // in 16-byte pieces
  bool always;
};
__device__ __forceinline__ void compact_row(const CompactArgs& a, int row, int used, int lane) {
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  const int at = a.position[row];
  const bool tail = row >= used && row < ((used + 63) & ~63);
  for (int p = lane; p < a.pieces; p += 32) {
    if (at >= 0) {
      a.x_compact[(long long)at * a.pitch + p] = __ldg(a.x + (long long)row * a.pieces + p);
    } else if (a.grad_x != nullptr) {
      a.grad_x[(long long)row * a.pieces + p] = zero;
    }
    if (tail) a.x_compact[(long long)row * a.pitch + p] = zero;
  }
  if (lane == 0 && at < 0) a.row_losses[row] = 0.f;
}
__global__ __launch_bounds__(256) void compact_kernel(CompactArgs a, const int* __restrict__ count) {
  chain_begin();
  const int used = *count, row = blockIdx.x * 8 + (threadIdx.x >> 5);
  if ((used == a.rows && !a.always) || row >= a.rows) return;
  compact_row(a, row, used, threadIdx.x & 31);
}

// What the plan leaves on the device for the other kernels.
struct Plan {
  int count;     // rows that take part
  int arrived;   // CTAs that have written their losses
  int splits_x, splits_w;
  float row_scale;  // the largest upstream gradient of a row loss by its magnitude, 1 where none is or all are 0
};
struct SplitSizes {
  int channels, vocab, most_x, most_w, pairs;
  int workers_x;     // pairs, or CTAs that work alone, for grad_x
  long long room_x;  // rows of fp32 parts of grad_x
  bool fixed;        // several pieces: what the host has chosen, whatever the count
};

// the cheapest number of parts, by one warp
__device__ int choose_splits(int most, float rows, float columns, float k, float pairs, int lane) {
  const float tiles = ceilf(rows / kTile) * ceilf(columns / kTile), blocks = ceilf(k / 64.f);
  float best = INFINITY;
  int which = 1;
  for (int s = lane + 1; s <= most; s += 32) {
    const float cost = s == 1 || blocks >= s * kLeastBlocks ? split_cost(s, tiles, blocks, rows * columns, pairs) : INFINITY;
    if (cost < best) {
      best = cost;
      which = s;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float c = __shfl_xor_sync(0xffffffffu, best, o);
    const int w = __shfl_xor_sync(0xffffffffu, which, o);
    if (c < best || (c == best && w < which)) {
      best = c;
      which = w;
    }
  }
  return which;
}

// One CTA numbers the rows in order (8192 in 7 us, most of it two round trips): position[row] = compact number or -1, row_map
// its inverse, main_column the label's column (the teacher's highest entry's) by compact number, -1 where it lies outside the
// vocabulary.
__global__ __launch_bounds__(1024) void plan_kernel(Labels labels, const int* __restrict__ highest, int* position,
                                                    int* __restrict__ row_map, int* __restrict__ main_column,
                                                    Plan* __restrict__ plan, SplitSizes sizes, CompactArgs compact,
                                                    const float* __restrict__ row_grads, int* __restrict__ error_flag,
                                                    int rows) {
  chain_begin();
  constexpr int kEach = 8;  // consecutive rows of a thread; what is in use comes in row order through shared memory
  __shared__ int warp_sums[32];
  __shared__ __align__(8) unsigned char flags[1024 * kEach];
  __shared__ int list[1024 * kEach];  // the rows in use of this round, so that they leave in whole lines
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int done = 0;
  float row_scale = 0.f;
  for (int begin = 0; begin < rows; begin += 1024 * kEach) {
    long long label[kEach];  // requested together: past the end the last row again
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int row = min(begin + i * 1024 + (int)threadIdx.x, rows - 1);
      if (labels.teacher != nullptr) {
        label[i] = __ldg(highest + row);
      } else if (labels.wide) {
        label[i] = __ldg(static_cast<const long long*>(labels.index) + row);
      } else {
        label[i] = __ldg(static_cast<const int*>(labels.index) + row);
      }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int at = i * 1024 + threadIdx.x;
      flags[at] = begin + at < rows && label[i] != (labels.teacher != nullptr ? -1 : labels.ignore_index);
    }
    __syncthreads();
    const uint2 mine8 = *reinterpret_cast<const uint2*>(flags + threadIdx.x * kEach);
    const int mine = __popc(mine8.x) + __popc(mine8.y);
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    const int others = warp_sums[lane];
    int at = __reduce_add_sync(0xffffffffu, lane < warp ? others : 0) + upto - mine;
    const int used_here = __reduce_add_sync(0xffffffffu, others);
    const int first = begin + threadIdx.x * kEach;
    int where[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const bool used = ((i < 4 ? mine8.x : mine8.y) >> (8 * (i & 3))) & 1u;
      where[i] = used ? done + at : -1;
      if (used) list[at++] = first + i;
    }
    if (first + kEach <= rows) {
      reinterpret_cast<int4*>(position + first)[0] = make_int4(where[0], where[1], where[2], where[3]);
      reinterpret_cast<int4*>(position + first)[1] = make_int4(where[4], where[5], where[6], where[7]);
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (first + i < rows) position[first + i] = where[i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < used_here; i += 1024) {
      const int row = list[i];
      const long long v = labels.teacher != nullptr ? labels.at((long long)row * labels.top + __ldg(highest + row)) : labels.at(row);
      row_map[done + i] = row;
      if (row_grads != nullptr) {
        const float g = fabsf(__ldg(row_grads + row));
        if (g <= FLT_MAX) row_scale = fmaxf(row_scale, g);  // one that is not finite stays its row's own affair
      }
      main_column[done + i] = v >= 0 && v < sizes.vocab ? (int)v : -1;
    }
    done += used_here;
    __syncthreads();
  }
  if (row_grads != nullptr) {
    // magnitudes order as their bits do
    const unsigned most = __reduce_max_sync(0xffffffffu, __float_as_uint(row_scale));
    if (lane == 0) warp_sums[warp] = (int)most;
    __syncthreads();
    row_scale = __uint_as_float(__reduce_max_sync(0xffffffffu, (unsigned)warp_sums[lane]));
  }
  if (warp == 0) {
    int most_x = sizes.most_x, splits_x = most_x, splits_w = sizes.most_w;
    if (!sizes.fixed && done > 0 && done < rows) {
      // fewer rows than the host has chosen for, which leave room for more parts
      if (most_x > 1) most_x = (int)min((long long)kMaxSplits, sizes.room_x / done);
      splits_x = choose_splits(most_x, (float)done, (float)sizes.channels, (float)sizes.vocab, (float)sizes.workers_x, lane);
      splits_w = choose_splits(sizes.most_w, (float)sizes.vocab, (float)sizes.channels, (float)done, (float)sizes.pairs, lane);
    }
    if (lane == 0) {
      *plan = Plan{done, 0, splits_x, splits_w, row_scale > 0.f ? row_scale : 1.f};
      *error_flag = 0;
    }
  }
  // a few rows are copied here, by a warp each, rather than by a launch of their own
  if (rows <= kFewRows && (done < rows || compact.always))
    for (int row = warp; row < rows; row += 32) compact_row(compact, row, done, lane);
}

// ---- finish: statistics to losses and logit gradients ------------------------------------------------------------------
__device__ __forceinline__ float block_reduce(float v, float* scratch, bool maximum) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = maximum ? fmaxf(v, w) : v + w;
  }
  __syncthreads();  // scratch may still be read from the reduction before
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
#pragma unroll
  for (int i = 1; i < kFinishThreads / 32; ++i) v = maximum ? fmaxf(v, scratch[i]) : v + scratch[i];
  return v;
}

// z of one label, a warp's fp32 dot product
__device__ __forceinline__ float label_logit(const bf16* x_row, const bf16* w_row, int pieces, int lane) {
  float dot = 0.f;
#pragma unroll 4
  for (int p = lane; p < pieces; p += 32) {
    const uint4 ux = __ldg(reinterpret_cast<const uint4*>(x_row) + p), uw = __ldg(reinterpret_cast<const uint4*>(w_row) + p);
    const uint32_t xs[4] = {ux.x, ux.y, ux.z, ux.w}, ws[4] = {uw.x, uw.y, uw.z, uw.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 fx = IO::unpack(xs[e]), fw = IO::unpack(ws[e]);
      dot = fmaf(fx.x, fw.x, dot);
      dot = fmaf(fx.y, fw.y, dot);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
  return dot;
}

constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;

// What a row's loss and gradients are made of, from the others' maximum and sum (in units of log2) and the label's z.
struct RowSums {
  float excess;    // log(1 + e^d) = -log q_t
  float missing;   // 1 - q_t
  float lse2;      // log2 of the sum over the whole vocabulary
};
__device__ __forceinline__ RowSums row_sums(float high, float sum, float z) {
  // z log2(e) in two parts, so that d does not lose to the size of either term
  const float z2 = z * kLog2e, z2_rest = fmaf(z, kLog2e, -z2) + z * 1.9259629911e-8f;
  const float others = log2f(sum);  // -inf where there are none
  const float d = ((high - z2) - z2_rest + others) * kLn2;
  RowSums r;
  const float e = expf(-fabsf(d)), small = log1pf(e);
  r.excess = d > 0.f ? d + small : small;
  r.missing = d > 0.f ? 1.f / (1.f + e) : e / (1.f + e);
  r.lse2 = z2 + r.excess * kLog2e;
  if (d != d) r.excess = r.missing = r.lse2 = d;
  return r;
}

struct FinishArgs {
  Rows rows;
  Labels labels;
  const bf16* x;
  const bf16* weight;
  const int* highest;        // of a teacher's entries, by row of x
  const float2* stats;       // [row of the piece][tiles]
  int vocab, channels;
  uint4* g;            // exponentials in, logit gradients out, ldg values per row; null without gradients
  long long ldg;
  bool mean;
  const float* row_grads;    // upstream gradients of the row losses, or null
  const float* row_scale;    // what they are divided by in g
  float* row_losses;
  float* loss;               // the last CTA of the last piece to arrive adds the row losses, in row order; or null
  int* arrived;
  int ctas;                  // of all pieces, the first part of a row each
};

// Called by every CTA that writes row losses.  The sum does not depend on who arrives last.  It runs in 64 bits and is rounded
// once, with the division of a mean: in fp32 the 65536 additions of a thread (2^24 rows), all rounded the same way where the
// row losses are alike, lose up to 1e-3 of it.
__device__ __forceinline__ void arrive_and_sum(const FinishArgs& a, int count) {
  if (a.loss == nullptr || blockIdx.y > 0) return;
  __shared__ bool last;
  __shared__ double sums[kFinishThreads / 32];
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(a.arrived, 1) == a.ctas - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double v = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < a.rows.total; i += kFinishThreads) v += (double)__ldcg(a.row_losses + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x > 0) return;
#pragma unroll
  for (int i = 1; i < kFinishThreads / 32; ++i) v += sums[i];
  *a.loss = (float)(a.mean && count > 0 ? v / (double)count : v);  // no row takes part: 0
}

// what a row's logit gradients are scaled by beside the factor that all rows share, NaN with its loss
__device__ __forceinline__ float grad_scale_of(const FinishArgs& a, long long n, float loss) {
  return loss != loss ? quiet_nan() : (a.row_grads != nullptr ? a.row_grads[n] / *a.row_scale : 1.f);
}
// eight fp16 exponentials to bf16 logit gradients
__device__ __forceinline__ uint4 scaled(const uint4& e, float f) {
  const uint32_t in[4] = {e.x, e.y, e.z, e.w};
  uint32_t out[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const float2 t = Io16<__half>::unpack(in[h]);
    out[h] = IO::pack(t.x * f, t.y * f);
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

// What finish_kernel does, by a warp per row and for labels alone: without gradients (4096 x 65536 in 13 us; a CTA per row took
// 51), and with them where rows are short and a CTA would mostly wait for its own reductions (short_rows).
__global__ __launch_bounds__(kFinishThreads) void finish_by_warps_kernel(const FinishArgs a) {
  chain_begin();
  const int tiles = (a.vocab + kStatsTile - 1) / kStatsTile, lane = threadIdx.x & 31;
  const int count = *a.rows.count, left = count - a.rows.piece_begin;
  const int rows_here = left < 0 ? 0 : (left < a.rows.piece_rows ? left : a.rows.piece_rows);
  const int r = blockIdx.x * (kFinishThreads / 32) + (threadIdx.x >> 5);
  const int groups = (int)(a.ldg / 8);
  uint4* g = a.g + (long long)r * groups;
  if (r < rows_here) {
    const long long n = a.rows.row_map[a.rows.piece_begin + r];
    const long long v = a.labels.at(n);
    const bool inside = v >= 0 && v < a.vocab;
    const float2* stats = a.stats + (long long)r * tiles;
    float high = -INFINITY, sum = 0.f;
#pragma unroll 4
    for (int t = lane; t < tiles; t += 32) high = fmaxf(high, __ldg(&stats[t].x));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    if (high == -INFINITY) high = 0.f;  // no others
#pragma unroll 4
    for (int t = lane; t < tiles; t += 32) {
      const float2 s = __ldg(stats + t);
      sum = fmaf(s.y, ex2_approx(s.x - high), sum);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float logit = inside ? label_logit(a.x + n * a.channels, a.weight + v * a.channels, a.channels / 8, lane) : 0.f;
    const RowSums row = row_sums(high, sum, logit);
    const float loss = inside ? row.excess : quiet_nan();
    if (lane == 0) a.row_losses[n] = loss;
    if (a.g != nullptr) {
      const float scale = grad_scale_of(a, n, loss);
      for (int begin = lane; begin < groups; begin += 128) {
        uint4 e[4];  // four pieces requested together
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (begin + 32 * j < groups) e[j] = g[begin + 32 * j];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = begin + 32 * j;
          if (i < groups) g[i] = scaled(e[j], scale * ex2_approx(__ldg(&stats[i / (kStatsTile / 8)].x) - row.lse2));
        }
      }
      __syncwarp();
      if (lane == 0 && inside) reinterpret_cast<bf16*>(g)[v] = IO::store(-scale * row.missing);
    }
  } else if (a.g != nullptr && r < a.rows.piece_rows && r < ((rows_here + 63) & ~63)) {
    for (int i = lane; i < groups; i += 32) g[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  arrive_and_sum(a, count);
}

// A row's loss, and with gradients its exponentials in place to logit gradients: bound by the bytes of the row there and back
// (8192 x 65536 in 0.37 ms, 5.8 TB/s), with a teacher by the rows of W that its entries gather as well (2048 x 65536 with 64
// entries in 0.18 ms, half of it these).  A CTA per row, more where rows are few.
__global__ __launch_bounds__(kFinishThreads) void finish_kernel(const FinishArgs a) {
  chain_begin();
  extern __shared__ float factor[];  // [tiles] then logit [top] and share [top]
  __shared__ float scratch[kFinishThreads / 32];
  const int tiles = (a.vocab + kStatsTile - 1) / kStatsTile, top = a.labels.top;
  float* logit = factor + tiles;
  float* share = logit + top;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int count = *a.rows.count, left = count - a.rows.piece_begin;
  const int rows_here = left < 0 ? 0 : (left < a.rows.piece_rows ? left : a.rows.piece_rows);
  // A row belongs to gridDim.y CTAs, which all take its statistics and labels and then scale a part of it each.
  const int r = blockIdx.x;
  const int groups = (int)(a.ldg / 8);
  const int part = (groups + gridDim.y - 1) / gridDim.y;
  const int from = min(groups, part * (int)blockIdx.y), to = min(groups, from + part);
  uint4* g = a.g + (long long)r * groups;
  if (r >= rows_here) {
    // zeros behind the last row, to the end of its block of the contraction over rows
    if (a.g != nullptr && r < ((rows_here + 63) & ~63))
      for (int i = from + tid; i < to; i += kFinishThreads) g[i] = make_uint4(0u, 0u, 0u, 0u);
    arrive_and_sum(a, count);
    return;
  }
  const long long n = a.rows.row_map[a.rows.piece_begin + r];

  // the softmax's normaliser, in units of log2
  const float2* stats = a.stats + (long long)r * tiles;
  float high = -INFINITY, sum = 0.f;
  for (int t = tid; t < tiles; t += kFinishThreads) high = fmaxf(high, stats[t].x);
  high = block_reduce(high, scratch, true);
  if (high == -INFINITY) high = 0.f;  // no others
  for (int t = tid; t < tiles; t += kFinishThreads) {
    const float2 s = stats[t];
    sum = fmaf(s.y, ex2_approx(s.x - high), sum);
  }
  sum = block_reduce(sum, scratch, false);

  // the labels' logits: a warp per entry
  const long long entry = n * top;
  bool bad = false;
  for (int k = warp; k < top; k += kFinishThreads / 32) {
    const bool there = a.labels.teacher == nullptr || !(a.labels.teacher[entry + k] == -INFINITY);
    const long long v = there ? a.labels.at(entry + k) : 0;
    const bool inside = v >= 0 && v < a.vocab;
    const float dot = there && inside ? label_logit(a.x + n * a.channels, a.weight + v * a.channels, a.channels / 8, lane) : 0.f;
    bad |= there && !inside;
    if (lane == 0) logit[k] = dot * a.labels.inv_temperature;
  }
  bad = __syncthreads_or(bad);

  const int main = a.labels.teacher != nullptr ? a.highest[n] : 0;
  const RowSums row = row_sums(high, sum, logit[main]);
  for (int t = tid; t < tiles; t += kFinishThreads) factor[t] = stats[t].x - row.lse2;

  float loss;
  if (a.labels.teacher == nullptr) {
    if (tid == 0) share[0] = 1.f;
    loss = row.excess;
  } else {
    // the difference before the temperature: it is as good as the logits are, wherever they lie, and of two that are the type's
    // lowest value it is 0
    const float most = a.labels.teacher[entry + main];
    float rest = 0.f;  // of the exponentials, beside the highest entry's 1
    for (int k = tid; k < top; k += kFinishThreads) {
      const float p = expf((a.labels.teacher[entry + k] - most) * a.labels.inv_temperature);
      share[k] = p;
      if (k != main) rest += p;
    }
    rest = block_reduce(rest, scratch, false);
    const float log_total = log1pf(rest);
    float part = 0.f;
    for (int k = tid; k < top; k += kFinishThreads) {
      const float p = share[k] / (1.f + rest);
      share[k] = p;
      const float log_p = (a.labels.teacher[entry + k] - most) * a.labels.inv_temperature - log_total;
      if (!(p == 0.f)) part = fmaf(p, (log_p + row.excess) - (logit[k] - logit[main]), part);  // an absent entry has p = 0
    }
    loss = a.labels.temperature * a.labels.temperature * block_reduce(part, scratch, false);
  }
  if (bad) loss = quiet_nan();  // a label outside the vocabulary
  if (tid == 0 && blockIdx.y == 0) a.row_losses[n] = loss;
  arrive_and_sum(a, count);
  if (a.g == nullptr) return;

  const float scale = grad_scale_of(a, n, loss);
  __syncthreads();  // the tiles' factors and the shares
  for (int begin = from + tid; begin < to; begin += 4 * kFinishThreads) {
    uint4 e[4];  // four pieces requested together
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (begin + j * kFinishThreads < to) e[j] = g[begin + j * kFinishThreads];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = begin + j * kFinishThreads;
      if (i < to) g[i] = scaled(e[j], scale * ex2_approx(factor[i / (kStatsTile / 8)]));
    }
  }
  __syncthreads();
  for (int k = tid; k < top && !bad; k += kFinishThreads) {
    if (a.labels.teacher != nullptr && a.labels.teacher[entry + k] == -INFINITY) continue;
    const long long v = a.labels.at(entry + k);
    if (v < 8ll * from || v >= 8ll * to) continue;
    // an index may occur more than once: each occurrence writes the same value
    const bool of_main = v == a.labels.at(entry + main);
    float here = 0.f, elsewhere = 0.f;
    for (int j = 0; j < top; ++j) {
      if (a.labels.teacher != nullptr && a.labels.teacher[entry + j] == -INFINITY) continue;
      if (a.labels.at(entry + j) == v)
        here += share[j];
      else
        elsewhere += share[j];
    }
    // q - p, or for the main column (1 - p) - (1 - q)
    const float slope = of_main ? elsewhere - row.missing : ex2_approx(logit[k] * kLog2e - row.lse2) - here;
    reinterpret_cast<bf16*>(g)[v] = IO::store(scale * slope);
  }
}

// ---- small passes ------------------------------------------------------------------------------------------------------
// out[row_map ? row_map[row_begin + row] : row][c] = sum of the parts, bound by their bytes (two of 8192 x 2048 in 38 us).  A
// thread takes four columns of every kWarps-th part; with eight warps to an output (many parts of few rows: 32 of 33 x 512 in 4
// us, 14 with one) their sums are added in warp order.
template <int kWarps>
__global__ __launch_bounds__(256) void sum_parts_kernel(const float4* __restrict__ partials, uint2* __restrict__ out,
                                                        const int* __restrict__ row_map, const Plan* __restrict__ plan,
                                                        bool of_x, int row_begin, int part_rows, int pieces) {
  chain_begin();
  constexpr int kOutputs = 256 / kWarps;
  __shared__ float4 sums[kWarps > 1 ? kWarps - 1 : 1][32];
  const int parts = of_x ? plan->splits_x : plan->splits_w;
  const int limit = of_x ? plan->count - row_begin : part_rows;
  const long long rows = limit < part_rows ? limit : part_rows;
  const long long total = rows * pieces;  // rows <= 0: nothing
  const int slice = kWarps > 1 ? threadIdx.x / 32 : 0, lane = threadIdx.x % kOutputs;
  for (long long first = (long long)blockIdx.x * kOutputs; first < total; first += (long long)gridDim.x * kOutputs) {
    const long long i = first + lane;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < total) {
      for (int s = slice; s < parts; s += 4 * kWarps) {  // four parts requested together (the first again where there are fewer)
        float4 u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = __ldg(partials + (s + j * kWarps < parts ? s + j * kWarps : s) * total + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (s + j * kWarps < parts) {
            a.x += u[j].x; a.y += u[j].y; a.z += u[j].z; a.w += u[j].w;
          }
        }
      }
    }
    if (kWarps > 1) {
      if (slice > 0) sums[slice - 1][lane] = a;
      __syncthreads();
      if (slice == 0) {
#pragma unroll
        for (int j = 0; j < kWarps - 1; ++j) {
          const float4 u = sums[j][lane];
          a.x += u.x; a.y += u.y; a.z += u.z; a.w += u.w;
        }
      }
      __syncthreads();
    }
    if (slice == 0 && i < total) {
      const long long row = i / pieces;
      const long long to = of_x ? (long long)row_map[row_begin + row] * pieces + (i - row * pieces) : i;
      out[to] = make_uint2(IO::pack(a.x, a.y), IO::pack(a.z, a.w));
    }
  }
}

int launch_sum_parts(const float* partials, void* out, const int* row_map, const Plan* plan, bool of_x, int row_begin,
                     int part_rows, int channels, int most, cudaStream_t s) {
  const long long outputs = (long long)part_rows * (channels / 4);
  if (most > 4) {
    const long long ctas = (outputs + 31) / 32;
    launch_chained(sum_parts_kernel<8>, dim3((unsigned)(ctas < 1184 ? ctas : 1184)), dim3(256), 0, s,
                   reinterpret_cast<const float4*>(partials), static_cast<uint2*>(out), row_map, plan, of_x, row_begin, part_rows,
                   channels / 4);
  } else {
    const long long ctas = (outputs + 255) / 256;
    launch_chained(sum_parts_kernel<1>, dim3((unsigned)(ctas < 1184 ? ctas : 1184)), dim3(256), 0, s,
                   reinterpret_cast<const float4*>(partials), static_cast<uint2*>(out), row_map, plan, of_x, row_begin, part_rows,
                   channels / 4);
  }
  return check_launch("sum_parts_kernel");
}

// Both arrays *= *scale, in place; nothing to do where the scale is one.
__global__ __launch_bounds__(256) void scale_kernel(uint4* __restrict__ first, long long first_pieces, uint4* __restrict__ second,
                                                    long long pieces, const float* __restrict__ scale) {
  chain_begin();
  const float f = *scale;
  if (f == 1.f) return;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (long long)gridDim.x * 256) {
    uint4* at = i < first_pieces ? first + i : second + (i - first_pieces);
    const uint4 u = *at;
    const uint32_t in[4] = {u.x, u.y, u.z, u.w};
    uint32_t out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = IO::unpack(in[j]);
      out[j] = IO::pack(t.x * f, t.y * f);
    }
    *at = make_uint4(out[0], out[1], out[2], out[3]);
  }
}

// ---- host side ---------------------------------------------------------------------------------------------------------
// The workspace of a call; sizes depend on the shapes and on which gradients are wanted, not on the labels.
struct Layout {
  long long ldg, ldx;
  int piece_rows, pieces, splits_x, splits_w;
  bool parts_x, parts_w;
  size_t position, row_map, highest, main_column, plan, x_compact, stats, power, partial_x, partial_w, bytes;
};

size_t take(size_t& at, size_t bytes) {
  const size_t here = at;
  at += (bytes + 255) & ~size_t(255);
  return here;
}

int splits_for(long long rows, long long columns, long long k, int workers) {
  const float tiles = (float)((rows + kTile - 1) / kTile * ((columns + kTile - 1) / kTile)), blocks = (float)((k + 63) / 64);
  const float pairs = (float)workers, elements = (float)rows * (float)columns;
  int best = 1;
  for (int s = 2; s <= kMaxSplits && blocks >= s * kLeastBlocks; ++s)
    if (split_cost(s, tiles, blocks, elements, pairs) < split_cost(best, tiles, blocks, elements, pairs)) best = s;
  return best;
}

Layout layout_of(long long rows, int channels, int vocab, bool grad_x, bool grad_weight) {
  Layout l{};
  const bool grads = grad_x || grad_weight;
  l.ldg = ((long long)vocab + 63) / 64 * 64;
  l.ldx = ((long long)channels + 63) / 64 * 64;
  const long long tiles = (vocab + kStatsTile - 1) / kStatsTile;
  long long most = kStatsBytes / (8 * tiles);
  if (grads && kPieceBytes / (2 * l.ldg) < most) most = kPieceBytes / (2 * l.ldg);
  most = most / kTile * kTile;
  if (most < kTile) most = kTile;
  l.pieces = (int)((rows + most - 1) / most);
  // pieces of equal size, whole tiles each; a single piece is the rows themselves
  l.piece_rows = l.pieces == 1 ? (int)rows : (int)(((rows + l.pieces - 1) / l.pieces + kTile - 1) / kTile * kTile);
  l.pieces = (int)((rows + l.piece_rows - 1) / l.piece_rows);
  l.splits_x = grad_x ? splits_for(l.piece_rows, channels, vocab, pair_count() * (one_cta(l.piece_rows) ? 2 : 1)) : 1;
  l.splits_w = grad_weight ? splits_for(vocab, channels, l.piece_rows, pair_count()) : 1;
  l.parts_x = l.splits_x > 1;
  l.parts_w = l.splits_w > 1 || l.pieces > 1;
  size_t at = 0;
  l.plan = take(at, sizeof(Plan));
  l.position = take(at, rows * 4);
  l.row_map = take(at, rows * 4);
  l.highest = take(at, rows * 4);
  l.main_column = take(at, rows * 4);
  l.x_compact = take(at, (size_t)rows * l.ldx * 2);
  l.stats = take(at, (size_t)tiles * l.piece_rows * 8);
  l.power = take(at, grads ? (size_t)l.piece_rows * l.ldg * 2 : 0);
  l.partial_x = take(at, grad_x && l.parts_x ? (size_t)l.splits_x * l.piece_rows * channels * 4 : 0);
  l.partial_w = take(at, grad_weight && l.parts_w ? (size_t)l.splits_w * vocab * channels * 4 : 0);
  l.bytes = at;
  return l;
}

bool aligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int check_shape(long long rows, int channels, int vocab) {
  FRWKV_REQUIRE(rows > 0 && channels > 0 && vocab > 0, "pretrain_head_loss: sizes must be positive");
  FRWKV_REQUIRE(rows <= (1 << 24), "pretrain_head_loss: at most 16777216 rows");
  FRWKV_REQUIRE(channels % 8 == 0 && channels <= 65536, "pretrain_head_loss: channels must be a multiple of 8 up to 65536");
  FRWKV_REQUIRE(vocab <= (1 << 20), "pretrain_head_loss: at most 1048576 vocabulary entries");
  return FRWKV_OK;
}

}  // namespace
}  // namespace head
}  // namespace frwkv

extern "C" size_t frwkv_pretrain_head_loss_workspace_bytes(long long rows, int channels, int vocab, int grad_x,
                                                           int grad_weight) {
  using namespace frwkv;
  if (head::check_shape(rows, channels, vocab) != FRWKV_OK) return 0;
  return head::layout_of(rows, channels, vocab, grad_x != 0, grad_weight != 0).bytes;
}

extern "C" int frwkv_pretrain_head_loss(const frwkv_head_loss_args* args, frwkv_stream_t stream) {
  using namespace frwkv;
  using namespace frwkv::head;
  clear_error();
  FRWKV_REQUIRE(args != nullptr, "pretrain_head_loss: null pointer argument");
  const frwkv_head_loss_args& a = *args;
  FRWKV_REQUIRE(a.x && a.weight && a.labels && a.row_losses && a.workspace && a.error_flag,
                "pretrain_head_loss: null pointer argument");
  if (int rc = check_shape(a.rows, a.channels, a.vocab)) return rc;
  FRWKV_REQUIRE(a.label_bytes == 4 || a.label_bytes == 8, "pretrain_head_loss: labels must be int32 or int64");
  FRWKV_REQUIRE(a.top >= 1 && a.top <= kMaxTop, "pretrain_head_loss: 1 to 512 entries per row");
  FRWKV_REQUIRE(a.teacher_logits != nullptr || a.top == 1, "pretrain_head_loss: one label per row");
  FRWKV_REQUIRE(a.temperature > 0.f && a.temperature - a.temperature == 0.f && 1.f / a.temperature - 1.f / a.temperature == 0.f,
                "pretrain_head_loss: temperature must be finite and positive");
  FRWKV_REQUIRE(a.teacher_logits != nullptr || a.temperature == 1.f, "pretrain_head_loss: labels go with temperature 1");
  FRWKV_REQUIRE(aligned(a.x, 16) && aligned(a.weight, 16) && aligned(a.grad_x, 16) && aligned(a.grad_weight, 16) &&
                    aligned(a.workspace, 256) && aligned(a.labels, a.label_bytes) && aligned(a.teacher_logits, 4),
                "pretrain_head_loss: x, weight and their gradients must be 16-byte aligned, the workspace 256-byte aligned");
  const bool grads = a.grad_x != nullptr || a.grad_weight != nullptr;
  const Layout l = layout_of(a.rows, a.channels, a.vocab, a.grad_x != nullptr, a.grad_weight != nullptr);
  FRWKV_REQUIRE(a.workspace_bytes >= l.bytes,
                "pretrain_head_loss: workspace is smaller than frwkv_pretrain_head_loss_workspace_bytes");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(a.workspace);
  Plan* plan = reinterpret_cast<Plan*>(ws + l.plan);
  const int* count = &plan->count;
  int* position = reinterpret_cast<int*>(ws + l.position);
  int* row_map = reinterpret_cast<int*>(ws + l.row_map);
  int* highest = reinterpret_cast<int*>(ws + l.highest);
  int* main_column = reinterpret_cast<int*>(ws + l.main_column);
  float2* stats = reinterpret_cast<float2*>(ws + l.stats);
  void* power = grads ? ws + l.power : nullptr;
  float* partial_x = l.parts_x ? reinterpret_cast<float*>(ws + l.partial_x) : nullptr;
  float* partial_w = l.parts_w ? reinterpret_cast<float*>(ws + l.partial_w) : nullptr;
  const int rows = (int)a.rows, tiles = (a.vocab + kStatsTile - 1) / kStatsTile;

  Labels labels{};
  labels.index = a.labels;
  labels.wide = a.label_bytes == 8;
  labels.teacher = a.teacher_logits;
  labels.ignore_index = a.ignore_index;
  labels.top = a.top;
  labels.temperature = a.temperature;
  labels.inv_temperature = 1.f / a.temperature;

  const dim3 by_warp((rows + 7) / 8);
  if (a.teacher_logits != nullptr) {
    launch_chained(teacher_rows_kernel, by_warp, dim3(256), 0, s, labels, highest, rows);
    if (int rc = check_launch("teacher_rows_kernel")) return rc;
  }
  const SplitSizes sizes{a.channels, a.vocab, l.splits_x, l.splits_w, pair_count(),
                         pair_count() * (one_cta(l.piece_rows) ? 2 : 1), (long long)l.splits_x * l.piece_rows, l.pieces > 1};
  CompactArgs compact{};
  compact.x = static_cast<const uint4*>(a.x);
  compact.position = position;
  compact.x_compact = reinterpret_cast<uint4*>(ws + l.x_compact);
  compact.grad_x = static_cast<uint4*>(a.grad_x);
  compact.row_losses = a.row_losses;
  compact.rows = rows;
  compact.pieces = a.channels / 8;
  compact.pitch = (int)(l.ldx / 8);
  compact.always = l.ldx != a.channels;
  launch_chained(plan_kernel, dim3(1), dim3(1024), 0, s, labels, highest, position, row_map, main_column, plan,
                 sizes, compact, a.row_grads, a.error_flag, rows);
  if (int rc = check_launch("plan_kernel")) return rc;
  if (rows > kFewRows) {
    launch_chained(compact_kernel, by_warp, dim3(256), 0, s, compact, count);
    if (int rc = check_launch("compact_kernel")) return rc;
  }

  const double lost = kTruncation * a.channels / parts_of_channels(a.channels);
  const float log2_scale = (float)(1.4426950408889634 * (1.0 + lost) * labels.inv_temperature);
  const GradFactor factor{labels.temperature, a.mean != 0, a.grad_scale, a.row_grads != nullptr ? &plan->row_scale : nullptr};
  const size_t finish_smem = (size_t)(tiles + 2 * a.top) * sizeof(float);
  for (int piece = 0; piece < l.pieces; ++piece) {
    const Rows here{count, row_map, rows, compact.always, l.ldx, piece * l.piece_rows, l.piece_rows};
    if (int rc = launch_logit_stats(a.x, ws + l.x_compact, a.weight, here, a.channels, a.vocab, log2_scale, main_column, stats,
                                    power, l.ldg, a.error_flag, s))
      return rc;
    FinishArgs f{};
    f.rows = here;
    f.labels = labels;
    f.x = static_cast<const bf16*>(a.x);
    f.weight = static_cast<const bf16*>(a.weight);
    f.highest = highest;
    f.stats = stats;
    f.vocab = a.vocab;
    f.channels = a.channels;
    f.g = static_cast<uint4*>(power);
    f.ldg = l.ldg;
    f.mean = a.mean != 0;
    f.row_grads = a.row_grads;
    f.row_scale = &plan->row_scale;
    f.row_losses = a.row_losses;
    f.loss = a.loss;
    f.arrived = &plan->arrived;
    const bool by_warps = a.teacher_logits == nullptr && (!grads || short_rows(l.ldg, l.piece_rows));
    // few rows are cut into parts, so that the device has two CTAs per SM to run (at most 16 parts of a row: one of 65536
    // entries then is two rounds of requests; 16 rows of 65536 take 10 us, 14 whole)
    const int parts = by_warps || !grads ? 1 : (l.piece_rows >= 148 ? 1 : (l.piece_rows > 18 ? 296 / l.piece_rows : 16));
    const int ctas = by_warps ? (l.piece_rows + kFinishThreads / 32 - 1) / (kFinishThreads / 32) : l.piece_rows;
    f.ctas = ctas * l.pieces;
    if (by_warps)
      launch_chained(finish_by_warps_kernel, dim3(ctas), dim3(kFinishThreads), 0, s, f);
    else
      launch_chained(finish_kernel, dim3(ctas, parts), dim3(kFinishThreads), finish_smem, s, f);
    if (int rc = check_launch("finish_kernel")) return rc;
    if (grads) {
      const GradTarget to_x{a.grad_x, partial_x, Splits{&plan->splits_x, l.splits_x}};
      const GradTarget to_weight{a.grad_weight, partial_w, Splits{&plan->splits_w, l.splits_w}};
      if (int rc = launch_gradients(power, l.ldg, a.x, ws + l.x_compact, a.weight, here, a.channels, a.vocab, to_x, to_weight,
                                    factor, piece > 0, a.error_flag, s))
        return rc;
      if (a.grad_x != nullptr && l.parts_x)
        if (int rc = launch_sum_parts(partial_x, a.grad_x, row_map, plan, true, here.piece_begin, l.piece_rows, a.channels,
                                      l.splits_x, s))
          return rc;
    }
  }
  if (a.grad_weight != nullptr && l.parts_w)
    if (int rc = launch_sum_parts(partial_w, a.grad_weight, row_map, plan, false, 0, a.vocab, a.channels, l.splits_w, s)) return rc;
  return FRWKV_OK;
}

extern "C" int frwkv_scale_bf16(void* first, long long first_numel, void* second, long long second_numel, const float* scale,
                                frwkv_stream_t stream) {
  using namespace frwkv;
  using namespace frwkv::head;
  clear_error();
  FRWKV_REQUIRE(scale && (first || second) && (first || first_numel == 0) && (second || second_numel == 0),
                "scale_bf16: null pointer argument");
  FRWKV_REQUIRE(first_numel >= 0 && second_numel >= 0 && first_numel % 8 == 0 && second_numel % 8 == 0,
                "scale_bf16: the numbers of values must be multiples of 8");
  FRWKV_REQUIRE(aligned(first, 16) && aligned(second, 16), "scale_bf16: values must be 16-byte aligned");
  const long long pieces = (first_numel + second_numel) / 8, blocks = (pieces + 255) / 256;
  if (pieces == 0) return FRWKV_OK;
  launch_chained(scale_kernel, dim3((unsigned)(blocks < 1184 ? blocks : 1184)), dim3(256), 0,
                 reinterpret_cast<cudaStream_t>(stream), static_cast<uint4*>(first), first_numel / 8,
                 static_cast<uint4*>(second), pieces, scale);
  return check_launch("scale_kernel");
}
