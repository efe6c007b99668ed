// Internal interface between the parts of the head's losses: head_loss.cu (plan of the rows, softmax statistics to losses
// and logit gradients, reductions, the C entries) and head_gemm.cu (the three products).
#pragma once

#include "frwkv_common.cuh"

namespace frwkv {
namespace head {

constexpr int kTile = 256;       // rows and columns of an output tile
constexpr int kStatsTile = 128;  // vocabulary columns of one maximum and sum of exponentials
// The tensor core truncates where it adds an instruction's 16 products to its fp32 accumulator, so a logit loses a share of its
// running sum with every addition: with all channels in one accumulator 1.0e-6, 2.2e-6, 4.3e-6 and 6.9e-5 of itself at 1024,
// 2048, 4096 and 65536 channels of random rows, 1.1e-5, 2.2e-5, 4.5e-5 and 7.2e-4 where the large products come first, nothing
// where the sums are exact.  So the contraction is cut into parts of equal length, of at most so many channels, that the
// epilogue adds in registers, rounding to nearest, and the loss grows no further than 1024 channels take it.  A part costs the
// epilogue one more read of the accumulator: statistics of 4096 x 65536 x 640 take 250 us with one part and 300 with two, of
// 2048 x 65536 x 2048 350 us with one, 355 with two, 390 with four.
constexpr int kPartChannels = 1024;
constexpr int parts_of_channels(int channels) { return (channels + kPartChannels - 1) / kPartChannels; }
// The gradients' contractions, over the vocabulary or the rows, are cut the same way before a sum loses what shows beside its
// rounding to bf16 (2^-8): 131072 rows that begin with the large ones were off by 1.6e-3 in one accumulator, by 8e-5 in parts.
// The time is the same (8192 x 65536 x 2048 5.3 to 5.4 ms either way).
constexpr int kGradPart = 4096;

// The rows that take part are numbered 0..count-1 ("compact rows"); the first *count entries of row_map are their numbers
// in x.  A product works on a piece of them: compact rows piece_begin .. piece_begin + piece_rows - 1, cut at *count.
struct Rows {
  const int* count;
  const int* row_map;
  int total;        // rows of x; where *count equals it and not `copied`, x itself is the compact form
  bool copied;      // x is copied in any case
  long long ldx;    // distance of the copied rows
  int piece_begin, piece_rows;
};

// Statistics of the logits z = x W^T / T: for every 128 vocabulary columns and every row of the piece
// stats[row][tile] = (max, sum exp2(z' - max)) with z' = z log2(e) / T, and, with `power`, the fp16 values
// exp2(z' - max) in power[row][ldp] (zeros behind the vocabulary).  The column main_column[compact row] of a row, its label,
// stays out of them (-1: none does); of no column at all they are (-inf, 0).
int launch_logit_stats(const void* x, const void* x_compact, const void* weight, const Rows& rows, int channels, int vocab,
                       float log2_scale, const int* main_column, float2* stats, void* power, long long ldp,
                       int* error_flag,
                       cudaStream_t stream);

// The time of a rows x columns product whose contraction of `blocks` blocks of 64 is cut into s parts: a wave of pairs takes
// one tile and part each (0.34 us per 256 x 256 x 64, as measured), and every part is written and read once more in fp32.
__host__ __device__ inline float split_cost(int s, float tiles, float blocks, float elements, float pairs) {
  const float waves = ceilf(tiles * (float)s / pairs);
  return waves * ceilf(blocks / (float)s) * 0.34f + (s > 1 ? 3.f + (float)s * elements * (8.f / 5.0e6f) : 0.f);
}
constexpr int kMaxSplits = 64;
constexpr float kLeastBlocks = 4.f;  // of a part

// The parts in use are chosen where the number of rows is known, by plan_kernel, from 1 to what the host has room for.
struct Splits {
  const int* chosen;  // device
  int most;           // partial sums have room for `most` parts of all rows; 1: none are kept
};

// Where a gradient goes: with room for one part bf16 straight to `grad` (null: not wanted), else fp32 parts to
// partials[part][rows of the product][channels].
struct GradTarget {
  void* grad;
  float* partials;
  Splits splits;
};

// What the gradients of all rows share: temperature * (mean ? 1 / *count : 1) * (scale ? *scale : 1) * (of_rows ? *of_rows : 1).
struct GradFactor {
  float temperature;
  bool mean;
  const float* scale;    // device
  const float* of_rows;  // device
};

// One launch for both gradients, each times `factor`: grad_x[row_map[row]] = g[row] W, contraction over the vocabulary (its
// parts have the rows that take part), and grad_weight = g^T x, contraction over the rows of the piece (its parts are added to
// what they hold where `add`).  The units of dW fill what the last units of dx leave of the device.
int launch_gradients(const void* g, long long ldg, const void* x, const void* x_compact, const void* weight, const Rows& rows,
                     int channels, int vocab, const GradTarget& to_x, const GradTarget& to_weight, const GradFactor& factor,
                     bool add, int* error_flag, cudaStream_t stream);

// Up to 128 rows one CTA works alone on a 128 x 256 tile: a pair's tile would be half empty, and the loads of W, which bound
// the product then, would wait for twice the tensor-core time per byte.  Steps alone / by pairs in us: 16 x 65536 x 4096 345 /
// 368, of x's gradient only 211 / 235; 128 x 65536 x 2048 232 / 239; 40 x 32000 x 768 62 / 67; 16 x 65536 x 1024 122 / 120 and
// 128 x 50277 x 1544 174 / 172 are the ones where pairs were ahead.
constexpr bool one_cta(long long rows) { return rows <= kTile / 2; }

int pair_count();  // of CTAs that the current device runs at once

}  // namespace head
}  // namespace frwkv
