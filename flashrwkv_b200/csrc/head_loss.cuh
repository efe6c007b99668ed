// Internal interface between the parts of the head's losses: head_loss.cu (plan of the rows, softmax statistics to losses
// and logit gradients, reductions, the C entries) and head_gemm.cu (the three products).
#pragma once

#include "frwkv_common.cuh"

namespace frwkv {
namespace head {

constexpr int kTile = 256;       // rows and columns of an output tile
constexpr int kStatsTile = 128;  // vocabulary columns of one maximum and sum of exponentials

// The rows that take part are numbered 0..count-1 ("compact rows"); the first *count entries of row_map are their numbers
// in x.  A product works on a piece of them: compact rows piece_begin .. piece_begin + piece_rows - 1, cut at *count.
struct Rows {
  const int* count;
  const int* row_map;
  int total;  // rows of x; where *count equals it, x itself is the compact form
  int piece_begin, piece_rows;
};

// Statistics of the logits z = x W^T / T: for every 128 vocabulary columns and every row of the piece
// stats[row][tile] = (max, sum exp2(z' - max)) with z' = z log2(e) / T, and, with `power`, the fp16 values
// exp2(z' - max) in power[row][ldp] (zeros behind the vocabulary).
int launch_logit_stats(const void* x, const void* x_compact, const void* weight, const Rows& rows, int channels, int vocab,
                       float log2_scale, float2* stats, void* power, long long ldp, int* error_flag,
                       cudaStream_t stream);

// How many parts the contraction of a rows x columns product over k is cut into.
int contraction_splits(long long rows, long long columns, long long k);

// grad_x[row_map[row]] = g[row] W, contraction over the vocabulary in `splits` parts: with one part bf16 rows go straight to
// grad_x, with more the fp32 parts go to partials[split][piece_rows][channels].
int launch_grad_x(const void* g, long long ldg, const void* weight, const Rows& rows, int channels, int vocab, int splits,
                  void* grad_x, float* partials, int* error_flag, cudaStream_t stream);

// grad_weight = g^T x, contraction over the rows of the piece in `splits` parts: bf16 straight to grad_weight, or (partials
// given) fp32 parts in partials[split][vocab][channels], added to what they hold where `add`.
int launch_grad_weight(const void* g, long long ldg, const void* x, const void* x_compact, const Rows& rows, int channels,
                       int vocab, int splits, void* grad_weight, float* partials, bool add, int* error_flag,
                       cudaStream_t stream);

}  // namespace head
}  // namespace frwkv
