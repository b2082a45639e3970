// Parameter blocks of the losses a language model is trained with (mss_linloss.hip: from the head's
// operands, logits not kept; mss_distill.hip: from logits). The host fills them after validation.
//
// A row (token) wants a distribution q over a few words: the one-hot of its target, or what a
// teacher's top logits make of its list. With s = logits / temperature and lse the log of the sum of exp s
// over the vocabulary,
//   loss = temperature^2 sum_k q_k (log q_k - s[word_k] + lse),
//   d loss / d logit_v = temperature (exp(s_v - lse) - q_v).
// Logarithms are kept to base 2: c = log2(e) / temperature takes a logit there.
#pragma once

#include "mss_common.h"

namespace mss {

constexpr int kLossMaxTop = 1024;
constexpr int kLinLossMaxima = 640;
constexpr int kLinLossTile = 256;  // largest side of a product's tile
enum { kLossNone = 0, kLossSum = 1, kLossMean = 2 };

// The rows' wanted words (of lists: launch_loss_rows). A row counts if it has one: live is 0 (no), 1 (yes), or NaN
// for one with a word outside the vocabulary, whose loss and gradients are NaN.
struct LossRows {
  int rows, top, vocab;
  float c;
  const long long* targets;  // [rows], or NULL where there are lists
  long long ignore;
  const long long* ids;      // [rows][top], negative: none
  const void* teacher;       // [rows][top] float32 or bf16
  int teacher_bf16;
  int* words;                // [rows][top], -1 where there is none; each word once
  float* q;                  // [rows][top]
  float* live;               // [rows]
  int* counts;               // [blocks] rows that count, by blocks of rows
  int blocks;
};

int loss_list_blocks(int rows);
int loss_target_blocks(int tokens);
hipError_t launch_loss_rows(const LossRows& r, hipStream_t stream);

// A matrix of bf16 in one plane, or of float32, a power of two's multiple of it, in two of half precision: the
// rounding to 11 bits, and that of what it leaves times 2^11.
struct LossMatrix {
  const bf16_t* base;
  long long ld, plane;  // elements from one row, one plane to the next
  long long end;        // elements of a plane from base on
};

struct LinLossParams {
  int tokens, features, vocab, width;  // width: features up to a multiple of 64, of 128 split
  int planes;                          // 1: bf16, 2: float32, split
  int reduction;
  float temperature, c;
  LossRows r;
  // x (features, tokens) and the weight (vocab, features) as given
  const void* x;
  long long sf, st;
  const void* w;
  long long ldw;
  int pack_w;
  bf16_t* xp;      // [planes][tokens][width]
  bf16_t* wp;      // [planes][vocab][width] where pack_w
  uint32_t* maxima;  // of float32 operands, kLinLossMaxima of them
  int* powers;       // [2]: of two, that x's planes and w's are taken times
  int* power_g;      // and the rows' upstream gradients
  float2* part;    // [parts][tokens]: a part's largest s and sum of 2^(s - largest), base 2
  int parts;
  float* picked;   // [rows][top] logits of the wanted words
  float2* stat;    // [tokens + kLinLossTile]: m, the largest s to base 2 or near it, and 1 / sum 2^(s - m), 0 where the row
                   // does not count: (their logarithm, in 32 bits, would cost a probability log2 |lse| of its bits)
  float* loss;     // [tokens]
  float* mean;     // the reduced loss
  float* by;       // 1 / (rows that count), for a mean
  // backward
  const float* grad;  // [1], or [tokens] without a reduction
  float2* scale;      // without a reduction: stat with the row's upstream gradient in its factor
  bf16_t* g;          // [planes][tokens][ldg] the logits' gradient for a piece of the vocabulary
  long long ldg;
  float* dx_sum;      // [features][ldx] where there are pieces
  long long ldx;
  float* partial;     // sums of tiles that several workgroups share
  int piece;          // words of a piece
  void* dx;           // [features][tokens] as x
  void* dw;           // [vocab][features]
  int dw_bf16;
  // both directions at once
  float* row_sums;    // [parts_both][block]
  float* dw_sum;      // [vocab][features] where there are blocks
  int* bad;           // [blocks]
  const int* only_if; // NULL, or nothing is done where this is 0
};

// What the call needs besides its operands; sizes depend on nothing but the arguments.
struct LinLossPlan {
  int shape, shape_x, shape_w;  // of the tiles: 0 small, 1 large, 2 thin, and of the logits' 3: of 192 tokens
  int parts, piece;
  long long ldg, ldx, partial;
  int both, block, parts_both;  // both directions at once: whether, tokens of a block
  long long lde, partial_both;
};
LinLossPlan linloss_plan(int tokens, int features, int vocab, int planes);

hipError_t launch_linloss_fwd(const LinLossParams& p, const LinLossPlan& plan, hipStream_t stream);
hipError_t launch_linloss_both(const LinLossParams& p, const LinLossPlan& plan, hipStream_t stream);
hipError_t launch_linloss_rescale(const LinLossParams& p, hipStream_t stream);
hipError_t launch_linloss_bwd(const LinLossParams& p, const LinLossPlan& plan, hipStream_t stream);

struct DistillParams {
  int vocab, io_bf16, reduction;
  float temperature;
  LossRows r;
  const void* logits;
  long long ld;
  float* loss;      // [rows]
  float2* stat;     // [rows]: largest logit, log2 of the sum of 2^((logit - largest) c)
  float* mean;      // the reduced loss
  float* by;        // 1 / (rows that count), for a mean
  const float* grad;  // [1], or [rows] without a reduction
  void* dlogits;      // [rows][vocab]
};

// The loss (kDsFwd), its gradient (kDsBwd), both from one reading of the logits for an upstream gradient of 1,
// or the gradient once more unless the upstream one is 1 (kDsAgain).
enum { kDsFwd = 1, kDsBwd = 2, kDsAgain = 4 };
hipError_t launch_distill(const DistillParams& p, int what, hipStream_t stream);
hipError_t launch_loss_mean(const float* loss, const LossRows& r, int reduction, float* mean, float* by, hipStream_t stream);

}  // namespace mss
