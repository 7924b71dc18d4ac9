// The operators at the two ends of a token model, reached as stablehlo.custom_call targets: embedding lookup and its
// gradient, counter-based dropout, log probabilities of given tokens and their gradient.  What a call needs to know
// (filled in by the planner) and the launches (rx_embedding.cu, rx_dropout.cu, rx_logprobs.cu).
//
//   @rx.embedding(table [V][D], ids [..]) {scale}                 -> [..][D]
//   @rx.embedding_grad(dy [..][D], ids [..]) {scale}              -> [V][D]
//   @rx.dropout(x, key [2] i32 [, residual]) {rate, site}         -> like x
//   @rx.token_logprobs(logits [..][V], ids [..]) {temperature, top_k}
//        -> logprob [..], entropy [..], lse [..] (f32) [, top log probabilities [..][k] f32, top tokens [..][k] i32]
//   @rx.token_logprobs_grad(logits, ids, lse, entropy, dlogprob, dentropy, dlse) {temperature} -> like logits
#pragma once
#include <stdint.h>

#include <string>
#include <vector>

#include "rx_ir.h"

namespace rx {

enum class CallK { None, Embedding, EmbeddingGrad, Dropout, LogProbs, LogProbsGrad };

constexpr int kMaxTopK = 64;

// Operands and results sit in the step's leaf_slot / out_slot, in the order of the call; an operand that is a constant
// zero and need not be read (a gradient that does not arrive) has slot -1.  All are dense, except that the rows of the
// first operand of the four row-wise calls may lie `ld` elements apart (a window of a wider array).
struct CallDesc {
  CallK op = CallK::None;
  int64_t rows = 0;               // tokens
  int64_t cols = 0;               // elements of a row: features, or the vocabulary of a logprobs call
  int64_t vocab = 0;              // rows of the embedding table
  int64_t ld = 0;                 // elements between the starts of two rows of the first operand
  std::vector<int64_t> off;       // element offset of each operand inside its slot
  DT in_dt = DT::F32, out_dt = DT::F32, ids_dt = DT::S32;
  double scale = 1;               // embedding: factor of a row; logprobs: 1 / temperature
  double rate = 0;                // dropout
  int64_t site = 0;
  bool sharded = false;           // dropout: this device's elements start at its place in the mesh * (rows * cols)
  int top_k = 0;
};

inline const char* call_name(CallK k) {
  switch (k) {
    case CallK::Embedding: return "embedding";
    case CallK::EmbeddingGrad: return "embedding_grad";
    case CallK::Dropout: return "dropout";
    case CallK::LogProbs: return "token_logprobs";
    case CallK::LogProbsGrad: return "token_logprobs_grad";
    default: return "call";
  }
}

// dropout: an element stays when its 16 bits reach this; 65536 - threshold of 65536 elements do
inline int64_t dropout_threshold(double rate) { return (int64_t)(rate * 65536.0 + 0.5); }

}  // namespace rx

#ifdef __CUDACC__
#include "rx_kernels.h"
namespace rx {
// in / out: the operands and results, offsets applied (null for an operand without a slot).
cudaError_t launch_embedding(const LaunchCtx& c, const CallDesc& d, const void* table, const void* ids, void* out);
cudaError_t launch_embedding_grad(const LaunchCtx& c, const CallDesc& d, const void* dy, const void* ids, void* out, void* workspace);
int64_t embedding_grad_workspace(const CallDesc& d, int sm_count);
// `first`: the index of x's first element in the array that all devices of a mesh hold together
cudaError_t launch_dropout(const LaunchCtx& c, const CallDesc& d, const void* x, const void* key, const void* residual, void* out, int64_t first);
struct LogProbsOut {
  float *logprob, *entropy, *lse, *top_value;
  int32_t* top_token;
};
cudaError_t launch_logprobs(const LaunchCtx& c, const CallDesc& d, const void* logits, const void* ids, const LogProbsOut& out);
struct LogProbsGradIn {
  const float *lse, *entropy, *dlogprob, *dentropy, *dlse;
};
cudaError_t launch_logprobs_grad(const LaunchCtx& c, const CallDesc& d, const void* logits, const void* ids, const LogProbsGradIn& in, void* out);
}  // namespace rx
#endif
