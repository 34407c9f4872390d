// Verification of drafted tokens against the target's probabilities.
//
//   DraftVerify  P, D, N, A, S[, Q] -> Tokens, Accepted
//     P  the target's probabilities [B, K + 1, C]     D  drafted tokens [B, K] (int32 / int64)
//     N  how many of the K are drafted [B]            A, S  uniform random numbers, float32 [B, K], [B]
//     Q  the draft's probabilities [B, K, C]; without it tokens were drafted without sampling
//
// Tokens [B, K + 1] = the accepted ones, one sampled where they end, -1 behind it. Has no
// gradient. No counterpart in the reference.
#pragma once

#include "core/operator.h"

namespace dragon {

template <class Context>
class DraftVerifyOp final : public Operator<Context> {
 public:
  DraftVerifyOp(const OperatorDef& def, Workspace* ws) : Operator<Context>(def, ws) {}
  USE_OPERATOR_FUNCTIONS;

  void Setup() override { this->CheckOutputsApart(); }
  void RunOnDevice() override { FloatingDispatch::Call(this, Input(0)); }

  template <typename T>
  void DoRunWithType();
  template <typename T, typename IndexT>
  void DoRunWithIndex();
};

} // namespace dragon
