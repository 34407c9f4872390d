// Distillation of a student's logits from a teacher's top logits (forward and gradient).
//
//   TopKDistillationLoss          X, I, T     -> L   X logits [..., C], I the classes of the teacher's
//                                                    top logits [..., K] (int32 / int64; an entry
//                                                    outside [0, C) is not listed), T those logits
//   TopKDistillationLossGradient  X, I, T, dL -> dX
//
// "temperature" divides both sides' logits; "reduction" is NONE, SUM, MEAN, BATCH_MEAN or VALID
// (default: divide by the rows that list a class), as for SoftmaxCrossEntropyLoss. The
// log-sum-exp of each row and the divisor are kept in the side tensor "X_stats". No counterpart
// in the reference.
#pragma once

#include "core/operator.h"

namespace dragon {

#define DECLARE_TOPK_DISTILLATION_OP(name)                                    \
  template <class Context>                                                    \
  class name##Op final : public Operator<Context> {                           \
   public:                                                                    \
    name##Op(const OperatorDef& def, Workspace* ws)                           \
        : Operator<Context>(def, ws),                                         \
          temperature_(OP_SINGLE_ARG(float, "temperature", 1.f)),             \
          reduction_(OP_SINGLE_ARG(string, "reduction", "VALID")) {}          \
    USE_OPERATOR_FUNCTIONS;                                                   \
    void Setup() override { this->CheckOutputsApart(); }                      \
    void RunOnDevice() override { FloatingDispatch::Call(this, Input(0)); }   \
    template <typename T>                                                     \
    void DoRunWithType();                                                     \
    template <typename T, typename IndexT>                                    \
    void DoRunWithIndex();                                                    \
                                                                              \
   protected:                                                                 \
    float temperature_;                                                       \
    string reduction_;                                                        \
  };

DECLARE_TOPK_DISTILLATION_OP(TopKDistillationLoss)
DECLARE_TOPK_DISTILLATION_OP(TopKDistillationLossGradient)
#undef DECLARE_TOPK_DISTILLATION_OP

} // namespace dragon
