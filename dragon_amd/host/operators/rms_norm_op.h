// RMSNorm with the residual's addition (forward and gradient), and its 8-bit form.
//
//   RMSNorm          X, W          -> Y            Y = X / sqrt(mean(X^2) + epsilon) * W
//                    X, W, R       -> Y, H         H = X + R, Y the norm of H
//   RMSNormGradient  X, W, dY      -> dX, dW
//                    H, W, dY[, dH] -> dX, dW, dR  dH: what arrives through H; dR equals dX
//   RMSNormSumGradient  dH, W     -> dX, dW, dR    where nothing arrives through Y: dX = dR = dH, dW = 0
//   RMSNormQuant     X, W[, R]     -> Q, S[, H]    Q e4m3 codes (uint8), S float32 scales: one per
//                                                  "group_size" columns, or per row for 0
//
// Everything from "axis" on is normalised; W is AccT as the affine parameters of LayerNorm. The
// reciprocal root is kept in the side tensor "X_rsig". No counterpart in the reference.
#pragma once

#include "core/operator.h"

namespace dragon {

#define DECLARE_RMS_NORM_OP(name, Dispatch)                                                     \
  template <class Context>                                                                      \
  class name##Op final : public Operator<Context> {                                             \
   public:                                                                                      \
    name##Op(const OperatorDef& def, Workspace* ws)                                             \
        : Operator<Context>(def, ws),                                                           \
          epsilon_(OP_SINGLE_ARG(double, "epsilon", 1e-5)),                                     \
          group_size_(OP_SINGLE_ARG(int64_t, "group_size", 0)) {}                               \
    USE_OPERATOR_FUNCTIONS;                                                                     \
    void Setup() override { this->CheckOutputsApart(); }                                        \
    void RunOnDevice() override { Dispatch::Call(this, Input(0)); }                             \
    template <typename T>                                                                       \
    void DoRunWithType();                                                                       \
                                                                                                \
   protected:                                                                                   \
    double epsilon_;                                                                            \
    int64_t group_size_;                                                                        \
  };

// float16, bfloat16 and float32: what an 8-bit output is made of.
struct QuantDispatch {
  template <class Op>
  static void Call(Op* op, const Tensor& tensor) {
    switch (tensor.meta()) {
      case DType::kFloat16: op->template DoRunWithType<float16>(); break;
      case DType::kBFloat16: op->template DoRunWithType<bfloat16>(); break;
      case DType::kFloat32: op->template DoRunWithType<float>(); break;
      default:
        LOG(FATAL) << op->MessageForUnsupported(NameOf(tensor.meta()),
                                                {"float16", "bfloat16", "float32"});
    }
  }
};

DECLARE_RMS_NORM_OP(RMSNorm, FloatingDispatch)
DECLARE_RMS_NORM_OP(RMSNormGradient, FloatingDispatch)
DECLARE_RMS_NORM_OP(RMSNormSumGradient, FloatingDispatch)
DECLARE_RMS_NORM_OP(RMSNormQuant, QuantDispatch)
#undef DECLARE_RMS_NORM_OP

} // namespace dragon
