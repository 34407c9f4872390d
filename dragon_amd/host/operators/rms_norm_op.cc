#include "operators/rms_norm_op.h"

#include <algorithm>

#include "core/gradient.h"
#include "kernels/op_kernels.h"

namespace dragon {

namespace {

// math::Copy counts in int; tensors of these operators may hold more elements.
template <typename T, class Context>
void CopyElements(const int64_t n, const T* x, T* y, Context* ctx) {
  constexpr int64_t kMost = int64_t(1) << 30;
  for (int64_t at = 0; at < n; at += kMost) {
    math::Copy(static_cast<int>(std::min(kMost, n - at)), x + at, y + at, ctx);
  }
}

} // namespace

template <class Context>
template <typename T>
void RMSNormOp<Context>::DoRunWithType() {
  using AccT = typename math::Traits<T>::accumulator_type;
  Tensor& X = Input(0);
  Tensor& W = Input(1);
  GET_OP_AXIS_ARG(axis, X.ndim(), -1);
  const int rows = KernelExtent("rows", X.count(0, axis)), width = KernelExtent("columns", X.count(axis));
  INITIALIZE_TENSOR_VIA_SPEC(W, vec64_t({width}), AccT);
  CHECK_EQ(OutputSize(), InputSize() - 1) << "\nA residual's sum is the second output.";
  const T* residual = nullptr;
  T* h = nullptr;
  if (InputSize() > 2) {
    INITIALIZE_TENSOR_VIA_SPEC(Input(2), X.dims(), T);
    residual = Input(2).template data<T, Context>(ctx());
    h = Output(1)->ReshapeLike(X)->template mutable_data<T, Context>(ctx());
  }
  kernels::RMSNorm(rows, width, static_cast<float>(epsilon_),
                   X.template data<T, Context>(ctx()), residual, W.template data<AccT, Context>(ctx()), h,
                   Output("X_rsig")->Reshape({rows})->template mutable_data<AccT, Context>(ctx()),
                   Output(0)->ReshapeLike(X)->template mutable_data<T, Context>(ctx()), ctx());
}

template <class Context>
template <typename T>
void RMSNormGradientOp<Context>::DoRunWithType() {
  using AccT = typename math::Traits<T>::accumulator_type;
  Tensor& H = Input(0);
  Tensor& W = Input(1);
  GET_OP_AXIS_ARG(axis, H.ndim(), -1);
  const int rows = KernelExtent("rows", H.count(0, axis)), width = KernelExtent("columns", H.count(axis));
  INITIALIZE_TENSOR_VIA_SPEC(W, vec64_t({width}), AccT);
  INITIALIZE_TENSOR_VIA_SPEC(Input(2), H.dims(), T);
  CHECK_EQ(Input("X_rsig").count(), rows) << "\nThe forward operator saw other rows.";
  const T* dh = nullptr;
  if (InputSize() > 3) {
    INITIALIZE_TENSOR_VIA_SPEC(Input(3), H.dims(), T);
    dh = Input(3).template data<T, Context>(ctx());
  }
  T* dx = Output(0)->ReshapeLike(H)->template mutable_data<T, Context>(ctx());
  kernels::RMSNormGrad(rows, width,
                       H.template data<T, Context>(ctx()),
                       Input("X_rsig").template data<AccT, Context>(ctx()),
                       W.template data<AccT, Context>(ctx()), Input(2).template data<T, Context>(ctx()), dh,
                       Output(1)->ReshapeLike(W)->template mutable_data<AccT, Context>(ctx()), dx, ctx());
  if (OutputSize() > 2) {  // X and the residual are summed: one gradient for both, in a tensor each
    CopyElements(H.count(), static_cast<const T*>(dx),
                 Output(2)->ReshapeLike(H)->template mutable_data<T, Context>(ctx()), ctx());
  }
}

template <class Context>
template <typename T>
void RMSNormSumGradientOp<Context>::DoRunWithType() {
  using AccT = typename math::Traits<T>::accumulator_type;
  Tensor& dH = Input(0);
  Tensor& W = Input(1);
  GET_OP_AXIS_ARG(axis, dH.ndim(), -1);
  const int width = KernelExtent("columns", dH.count(axis));
  INITIALIZE_TENSOR_VIA_SPEC(W, vec64_t({width}), AccT);
  const T* dh = dH.template data<T, Context>(ctx());
  CopyElements(dH.count(), dh, Output(0)->ReshapeLike(dH)->template mutable_data<T, Context>(ctx()), ctx());
  math::Set(width, AccT(0),
            Output(1)->ReshapeLike(W)->template mutable_data<AccT, Context>(ctx()), ctx());
  CopyElements(dH.count(), dh, Output(2)->ReshapeLike(dH)->template mutable_data<T, Context>(ctx()), ctx());
}

template <class Context>
template <typename T>
void RMSNormQuantOp<Context>::DoRunWithType() {
  Tensor& X = Input(0);
  Tensor& W = Input(1);
  GET_OP_AXIS_ARG(axis, X.ndim(), -1);
  const int rows = KernelExtent("rows", X.count(0, axis)), width = KernelExtent("columns", X.count(axis));
  INITIALIZE_TENSOR_VIA_SPEC(W, vec64_t({width}), float);
  CHECK_EQ(OutputSize(), InputSize()) << "\nA residual's sum is the third output.";
  CHECK_GE(group_size_, 0) << "\nExcepted a <group_size> of 0, 32, 64, 128 or 256.";
  const int group_size = KernelExtent("group_size", group_size_);
  const T* residual = nullptr;
  T* h = nullptr;
  if (InputSize() > 2) {
    INITIALIZE_TENSOR_VIA_SPEC(Input(2), X.dims(), T);
    residual = Input(2).template data<T, Context>(ctx());
    h = Output(2)->ReshapeLike(X)->template mutable_data<T, Context>(ctx());
  }
  vec64_t scale_dims(X.dims().begin(), X.dims().begin() + axis);
  scale_dims.push_back(group_size > 0 ? (int64_t(width) + group_size - 1) / group_size : 1);
  kernels::RMSNormQuant(
      rows, width, group_size,
      static_cast<float>(epsilon_), X.template data<T, Context>(ctx()), residual,
      W.template data<float, Context>(ctx()), h, static_cast<float*>(nullptr),
      Output(0)->ReshapeLike(X)->template mutable_data<uint8_t, Context>(ctx()),
      Output(1)->Reshape(scale_dims)->template mutable_data<float, Context>(ctx()), ctx());
}

DEPLOY_HIP_OPERATOR(RMSNorm);
DEPLOY_HIP_OPERATOR(RMSNormGradient);
DEPLOY_HIP_OPERATOR(RMSNormSumGradient);
DEPLOY_HIP_OPERATOR(RMSNormQuant);

OPERATOR_SCHEMA(RMSNorm).NumInputs(2, 3).NumOutputs(1, 2);          // X, W[, R] -> Y[, H]
OPERATOR_SCHEMA(RMSNormGradient).NumInputs(3, 4).NumOutputs(2, 3);  // H, W, dY[, dH] -> dX, dW[, dR]
OPERATOR_SCHEMA(RMSNormSumGradient).NumInputs(2).NumOutputs(3);     // dH, W -> dX, dW, dR
OPERATOR_SCHEMA(RMSNormQuant).NumInputs(2, 3).NumOutputs(2, 3);     // X, W[, R] -> Q, S[, H]

namespace {

class RMSNormGradientMaker final : public GradientMakerBase {
 public:
  using GradientMakerBase::GradientMakerBase;
  void CreateGradientDefs() override {
    if (def().input.size() < 3) {
      AddGradientDef("RMSNormGradient", {I(0), I(1), GO(0)}, {GI(0), GI(1)});
      return;
    }
    const bool from_y = Arrives(0), from_h = Arrives(1);
    CHECK(from_y || from_h) << "\nNo gradient arrives at Operator(" << def().type << ").";
    if (!from_y) {  // what arrives at the sum passes on as it is
      AddGradientDef("RMSNormSumGradient", {GO(1), I(1)}, {GI(0), GI(1), GI(2)});
      return;
    }
    vector<string> inputs = {O(1), I(1), GO(0)};
    if (from_h) inputs.push_back(GO(1));
    AddGradientDef("RMSNormGradient", inputs, {GI(0), GI(1), GI(2)});
  }

 private:
  bool Arrives(int i) const { return !GO(i).empty() && GO(i) != "NULL"; }
};

} // namespace

REGISTER_GRADIENT(RMSNorm, RMSNormGradientMaker);

} // namespace dragon
