#include "operators/topk_distillation_loss_op.h"

#include "core/gradient.h"
#include "kernels/op_kernels.h"

namespace dragon {

namespace {

// 0 keeps a loss per row, -1 divides by the rows that count. Logits without leading axes are one row.
float DistillationNormalizer(const string& reduction, int64_t rows, const Tensor& X) {
  if (reduction == "NONE") return 0.f;
  if (reduction == "VALID") return -1.f;
  if (reduction == "SUM") return 1.f;
  // of no rows, the sum is 0 whatever divides it
  if (reduction == "MEAN") return static_cast<float>(rows > 0 ? rows : 1);
  if (reduction == "BATCH_MEAN") return X.ndim() > 1 && X.dim(0) > 0 ? static_cast<float>(X.dim(0)) : 1.f;
  LOG(FATAL) << "Unknown reduction: " << reduction;
  return 0.f;
}

// X [..., C], I and T [..., K] with the same leading dimensions.
template <typename AccT>
void CheckShapes(const Tensor& X, const Tensor& I, const Tensor& T) {
  CHECK_GE(X.ndim(), 1) << "\nExcepted logits with a class axis.";
  CHECK_EQ(I.ndim(), X.ndim()) << "\nExcepted the classes' axes to be those of the logits.";
  for (int i = 0; i + 1 < X.ndim(); ++i) {
    CHECK_EQ(I.dim(i), X.dim(i)) << "\nAxis " << i << " of the classes and of the logits must be matched.";
  }
  CHECK(T.dims() == I.dims()) << "\nExcepted Tensor(" << T.name() << ")'s dimensions are "
                              << DimsToString(I.dims()) << ", got " << DimsToString(T.dims()) << ".";
  CHECK(T.meta() == TypeOf<AccT>::value)
      << "\nExcepted the type of Tensor(" << T.name() << ") is " << NameOf(TypeOf<AccT>::value) << ", got "
      << NameOf(T.meta()) << ".";
}

} // namespace

template <class Context>
template <typename T>
void TopKDistillationLossOp<Context>::DoRunWithType() {
  CHECK(Input(1).meta() == DType::kInt32 || Input(1).meta() == DType::kInt64)
      << this->MessageForUnsupported(NameOf(Input(1).meta()), {"int32", "int64"});
  if (Input(1).meta() == DType::kInt32) {
    DoRunWithIndex<T, int>();
  } else {
    DoRunWithIndex<T, int64_t>();
  }
}

template <class Context>
template <typename T, typename IndexT>
void TopKDistillationLossOp<Context>::DoRunWithIndex() {
  using AccT = typename math::Traits<T>::accumulator_type;
  Tensor& X = Input(0);
  Tensor& I = Input(1);
  CheckShapes<AccT>(X, I, Input(2));
  const int64_t rows = KernelExtent("rows", X.count(0, X.ndim() - 1));
  const int classes = KernelExtent("classes", X.dim(-1)), listed = KernelExtent("listed classes", I.dim(-1));
  vec64_t out_dims(X.dims().begin(), X.dims().end() - 1);
  if (reduction_ != "NONE") out_dims.clear();
  kernels::TopKDistillationLossForward(
      static_cast<int>(rows), classes, listed, temperature_,
      DistillationNormalizer(reduction_, rows, X), X.template data<T, Context>(ctx()),
      I.template data<IndexT, Context>(ctx()), Input(2).template data<AccT, Context>(ctx()),
      Output("X_stats")->Reshape({rows + 1})->template mutable_data<AccT, Context>(ctx()),
      Output(0)->Reshape(out_dims)->template mutable_data<AccT, Context>(ctx()), ctx());
}

template <class Context>
template <typename T>
void TopKDistillationLossGradientOp<Context>::DoRunWithType() {
  CHECK(Input(1).meta() == DType::kInt32 || Input(1).meta() == DType::kInt64)
      << this->MessageForUnsupported(NameOf(Input(1).meta()), {"int32", "int64"});
  if (Input(1).meta() == DType::kInt32) {
    DoRunWithIndex<T, int>();
  } else {
    DoRunWithIndex<T, int64_t>();
  }
}

template <class Context>
template <typename T, typename IndexT>
void TopKDistillationLossGradientOp<Context>::DoRunWithIndex() {
  using AccT = typename math::Traits<T>::accumulator_type;
  Tensor& X = Input(0);
  Tensor& I = Input(1);
  Tensor& dL = Input(3);
  CheckShapes<AccT>(X, I, Input(2));
  const int64_t rows = KernelExtent("rows", X.count(0, X.ndim() - 1));
  const int classes = KernelExtent("classes", X.dim(-1)), listed = KernelExtent("listed classes", I.dim(-1));
  CHECK_EQ(dL.count(), reduction_ == "NONE" ? rows : 1) << "\nNumel of L and dL must be matched.";
  CHECK_EQ(Input("X_stats").count(), rows + 1) << "\nThe forward operator saw other logits.";
  kernels::TopKDistillationLossBackward(
      static_cast<int>(rows), classes, listed, temperature_,
      DistillationNormalizer(reduction_, rows, X), X.template data<T, Context>(ctx()),
      I.template data<IndexT, Context>(ctx()), Input(2).template data<AccT, Context>(ctx()),
      Input("X_stats").template data<AccT, Context>(ctx()), dL.template data<AccT, Context>(ctx()),
      Output(0)->ReshapeLike(X)->template mutable_data<T, Context>(ctx()), ctx());
}

DEPLOY_HIP_OPERATOR(TopKDistillationLoss);
DEPLOY_HIP_OPERATOR(TopKDistillationLossGradient);

OPERATOR_SCHEMA(TopKDistillationLoss).NumInputs(3).NumOutputs(1);          // X, I, T -> L
OPERATOR_SCHEMA(TopKDistillationLossGradient).NumInputs(4).NumOutputs(1);  // X, I, T, dL -> dX

namespace {

class TopKDistillationLossGradientMaker final : public GradientMakerBase {
 public:
  using GradientMakerBase::GradientMakerBase;
  void CreateGradientDefs() override {
    AddGradientDef("TopKDistillationLossGradient", {I(0), I(1), I(2), GO(0)}, {GI(0)});
  }
};

} // namespace

REGISTER_GRADIENT(TopKDistillationLoss, TopKDistillationLossGradientMaker);

} // namespace dragon
