#include "operators/draft_verify_op.h"

#include "kernels/op_kernels.h"

namespace dragon {

template <class Context>
template <typename T>
void DraftVerifyOp<Context>::DoRunWithType() {
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
void DraftVerifyOp<Context>::DoRunWithIndex() {
  Tensor& P = Input(0);
  CHECK_EQ(P.ndim(), 3) << "\nExcepted probabilities of shape (B, K + 1, C).";
  const int64_t B = KernelExtent("sequences", P.dim(0)), K = KernelExtent("drafted tokens", P.dim(1) - 1);
  const int64_t C = KernelExtent("classes", P.dim(2));
  CHECK_GE(K, 0) << "\nExcepted probabilities at one position at least.";
  INITIALIZE_TENSOR_VIA_SPEC(Input(1), vec64_t({B, K}), IndexT);
  INITIALIZE_TENSOR_VIA_SPEC(Input(2), vec64_t({B}), IndexT);
  INITIALIZE_TENSOR_VIA_SPEC(Input(3), vec64_t({B, K}), float);
  INITIALIZE_TENSOR_VIA_SPEC(Input(4), vec64_t({B}), float);
  const T* draft = nullptr;
  if (InputSize() > 5) {
    INITIALIZE_TENSOR_VIA_SPEC(Input(5), vec64_t({B, K, C}), T);
    draft = Input(5).template data<T, Context>(ctx());
  }
  kernels::DraftVerify(
      static_cast<int>(B), static_cast<int>(K), static_cast<int>(C), P.template data<T, Context>(ctx()), draft,
      Input(1).template data<IndexT, Context>(ctx()), Input(2).template data<IndexT, Context>(ctx()),
      Input(3).template data<float, Context>(ctx()), Input(4).template data<float, Context>(ctx()),
      Output(0)->Reshape({B, K + 1})->template mutable_data<IndexT, Context>(ctx()),
      Output(1)->Reshape({B})->template mutable_data<IndexT, Context>(ctx()), ctx());
}

DEPLOY_HIP_OPERATOR(DraftVerify);

OPERATOR_SCHEMA(DraftVerify).NumInputs(5, 6).NumOutputs(2);  // P, D, N, A, S[, Q] -> Tokens, Accepted

} // namespace dragon
