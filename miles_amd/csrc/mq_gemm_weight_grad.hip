// The gradient of a linear layer's weight, dW = dz^T x, on the matrix cores (mq_gemm.hpp).  x may be an 8-bit copy: its values are
// exact in bf16, so they enter the product as they are, and the 16-bit tensor exists in shared memory only.
#include "mq_gemm.hpp"

using namespace mq;

template <int D>
static int weight_grad(GemmArgs& a, const GemmPlan& plan, float* ws, hipStream_t st) {
    return a.ps ? gemm_launch<D, kDownKept, kDown, false>(a, plan, ws, st) : gemm_launch<D, kDown, kDown, false>(a, plan, ws, st);
}
int mq_gemm_weight_grad(int dtype, GemmArgs& a, const GemmPlan& plan, float* ws, hipStream_t st) {
    return dtype == MQ_F16 ? weight_grad<MQ_F16>(a, plan, ws, st) : weight_grad<MQ_BF16>(a, plan, ws, st);
}
