// The gradient of a linear layer's input, dx = dz W, on the matrix cores (mq_gemm.hpp).
#include "mq_gemm.hpp"

using namespace mq;

int mq_gemm_input_grad(int dtype, GemmArgs& a, const GemmPlan& plan, float* ws, hipStream_t st) {
    return dtype == MQ_F16 ? gemm_launch<MQ_F16, kDown, kRows, false>(a, plan, ws, st) : gemm_launch<MQ_BF16, kDown, kRows, false>(a, plan, ws, st);
}
