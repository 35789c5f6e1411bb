// The forward product of a linear layer, y = act(x W^T + b) + r, on the matrix cores (mq_gemm.hpp).
#include "mq_gemm.hpp"

using namespace mq;

int mq_gemm_forward(int dtype, GemmArgs& a, const GemmPlan& plan, float* ws, hipStream_t st) {
    return dtype == MQ_F16 ? gemm_launch<MQ_F16, kRows, kRows, true>(a, plan, ws, st) : gemm_launch<MQ_BF16, kRows, kRows, true>(a, plan, ws, st);
}
