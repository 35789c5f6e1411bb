// The forward product of a linear layer, y = act(x W^T + b) + r, on the matrix cores (mq_gemm.hpp).
#include "mq_gemm.hpp"

using namespace mq;

template <int D>
static int forward(bool bounded, GemmArgs& a, const GemmPlan& plan, float* ws, hipStream_t st) {
    return bounded ? gemm_launch<D, kRowsAny, kRowsAny, true>(a, plan, ws, st) : gemm_launch<D, kRowsDirect, kRowsDirect, true>(a, plan, ws, st);
}
int mq_gemm_forward(int dtype, bool bounded, GemmArgs& a, const GemmPlan& plan, float* ws, hipStream_t st) {
    return dtype == MQ_F16 ? forward<MQ_F16>(bounded, a, plan, ws, st) : forward<MQ_BF16>(bounded, a, plan, ws, st);
}
