// The gradient of a linear layer's input, dx = dz W, on the matrix cores (mq_gemm.hpp).
#include "mq_gemm.hpp"

using namespace mq;

template <int D>
static int input_grad(bool bounded, GemmArgs& a, const GemmPlan& plan, float* ws, hipStream_t st) {
    return bounded ? gemm_launch<D, kDownAny, kRowsAny, false>(a, plan, ws, st) : gemm_launch<D, kDownDirect, kRowsDirect, false>(a, plan, ws, st);
}
int mq_gemm_input_grad(int dtype, bool bounded, GemmArgs& a, const GemmPlan& plan, float* ws, hipStream_t st) {
    return dtype == MQ_F16 ? input_grad<MQ_F16>(bounded, a, plan, ws, st) : input_grad<MQ_BF16>(bounded, a, plan, ws, st);
}
