#include "mq_attend.hpp"

int mq_attend_bf16_kept(const mq::AttendArgs& a, int nk, int nv, bool direct, unsigned grid, hipStream_t st) {
    return mq::attend_launch<MQ_BF16, true>(a, nk, nv, direct, grid, st);
}
