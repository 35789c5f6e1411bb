// Linear layers: which product runs how, the join of a product that was split along k, and the backward pass of the activation.
#include "mq_gemm.hpp"

int mq_column_sum_launch(const float* p0, void* out0, const float* p1, void* out1, int64_t parts, int64_t n, int dtype, hipStream_t st);

namespace mq {

// The sums of a product's splits, in their order, and what follows them.  Four columns a lane; the eight lanes of 32 columns are
// neighbours, because a row's units are counted in fours of eight.
template <int D>
__global__ __launch_bounds__(256) void gemm_join_kernel(const GemmArgs a, int splits) {
    const int64_t per_row = (a.np + 31) / 32 * 8, ldw = (a.np + 3) / 4 * 4;
    const int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x, row = unit / per_row, col = (unit - row * per_row) * 4;
    const bool inside = row < a.nq && col < a.np;
    float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (inside) {
        const float* from = a.ws + row * ldw + col;
        for (int s = 0; s < splits; s++) {
            const f32x4 v = *(const f32x4*)(from + (int64_t)s * a.nq * ldw);
#pragma unroll
            for (int i = 0; i < 4; i++) z[i] += v[i];
        }
        add_bias4<D>(a, col, z);
    }
    if (a.zq) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) m = umax(m, keep_magnitude(z[i]));
        m = group_max8(m);
        const uint32_t e = keep_exponent(m);
        if (inside) {
            *(uint32_t*)(a.zq + row * a.np + col) = keep_codes4(z[0], z[1], z[2], z[3], e8m0_inverse(e));
            if (col % 32 == 0) a.zs[row * (a.np / 32) + col / 32] = (uint8_t)e;
        }
    }
    if (inside) with_activation(a.act, [&](auto kind) { finish4<D, decltype(kind)::value>(a, row, col, z); });
}

struct ActGradArgs {
    const char* dy;
    const char* z;             // 16-bit, or (KEPT) e4m3 codes
    const uint8_t* zs;
    char* dz;                  // null: not wanted
    float* part;               // [gridDim.y][n], null: not wanted
    int64_t rows, n, lddy;
    int act;
};

// dz = dy act'(z) and the sums of its columns.  A wavefront goes down rows of 512 columns, eight to a lane, so that a column's sum
// stays in a register; the four wavefronts of a workgroup take turns and their sums meet in shared memory.
template <int D, int KEPT>
__global__ __launch_bounds__(256) void activation_bwd_kernel(const ActGradArgs a) {
    __shared__ float sums[4][8][kWave + 1];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int64_t col = ((int64_t)blockIdx.x * kWave + lane) * 8;
    float db[8];
#pragma unroll
    for (int j = 0; j < 8; j++) db[j] = 0.0f;
    with_activation(a.act, [&](auto kind) {
        constexpr int ACT = decltype(kind)::value;
        for (int64_t row = (int64_t)blockIdx.y * 4 + wave; row < a.rows; row += (int64_t)gridDim.y * 4) {
            float g[8];
            unpack<D>(ld_row<D>(a.dy + row * a.lddy * 2, col, a.n), g);
            if (ACT != MQ_ACT_NONE) {
                float z[8];
                if (KEPT) {
                    u32x2 c = {0u, 0u};
                    uint32_t e = 0;
                    if (col < a.n) {
                        c = *(const u32x2*)(a.z + row * a.n + col);
                        e = a.zs[row * (a.n / 32) + col / 32];
                    }
                    const float s = e8m0_value(e);
                    kept_values4(c.x, s, z);
                    kept_values4(c.y, s, z + 4);
                } else {
                    unpack<D>(ld_row<D>(a.z + row * a.n * 2, col, a.n), z);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) g[j] *= slope<ACT>(z[j]);
            }
            if (a.dz) st_row<D>(a.dz + row * a.n * 2, col, a.n, pack<D>(g));
#pragma unroll
            for (int j = 0; j < 8; j++) db[j] += g[j];
        }
    });
    if (!a.part) return;
#pragma unroll
    for (int j = 0; j < 8; j++) sums[wave][j][lane] = db[j];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int j = 0; j < 8; j++) db[j] = (sums[0][j][lane] + sums[1][j][lane]) + (sums[2][j][lane] + sums[3][j][lane]);
        float* to = a.part + (int64_t)blockIdx.y * a.n;
        st_row<MQ_F32>(to, col, a.n, pack<MQ_F32>(db));
        st_row<MQ_F32>(to, col + 4, a.n, pack<MQ_F32>(db + 4));
    }
}

}  // namespace mq

using namespace mq;

// How a product of np columns, nq rows and k runs: the tile, and into how many splits k is cut so that every compute unit has work.
// Each candidate's time is estimated from the rounds of workgroups that it takes and the bytes of its partial sums.
static GemmPlan gemm_plan(int64_t np, int64_t nq, int64_t k, bool bounded) {
    struct Tile {
        int bp, bq, per_cu;
        double step_us;                                   // of one step of one workgroup, with per_cu of them on a compute unit
    };
    static const Tile tiles[3] = {{256, 256, 1, 1.25}, {128, 128, 2, 0.85}, {128, 64, 3, 0.7}};
    const int64_t steps = (k + kStep - 1) / kStep;
    GemmPlan best{kTileMiddle, 1, (steps > 0 ? steps : 1) * kStep};
    double best_us = 1e30;
    for (int t = bounded ? kTileMiddle : kTileLarge; t <= (bounded ? kTileMiddle : kTileLow); t++) {
        const Tile& tile = tiles[t];
        const double count = (double)((np + tile.bp - 1) / tile.bp) * (double)((nq + tile.bq - 1) / tile.bq);
        for (int splits = 1; splits <= 64; splits = splits < 4 ? splits + 1 : splits + splits / 2) {
            const int64_t per = (steps + splits - 1) / splits;
            const int real = per > 0 ? (int)((steps + per - 1) / per) : 1;
            if (splits > 1 && (real != splits || per < 4)) continue;
            const double slots = 256.0 * tile.per_cu, rounds = (double)(int64_t)((count * real + slots - 1) / slots);
            double us = 3.0 + rounds * ((double)per * tile.step_us + 3.0);
            if (real > 1) us += 4.0 + (double)real * np * nq * 8 / 4e6;
            if (us < best_us) {
                best_us = us;
                best = GemmPlan{t, real, per * kStep};
            }
        }
    }
    return best;
}

static bool direct_ok(const void* p, int64_t ld, int64_t cols) {
    return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && cols % 8 == 0 && ld < (1 << 22);
}
static int check_sizes(int dtype, int64_t M, int64_t N, int64_t K) {
    if (dtype != MQ_BF16 && dtype != MQ_F16) return mq_fail(MQ_ERR_ARG, "linear: bf16 or fp16");
    if (M < 0 || N < 0 || K < 0) return mq_fail(MQ_ERR_ARG, "linear: bad argument");
    if (M > 0x7FFFFF00 || N > 0x7FFFFF00 || K > 0x7FFFFF00) return mq_fail(MQ_ERR_ARG, "linear: tensor too large");
    return MQ_OK;
}
static int check_rows(int64_t rows, int64_t cols, int64_t ld) {
    return rows > 1 && ld < cols ? mq_fail(MQ_ERR_ARG, "linear: rows overlap") : MQ_OK;
}
static int check_grid(const GemmPlan& plan, int64_t np, int64_t nq) {
    return ((np + 127) / 128) * ((nq + 63) / 64) * plan.splits > 0x7FFFFFF0 ? mq_fail(MQ_ERR_ARG, "linear: tensor too large") : MQ_OK;
}
// joins the splits, if there are any
static int join(int dtype, const GemmArgs& a, const GemmPlan& plan, hipStream_t st) {
    if (plan.splits > 1) {
        const int64_t blocks = (a.nq * ((a.np + 31) / 32 * 8) + 255) / 256;
        if (dtype == MQ_F16) hipLaunchKernelGGL(gemm_join_kernel<MQ_F16>, dim3((unsigned)blocks), dim3(256), 0, st, a, plan.splits);
        else hipLaunchKernelGGL(gemm_join_kernel<MQ_BF16>, dim3((unsigned)blocks), dim3(256), 0, st, a, plan.splits);
    }
    return mq_check_launch("linear");
}

extern "C" int mq_linear_workspace(int product, int64_t M, int64_t N, int64_t K, int64_t* floats) {
    if (!floats || product < MQ_LINEAR_FORWARD || product > MQ_LINEAR_WEIGHT_GRAD || M < 0 || N < 0 || K < 0) return mq_fail(MQ_ERR_ARG, "linear: bad argument");
    const int64_t np = product == MQ_LINEAR_FORWARD ? N : K, nq = product == MQ_LINEAR_WEIGHT_GRAD ? N : M;
    const int64_t k = product == MQ_LINEAR_FORWARD ? K : product == MQ_LINEAR_INPUT_GRAD ? N : M;
    *floats = 0;
    for (int bounded = 0; bounded < 2; bounded++) {
        const GemmPlan plan = gemm_plan(np, nq, k, bounded != 0);
        const int64_t need = plan.splits > 1 ? plan.splits * nq * ((np + 3) / 4 * 4) : 0;
        if (need > *floats) *floats = need;
    }
    return MQ_OK;
}

extern "C" int mq_linear_forward(const void* x, int dtype, int64_t ldx, const void* weight, int64_t ldw, const void* bias, int act,
                                 const void* residual, int64_t ldr, void* y, void* z, void* z8, uint8_t* z8_scale, int64_t M, int64_t N,
                                 int64_t K, float* ws, void* stream) {
    if (const int rc = check_sizes(dtype, M, N, K)) return rc;
    if (act < MQ_ACT_NONE || act > MQ_ACT_GELU_TANH) return mq_fail(MQ_ERR_ARG, "linear: unknown activation");
    if (check_rows(M, K, ldx) || check_rows(N, K, ldw) || (residual && check_rows(M, N, ldr))) return MQ_ERR_ARG;
    if (M == 0 || N == 0) return MQ_OK;
    if (!y || (K > 0 && (!x || !weight)) || !z8 != !z8_scale) return mq_fail(MQ_ERR_ARG, "linear: null pointer");
    if (z8 && (N % 32 != 0 || (uintptr_t)z8 % 4)) return mq_fail(MQ_ERR_ARG, "linear: columns kept in 8 bits are a multiple of 32, 4-byte aligned");
    const bool bounded = !direct_ok(x, M > 1 ? ldx : 8, K) || !direct_ok(weight, N > 1 ? ldw : 8, K);
    const GemmPlan plan = gemm_plan(N, M, K, bounded);
    if (const int rc = check_grid(plan, N, M)) return rc;
    if (plan.splits > 1 && (!ws || (uintptr_t)ws % 16)) return mq_fail(MQ_ERR_ARG, "linear: a 16-byte aligned workspace is needed");
    GemmArgs a{};
    a.p = (const char*)weight, a.q = (const char*)x, a.ldp = ldw, a.ldq = ldx, a.np = N, a.nq = M, a.k = K;
    a.out = (char*)y, a.bias = (const char*)bias, a.res = (const char*)residual, a.ldr = ldr;
    a.z = (char*)z, a.zq = (uint8_t*)z8, a.zs = z8_scale, a.act = act;
    const hipStream_t st = (hipStream_t)stream;
    if (const int rc = mq_gemm_forward(dtype, bounded, a, plan, ws, st)) return rc;
    return join(dtype, a, plan, st);
}

extern "C" int mq_linear_input_grad(const void* dz, int dtype, int64_t lddz, const void* weight, int64_t ldw, void* dx, int64_t M, int64_t N,
                                    int64_t K, float* ws, void* stream) {
    if (const int rc = check_sizes(dtype, M, N, K)) return rc;
    if (check_rows(M, N, lddz) || check_rows(N, K, ldw)) return MQ_ERR_ARG;
    if (M == 0 || K == 0) return MQ_OK;
    if (!dx || (N > 0 && (!dz || !weight))) return mq_fail(MQ_ERR_ARG, "linear: null pointer");
    const bool bounded = !direct_ok(dz, M > 1 ? lddz : 8, N) || !direct_ok(weight, N > 1 ? ldw : 8, K);
    const GemmPlan plan = gemm_plan(K, M, N, bounded);
    if (const int rc = check_grid(plan, K, M)) return rc;
    if (plan.splits > 1 && (!ws || (uintptr_t)ws % 16)) return mq_fail(MQ_ERR_ARG, "linear: a 16-byte aligned workspace is needed");
    GemmArgs a{};
    a.p = (const char*)weight, a.q = (const char*)dz, a.ldp = ldw, a.ldq = lddz, a.np = K, a.nq = M, a.k = N, a.out = (char*)dx;
    const hipStream_t st = (hipStream_t)stream;
    if (const int rc = mq_gemm_input_grad(dtype, bounded, a, plan, ws, st)) return rc;
    return join(dtype, a, plan, st);
}

extern "C" int mq_linear_weight_grad(const void* dz, int dtype, int64_t lddz, const void* x, int64_t ldx, const uint8_t* x_scale, void* dweight,
                                     int64_t M, int64_t N, int64_t K, float* ws, void* stream) {
    if (const int rc = check_sizes(dtype, M, N, K)) return rc;
    if (check_rows(M, N, lddz) || (!x_scale && check_rows(M, K, ldx))) return MQ_ERR_ARG;
    if (N == 0 || K == 0) return MQ_OK;
    if (!dweight || (M > 0 && (!dz || !x))) return mq_fail(MQ_ERR_ARG, "linear: null pointer");
    if (x_scale && (K % 32 != 0 || (uintptr_t)x % 16)) return mq_fail(MQ_ERR_ARG, "linear: an 8-bit copy has a multiple of 32 columns and is 16-byte aligned");
    const bool bounded = !direct_ok(dz, M > 1 ? lddz : 8, N) || (!x_scale && !direct_ok(x, M > 1 ? ldx : 8, K));
    const GemmPlan plan = gemm_plan(K, N, M, bounded);
    if (const int rc = check_grid(plan, K, N)) return rc;
    if (plan.splits > 1 && (!ws || (uintptr_t)ws % 16)) return mq_fail(MQ_ERR_ARG, "linear: a 16-byte aligned workspace is needed");
    GemmArgs a{};
    a.p = (const char*)x, a.ps = x_scale, a.q = (const char*)dz, a.ldp = x_scale ? K : ldx, a.ldq = lddz, a.np = K, a.nq = N, a.k = M;
    a.out = (char*)dweight;
    const hipStream_t st = (hipStream_t)stream;
    if (const int rc = mq_gemm_weight_grad(dtype, bounded, a, plan, ws, st)) return rc;
    return join(dtype, a, plan, st);
}

static int64_t act_parts(int64_t M, int64_t N) {
    const int64_t slabs = (N + 511) / 512, fours = (M + 3) / 4;
    int64_t parts = slabs > 0 ? 2048 / slabs : 1;
    parts = parts < 1 ? 1 : parts;
    return fours < parts ? (fours > 0 ? fours : 1) : parts;
}
extern "C" int mq_activation_backward_parts(int64_t M, int64_t N) { return (int)act_parts(M, N); }

extern "C" int mq_activation_backward(const void* dy, int dtype, int64_t lddy, const void* z, const uint8_t* z8_scale, int act, void* dz,
                                      void* dbias, float* ws, int64_t M, int64_t N, void* stream) {
    if (const int rc = check_sizes(dtype, M, N, 0)) return rc;
    if (act < MQ_ACT_NONE || act > MQ_ACT_GELU_TANH) return mq_fail(MQ_ERR_ARG, "linear: unknown activation");
    if (check_rows(M, N, lddy)) return MQ_ERR_ARG;
    if (N == 0 || (M == 0 && !dbias)) return MQ_OK;
    if ((M > 0 && (!dy || (act != MQ_ACT_NONE && !z))) || (dbias && !ws)) return mq_fail(MQ_ERR_ARG, "linear: null pointer");
    if (z8_scale && (N % 32 != 0 || (uintptr_t)z % 8)) return mq_fail(MQ_ERR_ARG, "linear: an 8-bit copy has a multiple of 32 columns and is 8-byte aligned");
    const int64_t parts = act_parts(M, N), slabs = (N + 511) / 512;
    const ActGradArgs a{(const char*)dy, (const char*)z, z8_scale, (char*)dz, dbias ? ws : nullptr, M, N, lddy, act};
    const dim3 grid((unsigned)slabs, (unsigned)parts);
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == MQ_F16 && z8_scale) hipLaunchKernelGGL((activation_bwd_kernel<MQ_F16, 1>), grid, dim3(256), 0, st, a);
    else if (dtype == MQ_F16) hipLaunchKernelGGL((activation_bwd_kernel<MQ_F16, 0>), grid, dim3(256), 0, st, a);
    else if (z8_scale) hipLaunchKernelGGL((activation_bwd_kernel<MQ_BF16, 1>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((activation_bwd_kernel<MQ_BF16, 0>), grid, dim3(256), 0, st, a);
    if (const int rc = mq_check_launch("activation backward")) return rc;
    return dbias ? mq_column_sum_launch(ws, dbias, nullptr, nullptr, parts, N, dtype, st) : MQ_OK;
}
