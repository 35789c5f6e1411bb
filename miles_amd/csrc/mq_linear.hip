// Linear layers: which product runs how, the join of a product that was split along k, and the backward pass of the activation.
#include "mq_gemm.hpp"

int mq_column_sum_launch(const float* p0, void* out0, const float* p1, void* out1, int64_t parts, int64_t n, int dtype, hipStream_t st);

namespace mq {

// The sums of the parts of the tiles that were cut along k, in the parts' order, and what follows them.  Four columns a lane; the eight
// lanes of 32 columns are neighbours.
template <int D>
__global__ __launch_bounds__(256) void gemm_join_kernel(const GemmArgs a, int bp, int bq) {
    const int units = bp * bq / 4, blocks = units / 256, nth = (int)blockIdx.x / blocks, unit = ((int)blockIdx.x - nth * blocks) * 256 + (int)threadIdx.x;
    int tp, tq;
    place_of(a, a.whole + nth, tp, tq);
    const int r = unit / (bp / 4), c = (unit - r * (bp / 4)) * 4;
    const int64_t row = (int64_t)tq * bq + r, col = (int64_t)tp * bp + c;
    const bool inside = row < a.nq && col < a.np;
    float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (inside) {
        const float* from = a.ws + (int64_t)nth * a.splits * bp * bq + r * bp + c;
        // eight parts' loads at once (48 x 2560 x 9728 in twelve parts: 4.8 us, and 8.8 by one load after the other)
        constexpr int kAtOnce = 8;
        for (int s0 = 0; s0 < a.splits; s0 += kAtOnce) {
            f32x4 v[kAtOnce];
#pragma unroll
            for (int s = 0; s < kAtOnce; s++) {
                v[s] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (s0 + s < a.splits) v[s] = *(const f32x4*)(from + (int64_t)(s0 + s) * bp * bq);
            }
#pragma unroll
            for (int s = 0; s < kAtOnce; s++)
#pragma unroll
                for (int i = 0; i < 4; i++) z[i] += v[s][i];
        }
        add_bias4<D>(a, col, z);
    }
    if (a.zq) {
        const uint32_t m = group_max8(f2u(keep_larger(keep_larger(keep_larger(keep_larger(0.0f, z[0]), z[1]), z[2]), z[3]))), e = keep_exponent(m);
        if (inside) {
            *(uint32_t*)(a.zq + row * a.np + col) = keep_codes4(z[0], z[1], z[2], z[3], e8m0_inverse(e), m == kInfinity);
            if (col % 32 == 0) a.zs[row * (a.np / 32) + col / 32] = (uint8_t)e;
        }
    }
    if (inside) with_activation(a.act, [&](auto kind) { finish4<D, decltype(kind)::value>(a, row, col, z); });
}

// Operands whose rows do not begin at multiples of 16 bytes, or do not end with a whole piece of eight elements, copied so that they do,
// zeros behind a row's end; blockIdx.y: which of the two.  A wavefront to a row: 777 x 1545 and 1003 x 1545 in 5.8 us.
struct PadArgs {
    const char* from[2];
    char* to[2];
    int64_t rows[2], cols[2], ld[2];
};
__global__ __launch_bounds__(256) void pad_rows_kernel(const PadArgs a) {
    const int which = blockIdx.y;
    if (!a.to[which]) return;
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t cols = a.cols[which], pieces = (cols + 7) / 8, step = (int64_t)gridDim.x * 4;
    for (int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave; row < a.rows[which]; row += step) {
        const char* from = a.from[which] + row * a.ld[which] * 2;
        char* to = a.to[which] + row * pieces * 16;
        constexpr int kAtOnce = 4;
        for (int64_t i = lane; i < pieces; i += kWave * kAtOnce) {
            u32x4 v[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; u++) v[u] = ld_row<MQ_BF16>(from, (i + u * kWave) * 8, cols);
#pragma unroll
            for (int u = 0; u < kAtOnce; u++)
                if (i + u * kWave < pieces) *(u32x4*)(to + (i + u * kWave) * 16) = v[u];
        }
    }
}

// A few tokens (nq <= 16): what counts is reading the weight once, as fast as memory gives it.  A wavefront has 16 rows of the weight and
// a share of k, in steps of 64, and the wavefronts' sums meet in shared memory.  A step's 128 bytes of each row come into shared memory,
// in a ring of the wavefront's own (no barrier), eight lanes to a row: loads straight into the operands of the matrix instruction have
// neighbouring lanes in different rows and pay for each.  Those took, with a weight of 9728 x 2560 that comes from memory, 13.6 us for one
// token and 20.7 us for sixteen; this takes 12.2 and 14.5 (4.1 and 3.4 TB/s); with 151936 x 2560 141 us and 125 (6.2 TB/s).
// DIRECT (aligned rows): straight into shared memory, three steps ahead of the one that is worked on.  Rings of three steps took 16.1 us
// instead of 12.6 with 2560 x 9728, rings of eight 15.2 instead of 12.2 with 9728 x 2560 and 169 instead of 125 with 151936 x 2560, where
// fewer workgroups are on a compute unit; eight wavefronts 15.2 instead of 12.2.  Rows at other addresses come through registers, four
// steps at a time: 9727 x 2559 in 27 us for one token and 35 for sixteen, 2560 x 9729 in 25 and 28, where a copy with aligned rows and the
// tiles of the other kernels take 36 to 37 (the operand's own layout straight from memory: 28, 49, 33 and 60).
struct FewArgs {
    GemmArgs g;
    int64_t k_wave;            // k of a wavefront, a multiple of 64
};
constexpr int kFewWaves = 4, kFewRing = 4;
template <int D, bool DIRECT>
__global__ __launch_bounds__(kFewWaves * kWave) void few_rows_kernel(const FewArgs f) {
    const GemmArgs& a = f.g;
    constexpr int kOperand = 16 * 128, kBuffer = 2 * kOperand;
    __shared__ __attribute__((aligned(1024))) char shared[kFewWaves * kFewRing * kBuffer];
    static_assert(sizeof(shared) >= kFewWaves * 16 * 17 * 4, "the sums fit");
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), j = lane & 15, g = lane >> 4;
    const int64_t p0 = (int64_t)blockIdx.x * 16;
    const int64_t k0 = wave * f.k_wave < a.k ? wave * f.k_wave : a.k, k1 = k0 + f.k_wave < a.k ? k0 + f.k_wave : a.k;
    const int span = (int)(k1 - k0), steps = (span + 63) / 64;
    const char *p = a.p + (p0 * a.ldp + k0) * 2, *q = a.q + k0 * 2;
    MQ_LDS char* lds = (MQ_LDS char*)shared + wave * (kFewRing * kBuffer);
    // 16 bytes for each lane, eight rows at a time; the pieces of a row are in an order that spreads the reads over the banks
    int64_t at_p[2], at_q[2];
    int piece[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const int at = lane + u * kWave, row = at >> 3;
        piece[u] = (at & 7) ^ (at >> 4 & 7);
        at_p[u] = (p0 + row < a.np ? row : a.np - 1 - p0) * a.ldp * 2;
        at_q[u] = (row < a.nq ? row : a.nq - 1) * a.ldq * 2;
    }
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    auto products = [&](MQ_LDS char* from) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t at = (uint32_t)(j * 128 + ((g + 4 * h) ^ (j >> 1 & 7)) * 16);
            acc = mfma<D>(*(MQ_LDS const u32x4*)(from + at), *(MQ_LDS const u32x4*)(from + kOperand + at), acc);
        }
    };
    if (DIRECT) {
        const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
        auto ask = [&](int t) {                            // the same number of accesses for every step, also behind the last
            const int left = span - t * 64;
            const uint32_t to = lds0 + (uint32_t)(t % kFewRing) * kBuffer;
            const u32x4 from_p = buffer_of(p + (int64_t)t * 128), from_q = buffer_of(q + (int64_t)t * 128);
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const bool inside = piece[u] * 8 < left, is_row = ((lane + u * kWave) >> 3) < a.nq;
                direct16(to + u * 1024, from_p, inside ? (uint32_t)at_p[u] + piece[u] * 16 : kNowhere);
                direct16(to + kOperand + u * 1024, from_q, inside && is_row ? (uint32_t)at_q[u] + piece[u] * 16 : kNowhere);
            }
        };
#pragma unroll
        for (int t = 0; t < kFewRing - 1; t++) ask(t);
        for (int t = 0; t < steps; t++) {
            // this step has arrived, and the reads of the one before are done, whose buffer is the next to be filled
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"((kFewRing - 2) * 4) : "memory");
            __builtin_amdgcn_sched_barrier(0);
            ask(t + kFewRing - 1);
            products(lds + (t % kFewRing) * kBuffer);
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    } else {
        u32x4 vp[kFewRing][2], vq[kFewRing][2];
        auto ask = [&](int t) {
            if (t >= steps) return;
            const bool whole = (t + kFewRing) * 64 <= span;
#pragma unroll
            for (int i = 0; i < kFewRing; i++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int64_t c = (t + i) * 64 + piece[u] * 8;
                    vp[i][u] = whole ? ld16_at2(p + at_p[u] + c * 2) : ld_row<D>(p + at_p[u], c, span);
                    vq[i][u] = whole ? ld16_at2(q + at_q[u] + c * 2) : ld_row<D>(q + at_q[u], c, span);
                }
        };
        ask(0);
        for (int t = 0; t < steps; t += kFewRing) {
#pragma unroll
            for (int i = 0; i < kFewRing; i++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    *(MQ_LDS u32x4*)(lds + i * kBuffer + (lane + u * kWave) * 16) = vp[i][u];
                    *(MQ_LDS u32x4*)(lds + i * kBuffer + kOperand + (lane + u * kWave) * 16) = vq[i][u];
                }
            ask(t + kFewRing);
            lanes_meet();
#pragma unroll
            for (int i = 0; i < kFewRing; i++) products(lds + i * kBuffer);
            lanes_meet();
        }
    }
    __syncthreads();
    float* sums = (float*)shared;                          // [wave][row of x][17]
#pragma unroll
    for (int x = 0; x < 4; x++) sums[(wave * 16 + j) * 17 + g * 4 + x] = acc[x];
    __syncthreads();
    const int row = threadIdx.x / 16, c = threadIdx.x % 16;
    static_assert(kFewWaves * kWave == 256, "a thread for each output");
    if (row >= a.nq || p0 + c >= a.np) return;
    float z = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewWaves; w++) z += sums[(w * 16 + row) * 17 + c];
    const int64_t at = row * a.np + p0 + c;
    if (a.bias) z += one_elem<D>(a.bias, p0 + c);
    if (a.z) store_dtype(a.z, at, z, D);
    float y = z;
    with_activation(a.act, [&](auto kind) { y = activate<decltype(kind)::value>(z); });
    if (a.res) y += one_elem<D>(a.res, row * a.ldr + p0 + c);
    store_dtype(a.out, at, y, D);
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

// dz = dy act'(z) and the sums of its columns.  dz is rounded to the tensors' type, because the matrix instructions that take it further
// have 16-bit operands (a gradient's error is then that of two such roundings, 2.3e-3 of its size in bf16 where one makes 1.7e-3); the
// sums are of what was not rounded.  A wavefront goes down rows of 512 columns, eight to a lane, so that a column's sum
// stays in a register; the four wavefronts of a workgroup take turns and their sums meet in shared memory.  Near what
// memory allows, the slope's arithmetic close behind it: 8192 x 9728 bf16, GELU from 8 bits 82 us (4.9 TB/s), from 16 bits 99 (4.8), the
// bias alone 31 (5.2); two or four rows' loads at once are no faster.
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
            float g[8], z[8];
            unpack<D>(ld_row<D>(a.dy + row * a.lddy * 2, col, a.n), g);
            if (ACT != MQ_ACT_NONE) {
                if (!KEPT) {
                    unpack<D>(ld_row<D>(a.z + row * a.n * 2, col, a.n), z);
                } else {
                    u32x2 c = {0u, 0u};
                    float s = 0.0f;
                    if (col < a.n) {
                        c = *(const u32x2*)(a.z + row * a.n + col);
                        s = e8m0_value(a.zs[row * (a.n / 32) + col / 32]);
                    }
                    kept_values4(c.x, s, z);
                    kept_values4(c.y, s, z + 4);
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

// How a product of np columns, nq rows and k runs: the tile, and which tiles are cut along k.  Tiles that fill every place on the card
// run whole, round by round; those of a last round that would leave places empty (all of them, of a small product) are cut into as
// many parts as fill it.  Each candidate's time is estimated from its rounds and the bytes of its partial sums; the constants were
// fitted to 44 products measured with every tile and up to ten numbers of parts, where the choice loses 1 % against the best.  Some of
// them (M x N x K, us by 256 x 256, 128 x 128, 128 x 64): 4099 x 2560 x 4096 92, 105, 116; 12544 x 1152 x 2192 70, 85, 104;
// 2048 x 2048 x 2048 41, 32, 25; 512 x 4096 x 4096 40, 36, 34, and uncut 76, 54, 35; 48 x 2560 x 9728 26, 21, 17, and uncut 156, 114, 70.
static GemmPlan gemm_plan(bool weight_grad, int64_t np, int64_t nq, int64_t k) {
    struct Cost {
        int per_cu;
        double least_us, step_us, tile_us;                // of a step, of a step for each workgroup on the compute unit, and besides the steps
    };
    static const Cost costs[4] = {{1, 0.79, 0.93, 8.5}, {2, 0.68, 0.48, 3.2}, {2, 0.32, 0.32, 2.0}, {3, 0.49, 0.34, 1.6}};
    const int64_t steps = k > 0 ? (k + kStep - 1) / kStep : 1;
    GemmPlan best{};
    double best_us = 1e30;
    for (int t = kTileLarge; t <= kTileLow; t++) {
        const Cost& cost = costs[t == kTileLow && weight_grad ? 3 : t];
        const int64_t tiles_p = (np + kTileP[t] - 1) / kTileP[t], tiles_q = (nq + kTileQ[t] - 1) / kTileQ[t];
        const int64_t tiles = tiles_p * tiles_q, places = 256 * cost.per_cu, rest = tiles % places;
        auto round_us = [&](int64_t count, int64_t n_steps) {      // so many workgroups at once, of so many steps
            const double step = cost.step_us * (double)((count + 255) / 256);
            return (double)n_steps * (step > cost.least_us ? step : cost.least_us) + cost.tile_us;
        };
        const double whole_us = (double)(tiles / places) * round_us(places, steps);
        for (int64_t splits = 1; splits <= 64; splits++) {
            const int64_t per = (steps + splits - 1) / splits;
            if (splits > 1 && (rest == 0 || per < 2 || (steps + per - 1) / per != splits)) continue;
            const int64_t parts = rest * splits;
            double us = whole_us + (double)(parts / places) * round_us(places, per);
            if (parts % places) us += round_us(parts % places, per);
            if (splits > 1) us += 2.5 + (double)parts * kTileP[t] * (double)(nq < kTileQ[t] ? nq : kTileQ[t]) * 8 / 5.3e6;
            if (us < best_us) {
                best_us = us;
                best = GemmPlan{t, (int)tiles_p, (int)tiles_q, (int)(splits > 1 ? tiles - rest : tiles), (int)splits, per * kStep};
            }
        }
    }
    return best;
}
static int64_t partial_floats(const GemmPlan& plan) {
    return (int64_t)(plan.tiles_p * plan.tiles_q - plan.whole) * plan.splits * kTileP[plan.tile] * kTileQ[plan.tile];
}

static bool direct_ok(const void* p, int64_t ld, int64_t cols) {
    return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && cols % 8 == 0 && ld < (1 << 22);
}
// joins the parts, if there are any
static int join(int dtype, const GemmArgs& a, const GemmPlan& plan, hipStream_t st) {
    const int cut = plan.tiles_p * plan.tiles_q - plan.whole, bp = kTileP[plan.tile], bq = kTileQ[plan.tile];
    if (cut > 0) {
        const dim3 grid((unsigned)(cut * (bp * bq / 1024)));
        if (dtype == MQ_F16) hipLaunchKernelGGL(gemm_join_kernel<MQ_F16>, grid, dim3(256), 0, st, a, bp, bq);
        else hipLaunchKernelGGL(gemm_join_kernel<MQ_BF16>, grid, dim3(256), 0, st, a, bp, bq);
    }
    return mq_check_launch("linear");
}

// A product as it is run: sizes and operands (P the first, p_rows x p_cols in memory), and what of the workspace is whose.
struct Product {
    const void *p, *q;
    int64_t ldp, ldq, p_rows, p_cols, q_rows, q_cols, np, nq, k;
    bool kept, few;
    GemmPlan plan;
    int64_t p_at, q_at, bytes;     // where the operands' copies are, -1 for none

    Product(int product, const void* a, int64_t lda, const void* b, int64_t ldb, bool kept_, bool few_, int64_t M, int64_t N, int64_t K)
        : p(b), q(a), ldp(ldb), ldq(lda), kept(kept_), few(few_) {
        const bool weight_grad = product == MQ_LINEAR_WEIGHT_GRAD, forward = product == MQ_LINEAR_FORWARD;
        p_rows = weight_grad ? M : N, p_cols = K;
        q_rows = M, q_cols = forward ? K : N;
        np = forward ? N : K, nq = weight_grad ? N : M, k = forward ? K : weight_grad ? M : N;
        plan = few ? GemmPlan{} : gemm_plan(weight_grad, np, nq, k);
        bytes = few ? 0 : partial_floats(plan) * 4;
        p_at = few || kept ? -1 : copy_at(p, ldp, p_rows, p_cols);
        q_at = few ? -1 : copy_at(q, ldq, q_rows, q_cols);
    }
    int64_t copy_at(const void* at, int64_t ld, int64_t rows, int64_t cols) {
        if (direct_ok(at, rows > 1 ? ld : 8, cols)) return -1;
        const int64_t here = bytes;
        bytes += rows * ((cols + 7) / 8 * 8) * 2;          // (a multiple of 16)
        return here;
    }
    // the arguments, with the operands copied into the workspace where that is needed
    int arguments(GemmArgs& a, char* ws, hipStream_t st) const {
        if (bytes > 0 && (!ws || (uintptr_t)ws % 16)) return mq_fail(MQ_ERR_ARG, "linear: a 16-byte aligned workspace is needed");
        a.p = (const char*)p, a.q = (const char*)q, a.ldp = ldp, a.ldq = ldq, a.np = np, a.nq = nq, a.k = k;
        PadArgs pad{};
        int64_t most = 0;
        auto copy = [&](int i, const char*& operand, int64_t& ld, int64_t at, int64_t rows, int64_t cols) {
            if (at < 0) return;
            pad.from[i] = operand, pad.ld[i] = ld, pad.rows[i] = rows, pad.cols[i] = cols, pad.to[i] = ws + at;
            operand = ws + at, ld = (cols + 7) / 8 * 8;
            if (rows > most) most = rows;
        };
        copy(0, a.p, a.ldp, p_at, p_rows, p_cols);
        copy(1, a.q, a.ldq, q_at, q_rows, q_cols);
        if (most > 0) {
            const int64_t blocks = (most + 3) / 4;
            hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096), 2), dim3(256), 0, st, pad);
        }
        return MQ_OK;
    }
};
// few tokens, and nothing that needs 32 columns at once (sixteen, with 9728 x 2560: 14.5 us, by tiles 17.1; the same kernel with two
// such operands took 20.9 us for 32 with 2560 x 9728, where tiles take 15.8 for 17 and 17.0 for 48)
static bool few_rows(int product, int64_t M, bool z8) { return product == MQ_LINEAR_FORWARD && M <= 16 && !z8; }

static int check_product(int product, const void* a, int64_t lda, const void* b, int64_t ldb, bool kept, int64_t M, int64_t N, int64_t K) {
    if (M < 0 || N < 0 || K < 0) return mq_fail(MQ_ERR_ARG, "linear: bad argument");
    // (a lane's offsets into 256 rows of an operand are 32-bit numbers)
    if (M > 0x7FFFFF00 || N >= 1 << 22 || K >= 1 << 22) return mq_fail(MQ_ERR_ARG, "linear: tensor too large");
    const bool forward = product == MQ_LINEAR_FORWARD, weight_grad = product == MQ_LINEAR_WEIGHT_GRAD;
    if ((M > 1 && lda < (forward ? K : N)) || (!kept && (weight_grad ? M : N) > 1 && ldb < K)) return mq_fail(MQ_ERR_ARG, "linear: rows overlap");
    const int64_t np = forward ? N : K, nq = weight_grad ? N : M;
    if (((np + 127) / 128) * ((nq + 63) / 64) > 0x7FFFFF) return mq_fail(MQ_ERR_ARG, "linear: tensor too large");
    return MQ_OK;
}
static int check_dtype(int dtype) { return dtype != MQ_BF16 && dtype != MQ_F16 ? mq_fail(MQ_ERR_ARG, "linear: bf16 or fp16") : MQ_OK; }

extern "C" int mq_linear_workspace(int product, const void* a, int64_t lda, const void* b, int64_t ldb, int kept8, int64_t M, int64_t N, int64_t K,
                                   int64_t* bytes) {
    if (!bytes || product < MQ_LINEAR_FORWARD || product > MQ_LINEAR_WEIGHT_GRAD) return mq_fail(MQ_ERR_ARG, "linear: bad argument");
    const bool kept = product == MQ_LINEAR_WEIGHT_GRAD && kept8;
    if (const int rc = check_product(product, a, lda, b, ldb, kept, M, N, K)) return rc;
    *bytes = 0;
    if ((product != MQ_LINEAR_WEIGHT_GRAD && M == 0) || (product != MQ_LINEAR_INPUT_GRAD && N == 0) || (product != MQ_LINEAR_FORWARD && K == 0)) return MQ_OK;
    *bytes = Product(product, a, lda, b, ldb, kept, few_rows(product, M, kept8 != 0), M, N, K).bytes;
    return MQ_OK;
}

extern "C" int mq_linear_forward(const void* x, int dtype, int64_t ldx, const void* weight, int64_t ldw, const void* bias, int act,
                                 const void* residual, int64_t ldr, void* y, void* z, void* z8, uint8_t* z8_scale, int64_t M, int64_t N,
                                 int64_t K, void* ws, void* stream) {
    if (const int rc = check_dtype(dtype)) return rc;
    if (const int rc = check_product(MQ_LINEAR_FORWARD, x, ldx, weight, ldw, false, M, N, K)) return rc;
    if (act < MQ_ACT_NONE || act > MQ_ACT_GELU_TANH) return mq_fail(MQ_ERR_ARG, "linear: unknown activation");
    if (residual && M > 1 && ldr < N) return mq_fail(MQ_ERR_ARG, "linear: rows overlap");
    if (M == 0 || N == 0) return MQ_OK;
    if (!y || (K > 0 && (!x || !weight)) || !z8 != !z8_scale) return mq_fail(MQ_ERR_ARG, "linear: null pointer");
    if (z8 && (N % 32 != 0 || (uintptr_t)z8 % 4)) return mq_fail(MQ_ERR_ARG, "linear: columns kept in 8 bits are a multiple of 32, 4-byte aligned");
    const hipStream_t st = (hipStream_t)stream;
    const Product product(MQ_LINEAR_FORWARD, x, ldx, weight, ldw, false, few_rows(MQ_LINEAR_FORWARD, M, z8 != nullptr), M, N, K);
    FewArgs few{};
    GemmArgs& a = few.g;
    if (const int rc = product.arguments(a, (char*)ws, st)) return rc;
    a.out = (char*)y, a.bias = (const char*)bias, a.res = (const char*)residual, a.ldr = ldr;
    a.z = (char*)z, a.zq = (uint8_t*)z8, a.zs = z8_scale, a.act = act;
    if (product.few) {
        few.k_wave = (K + kFewWaves * 64 - 1) / (kFewWaves * 64) * 64;
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)((N + 15) / 16)), dim3(kFewWaves * kWave), 0, st, few); };
        if (direct_ok(x, M > 1 ? ldx : 8, K) && direct_ok(weight, N > 1 ? ldw : 8, K)) {
            go(dtype == MQ_F16 ? few_rows_kernel<MQ_F16, true> : few_rows_kernel<MQ_BF16, true>);
        } else {
            go(dtype == MQ_F16 ? few_rows_kernel<MQ_F16, false> : few_rows_kernel<MQ_BF16, false>);
        }
        return mq_check_launch("linear");
    }
    if (const int rc = mq_gemm_forward(dtype, a, product.plan, (float*)ws, st)) return rc;
    return join(dtype, a, product.plan, st);
}

extern "C" int mq_linear_input_grad(const void* dz, int dtype, int64_t lddz, const void* weight, int64_t ldw, void* dx, int64_t M, int64_t N,
                                    int64_t K, void* ws, void* stream) {
    if (const int rc = check_dtype(dtype)) return rc;
    if (const int rc = check_product(MQ_LINEAR_INPUT_GRAD, dz, lddz, weight, ldw, false, M, N, K)) return rc;
    if (M == 0 || K == 0) return MQ_OK;
    if (!dx || (N > 0 && (!dz || !weight))) return mq_fail(MQ_ERR_ARG, "linear: null pointer");
    const hipStream_t st = (hipStream_t)stream;
    const Product product(MQ_LINEAR_INPUT_GRAD, dz, lddz, weight, ldw, false, false, M, N, K);
    GemmArgs a{};
    if (const int rc = product.arguments(a, (char*)ws, st)) return rc;
    a.out = (char*)dx;
    if (const int rc = mq_gemm_input_grad(dtype, a, product.plan, (float*)ws, st)) return rc;
    return join(dtype, a, product.plan, st);
}

extern "C" int mq_linear_weight_grad(const void* dz, int dtype, int64_t lddz, const void* x, int64_t ldx, const uint8_t* x_scale, void* dweight,
                                     int64_t M, int64_t N, int64_t K, void* ws, void* stream) {
    if (const int rc = check_dtype(dtype)) return rc;
    if (x_scale) ldx = K;
    if (const int rc = check_product(MQ_LINEAR_WEIGHT_GRAD, dz, lddz, x, ldx, x_scale != nullptr, M, N, K)) return rc;
    if (N == 0 || K == 0) return MQ_OK;
    if (!dweight || (M > 0 && (!dz || !x))) return mq_fail(MQ_ERR_ARG, "linear: null pointer");
    if (x_scale && (K % 32 != 0 || (uintptr_t)x % 16)) return mq_fail(MQ_ERR_ARG, "linear: an 8-bit copy has a multiple of 32 columns and is 16-byte aligned");
    const hipStream_t st = (hipStream_t)stream;
    const Product product(MQ_LINEAR_WEIGHT_GRAD, dz, lddz, x, ldx, x_scale != nullptr, false, M, N, K);
    GemmArgs a{};
    if (const int rc = product.arguments(a, (char*)ws, st)) return rc;
    a.ps = x_scale, a.out = (char*)dweight;
    if (const int rc = mq_gemm_weight_grad(dtype, a, product.plan, (float*)ws, st)) return rc;
    return join(dtype, a, product.plan, st);
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
    if (const int rc = check_dtype(dtype)) return rc;
    if (M < 0 || N < 0) return mq_fail(MQ_ERR_ARG, "linear: bad argument");
    if (M > 0x7FFFFF00 || N > 0x1FFFFF00) return mq_fail(MQ_ERR_ARG, "linear: tensor too large");      // (eight lanes to a column of the sums, 2^32 to a launch)
    if (act < MQ_ACT_NONE || act > MQ_ACT_GELU_TANH) return mq_fail(MQ_ERR_ARG, "linear: unknown activation");
    if (M > 1 && lddy < N) return mq_fail(MQ_ERR_ARG, "linear: rows overlap");
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
