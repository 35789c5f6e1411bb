// Layer norm and RMS norm, forward and backward, for gfx950.
//
//   mean = sum(x) / n (0 for RMS norm), var = sum((x - mean)^2) / n, rstd = 1 / sqrt(var + eps),
//   xhat = (x - mean) rstd, y = xhat w + b;
//   g = dy w, dx = rstd (g - mean(g) - xhat mean(g xhat)) (no mean(g) for RMS norm), dw = sum over rows of dy xhat, db of dy.
//
// Both directions are bound by HBM: a row is read once, stays in the registers of one wavefront (rows of at most two accesses a
// lane) or one workgroup, and both statistics are taken from there, the variance around the mean of the row itself.
// Sums and statistics are fp32.  Kept for the backward pass: x, mean and rstd; or xhat in 8 bits (e4m3, an exponent for each
// 32 columns) and rstd, which is 1.03 bytes per element instead of two or four.
#include "mq_rows.hpp"

namespace mq {

struct NormArgs {
    const void* x;
    const void* w;             // null: no weight
    const void* b;             // null: no bias
    void* y;
    uint8_t *xq, *xs;          // xhat in 8 bits, or null
    uint8_t *yq, *ys;          // y in 8 bits, or null
    float *mean, *rstd;        // null: not kept
    int64_t rows, n, ldx;
    float eps;
    int rms;
};

// the sum over the LANES lanes of a row, in every one of them; `part`: LANES / 64 words for this use alone
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* part) {
    v = wave_sum(v);
    if (LANES == kWave) return v;
    const int wave = threadIdx.x / kWave;
    if ((threadIdx.x & (kWave - 1)) == 0) part[wave] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < LANES / kWave; i++) s += part[i];
    return s;
}

// An 8-bit copy of the V values that a lane holds of a row: the lanes of 32 neighbouring columns are neighbours.  n is a multiple of
// 32, so that a group's lanes are inside the row or outside together.
template <int D>
__device__ __forceinline__ void keep_row(const float* f, int64_t c, int64_t n, uint8_t* q, uint8_t* s) {
    constexpr int V = kVec<D>;
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < V; j++) m = umax(m, keep_magnitude(f[j]));
    m = D == MQ_F32 ? group_max8(m) : group_max4(m);
    const uint32_t e = keep_exponent(m);
    const float inv = e8m0_inverse(e);
    if (c < n) {
        const uint32_t lo = keep_codes4(f[0], f[1], f[2], f[3], inv);
        if (D == MQ_F32) {
            *(uint32_t*)(q + c) = lo;
        } else {
            *(u32x2*)(q + c) = u32x2{lo, keep_codes4(f[V - 4], f[V - 3], f[V - 2], f[V - 1], inv)};
        }
        if (c % 32 == 0) s[c / 32] = (uint8_t)e;
    }
}

template <int D, int WF32, int LANES, int UNITS>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void norm_fwd_kernel(const NormArgs a) {
    constexpr int V = kVec<D>, kRows = LANES < 256 ? 256 / LANES : 1;
    __shared__ float part[2][LANES / kWave];
    const int lane = threadIdx.x % LANES;
    const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / LANES;
    if (row >= a.rows) return;           // (only where a row has a wavefront of its own: nobody waits for it)
    const char* x = (const char*)a.x + row * a.ldx * kElem<D>;
    float v[UNITS][V];
#pragma unroll
    for (int u = 0; u < UNITS; u++) unpack<D>(ld_row<D>(x, (int64_t)(u * LANES + lane) * V, a.n), v[u]);
    const float inv_n = 1.0f / (float)a.n;
    float mean = 0.0f;
    if (!a.rms) {
        float s = 0.0f;
#pragma unroll
        for (int u = 0; u < UNITS; u++)
#pragma unroll
            for (int j = 0; j < V; j++) s += v[u][j];
        mean = row_sum<LANES>(s, part[0]) * inv_n;
    }
    float s2 = 0.0f;
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
        const int64_t c = (int64_t)(u * LANES + lane) * V;
#pragma unroll
        for (int j = 0; j < V; j++) {
            v[u][j] = c + j < a.n ? v[u][j] - mean : 0.0f;
            s2 += v[u][j] * v[u][j];
        }
    }
    const float rstd = 1.0f / __builtin_sqrtf(row_sum<LANES>(s2, part[1]) * inv_n + a.eps);
    if (lane == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
        const int64_t c = (int64_t)(u * LANES + lane) * V;
        float f[V], w[V];
#pragma unroll
        for (int j = 0; j < V; j++) f[j] = v[u][j] * rstd;
        if (a.xq) keep_row<D>(f, c, a.n, a.xq + row * a.n, a.xs + row * (a.n / 32));
        if (a.w) {
            ld_vector<D, WF32>(a.w, c, a.n, w);
#pragma unroll
            for (int j = 0; j < V; j++) f[j] *= w[j];
        }
        if (a.b) {
            ld_vector<D, WF32>(a.b, c, a.n, w);
#pragma unroll
            for (int j = 0; j < V; j++) f[j] += w[j];
        }
        const u32x4 out = pack<D>(f);
        st_row<D>((char*)a.y + row * a.n * kElem<D>, c, a.n, out);
        if (a.yq) {
            unpack<D>(out, f);           // the copy stands for y as it is stored
            keep_row<D>(f, c, a.n, a.yq + row * a.n, a.ys + row * (a.n / 32));
        }
    }
}

// Rows too long for the registers of a workgroup: three passes over the row, which the caches hold.
template <int D, int WF32>
__global__ __launch_bounds__(1024) void norm_fwd_long_kernel(const NormArgs a) {
    constexpr int V = kVec<D>, kLanes = 1024;
    __shared__ float part[2][kLanes / kWave];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const char* x = (const char*)a.x + row * a.ldx * kElem<D>;
    const float inv_n = 1.0f / (float)a.n;
    float mean = 0.0f, f[V], w[V];
    if (!a.rms) {
        float s = 0.0f;
        for (int64_t c = (int64_t)lane * V; c < a.n; c += kLanes * V) {
            unpack<D>(ld_row<D>(x, c, a.n), f);
#pragma unroll
            for (int j = 0; j < V; j++) s += f[j];
        }
        mean = row_sum<kLanes>(s, part[0]) * inv_n;
    }
    float s2 = 0.0f;
    for (int64_t c = (int64_t)lane * V; c < a.n; c += kLanes * V) {
        unpack<D>(ld_row<D>(x, c, a.n), f);
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float d = c + j < a.n ? f[j] - mean : 0.0f;
            s2 += d * d;
        }
    }
    const float rstd = 1.0f / __builtin_sqrtf(row_sum<kLanes>(s2, part[1]) * inv_n + a.eps);
    if (lane == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
    // whole wavefronts stay together: the 8-bit copies take maxima over lanes
    for (int64_t c0 = 0; c0 < a.n; c0 += kLanes * V) {
        const int64_t c = c0 + (int64_t)lane * V;
        unpack<D>(ld_row<D>(x, c, a.n), f);
#pragma unroll
        for (int j = 0; j < V; j++) f[j] = c + j < a.n ? (f[j] - mean) * rstd : 0.0f;
        if (a.xq) keep_row<D>(f, c, a.n, a.xq + row * a.n, a.xs + row * (a.n / 32));
        if (a.w) {
            ld_vector<D, WF32>(a.w, c, a.n, w);
#pragma unroll
            for (int j = 0; j < V; j++) f[j] *= w[j];
        }
        if (a.b) {
            ld_vector<D, WF32>(a.b, c, a.n, w);
#pragma unroll
            for (int j = 0; j < V; j++) f[j] += w[j];
        }
        const u32x4 out = pack<D>(f);
        st_row<D>((char*)a.y + row * a.n * kElem<D>, c, a.n, out);
        if (a.yq) {
            unpack<D>(out, f);
            keep_row<D>(f, c, a.n, a.yq + row * a.n, a.ys + row * (a.n / 32));
        }
    }
}

struct NormGradArgs {
    const void* dy;
    const void* x;             // the input, or (KEPT) the 8-bit xhat
    const uint8_t* xs;
    const float *mean, *rstd;
    const void* w;
    void* dx;                  // null: not wanted
    float *dw, *db;            // partial sums [parts][n], null: not wanted
    int64_t rows, n, lddy, ldx, parts;
    int rms;
};

// the kVec normalized values of a row from column c on, zero outside
template <int D, int KEPT>
__device__ __forceinline__ void ld_xhat(const NormGradArgs& a, int64_t row, int64_t c, float mean, float rstd, float* f) {
    constexpr int V = kVec<D>;
    if (KEPT) {
#pragma unroll
        for (int j = 0; j < V; j++) f[j] = 0.0f;
        if (c < a.n) {
            const float scale = e8m0_value(a.xs[row * (a.n / 32) + c / 32]);
            const uint8_t* q = (const uint8_t*)a.x + row * a.n + c;
            if (D == MQ_F32) kept_values4(*(const uint32_t*)q, scale, f);
            else {
                const u32x2 v = *(const u32x2*)q;
                kept_values4(v.x, scale, f);
                kept_values4(v.y, scale, f + (V - 4));
            }
        }
    } else {
        unpack<D>(ld_row<D>((const char*)a.x + row * a.ldx * kElem<D>, c, a.n), f);
#pragma unroll
        for (int j = 0; j < V; j++) f[j] = c + j < a.n ? (f[j] - mean) * rstd : 0.0f;
    }
}

// A workgroup goes through rows far apart (`parts` sets of lanes in all) and keeps its columns' sums in registers; the partial
// sums are added by column_sum_kernel in a fixed order.
template <int D, int WF32, int KEPT, int LANES, int UNITS>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void norm_bwd_kernel(const NormGradArgs a) {
    constexpr int V = kVec<D>, kRows = LANES < 256 ? 256 / LANES : 1;
    __shared__ float part[2][2][LANES / kWave];
    const int lane = threadIdx.x % LANES;
    const int64_t mine = (int64_t)blockIdx.x * kRows + threadIdx.x / LANES;
    const float inv_n = 1.0f / (float)a.n;
    float dw[UNITS][V], db[UNITS][V], w[UNITS][V];
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
        if (a.w) ld_vector<D, WF32>(a.w, (int64_t)(u * LANES + lane) * V, a.n, w[u]);
#pragma unroll
        for (int j = 0; j < V; j++) {
            dw[u][j] = db[u][j] = 0.0f;
            if (!a.w) w[u][j] = 1.0f;
        }
    }
    int turn = 0;
    for (int64_t row = mine; row < a.rows; row += a.parts, turn ^= 1) {
        const float mean = KEPT || a.rms ? 0.0f : a.mean[row], rstd = a.rstd[row];
        float g[UNITS][V], xh[UNITS][V], sg = 0.0f, sgx = 0.0f;
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            const int64_t c = (int64_t)(u * LANES + lane) * V;
            unpack<D>(ld_row<D>((const char*)a.dy + row * a.lddy * kElem<D>, c, a.n), g[u]);
            ld_xhat<D, KEPT>(a, row, c, mean, rstd, xh[u]);
        }
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                dw[u][j] += g[u][j] * xh[u][j];
                db[u][j] += g[u][j];
                g[u][j] *= w[u][j];
                sg += g[u][j];
                sgx += g[u][j] * xh[u][j];
            }
        }
        if (!a.dx) continue;
        // two sums with one wait between the wavefronts; the words are used every other row, so that a fast wavefront's next
        // sums do not meet a slow one's reading of these
        sg = wave_sum(sg);
        sgx = wave_sum(sgx);
        if (LANES > kWave) {
            if ((threadIdx.x & (kWave - 1)) == 0) {
                part[turn][0][threadIdx.x / kWave] = sg;
                part[turn][1][threadIdx.x / kWave] = sgx;
            }
            __syncthreads();
            sg = sgx = 0.0f;
#pragma unroll
            for (int i = 0; i < LANES / kWave; i++) {
                sg += part[turn][0][i];
                sgx += part[turn][1][i];
            }
        }
        const float mg = a.rms ? 0.0f : sg * inv_n, mgx = sgx * inv_n;
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            float f[V];
#pragma unroll
            for (int j = 0; j < V; j++) f[j] = (g[u][j] - mg - xh[u][j] * mgx) * rstd;
            st_row<D>((char*)a.dx + row * a.n * kElem<D>, (int64_t)(u * LANES + lane) * V, a.n, pack<D>(f));
        }
    }
    if (mine < a.parts) {
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            const int64_t c = (int64_t)(u * LANES + lane) * V;
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                if (a.dw) st_row<MQ_F32>(a.dw + mine * a.n, c + j, a.n, pack<MQ_F32>(&dw[u][j]));
                if (a.db) st_row<MQ_F32>(a.db + mine * a.n, c + j, a.n, pack<MQ_F32>(&db[u][j]));
            }
        }
    }
}

// Long rows: dx by three passes over the row; the columns' sums by norm_bwd_long_sums_kernel, which goes down the columns.
template <int D, int WF32, int KEPT>
__global__ __launch_bounds__(1024) void norm_bwd_long_kernel(const NormGradArgs a) {
    constexpr int V = kVec<D>, kLanes = 1024;
    __shared__ float part[2][kLanes / kWave];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const float inv_n = 1.0f / (float)a.n, mean = KEPT || a.rms ? 0.0f : a.mean[row], rstd = a.rstd[row];
    float g[V], xh[V], w[V], sg = 0.0f, sgx = 0.0f;
#pragma unroll
    for (int j = 0; j < V; j++) w[j] = 1.0f;
    for (int64_t c = (int64_t)lane * V; c < a.n; c += kLanes * V) {
        unpack<D>(ld_row<D>((const char*)a.dy + row * a.lddy * kElem<D>, c, a.n), g);
        ld_xhat<D, KEPT>(a, row, c, mean, rstd, xh);
        if (a.w) ld_vector<D, WF32>(a.w, c, a.n, w);
#pragma unroll
        for (int j = 0; j < V; j++) {
            sg += g[j] * w[j];
            sgx += g[j] * w[j] * xh[j];
        }
    }
    const float mg = row_sum<kLanes>(sg, part[0]) * inv_n, mgx = row_sum<kLanes>(sgx, part[1]) * inv_n;
    for (int64_t c = (int64_t)lane * V; c < a.n; c += kLanes * V) {
        unpack<D>(ld_row<D>((const char*)a.dy + row * a.lddy * kElem<D>, c, a.n), g);
        ld_xhat<D, KEPT>(a, row, c, mean, rstd, xh);
        if (a.w) ld_vector<D, WF32>(a.w, c, a.n, w);
#pragma unroll
        for (int j = 0; j < V; j++) g[j] = (g[j] * w[j] - (a.rms ? 0.0f : mg) - xh[j] * mgx) * rstd;
        st_row<D>((char*)a.dx + row * a.n * kElem<D>, c, a.n, pack<D>(g));
    }
}
template <int D, int KEPT>
__global__ __launch_bounds__(256) void norm_bwd_long_sums_kernel(const NormGradArgs a) {
    constexpr int V = kVec<D>;
    const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V, mine = blockIdx.y;
    if (c >= a.n) return;
    float dw[V], db[V], g[V], xh[V];
#pragma unroll
    for (int j = 0; j < V; j++) dw[j] = db[j] = 0.0f;
    for (int64_t row = mine; row < a.rows; row += a.parts) {
        const float mean = KEPT || a.rms ? 0.0f : a.mean[row];
        unpack<D>(ld_row<D>((const char*)a.dy + row * a.lddy * kElem<D>, c, a.n), g);
        ld_xhat<D, KEPT>(a, row, c, mean, a.rstd[row], xh);
#pragma unroll
        for (int j = 0; j < V; j++) {
            dw[j] += g[j] * xh[j];
            db[j] += g[j];
        }
    }
#pragma unroll
    for (int j = 0; j < V; j += 4) {
        if (a.dw) st_row<MQ_F32>(a.dw + mine * a.n, c + j, a.n, pack<MQ_F32>(&dw[j]));
        if (a.db) st_row<MQ_F32>(a.db + mine * a.n, c + j, a.n, pack<MQ_F32>(&db[j]));
    }
}

// out[c] = sum over `parts` rows of partial sums [parts][n], blockIdx.y the first or the second set.  Eight lanes own 32 columns (a
// line), 32 of them go down the rows, and their sums meet in shared memory.
struct ColumnSumArgs {
    const float* part[2];
    void* out[2];
    int64_t parts, n;
    int dtype;
};
__global__ __launch_bounds__(256) void column_sum_kernel(const ColumnSumArgs a) {
    __shared__ float sums[32][33];
    const float* p = a.part[blockIdx.y];
    const int col = threadIdx.x % 8 * 4, down = threadIdx.x / 8;
    const int64_t c = (int64_t)blockIdx.x * 32 + col;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f}, f[4];
    for (int64_t r = down; r < a.parts; r += 32) {
        unpack<MQ_F32>(ld_row<MQ_F32>(p + r * a.n, c, a.n), f);
#pragma unroll
        for (int j = 0; j < 4; j++) s[j] += f[j];
    }
#pragma unroll
    for (int j = 0; j < 4; j++) sums[down][col + j] = s[j];
    __syncthreads();
    if (threadIdx.x < 32) {
        float total = 0.0f;
        for (int i = 0; i < 32; i++) total += sums[i][threadIdx.x];
        const int64_t at = (int64_t)blockIdx.x * 32 + threadIdx.x;
        if (at < a.n) store_dtype(a.out[blockIdx.y], at, total, a.dtype);
    }
}

}  // namespace mq

using namespace mq;

int mq_column_sum_launch(const float* p0, void* out0, const float* p1, void* out1, int64_t parts, int64_t n, int dtype, hipStream_t st) {
    ColumnSumArgs a{{out0 ? p0 : p1, p1}, {out0 ? out0 : out1, out1}, parts, n, dtype};
    const unsigned sets = (out0 ? 1 : 0) + (out1 ? 1 : 0);
    if (sets == 0) return MQ_OK;
    hipLaunchKernelGGL(column_sum_kernel, dim3((unsigned)((n + 31) / 32), sets), dim3(256), 0, st, a);
    return mq_check_launch("column sums");
}

// Lanes and accesses of a row of n elements, V to an access: the fewest registers that hold it, a wavefront for short rows (no
// wait between wavefronts), and beyond 1024 lanes of four accesses the long forms.
template <class F>
static void norm_shape(int64_t n, int V, F&& f) {
    const int64_t units = (n + V - 1) / V;
    if (units <= 64) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    else if (units <= 128) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    else if (units <= 256) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
    else if (units <= 512) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    else if (units <= 1024) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
    else if (units <= 2048) f(std::integral_constant<int, 512>{}, std::integral_constant<int, 4>{});
    else if (units <= 4096) f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 4>{});
    else f(std::integral_constant<int, 0>{}, std::integral_constant<int, 0>{});
}

template <class F>
static void norm_types(int dtype, int wdtype, F&& f) {
    const bool wide = wdtype == MQ_F32;
    if (dtype == MQ_F32) f(std::integral_constant<int, MQ_F32>{}, std::integral_constant<int, 1>{});
    else if (dtype == MQ_F16 && wide) f(std::integral_constant<int, MQ_F16>{}, std::integral_constant<int, 1>{});
    else if (dtype == MQ_F16) f(std::integral_constant<int, MQ_F16>{}, std::integral_constant<int, 0>{});
    else if (wide) f(std::integral_constant<int, MQ_BF16>{}, std::integral_constant<int, 1>{});
    else f(std::integral_constant<int, MQ_BF16>{}, std::integral_constant<int, 0>{});
}

static int norm_check(int dtype, int wdtype, int64_t rows, int64_t n, int64_t ld) {
    if (dtype < MQ_BF16 || dtype > MQ_F32 || rows < 0 || n < 0) return mq_fail(MQ_ERR_ARG, "norm: bad argument");
    if (wdtype != dtype && wdtype != MQ_F32) return mq_fail(MQ_ERR_ARG, "norm: the weight has the input's type or is fp32");
    if (rows > 1 && ld < n) return mq_fail(MQ_ERR_ARG, "norm: rows overlap");
    if (rows > 0x7FFFFFF0 || n > 0x7FFFFFF0) return mq_fail(MQ_ERR_ARG, "norm: tensor too large");
    return MQ_OK;
}

extern "C" int mq_norm_forward(const void* x, int dtype, int64_t ldx, const void* weight, const void* bias, int wdtype, void* y, void* xhat8,
                               uint8_t* xhat8_scale, void* y8, uint8_t* y8_scale, float* mean, float* rstd, int64_t rows, int64_t n,
                               float eps, int rms, void* stream) {
    if (const int rc = norm_check(dtype, wdtype, rows, n, ldx)) return rc;
    if (rows == 0 || n == 0) return MQ_OK;
    if (!x || !y || !xhat8 != !xhat8_scale || !y8 != !y8_scale) return mq_fail(MQ_ERR_ARG, "norm: null pointer");
    if ((xhat8 || y8) && n % 32 != 0) return mq_fail(MQ_ERR_ARG, "norm: rows kept in 8 bits are a multiple of 32 long");
    if (((uintptr_t)xhat8 | (uintptr_t)y8) % 8) return mq_fail(MQ_ERR_ARG, "norm: 8-bit copies start at a multiple of 8 bytes");
    const NormArgs a{x, weight, bias, y, (uint8_t*)xhat8, xhat8_scale, (uint8_t*)y8, y8_scale, mean, rstd, rows, n, ldx, eps, rms};
    const hipStream_t st = (hipStream_t)stream;
    norm_types(dtype, wdtype, [&](auto d, auto wf) {
        constexpr int D = decltype(d)::value, WF = decltype(wf)::value;
        norm_shape(n, kVec<D>, [&](auto l, auto u) {
            constexpr int L = decltype(l)::value, U = decltype(u)::value;
            if constexpr (L == 0) {
                hipLaunchKernelGGL((norm_fwd_long_kernel<D, WF>), dim3((unsigned)rows), dim3(1024), 0, st, a);
            } else {
                constexpr int kRows = L < 256 ? 256 / L : 1;
                hipLaunchKernelGGL((norm_fwd_kernel<D, WF, L, U>), dim3((unsigned)((rows + kRows - 1) / kRows)), dim3(L < 256 ? 256 : L), 0, st, a);
            }
        });
    });
    return mq_check_launch("norm forward");
}

// Sets of lanes that share the rows of a backward pass, and rows of its partial sums
static int64_t norm_parts(int64_t rows, int64_t n) {
    const int64_t most = n <= 1024 ? 4096 : 1024;
    return rows < most ? (rows > 0 ? rows : 1) : most;
}
extern "C" int mq_norm_backward_parts(int64_t rows, int64_t n) { return (int)norm_parts(rows, n); }

extern "C" int mq_norm_backward(const void* dy, int dtype, int64_t lddy, const void* x, int64_t ldx, const uint8_t* xhat8_scale, const float* mean,
                                const float* rstd, const void* weight, int wdtype, void* dx, void* dweight, void* dbias, float* ws,
                                int64_t rows, int64_t n, int rms, void* stream) {
    if (const int rc = norm_check(dtype, wdtype, rows, n, ldx)) return rc;
    if (rows > 1 && lddy < n) return mq_fail(MQ_ERR_ARG, "norm: rows overlap");
    if (n == 0) return MQ_OK;
    if ((dweight || dbias) && !ws) return mq_fail(MQ_ERR_ARG, "norm: null pointer");
    if (rows > 0 && (!dy || !x || !rstd || (!mean && !rms && !xhat8_scale))) return mq_fail(MQ_ERR_ARG, "norm: null pointer");
    if (xhat8_scale && (n % 32 != 0 || (uintptr_t)x % 8)) return mq_fail(MQ_ERR_ARG, "norm: rows kept in 8 bits are a multiple of 32 long, 8-byte aligned");
    const int64_t parts = norm_parts(rows, n);
    float* dw = dweight ? ws : nullptr;
    float* db = dbias ? ws + (dweight ? parts * n : 0) : nullptr;
    const NormGradArgs a{dy, x, xhat8_scale, mean, rstd, weight, dx, dw, db, rows, n, lddy, ldx, parts, rms};
    const hipStream_t st = (hipStream_t)stream;
    norm_types(dtype, wdtype, [&](auto d, auto wf) {
        constexpr int D = decltype(d)::value, WF = decltype(wf)::value;
        auto launch = [&](auto kept) {
            constexpr int KEPT = decltype(kept)::value;
            norm_shape(n, kVec<D>, [&](auto l, auto u) {
                constexpr int L = decltype(l)::value, U = decltype(u)::value;
                if constexpr (L == 0) {
                    if (dx && rows > 0) hipLaunchKernelGGL((norm_bwd_long_kernel<D, WF, KEPT>), dim3((unsigned)rows), dim3(1024), 0, st, a);
                    if (dw || db) {
                        const int64_t per = 256 * kVec<D>;
                        hipLaunchKernelGGL((norm_bwd_long_sums_kernel<D, KEPT>), dim3((unsigned)((n + per - 1) / per), (unsigned)parts), dim3(256), 0, st, a);
                    }
                } else {
                    constexpr int kRows = L < 256 ? 256 / L : 1;
                    hipLaunchKernelGGL((norm_bwd_kernel<D, WF, KEPT, L, U>), dim3((unsigned)((parts + kRows - 1) / kRows)), dim3(L < 256 ? 256 : L), 0,
                                       st, a);
                }
            });
        };
        if (xhat8_scale) launch(std::integral_constant<int, 1>{});
        else launch(std::integral_constant<int, 0>{});
    });
    if (const int rc = mq_check_launch("norm backward")) return rc;
    return mq_column_sum_launch(dw, dweight, db, dbias, parts, n, wdtype, st);
}
