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
//
// Measured in bf16 with inputs from memory, forward and backward: 16384 x 2048 layer norm 23 and 50 us (5.8 and 4.0 TB/s), 16384 x 4096
// 51 and 78 (5.3 and 5.2), 16384 x 7168 RMS norm with 8-bit xhat 103 and 110 (5.7 and 5.4).
#include "mq_rows.hpp"

namespace mq {

// A row in aligned pieces of 16 bytes: `base` is the multiple of 16 at or below the row's first element, which is `shift` elements
// behind it.  Piece i holds the columns i V - shift and on, of which the first and the last piece may lie partly outside the row.
// A load reads a piece whole where it holds any element of the row -- bytes of one aligned 16 that the row has a share in -- and what
// is outside counts as zero; a store writes the row's elements alone.
// (The backward pass of 16384 x 4095 bf16 by loads at each row's own offset instead: 194 us, and 107 by these.)
struct Span {
    int shift, end;            // elements: the row's first and the one behind its last, from the base

    // rows of n elements of `size` bytes; every operand's rows have the same offset
    __device__ __forceinline__ Span(const void* row, int n, int size) : shift((int)((uintptr_t)row & 15) / size), end(shift + n) {}
    template <int V>
    __device__ __forceinline__ bool any(int piece) const { return piece * V < end; }
    template <int V>
    __device__ __forceinline__ bool all(int piece) const { return piece * V >= shift && piece * V + V <= end; }
    template <int V>
    __device__ __forceinline__ bool has(int piece, int j) const { return piece * V + j >= shift && piece * V + j < end; }
};
__device__ __forceinline__ const char* base_of(const void* row) { return (const char*)((uintptr_t)row & ~(uintptr_t)15); }

template <int D>
__device__ __forceinline__ u32x4 ld_piece(const char* base, const Span& s, int piece) {
    u32x4 v = {0u, 0u, 0u, 0u};
    if (s.any<kVec<D>>(piece)) v = *(const u32x4*)(base + (uint32_t)piece * 16u);
    return v;
}
template <int D>
__device__ __forceinline__ void st_piece(char* base, const Span& s, int piece, u32x4 v) {
    constexpr int V = kVec<D>;
    if (s.all<V>(piece)) {
        st16(base + (uint32_t)piece * 16u, v);
        return;
    }
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < V; j++) {
        if (s.has<V>(piece, j)) {
            if (D == MQ_F32) ((uint32_t*)base)[piece * V + j] = u[j & 3];
            else ((uint16_t*)base)[piece * V + j] = (uint16_t)(u[j / 2] >> (16 * (j & 1)));
        }
    }
}
// the same columns of a vector that is fp32 (WF32) or of type D, from any element boundary, zero outside
template <int D>
__device__ __forceinline__ u32x4 ld_columns(const void* p, int first, int n) {
    constexpr int V = kVec<D>;
    if (first >= 0 && first + V <= n) return ld16_at2((const char*)p + first * kElem<D>);
    uint32_t u[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < V; j++) {
        if (first + j >= 0 && first + j < n) {
            if (D == MQ_F32) u[j & 3] = ((const uint32_t*)p)[first + j];
            else u[j / 2] |= (uint32_t)((const uint16_t*)p)[first + j] << (16 * (j & 1));
        }
    }
    return u32x4{u[0], u[1], u[2], u[3]};
}
template <int D, int WF32>
struct WeightPiece {
    static constexpr int kTwo = WF32 && D != MQ_F32;
    u32x4 v[kTwo + 1];
    __device__ __forceinline__ void load(const void* p, const Span& s, int piece) {
        const int first = piece * kVec<D> - s.shift, n = s.end - s.shift;
        v[0] = kTwo ? ld_columns<MQ_F32>(p, first, n) : ld_columns<D>(p, first, n);
        if (kTwo) v[kTwo] = ld_columns<MQ_F32>(p, first + 4, n);
    }
    // The same with anything in the place of what is outside, by aligned loads: of the two pieces that hold the columns, whichever
    // hold any of the vector, shifted into place by a distance that is the same for all lanes (16384 x 4095 bf16 forward: 81 us,
    // and 88 by loads off 16 bytes).
    __device__ __forceinline__ void load_near(const void* p, const Span& s, int piece) {
        if (kTwo) {
            load(p, s, piece);
            return;
        }
        const char *begin = (const char*)p, *end = begin + (int64_t)(s.end - s.shift) * kElem<D>;
        const char* at = begin - s.shift * kElem<D>;
        const int off = (int)((uintptr_t)at & 15);
        const char* lo = at - off + (int64_t)piece * 16;
        u32x4 x = {0u, 0u, 0u, 0u}, y = {0u, 0u, 0u, 0u};
        if (lo + 16 > begin && lo < end) x = *(const u32x4*)lo;
        if (off == 0) {
            v[0] = x;
            return;
        }
        if (lo + 32 > begin && lo + 16 < end) y = *(const u32x4*)(lo + 16);
        uint32_t d[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        if (off & 8)
#pragma unroll
            for (int i = 0; i < 6; i++) d[i] = d[i + 2];
        if (off & 4)
#pragma unroll
            for (int i = 0; i < 5; i++) d[i] = d[i + 1];
        if (off & 2)
#pragma unroll
            for (int i = 0; i < 4; i++) d[i] = (d[i] >> 16) | (d[i + 1] << 16);
        v[0] = u32x4{d[0], d[1], d[2], d[3]};
    }
    __device__ __forceinline__ void get(float* f) const {
        if (kTwo) {
            unpack<MQ_F32>(v[0], f);
            unpack<MQ_F32>(v[kTwo], f + (kVec<D> - 4));
        } else {
            unpack<D>(v[0], f);
        }
    }
};
// fp32 partial sums of the same columns
template <int V>
__device__ __forceinline__ void st_sums(float* row, const Span& s, int piece, const float* f) {
    const int first = piece * V - s.shift;
#pragma unroll
    for (int j = 0; j < V; j += 4) {
        if (s.all<V>(piece)) {
            st16_at2(row + first + j, pack<MQ_F32>(f + j));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (s.has<V>(piece, j + i)) row[first + j + i] = f[j + i];
        }
    }
}

struct NormArgs {
    const void* x;
    const void* w;             // null: no weight
    const void* b;             // null: no bias
    void* y;
    uint8_t *xq, *xs;          // xhat in 8 bits, or null
    uint8_t *yq, *ys;          // y in 8 bits, or null
    float *mean, *rstd;        // null: not kept
    int64_t rows, ldx;
    int n;
    float eps;
    int rms;
};

// the sum over a row's lanes, in every one of them: a wavefront's (WAVE), or the workgroup's, through `part`, a word for each of up to
// 16 wavefronts that is this sum's alone
template <int WAVE>
__device__ __forceinline__ float row_sum(float v, float* part) {
    v = wave_sum(v);
    if (WAVE) return v;
    const int waves = (int)blockDim.x / kWave;
    if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    float s = 0.0f;
    for (int i = 0; i < waves; i++) s += part[i];
    return s;
}
// sum / n, exact where n goes into the sum: a row of one value has that as its mean, and no spread.  (The product with 1 / n is a
// rounding off, and put right by what it leaves.)
__device__ __forceinline__ float quotient(float sum, int n, float inv_n) {
    const float q = sum * inv_n;
    return __builtin_fmaf(__builtin_fmaf(-q, (float)n, sum), inv_n, q);
}
// the row (or the set of rows) of a lane, and the lane's place in it
template <int WAVE>
__device__ __forceinline__ int64_t row_of() {
    return WAVE ? (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave) : (int64_t)blockIdx.x;
}
template <int WAVE>
__device__ __forceinline__ int lane_of() { return WAVE ? (int)threadIdx.x & (kWave - 1) : (int)threadIdx.x; }
template <int WAVE>
__device__ __forceinline__ int lanes() { return WAVE ? kWave : (int)blockDim.x; }

// An 8-bit copy of the V values that a lane holds of a row: the lanes of 32 neighbouring columns are neighbours.  n is a multiple of
// 32 and the row begins with a piece, so that a group's lanes are inside the row or outside together.
template <int D>
__device__ __forceinline__ void keep_piece(const float* f, int piece, int n, uint8_t* q, uint8_t* s) {
    constexpr int V = kVec<D>;
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < V; j++) top = keep_larger(top, f[j]);
    const uint32_t m = D == MQ_F32 ? group_max8(f2u(top)) : group_max4(f2u(top)), e = keep_exponent(m);
    const float inv = e8m0_inverse(e);
    const int c = piece * V;
    if (c < n) {
        const uint32_t lo = keep_codes4(f[0], f[1], f[2], f[3], inv, m == kInfinity);
        if (D == MQ_F32) {
            *(uint32_t*)(q + c) = lo;
        } else {
            *(u32x2*)(q + c) = u32x2{lo, keep_codes4(f[V - 4], f[V - 3], f[V - 2], f[V - 1], inv, m == kInfinity)};
        }
        if (c % 32 == 0) s[c / 32] = (uint8_t)e;
    }
}

// y of a piece and what is kept of it, from the normalized values
template <int D, int WF32>
__device__ __forceinline__ void finish_piece(const NormArgs& a, const Span& s, int64_t row, char* y, int piece, float* f) {
    constexpr int V = kVec<D>;
    if (a.xq) keep_piece<D>(f, piece, a.n, a.xq + row * a.n, a.xs + row * (a.n / 32));
    WeightPiece<D, WF32> wp;
    float w[V];
    if (a.w) {
        wp.load_near(a.w, s, piece);
        wp.get(w);
#pragma unroll
        for (int j = 0; j < V; j++) f[j] *= w[j];
    }
    if (a.b) {
        wp.load_near(a.b, s, piece);
        wp.get(w);
#pragma unroll
        for (int j = 0; j < V; j++) f[j] += w[j];
    }
    const u32x4 out = pack<D>(f);
    st_piece<D>(y, s, piece, out);
    if (a.yq) {
        unpack<D>(out, f);               // the copy stands for y as it is stored
        keep_piece<D>(f, piece, a.n, a.yq + row * a.n, a.ys + row * (a.n / 32));
    }
}

template <int D, int WF32, int WAVE, int UNITS>
__global__ __launch_bounds__(WAVE ? 256 : 1024) void norm_fwd_kernel(const NormArgs a) {
    constexpr int V = kVec<D>;
    __shared__ float part[2][16];
    const int lane = lane_of<WAVE>(), apart = lanes<WAVE>();
    const int64_t row = row_of<WAVE>();
    if (row >= a.rows) return;           // (only where a row has a wavefront of its own: nobody waits for it)
    const char* x = (const char*)a.x + row * a.ldx * kElem<D>;
    char* y = const_cast<char*>(base_of((const char*)a.y + row * a.n * kElem<D>));
    const Span s(x, a.n, kElem<D>);
    const char* base = base_of(x);
    float v[UNITS][V];
#pragma unroll
    for (int u = 0; u < UNITS; u++) unpack<D>(ld_piece<D>(base, s, u * apart + lane), v[u]);
    const float inv_n = 1.0f / (float)a.n;
    const bool whole = s.shift == 0 && a.n % V == 0;       // no piece is partly outside
    auto outside = [&](float with) {                       // in the row's elements' place where there are none
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            const int piece = u * apart + lane;
            if (!s.all<V>(piece)) {                        // (most wavefronts have no such piece)
#pragma unroll
                for (int j = 0; j < V; j++) v[u][j] = s.has<V>(piece, j) ? v[u][j] : with;
            }
        }
    };
    float mean = 0.0f;
    if (!whole) outside(0.0f);                             // (pieces wholly outside are zero as they come)
    if (!a.rms) {
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < UNITS; u++)
#pragma unroll
            for (int j = 0; j < V; j++) sum += v[u][j];
        mean = quotient(row_sum<WAVE>(sum, part[0]), a.n, inv_n);
        outside(mean);
#pragma unroll
        for (int u = 0; u < UNITS; u++)
#pragma unroll
            for (int j = 0; j < V; j++) v[u][j] -= mean;
    }
    float s2 = 0.0f;
#pragma unroll
    for (int u = 0; u < UNITS; u++)
#pragma unroll
        for (int j = 0; j < V; j++) s2 = __builtin_fmaf(v[u][j], v[u][j], s2);
    const float rstd = 1.0f / __builtin_sqrtf(row_sum<WAVE>(s2, part[1]) * inv_n + a.eps);
    if (lane == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
#pragma unroll
        for (int j = 0; j < V; j++) v[u][j] *= rstd;
        finish_piece<D, WF32>(a, s, row, y, u * apart + lane, v[u]);
    }
}

// Rows too long for the registers of a workgroup: three passes over the row, which the caches hold.
template <int D, int WF32>
__global__ __launch_bounds__(1024) void norm_fwd_long_kernel(const NormArgs a) {
    constexpr int V = kVec<D>, kLanes = 1024;
    __shared__ float part[2][16];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const char* x = (const char*)a.x + row * a.ldx * kElem<D>;
    char* y = const_cast<char*>(base_of((const char*)a.y + row * a.n * kElem<D>));
    const Span s(x, a.n, kElem<D>);
    const char* base = base_of(x);
    const float inv_n = 1.0f / (float)a.n;
    float mean = 0.0f, f[V];
    if (!a.rms) {
        float sum = 0.0f;
        for (int i = lane; s.any<V>(i); i += kLanes) {
            unpack<D>(ld_piece<D>(base, s, i), f);
#pragma unroll
            for (int j = 0; j < V; j++) sum += s.has<V>(i, j) ? f[j] : 0.0f;
        }
        mean = quotient(row_sum<0>(sum, part[0]), a.n, inv_n);
    }
    float s2 = 0.0f;
    for (int i = lane; s.any<V>(i); i += kLanes) {
        unpack<D>(ld_piece<D>(base, s, i), f);
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float d = s.has<V>(i, j) ? f[j] - mean : 0.0f;
            s2 = __builtin_fmaf(d, d, s2);
        }
    }
    const float rstd = 1.0f / __builtin_sqrtf(row_sum<0>(s2, part[1]) * inv_n + a.eps);
    if (lane == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
    // whole wavefronts stay together: the 8-bit copies take maxima over lanes
    for (int i0 = 0; s.any<V>(i0); i0 += kLanes) {
        const int i = i0 + lane;
        unpack<D>(ld_piece<D>(base, s, i), f);
#pragma unroll
        for (int j = 0; j < V; j++) f[j] = s.has<V>(i, j) ? (f[j] - mean) * rstd : 0.0f;
        finish_piece<D, WF32>(a, s, row, y, i, f);
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
    int64_t rows, lddy, ldx, parts;
    int n, rms;
};

// What a lane reads of a row for one piece: the gradient, and the input or the codes of xhat with their exponent
template <int D, int KEPT>
struct RowPiece {
    static constexpr int V = kVec<D>;
    u32x4 dy, x;
    uint32_t e;

    __device__ __forceinline__ void load(const NormGradArgs& a, const Span& s, int64_t row, int piece) {
        dy = ld_piece<D>(base_of((const char*)a.dy + row * a.lddy * kElem<D>), s, piece);
        if (KEPT) {
            x = u32x4{0u, 0u, 0u, 0u};
            e = 0;
            if (s.any<V>(piece)) {
                const char* q = (const char*)a.x + row * a.n;
                if (D == MQ_F32) x.x = *(const uint32_t*)(q + (uint32_t)(piece * V));
                else {
                    const u32x2 v = *(const u32x2*)(q + (uint32_t)(piece * V));
                    x.x = v.x, x.y = v.y;
                }
                e = (a.xs + row * (a.n / 32))[(uint32_t)(piece * V / 32)];
            }
        } else {
            x = ld_piece<D>(base_of((const char*)a.x + row * a.ldx * kElem<D>), s, piece);
        }
    }
    // The gradient and the normalized values, zero outside the row; whole: no piece is partly outside.  The values are the forward pass's,
    // subtraction first: as x rstd - mean rstd, in one instruction, those of a row of 1000s came out as 0.02 instead of 0 (8191 x 4096 fp16
    // forward and backward 73.0 us, and 74.0 like this).
    __device__ __forceinline__ void get(const Span& s, bool whole, int piece, float mean, float rstd, float* g, float* xh) const {
        unpack<D>(dy, g);
        if (KEPT) {
            const float scale = e8m0_value(e);
            kept_values4(x.x, scale, xh);
            if (D != MQ_F32) kept_values4(x.y, scale, xh + (V - 4));
        } else {
            unpack<D>(x, xh);
#pragma unroll
            for (int j = 0; j < V; j++) xh[j] = (xh[j] - mean) * rstd;
            if (!whole && !s.all<V>(piece)) {
#pragma unroll
                for (int j = 0; j < V; j++)
                    if (!s.has<V>(piece, j)) g[j] = xh[j] = 0.0f;
            }
        }
    }
};

// A wavefront (WAVE) or a workgroup goes through rows far apart, `parts` of them in all, and keeps its columns' sums in registers; the
// partial sums are added by column_sum_kernel in a fixed order.  Bound by HBM, with the vector unit not far behind (some twelve
// instructions an element of the forty that the bytes leave time for): a row's products stay in registers between its two passes,
// and the next row's pieces are on their way meanwhile.
template <int D, int WF32, int KEPT, int RMS, int WAVE, int UNITS>
__global__ __launch_bounds__(WAVE ? 256 : 512) void norm_bwd_kernel(const NormGradArgs a) {
    constexpr int V = kVec<D>;
    __shared__ float part[2][2][8];
    const int lane = lane_of<WAVE>(), apart = lanes<WAVE>();
    const int64_t mine = row_of<WAVE>();
    if (mine >= a.parts) return;         // (only where a row has a wavefront of its own)
    const float inv_n = 1.0f / (float)a.n;
    // the rows of a set have one offset: there are eight times as many elements from one to the next as one begins with
    const Span s((const char*)a.dy + mine * a.lddy * kElem<D>, a.n, kElem<D>);
    const bool whole = s.shift == 0 && a.n % V == 0;
    float dw[UNITS][V], db[UNITS][V];
    WeightPiece<D, WF32> w[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
        if (a.w) w[u].load(a.w, s, u * apart + lane);
#pragma unroll
        for (int j = 0; j < V; j++) dw[u][j] = db[u][j] = 0.0f;
    }
    RowPiece<D, KEPT> next[UNITS];
    float next_mean = 0.0f, next_rstd = 0.0f;
    auto load = [&](int64_t row) {
#pragma unroll
        for (int u = 0; u < UNITS; u++) next[u].load(a, s, row, u * apart + lane);
        if (!KEPT && !RMS) next_mean = a.mean[row];
        next_rstd = a.rstd[row];
    };
    if (mine < a.rows) load(mine);
    int turn = 0;
    for (int64_t row = mine; row < a.rows; row += a.parts, turn ^= 1) {
        const float mean = next_mean, rstd = next_rstd;
        float g[UNITS][V], xh[UNITS][V], sg = 0.0f, sgx = 0.0f;
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            next[u].get(s, whole, u * apart + lane, mean, rstd, g[u], xh[u]);
            float f[V];
            if (a.w) w[u].get(f);
#pragma unroll
            for (int j = 0; j < V; j++) {
                dw[u][j] = __builtin_fmaf(g[u][j], xh[u][j], dw[u][j]);
                if (!RMS) db[u][j] += g[u][j];
                if (a.w) g[u][j] *= f[j];
                if (!RMS) sg += g[u][j];
                sgx = __builtin_fmaf(g[u][j], xh[u][j], sgx);
            }
        }
        if (row + a.parts < a.rows) load(row + a.parts);
        if (!a.dx) continue;
        // two sums with one wait between the wavefronts; the words are used every other row, so that a fast wavefront's next
        // sums do not meet a slow one's reading of these
        if (!RMS) sg = wave_sum(sg);
        sgx = wave_sum(sgx);
        if (!WAVE) {
            if ((threadIdx.x & (kWave - 1)) == 0) {
                part[turn][0][threadIdx.x / kWave] = sg;
                part[turn][1][threadIdx.x / kWave] = sgx;
            }
            __syncthreads();
            sg = sgx = 0.0f;
            for (int i = 0; i < apart / kWave; i++) {
                if (!RMS) sg += part[turn][0][i];
                sgx += part[turn][1][i];
            }
        }
        // dx = rstd g - rstd mean(g) - rstd mean(g xhat) xhat
        const float flat = RMS ? 0.0f : -rstd * (sg * inv_n), along = -rstd * (sgx * inv_n);
        char* dx = const_cast<char*>(base_of((const char*)a.dx + row * a.n * kElem<D>));
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                g[u][j] = RMS ? rstd * g[u][j] : __builtin_fmaf(rstd, g[u][j], flat);
                g[u][j] = __builtin_fmaf(along, xh[u][j], g[u][j]);
            }
            st_piece<D>(dx, s, u * apart + lane, pack<D>(g[u]));
        }
    }
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
        if (a.dw) st_sums<V>(a.dw + mine * a.n, s, u * apart + lane, dw[u]);
        if (!RMS && a.db) st_sums<V>(a.db + mine * a.n, s, u * apart + lane, db[u]);
    }
}

// Long rows: dx by three passes over the row; the columns' sums by norm_bwd_long_sums_kernel, which goes down the columns.
template <int D, int WF32, int KEPT>
__global__ __launch_bounds__(1024) void norm_bwd_long_kernel(const NormGradArgs a) {
    constexpr int V = kVec<D>, kLanes = 1024;
    __shared__ float part[2][16];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const Span s((const char*)a.dy + row * a.lddy * kElem<D>, a.n, kElem<D>);
    const float inv_n = 1.0f / (float)a.n, mean = KEPT || a.rms ? 0.0f : a.mean[row], rstd = a.rstd[row];
    float g[V], xh[V], w[V], sg = 0.0f, sgx = 0.0f;
    auto get = [&](int i) {
        RowPiece<D, KEPT> piece;
        piece.load(a, s, row, i);
        piece.get(s, false, i, mean, rstd, g, xh);
        if (a.w) {
            WeightPiece<D, WF32> wp;
            wp.load(a.w, s, i);
            wp.get(w);
#pragma unroll
            for (int j = 0; j < V; j++) g[j] *= w[j];
        }
    };
    for (int i = lane; s.any<V>(i); i += kLanes) {
        get(i);
#pragma unroll
        for (int j = 0; j < V; j++) {
            sg += g[j];
            sgx = __builtin_fmaf(g[j], xh[j], sgx);
        }
    }
    const float mg = row_sum<0>(sg, part[0]) * inv_n, mgx = row_sum<0>(sgx, part[1]) * inv_n;
    char* dx = const_cast<char*>(base_of((const char*)a.dx + row * a.n * kElem<D>));
    for (int i = lane; s.any<V>(i); i += kLanes) {
        get(i);
#pragma unroll
        for (int j = 0; j < V; j++) g[j] = (__builtin_fmaf(-xh[j], mgx, g[j]) - (a.rms ? 0.0f : mg)) * rstd;
        st_piece<D>(dx, s, i, pack<D>(g));
    }
}
template <int D, int KEPT>
__global__ __launch_bounds__(256) void norm_bwd_long_sums_kernel(const NormGradArgs a) {
    constexpr int V = kVec<D>;
    const int piece = (int)blockIdx.x * 256 + (int)threadIdx.x;
    const int64_t mine = blockIdx.y;
    const Span s((const char*)a.dy + mine * a.lddy * kElem<D>, a.n, kElem<D>);
    if (!s.any<V>(piece)) return;
    float dw[V], db[V], g[V], xh[V];
#pragma unroll
    for (int j = 0; j < V; j++) dw[j] = db[j] = 0.0f;
    for (int64_t row = mine; row < a.rows; row += a.parts) {
        const float mean = KEPT || a.rms ? 0.0f : a.mean[row];
        RowPiece<D, KEPT> p;
        p.load(a, s, row, piece);
        p.get(s, false, piece, mean, a.rstd[row], g, xh);
#pragma unroll
        for (int j = 0; j < V; j++) {
            dw[j] = __builtin_fmaf(g[j], xh[j], dw[j]);
            db[j] += g[j];
        }
    }
    if (a.dw) st_sums<V>(a.dw + mine * a.n, s, piece, dw);
    if (a.db) st_sums<V>(a.db + mine * a.n, s, piece, db);
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
#pragma unroll 4
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

// How a row of so many pieces is shared: by a wavefront up to two pieces a lane (no wait between wavefronts), by the wavefronts of a
// workgroup as many as it needs beyond; f gets whether it is a wavefront, the pieces of a lane (0: the long forms), and the lanes.
// Measured in bf16: 32768 x 1024 forward 22 us by a wavefront of two pieces a lane, 28 by a workgroup of one; 16384 x 2048 forward by a
// workgroup of two pieces a lane 23 us, of one 28; backward with 8-bit xhat 46 and 43, so that there one comes first.  Forward passes hold
// a row, a backward pass two and the columns' sums, so that its workgroups are smaller (16384 x 7168, 8-bit xhat: two pieces a lane, 448
// lanes, 110 us backward; four pieces, 256 lanes, 164).  Forward, four pieces a lane from 513 pieces on instead of from 2049: 16384 x 7168
// 84 us instead of 94, but 8192 x 8192 63 instead of 59 where xhat is kept in 8 bits and one row of 7168 4.7 instead of 4.2; a rule on what
// is kept or on the number of rows would make a row's result depend on them.  Four pieces a lane spill in the backward pass of
// layer norm in 16 bits: 16384 x 14336 532 us, and 722 from 8-bit xhat, where the long forms take 520 and 466; of RMS norm 307 and 500, and
// of fp32 rows (16384 x 7168) 304 and 495.
template <int BACKWARD, class F>
static void norm_shape(int64_t pieces, F&& f) {
    constexpr int kMost = BACKWARD ? 512 : 1024;
    constexpr std::integral_constant<int, 0> no{};
    constexpr std::integral_constant<int, 1> yes{}, one{};
    constexpr std::integral_constant<int, 2> two{};
    constexpr std::integral_constant<int, 3> three{};
    constexpr std::integral_constant<int, 4> four{};
    auto lanes = [&](int64_t units) { return (unsigned)((pieces + units * kWave - 1) / (units * kWave) * kWave); };
    if (pieces <= 64) f(yes, one, 256u);
    else if (pieces <= 128) f(yes, two, 256u);
    else if (BACKWARD && pieces <= 256) f(no, one, lanes(1));
    else if (pieces <= 2 * kMost) f(no, two, lanes(2));
    else if (BACKWARD && pieces <= 3 * kMost) f(no, three, lanes(3));
    else if (pieces <= 4 * kMost) f(no, four, lanes(4));
    else f(no, no, 1024u);
}
// pieces of a row: one more where rows begin inside one
static int64_t norm_pieces(const void* at, int64_t ld, int64_t n, int dtype) {
    const int size = dtype == MQ_F32 ? 4 : 2, V = 16 / size;
    const bool inside = (uintptr_t)at % 16 != 0 || ld * size % 16 != 0;
    return (n + (inside ? V - 1 : 0) + V - 1) / V;
}
// whether rows that begin at a and at b have the same offset in 16 bytes, all of them
static bool same_offsets(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t rows, int dtype) {
    const int size = dtype == MQ_F32 ? 4 : 2;
    return ((uintptr_t)a - (uintptr_t)b) % 16 == 0 && (rows <= 1 || (lda - ldb) * size % 16 == 0);
}
static int norm_offsets() { return mq_fail(MQ_ERR_ARG, "norm: rows of the operands have different offsets in 16 bytes"); }

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
    if (rows > 0x7FFFFFF0 || n > 0x1FFFFF00) return mq_fail(MQ_ERR_ARG, "norm: tensor too large");
    return MQ_OK;
}

extern "C" int mq_norm_forward(const void* x, int dtype, int64_t ldx, const void* weight, const void* bias, int wdtype, void* y, void* xhat8,
                               uint8_t* xhat8_scale, void* y8, uint8_t* y8_scale, float* mean, float* rstd, int64_t rows, int64_t n,
                               float eps, int rms, void* stream) {
    if (const int rc = norm_check(dtype, wdtype, rows, n, ldx)) return rc;
    if (rows == 0 || n == 0) return MQ_OK;
    if (!x || !y || !xhat8 != !xhat8_scale || !y8 != !y8_scale) return mq_fail(MQ_ERR_ARG, "norm: null pointer");
    if (rms && bias) return mq_fail(MQ_ERR_ARG, "norm: RMS norm has no bias");
    if ((xhat8 || y8) && n % 32 != 0) return mq_fail(MQ_ERR_ARG, "norm: rows kept in 8 bits are a multiple of 32 long");
    if (((uintptr_t)xhat8 | (uintptr_t)y8) % 8) return mq_fail(MQ_ERR_ARG, "norm: 8-bit copies start at a multiple of 8 bytes");
    const int64_t ldy = rows > 1 ? n : ldx;
    if (!same_offsets(x, ldx, y, ldy, rows, dtype) || ((xhat8 || y8) && ((uintptr_t)x % 16 || !same_offsets(x, ldx, y, 0, rows, dtype)))) return norm_offsets();
    const hipStream_t st = (hipStream_t)stream;
    const int64_t pieces = norm_pieces(x, rows > 1 ? ldx : 0, n, dtype);
    norm_types(dtype, wdtype, [&](auto d, auto wf) {
        constexpr int D = decltype(d)::value, WF = decltype(wf)::value;
        norm_shape<0>(pieces, [&](auto wave, auto units, unsigned lanes) {
            constexpr int W = decltype(wave)::value, U = decltype(units)::value;
            // A launch has fewer than 2^32 lanes, 64 to a row or up to 1024.  (The rows of a launch are a multiple of eight, so that those of the
            // next begin at the offsets in 16 bytes that the first launch's have.)
            constexpr int64_t kMost = W ? 1 << 25 : 1 << 21;
            for (int64_t at = 0; at < rows; at += kMost) {
                const int64_t count = rows - at < kMost ? rows - at : kMost;
                auto from = [&](auto* p, int64_t row) { return p ? p + at * row : p; };
                const NormArgs a{(const char*)x + at * ldx * kElem<D>, weight, bias, (char*)y + at * n * kElem<D>, from((uint8_t*)xhat8, n), from(xhat8_scale, n / 32),
                                 from((uint8_t*)y8, n), from(y8_scale, n / 32), from(mean, 1), from(rstd, 1), count, ldx, (int)n, eps, rms};
                if constexpr (U == 0) hipLaunchKernelGGL((norm_fwd_long_kernel<D, WF>), dim3((unsigned)count), dim3(lanes), 0, st, a);
                else hipLaunchKernelGGL((norm_fwd_kernel<D, WF, W, U>), dim3((unsigned)(W ? (count + 3) / 4 : count)), dim3(lanes), 0, st, a);
            }
        });
    });
    return mq_check_launch("norm forward");
}

// Sets of lanes that share the rows of a backward pass, and rows of its partial sums: a multiple of eight wherever a set has more
// than one row, so that all of a set's rows have one offset in 16 bytes.  More sets hide more latency and write more sums: 32768 x 1024
// bf16 50 us with 2048 sets and 71 with 512, 16384 x 2048 54 and 50, 16384 x 4096 92 and 78.
static int64_t norm_parts(int64_t rows, int64_t n) {
    const int64_t most = n <= 1024 ? 2048 : 512;
    return rows < most ? (rows > 0 ? rows : 1) : most;
}
extern "C" int mq_norm_backward_parts(int64_t rows, int64_t n) { return (int)norm_parts(rows, n); }

extern "C" int mq_norm_backward(const void* dy, int dtype, int64_t lddy, const void* x, int64_t ldx, const uint8_t* xhat8_scale, const float* mean,
                                const float* rstd, const void* weight, int wdtype, void* dx, void* dweight, void* dbias, float* ws,
                                int64_t rows, int64_t n, int rms, void* stream) {
    if (const int rc = norm_check(dtype, wdtype, rows, n, ldx)) return rc;
    if (rows > 1 && lddy < n) return mq_fail(MQ_ERR_ARG, "norm: rows overlap");
    if (n == 0) return MQ_OK;
    if (rms && dbias) return mq_fail(MQ_ERR_ARG, "norm: RMS norm has no bias");
    if ((dweight || dbias) && !ws) return mq_fail(MQ_ERR_ARG, "norm: null pointer");
    if (rows > 0 && (!dy || !x || !rstd || (!mean && !rms && !xhat8_scale))) return mq_fail(MQ_ERR_ARG, "norm: null pointer");
    if (xhat8_scale && (n % 32 != 0 || (uintptr_t)x % 8)) return mq_fail(MQ_ERR_ARG, "norm: rows kept in 8 bits are a multiple of 32 long, 8-byte aligned");
    const int64_t parts = norm_parts(rows, n);
    float* dw = dweight ? ws : nullptr;
    float* db = dbias ? ws + (dweight ? parts * n : 0) : nullptr;
    if (rows > 0) {
        const int64_t mine = rows > 1 ? lddy : 0;
        if (xhat8_scale ? (uintptr_t)dy % 16 != 0 || !same_offsets(dy, mine, dy, 0, rows, dtype) : !same_offsets(dy, mine, x, rows > 1 ? ldx : 0, rows, dtype))
            return norm_offsets();
        if (dx && !same_offsets(dy, mine, dx, rows > 1 ? n : 0, rows, dtype)) return norm_offsets();
    }
    const NormGradArgs a{dy, x, xhat8_scale, mean, rstd, weight, dx, dw, db, rows, lddy, ldx, parts, (int)n, rms};
    const hipStream_t st = (hipStream_t)stream;
    norm_types(dtype, wdtype, [&](auto d, auto wf) {
        constexpr int D = decltype(d)::value, WF = decltype(wf)::value;
        auto launch = [&](auto kept, auto without_mean) {
            constexpr int KEPT = decltype(kept)::value, RMS = decltype(without_mean)::value;
            const int64_t pieces = norm_pieces(dy, rows > 1 ? lddy : 0, n, dtype);
            norm_shape<1>(pieces, [&](auto wave, auto units, unsigned lanes) {
                constexpr int W = decltype(wave)::value, U = decltype(units)::value;
                if constexpr (U == 0) {
                    if (dx && rows > 0) hipLaunchKernelGGL((norm_bwd_long_kernel<D, WF, KEPT>), dim3((unsigned)rows), dim3(lanes), 0, st, a);
                    if (dw || db) {
                        hipLaunchKernelGGL((norm_bwd_long_sums_kernel<D, KEPT>), dim3((unsigned)((pieces + 255) / 256), (unsigned)parts), dim3(256), 0, st, a);
                    }
                } else {
                    hipLaunchKernelGGL((norm_bwd_kernel<D, WF, KEPT, RMS, W, U>), dim3((unsigned)(W ? (parts + 3) / 4 : parts)), dim3(lanes), 0, st, a);
                }
            });
        };
        constexpr std::integral_constant<int, 0> no{};
        constexpr std::integral_constant<int, 1> yes{};
        if (xhat8_scale && rms) launch(yes, yes);
        else if (xhat8_scale) launch(yes, no);
        else if (rms) launch(no, yes);
        else launch(no, no);
    });
    if (const int rc = mq_check_launch("norm backward")) return rc;
    return mq_column_sum_launch(dw, dweight, db, dbias, parts, n, wdtype, st);
}
