// Matrix products of 16-bit operands on the matrix cores, fp32 sums: out[q][p] = sum over k of Q(q, k) P(p, k).
//
// The three products of a linear layer y = x W^T differ in how the operands lie in memory:
//   forward          P = W [N][K], Q = x [M][K]          both with k along the rows
//   input gradient   P = W [N][K] read as (k of W, n), Q = dz [M][N]
//   weight gradient  P = x [M][K] or its 8-bit copy, Q = dz [M][N], both with the sum going down the rows
// A workgroup computes a BP x BQ tile of the output in steps of 64 along k, through two buffers in shared memory: while the matrix
// cores work on one, the next step's operands go into the other.
//
// Operands with k along the rows lie in shared memory as rows of 64 elements (eight 16-byte slots; slot s of row r holds the
// row's piece s ^ (r & 7), so that the 16 rows of a fragment read from all banks); a lane's eight k are one 16-byte read.  Operands
// whose sum goes down the rows lie as 64 rows of BP or BQ elements (32-byte slots, slot c of row k holds piece c ^ swizzle(k)); a
// lane's eight k come by two transposing reads of four rows by 16 columns for each 16 lanes.
// The P operand is the first of v_mfma_f32_16x16x32: a lane's four results are neighbours along p, the rows of the output.
#pragma once
#include "mq_act.hpp"
#include "mq_rows.hpp"

namespace mq {

constexpr int kStep = 64;                 // k of a step

// how an operand is staged: k along its rows or down them; straight into shared memory (16-byte aligned rows, sizes a multiple of
// eight), through registers with every bound checked, or from an 8-bit copy (then 16-bit values are made on the way)
enum { kRowsDirect = 0, kRowsAny = 1, kDownDirect = 2, kDownAny = 3, kDownKept = 4 };

struct GemmArgs {
    const char* p;
    const char* q;
    const uint8_t* ps;                    // exponent bytes of a P kept in 8 bits
    int64_t ldp, ldq;                     // elements
    int64_t np, nq, k;
    char* out;                            // [nq][np]
    const char* bias;                     // [np], null: none
    const char* res;                      // [nq][np], rows ldr apart, null: none
    int64_t ldr;
    char* z;                              // what the activation is applied to, in the output's type, null: not kept
    uint8_t *zq, *zs;                     // the same in 8 bits, null: not kept
    float* ws;                            // partial sums [splits][nq][round up np to 4], null: one split
    int64_t k_split;                      // k of a split, a multiple of the step
    int tiles_p, tiles_q, act;
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
#define MQ_LDS __attribute__((address_space(3)))

template <int D>
__device__ __forceinline__ f32x4 mfma(u32x4 p, u32x4 q, f32x4 c) {
    if (D == MQ_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, p), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
}

// 16 bytes from memory straight into shared memory: lane i's go to `lds` + 16 i (lds uniform), from rsrc's base + offset, zeros where
// the offset is not below 2^31 - 1.  The instruction has no register result; the caller waits for it.
__device__ __forceinline__ void direct16(uint32_t lds, u32x4 rsrc, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(rsrc) : "memory");
}
constexpr uint32_t kNowhere = 0x80000000u;

__device__ __forceinline__ u32x4 buffer_of(const char* base) {
    const uint64_t a = (uint64_t)base;
    u32x4 r;
    r.x = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
    r.y = (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xFFFFu));
    r.z = 0x7FFFFFFFu;
    r.w = 0x00027000u;
    return r;
}

// piece order of row k of an operand that lies down the rows, 32-byte pieces, B elements to a row
template <int B>
__device__ __forceinline__ int down_swizzle(int k) { return ((k & 3) | ((k >> 1) & 4)) & (B / 16 - 1); }

// One operand's way into shared memory.  A buffer is B x 64 elements; thread t's unit u is the 16 bytes at (t + u THREADS) 16.
template <int MODE, int D, int B, int THREADS>
struct Stage {
    static constexpr bool kDirect = MODE == kRowsDirect || MODE == kDownDirect;
    static constexpr bool kDown = MODE >= kDownDirect;
    static constexpr bool kKept = MODE == kDownKept;
    static constexpr int kUnits = B * 8 / THREADS;
    static constexpr int kPieces = kKept ? kUnits / 2 : kUnits;       // accesses to memory: 16 codes fill two units
    static_assert(B * 8 % (THREADS * (kKept ? 2 : 1)) == 0, "whole units");

    const char* base;                     // the tile's first element at the next step's first k
    const uint8_t* scales;
    int64_t ld, n;                        // n: outputs from the tile's first on
    int64_t advance;
    uint32_t offset[kPieces];
    u32x4 v[kPieces];
    uint32_t e[kPieces];

    static __device__ __forceinline__ int down_k(int at) { return at / (B / 8); }
    static __device__ __forceinline__ int down_col(int at) {
        const int unit = at % (B / 8);
        return ((unit >> 1) ^ down_swizzle<B>(down_k(at))) * 16 + (unit & 1) * 8;
    }

    __device__ __forceinline__ void init(const char* op, const uint8_t* s, int64_t ld_, int64_t first, int64_t count, int64_t k0) {
        ld = ld_;
        n = count - first;
        constexpr int kSize = kKept ? 1 : 2;
        base = op + (kDown ? k0 * ld + first : first * ld + k0) * kSize;
        advance = (kDown ? kStep * ld : kStep) * kSize;
        if (kKept) scales = s + k0 * (ld / 32) + first / 32;
        if (kDirect) {
#pragma unroll
            for (int u = 0; u < kUnits; u++) {
                const int at = (int)threadIdx.x + u * THREADS;
                if (kDown) {
                    const int k = down_k(at), c = down_col(at);
                    offset[u] = (uint32_t)((int64_t)k * ld * 2 + (c < n ? c : 0) * 2);
                } else {
                    const int row = at >> 3, c = (at & 7) ^ (row & 7);
                    offset[u] = (uint32_t)((row < n ? row : n - 1) * ld * 2 + c * 16);
                }
            }
        }
    }
    // the next step's operand: on its way to `lds` (direct), or into registers; left: k that are left from the step's first on
    __device__ __forceinline__ void fetch(uint32_t lds, int64_t left) {
        if (kDirect) {
            const u32x4 rsrc = buffer_of(base);
            const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave) * (kWave * 16);
            if (left >= kStep) {
#pragma unroll
                for (int u = 0; u < kUnits; u++) direct16(lds + wave + u * (THREADS * 16), rsrc, offset[u]);
            } else {
#pragma unroll
                for (int u = 0; u < kUnits; u++) {
                    const int at = (int)threadIdx.x + u * THREADS;
                    const int k = kDown ? down_k(at) : ((at & 7) ^ ((at >> 3) & 7)) * 8;
                    direct16(lds + wave + u * (THREADS * 16), rsrc, k < left ? offset[u] : kNowhere);
                }
            }
        } else if (kKept) {
#pragma unroll
            for (int i = 0; i < kPieces; i++) {
                const int at = ((int)threadIdx.x + i * THREADS) * 2, k = down_k(at), c = down_col(at);
                v[i] = u32x4{0u, 0u, 0u, 0u};
                e[i] = 0;
                if (k < left && c < n) {
                    v[i] = *(const u32x4*)(base + k * ld + c);
                    e[i] = scales[k * (ld / 32) + c / 32];
                }
            }
            scales += kStep * (ld / 32);
        } else {
#pragma unroll
            for (int u = 0; u < kUnits; u++) {
                const int at = (int)threadIdx.x + u * THREADS;
                v[u] = u32x4{0u, 0u, 0u, 0u};
                if (kDown) {
                    const int k = down_k(at), c = down_col(at);
                    if (k < left) v[u] = ld_row<MQ_BF16>(base + (int64_t)k * ld * 2, c, n);
                } else {
                    const int row = at >> 3, c = ((at & 7) ^ (row & 7)) * 8;
                    if (row < n) v[u] = ld_row<MQ_BF16>(base + (int64_t)row * ld * 2, c, left);
                }
            }
        }
        base += advance;
    }
    // what came through registers, into shared memory
    __device__ __forceinline__ void put(MQ_LDS char* lds) {
        if (kDirect) return;
        if (kKept) {
#pragma unroll
            for (int i = 0; i < kPieces; i++) {
                const float s = e8m0_value(e[i]);
                const uint32_t c[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
                float f[16];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    kept_values4(c[j], s, f + 4 * j);
                    if (D == MQ_F16)
                        for (int m = 0; m < 4; m++) f[4 * j + m] = clamp_keep_nan(f[4 * j + m], -65504.0f, 65504.0f);
                }
                MQ_LDS u32x4* to = (MQ_LDS u32x4*)(lds + ((int)threadIdx.x + i * THREADS) * 32);
                to[0] = pack<D>(f);
                to[1] = pack<D>(f + 8);
            }
        } else {
#pragma unroll
            for (int u = 0; u < kUnits; u++) *(MQ_LDS u32x4*)(lds + ((int)threadIdx.x + u * THREADS) * 16) = v[u];
        }
    }
};

// Addresses of a wavefront's fragments of an operand in shared memory: F fragments of 16 outputs from `first` on
template <int MODE, int B, int F>
struct Fragments {
    static constexpr bool kDown = MODE >= kDownDirect;
    uint32_t at[kDown ? F : 2];

    __device__ __forceinline__ void init(int first) {
        const int lane = threadIdx.x & (kWave - 1), j = lane & 15, g = lane >> 4;
        if (kDown) {
            const int k = g * 8 + (j >> 2);
#pragma unroll
            for (int f = 0; f < F; f++) at[f] = (uint32_t)(k * (B * 2) + ((first / 16 + f) ^ down_swizzle<B>(k)) * 32 + (j & 3) * 8);
        } else {
#pragma unroll
            for (int s = 0; s < 2; s++) at[s] = (uint32_t)((first + j) * 128 + ((g + 4 * s) ^ (j & 7)) * 16);
        }
    }
    // fragment f of the 32 k from 32 s on
    __device__ __forceinline__ u32x4 get(MQ_LDS char* lds, int s, int f) const {
        if (kDown) {
            MQ_LDS char* from = lds + at[f] + s * (32 * B * 2);
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MQ_LDS s16x4*)from);
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MQ_LDS s16x4*)(from + 4 * B * 2));
            const u32x2 x = __builtin_bit_cast(u32x2, a), y = __builtin_bit_cast(u32x2, b);
            return u32x4{x.x, x.y, y.x, y.y};
        }
        return *(MQ_LDS const u32x4*)(lds + at[s] + f * 2048);
    }
};

// Four neighbouring 16-bit elements of a row, from any element boundary, zero from column n on
typedef u32x2 u32x2_at2 __attribute__((aligned(2)));
__device__ __forceinline__ u32x2 ld4_row(const char* row, int64_t c, int64_t n) {
    if (c + 4 <= n) return *(const u32x2_at2*)(row + c * 2);
    u32x2 v = {0u, 0u};
    if (c < n) v.x = ((const uint16_t*)row)[c];
    if (c + 1 < n) v.x |= (uint32_t)((const uint16_t*)row)[c + 1] << 16;
    if (c + 2 < n) v.y = ((const uint16_t*)row)[c + 2];
    return v;
}
__device__ __forceinline__ void st4_row(char* row, int64_t c, int64_t n, u32x2 v) {
    if (c + 4 <= n) {
        *(u32x2_at2*)(row + c * 2) = v;
        return;
    }
    if (c < n) ((uint16_t*)row)[c] = (uint16_t)v.x;
    if (c + 1 < n) ((uint16_t*)row)[c + 1] = (uint16_t)(v.x >> 16);
    if (c + 2 < n) ((uint16_t*)row)[c + 2] = (uint16_t)v.y;
}

// What follows a product's sums of one row and four columns: bias, the copy of z in its own type, activation, residual, store.
template <int D, int ACT>
__device__ __forceinline__ void finish4(const GemmArgs& a, int64_t row, int64_t col, const float* z) {
    if (a.z) st4_row(a.z + row * a.np * 2, col, a.np, u32x2{pack2<D>(z[0], z[1]), pack2<D>(z[2], z[3])});
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = activate<ACT>(z[i]);
    if (a.res) {
        const u32x2 r = ld4_row(a.res + row * a.ldr * 2, col, a.np);
        y[0] += elem_lo<D == MQ_F16>(r.x);
        y[1] += elem_hi<D == MQ_F16>(r.x);
        y[2] += elem_lo<D == MQ_F16>(r.y);
        y[3] += elem_hi<D == MQ_F16>(r.y);
    }
    st4_row(a.out + row * a.np * 2, col, a.np, u32x2{pack2<D>(y[0], y[1]), pack2<D>(y[2], y[3])});
}
template <int D>
__device__ __forceinline__ void add_bias4(const GemmArgs& a, int64_t col, float* z) {
    if (!a.bias) return;
    const u32x2 b = ld4_row(a.bias, col, a.np);
    z[0] += elem_lo<D == MQ_F16>(b.x);
    z[1] += elem_hi<D == MQ_F16>(b.x);
    z[2] += elem_lo<D == MQ_F16>(b.y);
    z[3] += elem_hi<D == MQ_F16>(b.y);
}

// the tile of a workgroup: the eight XCDs take turns on the ids, so each is given a run of tiles of its own, and a run goes down four
// tiles of q before it goes on along p, so that the 32 tiles that an XCD works on share their operands in its L2
__device__ __forceinline__ void tile_of(const GemmArgs& a, int& tp, int& tq, int& split) {
    const int tiles = a.tiles_p * a.tiles_q, total = (int)gridDim.x, id = (int)blockIdx.x;
    const int xcd = id & 7, nth = id >> 3, per = total >> 3, more = total & 7;
    int t = xcd * per + (xcd < more ? xcd : more) + nth;
    split = t / tiles;
    t -= split * tiles;
    const int band = 4 * a.tiles_p, b = t / band, in = t - b * band;
    const int high = a.tiles_q - b * 4 < 4 ? a.tiles_q - b * 4 : 4;
    tp = in / high;
    tq = b * 4 + in - tp * high;
}

template <int D, int PM, int QM, int BP, int BQ, int WP, int WQ, bool EPILOGUE>
__global__ __launch_bounds__(WP* WQ* kWave) void gemm_kernel(const GemmArgs a) {
    constexpr int kThreads = WP * WQ * kWave, TP = BP / WP, TQ = BQ / WQ, FP = TP / 16, FQ = TQ / 16;
    constexpr int kPBytes = BP * kStep * 2, kQBytes = BQ * kStep * 2, kBuffer = kPBytes + kQBytes;
    __shared__ __attribute__((aligned(1024))) char shared[2 * kBuffer];
    MQ_LDS char* lds = (MQ_LDS char*)shared;
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
    int tp, tq, split;
    tile_of(a, tp, tq, split);
    const int64_t p0 = (int64_t)tp * BP, q0 = (int64_t)tq * BQ, k0 = split * a.k_split;
    const int64_t k1 = k0 + a.k_split < a.k ? k0 + a.k_split : a.k;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), wp = wave % WP, wq = wave / WP;
    const int lane = threadIdx.x & (kWave - 1);

    Stage<PM, D, BP, kThreads> sp;
    Stage<QM, D, BQ, kThreads> sq;
    sp.init(a.p, a.ps, a.ldp, p0, a.np, k0);
    sq.init(a.q, nullptr, a.ldq, q0, a.nq, k0);
    Fragments<PM, BP, FP> fp;
    Fragments<QM, BQ, FQ> fq;
    fp.init(wp * TP);
    fq.init(wq * TQ);

    f32x4 acc[FP][FQ];
#pragma unroll
    for (int i = 0; i < FP; i++)
#pragma unroll
        for (int j = 0; j < FQ; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    if (k0 < k1) {
        sp.fetch(lds0, k1 - k0);
        sq.fetch(lds0 + kPBytes, k1 - k0);
        sp.put(lds);
        sq.put(lds + kPBytes);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int now = 0;
    for (int64_t k = k0; k < k1; k += kStep) {
        const int next = now ^ kBuffer;                  // (the buffers lie at 0 and kBuffer)
        const bool more = k + kStep < k1;
        if (more) {
            sp.fetch(lds0 + next, k1 - k - kStep);
            sq.fetch(lds0 + next + kPBytes, k1 - k - kStep);
        }
#pragma unroll
        for (int s = 0; s < 2; s++) {
            u32x4 p[FP], q[FQ];
#pragma unroll
            for (int i = 0; i < FP; i++) p[i] = fp.get(lds + now, s, i);
#pragma unroll
            for (int j = 0; j < FQ; j++) q[j] = fq.get(lds + now + kPBytes, s, j);
#pragma unroll
            for (int i = 0; i < FP; i++)
#pragma unroll
                for (int j = 0; j < FQ; j++) acc[i][j] = mfma<D>(p[i], q[j], acc[i][j]);
        }
        if (more) {
            sp.put(lds + next);
            sq.put(lds + next + kPBytes);
        }
        // the next step's operands have arrived, and every wavefront is done with this step's, whose buffer is filled next
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        now = next;
    }

    const int64_t row0 = q0 + wq * TQ + (lane & 15), col0 = p0 + wp * TP + (lane >> 4) * 4;
    if (a.ws) {
        const int64_t ldw = (a.np + 3) / 4 * 4;
#pragma unroll
        for (int j = 0; j < FQ; j++) {
            const int64_t row = row0 + j * 16;
            if (row >= a.nq) continue;
            float* to = a.ws + ((int64_t)split * a.nq + row) * ldw;
#pragma unroll
            for (int i = 0; i < FP; i++) {
                const int64_t col = col0 + i * 16;
                if (col < a.np) *(f32x4*)(to + col) = acc[i][j];
            }
        }
        return;
    }
    if (!EPILOGUE) {
#pragma unroll
        for (int j = 0; j < FQ; j++) {
            const int64_t row = row0 + j * 16;
            if (row >= a.nq) continue;
#pragma unroll
            for (int i = 0; i < FP; i++)
                st4_row(a.out + row * a.np * 2, col0 + i * 16, a.np, u32x2{pack2<D>(acc[i][j][0], acc[i][j][1]), pack2<D>(acc[i][j][2], acc[i][j][3])});
        }
        return;
    }
    with_activation(a.act, [&](auto kind) {
        constexpr int ACT = decltype(kind)::value;
#pragma unroll
        for (int i = 0; i < FP; i += 2) {
#pragma unroll
            for (int j = 0; j < FQ; j++) {
                const int64_t row = row0 + j * 16;
                float z[2][4];
                uint32_t m = 0;
#pragma unroll
                for (int h = 0; h < 2; h++) {
#pragma unroll
                    for (int x = 0; x < 4; x++) z[h][x] = acc[i + h][j][x];
                    add_bias4<D>(a, col0 + (i + h) * 16, z[h]);
#pragma unroll
                    for (int x = 0; x < 4; x++) m = umax(m, keep_magnitude(z[h][x]));
                }
                if (a.zq) {                              // 32 columns: two fragments of the four lanes with this row
                    m = umax(m, (uint32_t)__shfl_xor((int)m, 16));
                    m = umax(m, (uint32_t)__shfl_xor((int)m, 32));
                    const uint32_t e = keep_exponent(m);
                    const float inv = e8m0_inverse(e);
                    if (row < a.nq && col0 + i * 16 < a.np) {
                        uint8_t* to = a.zq + row * a.np + col0 + i * 16;
                        *(uint32_t*)to = keep_codes4(z[0][0], z[0][1], z[0][2], z[0][3], inv);
                        *(uint32_t*)(to + 16) = keep_codes4(z[1][0], z[1][1], z[1][2], z[1][3], inv);
                        if (lane < 16) a.zs[row * (a.np / 32) + (col0 + i * 16) / 32] = (uint8_t)e;
                    }
                }
                if (row < a.nq) {
                    finish4<D, ACT>(a, row, col0 + i * 16, z[0]);
                    finish4<D, ACT>(a, row, col0 + (i + 1) * 16, z[1]);
                }
            }
        }
    });
}

// ---- the host's side ---------------------------------------------------------------------------------------------------------
enum { kTileLarge = 0, kTileMiddle = 1, kTileLow = 2 };       // 256 x 256, 128 x 128, 128 (p) x 64 (q)
struct GemmPlan {
    int tile, splits;
    int64_t k_split;
};

template <int D, int PM, int QM, bool EPILOGUE>
int gemm_launch(GemmArgs& a, const GemmPlan& plan, float* ws, hipStream_t st) {
    a.ws = plan.splits > 1 ? ws : nullptr;
    a.k_split = plan.k_split;
    const int bp = plan.tile == kTileLarge ? 256 : 128, bq = plan.tile == kTileLarge ? 256 : plan.tile == kTileMiddle ? 128 : 64;
    a.tiles_p = (int)((a.np + bp - 1) / bp);
    a.tiles_q = (int)((a.nq + bq - 1) / bq);
    const dim3 grid((unsigned)((int64_t)a.tiles_p * a.tiles_q * plan.splits));
    constexpr bool kBounded = PM == kRowsAny || PM == kDownAny || QM == kRowsAny || QM == kDownAny;
    if constexpr (kBounded) {
        hipLaunchKernelGGL((gemm_kernel<D, PM, QM, 128, 128, 2, 2, EPILOGUE>), grid, dim3(256), 0, st, a);
    } else if (plan.tile == kTileLarge) {
        hipLaunchKernelGGL((gemm_kernel<D, PM, QM, 256, 256, 2, 4, EPILOGUE>), grid, dim3(512), 0, st, a);
    } else if (plan.tile == kTileMiddle) {
        hipLaunchKernelGGL((gemm_kernel<D, PM, QM, 128, 128, 2, 2, EPILOGUE>), grid, dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL((gemm_kernel<D, PM, QM, 128, 64, 2, 2, EPILOGUE>), grid, dim3(256), 0, st, a);
    }
    return MQ_OK;
}

}  // namespace mq

// the three products, each in a file of its own: launched as planned, the partial sums of several splits left in ws
int mq_gemm_forward(int dtype, bool bounded, mq::GemmArgs& a, const mq::GemmPlan& plan, float* ws, hipStream_t st);
int mq_gemm_input_grad(int dtype, bool bounded, mq::GemmArgs& a, const mq::GemmPlan& plan, float* ws, hipStream_t st);
int mq_gemm_weight_grad(int dtype, bool bounded, mq::GemmArgs& a, const mq::GemmPlan& plan, float* ws, hipStream_t st);
