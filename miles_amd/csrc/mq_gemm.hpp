// Matrix products of 16-bit operands on the matrix cores, fp32 sums: out[q][p] = sum over k of Q(q, k) P(p, k).
//
// The three products of a linear layer y = x W^T differ in how the operands lie in memory:
//   forward          P = W [N][K], Q = x [M][K]          both with k along the rows
//   input gradient   P = W [N][K] read as (k of W, n), Q = dz [M][N]
//   weight gradient  P = x [M][K] or its 8-bit copy, Q = dz [M][N], both with the sum going down the rows
// A workgroup computes a BP x BQ tile of the output in steps of 64 along k: the operands of a step lie in shared memory while those
// of the next steps are on their way.
//
// Operands with k along the rows lie in shared memory as rows of 64 elements, a cache line of memory each (eight 16-byte slots; slot s
// of row r holds the row's piece s ^ (r / 2 & 7), so that the rows of a fragment are read from all banks); a lane's eight k are
// one 16-byte read.  Operands whose sum goes down the rows lie as 64 rows of BP or BQ elements (32-byte slots, slot c of row k holds
// piece c ^ swizzle(k)); a lane's eight k come by two transposing reads of four rows by 16 columns for each 16 lanes.
// The P operand is the first of the matrix instruction (32 x 32 x 16 in the largest tile, 16 x 16 x 32 in the others): four of a lane's
// results are neighbours along p, the rows of the output.
//
// Large products are bound by the matrix cores: 8192^3 in bf16 783 us (1405 TFLOP/s at the clock that the card holds then; matrix
// instructions take 76 % of the cycles), 8192 x 9728 x 2560 forward 346, input gradient 330, weight gradient 336, from 8 bits 375, and
// forward with GELU and 8 bits of its argument 428, whose epilogue has one wavefront a SIMD to run on.  With zeros, at full clock, 8192^3
// takes 580 us, and 546 in a copy where every step reads the same operands again, from the nearest cache: the way from memory costs 8 % (13 % at
// 16384 x 2048 x 7168), since a buffer of the next step but one is free only when this step's last fragments have been read.  Small
// products are bound by that way throughout: 2048^3 25 us.
#pragma once
#include "mq_act.hpp"
#include "mq_rows.hpp"

namespace mq {

constexpr int kStep = 64;                 // k of a step

// How an operand is staged: k along its rows or down them, straight into shared memory; or from an 8-bit copy, whose 16-bit values are
// made on the way.  Rows begin at multiples of 16 bytes, and the last piece of eight of a row is read whole: what lies behind the
// operand's end along k has to be zero there (an operand that is not like that is copied first).
enum { kRows = 0, kDown = 1, kDownKept = 2 };

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
    // Tiles from `whole` on are cut along k into `splits` parts of k_split (a multiple of the step); part s of tile t leaves its sums
    // at ws + ((t - whole) splits + s) BP BQ, row by row.
    float* ws;
    int64_t k_split;
    int tiles_p, tiles_q, whole, splits, act;
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
#define MQ_LDS __attribute__((address_space(3)))

template <int D>
__device__ __forceinline__ f32x4 mfma(u32x4 p, u32x4 q, f32x4 c) {
    if (D == MQ_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, p), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
}

// 32 x 32 outputs, 16 k
template <int D>
__device__ __forceinline__ f32x16 mfma(u32x4 p, u32x4 q, f32x16 c) {
    if (D == MQ_F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, p), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
}

// 16 bytes from memory straight into shared memory: lane i's go to `lds` + 16 i (lds uniform), from rsrc's base + offset, zeros where
// the offset is not below 2^31 - 1.  The instruction has no register result; the caller waits for it.  It writes m0 and says so: that is
// one of the compiler's reserved registers, which sets it before each instruction of its own that reads it and merges settings that
// nothing between them is declared to change.  (The warning is about reserved registers in general.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void direct16(uint32_t lds, u32x4 rsrc, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(rsrc) : "m0", "memory");
}
#pragma clang diagnostic pop
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

// the same into registers, and one byte
__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource_of(const void* base) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7FFFFFFF, 0x00027000);
}
__device__ __forceinline__ u32x4 read16(const void* base, uint32_t offset) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(resource_of(base), (int)offset, 0, 0));
}
__device__ __forceinline__ uint32_t read1(const void* base, uint32_t offset) {
    return __builtin_amdgcn_raw_buffer_load_b8(resource_of(base), (int)offset, 0, 0);
}

// piece order of row k of an operand that lies down the rows, 32-byte pieces, B elements to a row
template <int B>
__device__ __forceinline__ int down_swizzle(int k) { return ((k & 3) | ((k >> 1) & 4)) & (B / 16 - 1); }

// One operand's way into shared memory.  A buffer is B x 64 elements; thread t's unit u is the 16 bytes at (t + u THREADS) 16.
template <int MODE, int D, int B, int THREADS>
struct Stage {
    static constexpr bool kAcross = MODE == kRows;
    static constexpr bool kKept = MODE == kDownKept;
    static constexpr bool kDirect = !kKept;
    static constexpr int kUnits = B * 8 / THREADS;
    static constexpr int kPieces = kKept ? kUnits / 2 : kUnits;       // accesses to memory: 16 codes fill two units
    static_assert(B * 8 % (THREADS * (kKept ? 2 : 1)) == 0, "whole units");

    const char* base;                     // the tile's first element at the next step's first k
    const uint8_t* scales;
    int64_t ld, n;                        // n: outputs from the tile's first on
    int64_t step_bytes;
    uint32_t offset[kPieces];
    u32x4 coming[kKept ? kPieces : 1], v[kKept ? kPieces : 1];        // codes on their way, and those that have arrived
    uint32_t coming_e[kKept ? kPieces : 1], e[kKept ? kPieces : 1];

    static __device__ __forceinline__ int row_piece(int at) { return (at & 7) ^ (at >> 4 & 7); }
    static __device__ __forceinline__ int down_k(int at) { return at / (B / 8); }
    static __device__ __forceinline__ int down_col(int at) {
        const int unit = at % (B / 8);
        return ((unit >> 1) ^ down_swizzle<B>(down_k(at))) * 16 + (unit & 1) * 8;
    }

    __device__ __forceinline__ void init(const char* op, const uint8_t* s, int64_t ld_, int64_t first, int64_t count, int64_t k0) {
        ld = ld_;
        n = count - first;
        constexpr int kSize = kKept ? 1 : 2;
        base = op + (kAcross ? first * ld + k0 : k0 * ld + first) * kSize;
        step_bytes = (kAcross ? kStep : kStep * ld) * kSize;
        if (kKept) scales = s + k0 * (ld / 32) + first / 32;
        if (kDirect) {
#pragma unroll
            for (int u = 0; u < kUnits; u++) {
                const int at = (int)threadIdx.x + u * THREADS;
                if (kAcross) {
                    const int row = at >> 3, c = row_piece(at);
                    offset[u] = (uint32_t)((row < n ? row : n - 1) * ld * 2 + c * 16);
                } else {
                    const int k = down_k(at), c = down_col(at);
                    offset[u] = (uint32_t)((int64_t)k * ld * 2 + (c < n ? c : 0) * 2);
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < kPieces; u++) {
                const int at = ((int)threadIdx.x + u * THREADS) * 2, c = down_col(at);
                offset[u] = (uint32_t)(down_k(at) * ld + (c < n ? c : 0));
            }
        }
    }
    // The next step's operand, piece by piece: on its way to `lds` (direct), or into registers.  left: k that are left from the step's
    // first on, from zero down for a step behind the last, whose operands are zeros.  All pieces of a step, then `advance`.
    __device__ __forceinline__ void fetch_piece(int u, uint32_t lds, int left) {
        if (kDirect) {
            const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave) * (kWave * 16);
            const int at = (int)threadIdx.x + u * THREADS, k = kAcross ? row_piece(at) * 8 : down_k(at);
            direct16(lds + wave + u * (THREADS * 16), buffer_of(base), k < left ? offset[u] : kNowhere);
        } else {
            const bool inside = down_k(((int)threadIdx.x + u * THREADS) * 2) < left;
            coming[u] = read16(base, inside ? offset[u] : kNowhere);
            coming_e[u] = read1(scales, inside ? offset[u] / 32 : kNowhere);                  // (ld is a multiple of 32)
        }
    }
    __device__ __forceinline__ void advance() {
        base += step_bytes;
        if (kKept) scales += kStep * (ld / 32);
    }
    // The codes have arrived: said where the wavefront has waited for them anyway, because a wait that the compiler put in front of
    // their use would also wait for the accesses issued since, which it does not know of.
    __device__ __forceinline__ void settle() {
        if (kDirect) return;
#pragma unroll
        for (int u = 0; u < kPieces; u++) {
            asm volatile("" : "+v"(coming[u].x), "+v"(coming[u].y), "+v"(coming[u].z), "+v"(coming[u].w), "+v"(coming_e[u]));
            v[u] = coming[u];
            e[u] = coming_e[u];
        }
    }
    // Half of an 8-bit piece, eight values, that came through registers, into shared memory: which half first depends on the lane, so
    // that lanes whose slots lie in the same banks write different halves.
    __device__ __forceinline__ void put_half(int u, int turn, MQ_LDS char* lds) {
        if (kDirect) return;
        const bool high = (turn != 0) != ((threadIdx.x & 8) != 0);
        const u32x2 a = kept_pack4<D>(high ? v[u].z : v[u].x, e[u]), b = kept_pack4<D>(high ? v[u].w : v[u].y, e[u]);
        *(MQ_LDS u32x4*)(lds + ((int)threadIdx.x + u * THREADS) * 32 + (high ? 16 : 0)) = u32x4{a.x, a.y, b.x, b.y};
    }
};

// Addresses of a wavefront's fragments of an operand in shared memory: F fragments of 16 outputs from `first` on
template <int MODE, int B, int F>
struct Fragments {
    static constexpr bool kAcross = MODE == kRows;
    uint32_t at[kAcross ? 2 : F];

    __device__ __forceinline__ void init(int first) {
        const int lane = threadIdx.x & (kWave - 1), j = lane & 15, g = lane >> 4;
        if (!kAcross) {
            const int k = g * 8 + (j >> 2);
#pragma unroll
            for (int f = 0; f < F; f++) at[f] = (uint32_t)(k * (B * 2) + ((first / 16 + f) ^ down_swizzle<B>(k)) * 32 + (j & 3) * 8);
        } else {
#pragma unroll
            for (int s = 0; s < 2; s++) at[s] = (uint32_t)((first + j) * 128 + ((g + 4 * s) ^ (j >> 1 & 7)) * 16);
        }
    }
    // fragment f of the 32 k from 32 s on
    __device__ __forceinline__ u32x4 get(MQ_LDS char* lds, int s, int f) const {
        if (!kAcross) {
            MQ_LDS char* from = lds + at[f] + s * (32 * B * 2);
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MQ_LDS s16x4*)from);
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MQ_LDS s16x4*)(from + 4 * B * 2));
            const u32x2 x = __builtin_bit_cast(u32x2, a), y = __builtin_bit_cast(u32x2, b);
            return u32x4{x.x, x.y, y.x, y.y};
        }
        return *(MQ_LDS const u32x4*)(lds + at[s] + f * 2048);
    }
};

// The same for fragments of 32 outputs and 16 k, four of them along k in a step
template <int MODE, int B, int F>
struct WideFragments {
    static constexpr bool kAcross = MODE == kRows;
    uint32_t at[4];
    static_assert(F == 4, "addresses for fragments, or for the parts of a step");

    __device__ __forceinline__ void init(int first) {
        const int lane = threadIdx.x & (kWave - 1);
        if (!kAcross) {
            const int j = lane & 15, g = lane >> 4, k = (g >> 1) * 8 + (j >> 2);
#pragma unroll
            for (int f = 0; f < F; f++) at[f] = (uint32_t)(k * (B * 2) + ((first / 16 + f * 2 + (g & 1)) ^ down_swizzle<B>(k)) * 32 + (j & 3) * 8);
        } else {
            const int j = lane & 31, g = lane >> 5;
#pragma unroll
            for (int h = 0; h < 4; h++) at[h] = (uint32_t)((first + j) * 128 + ((g + 2 * h) ^ (j >> 1 & 7)) * 16);
        }
    }
    // fragment f of the 16 k from 16 h on
    __device__ __forceinline__ u32x4 get(MQ_LDS char* lds, int h, int f) const {
        if (!kAcross) {
            MQ_LDS char* from = lds + at[f] + h * (16 * B * 2);
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MQ_LDS s16x4*)from);
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MQ_LDS s16x4*)(from + 4 * B * 2));
            const u32x2 x = __builtin_bit_cast(u32x2, a), y = __builtin_bit_cast(u32x2, b);
            return u32x4{x.x, x.y, y.x, y.y};
        }
        return *(MQ_LDS const u32x4*)(lds + at[h] + f * 4096);
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

// Where tile t lies: down four tiles of q before it goes on along p, so that the 32 tiles that an XCD works on share their operands
// in its L2.
__device__ __forceinline__ void place_of(const GemmArgs& a, int t, int& tp, int& tq) {
    const int band = 4 * a.tiles_p, b = t / band, in = t - b * band;
    const int high = a.tiles_q - b * 4 < 4 ? a.tiles_q - b * 4 : 4;
    tp = in / high;
    tq = b * 4 + in - tp * high;
}
// the tile and part of a workgroup: whole tiles first; the eight XCDs take turns on the ids, so each is given a run of tiles of its own
__device__ __forceinline__ void tile_of(const GemmArgs& a, int& tile, int& part) {
    const int id = (int)blockIdx.x, tail = id >= a.whole, total = tail ? (int)gridDim.x - a.whole : a.whole, mine = tail ? id - a.whole : id;
    const int xcd = mine & 7, nth = mine >> 3, per = total >> 3, more = total & 7;
    const int t = xcd * per + (xcd < more ? xcd : more) + nth;
    tile = tail ? a.whole + t / a.splits : t;
    part = tail ? t % a.splits : -1;
}

// every wavefront of the workgroup has come this far, with its reads and writes of shared memory done; nothing is moved across
__device__ __forceinline__ void meet() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

// what a wavefront's lanes have written to shared memory is there for its other lanes, and what they have read may be overwritten
__device__ __forceinline__ void lanes_meet() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// What follows the sums, from shared memory: 64 columns of ROWS rows of one wavefront, in fp32, four columns at position
// (column / 4) ^ (row & 15) of a row's sixteen.  A lane has eight columns, so that eight lanes store whole lines.
__device__ __forceinline__ int stage_at(int row, int four) { return row * 256 + ((four ^ (row & 15)) * 16); }

template <int D, bool EPILOGUE, int ROWS>
__device__ __forceinline__ void finish_block(const GemmArgs& a, float* sums, int pitch, int64_t row0, int64_t col0, MQ_LDS const char* stage) {
    const int lane = threadIdx.x & (kWave - 1), mine = lane & 7;
    const int64_t col = col0 + mine * 8;
    if (!EPILOGUE || sums) {                               // sums: where a part's go, rows `pitch` apart
        for (int r = lane >> 3; r < ROWS; r += 8) {
            const int64_t row = row0 + r;
            if (row >= a.nq) break;
            const f32x4 lo = *(MQ_LDS const f32x4*)(stage + stage_at(r, 2 * mine)), hi = *(MQ_LDS const f32x4*)(stage + stage_at(r, 2 * mine + 1));
            if (sums) {
                f32x4* to = (f32x4*)(sums + r * pitch + mine * 8);
                to[0] = lo;
                to[1] = hi;
            } else {
                const float z[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                st_row<D>(a.out + row * a.np * 2, col, a.np, pack<D>(z));
            }
        }
        return;
    }
    float bias[8];
    if (a.bias) {
        unpack<D>(ld_row<D>(a.bias, col, a.np), bias);
    } else {
#pragma unroll
        for (int x = 0; x < 8; x++) bias[x] = 0.0f;
    }
    // four rows at a time, whose loads are issued together: one wavefront on a SIMD has nobody to wait behind
    constexpr int kAtOnce = 4;
    static_assert(ROWS % (8 * kAtOnce) == 0, "whole rounds");
    with_activation(a.act, [&](auto kind) {
        constexpr int ACT = decltype(kind)::value;
        for (int r0 = lane >> 3; r0 < ROWS; r0 += 8 * kAtOnce) {
            float z[kAtOnce][8];
            u32x4 res[kAtOnce];
            if (row0 + r0 >= a.nq) break;                  // (the four lanes of 32 columns have one row)
#pragma unroll
            for (int i = 0; i < kAtOnce; i++) {
                const int r = r0 + 8 * i;
                if (a.res && row0 + r < a.nq) res[i] = ld_row<D>(a.res + (row0 + r) * a.ldr * 2, col, a.np);
                const f32x4 lo = *(MQ_LDS const f32x4*)(stage + stage_at(r, 2 * mine)), hi = *(MQ_LDS const f32x4*)(stage + stage_at(r, 2 * mine + 1));
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    z[i][x] = lo[x];
                    z[i][4 + x] = hi[x];
                }
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; i++) {
                const int64_t row = row0 + r0 + 8 * i;
                if (row >= a.nq) break;
#pragma unroll
                for (int x = 0; x < 8; x++) z[i][x] += bias[x];
                if (a.zq) {
                    float top = 0.0f;
#pragma unroll
                    for (int x = 0; x < 8; x++) top = keep_larger(top, z[i][x]);
                    const uint32_t m = group_max4(f2u(top)), e = keep_exponent(m);
                    const float inv = e8m0_inverse(e);
                    if (col < a.np) {
                        uint32_t* to = (uint32_t*)(a.zq + row * a.np + col);
                        to[0] = keep_codes4(z[i][0], z[i][1], z[i][2], z[i][3], inv, m == kInfinity);
                        to[1] = keep_codes4(z[i][4], z[i][5], z[i][6], z[i][7], inv, m == kInfinity);
                        if ((lane & 3) == 0) a.zs[row * (a.np / 32) + col / 32] = (uint8_t)e;
                    }
                }
                if (a.z) st_row<D>(a.z + row * a.np * 2, col, a.np, pack<D>(z[i]));
#pragma unroll
                for (int x = 0; x < 8; x++) z[i][x] = activate<ACT>(z[i][x]);
                if (a.res) {
                    float f[8];
                    unpack<D>(res[i], f);
#pragma unroll
                    for (int x = 0; x < 8; x++) z[i][x] += f[x];
                }
                st_row<D>(a.out + row * a.np * 2, col, a.np, pack<D>(z[i]));
            }
        }
    });
}

// Buffers of a smaller tile: three of the 128 x 64 one and two workgroups on a compute unit, except in the weight gradient, whose sum is
// short where this tile is chosen, two and three.  (48 x 2560 x 9728 in us with two and three buffers: forward 18.6 and 16.6, input
// gradient 17.7 and 16.0, weight gradient 18 and 23; 512 x 2048 x 2048 forward 20.7 and 18.4.  Four and six buffers leave one workgroup:
// 48 x 2560 x 9728 forward 17 and 18, 2048^3 35 and 37 where three take 25.  The 128 x 128 tile with three: weight gradient of
// 200 x 2560 x 2560 14.8 for 10.7.)
constexpr int small_ring(int bq, bool weight_grad) { return bq == 64 && !weight_grad ? 3 : 2; }

template <int D, int PM, int QM, int BP, int BQ, int WP, int WQ, bool EPILOGUE>
__global__ __launch_bounds__(WP* WQ* kWave) __attribute__((amdgpu_waves_per_eu(1))) void gemm_kernel(const GemmArgs a) {
    constexpr int kThreads = WP * WQ * kWave, TP = BP / WP, TQ = BQ / WQ, FP = TP / 16, FQ = TQ / 16;
    constexpr int kPBytes = BP * kStep * 2, kQBytes = BQ * kStep * 2, kBuffer = kPBytes + kQBytes;
    constexpr int kRing = small_ring(BQ, QM == kDown);     // buffers of a smaller tile
    __shared__ __attribute__((aligned(1024))) char shared[BP == 256 ? 5 * kPBytes : kRing * kBuffer];
    MQ_LDS char* lds = (MQ_LDS char*)shared;
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
    int tile, part, tp, tq;
    tile_of(a, tile, part);
    place_of(a, tile, tp, tq);
    const int64_t p0 = (int64_t)tp * BP, q0 = (int64_t)tq * BQ, k0 = part < 0 ? 0 : part * a.k_split;
    const int64_t k1 = part >= 0 && k0 + a.k_split < a.k ? k0 + a.k_split : a.k;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), wp = wave % WP, wq = wave / WP;
    float* sums = part < 0 ? nullptr : a.ws + ((int64_t)(tile - a.whole) * a.splits + part) * (BP * BQ) + wq * TQ * BP + wp * TP;
    const int lane = threadIdx.x & (kWave - 1);

    Stage<PM, D, BP, kThreads> sp;
    Stage<QM, D, BQ, kThreads> sq;
    sp.init(a.p, a.ps, a.ldp, p0, a.np, k0);
    sq.init(a.q, nullptr, a.ldq, q0, a.nq, k0);
    const int steps = (int)((k1 - k0 + kStep - 1) / kStep);
    const int span = (int)(k1 - k0);
    auto left_of = [&](int t) { return span - t * kStep; };
    // A step's pieces of one operand, on their way to buffer `to`.  The same number of accesses for every step, also behind the last
    // (there they read nothing), so that a wavefront knows by counting which have arrived.
    auto fetch_p = [&](int t, uint32_t to) {
        const int left = left_of(t);
#pragma unroll
        for (int u = 0; u < sp.kPieces; u++) sp.fetch_piece(u, to, left);
        sp.advance();
    };
    auto fetch_q = [&](int t, uint32_t to) {
        const int left = left_of(t);
#pragma unroll
        for (int u = 0; u < sq.kPieces; u++) sq.fetch_piece(u, to, left);
        sq.advance();
    };
    auto put_p = [&](MQ_LDS char* to) {                    // what has arrived in registers
#pragma unroll
        for (int u = 0; u < sp.kPieces; u++)
#pragma unroll
            for (int turn = 0; turn < 2; turn++) sp.put_half(u, turn, to);
    };
    constexpr bool kPDirect = PM != kDownKept;
    static_assert(QM != kDownKept, "the first operand may be an 8-bit copy");
    if constexpr (BP == 256) {
        // One wavefront on each SIMD, 128 x 128 outputs each: four of them read half of what eight would from shared memory.  The
        // next 16 k's fragments are read between the products of these.  Halfway through a step every wavefront has the rest of its
        // fragments, so that its buffer is free for the step after the next three, and has seen its part of the next step arrive.
        constexpr int F = 4;
        WideFragments<PM, BP, F> fp;
        WideFragments<QM, BQ, F> fq;
        fp.init(wp * TP);
        fq.init(wq * TQ);
        f32x16 acc[F][F];
#pragma unroll
        for (int i = 0; i < F; i++)
#pragma unroll
            for (int j = 0; j < F; j++)
#pragma unroll
                for (int x = 0; x < 16; x++) acc[i][j][x] = 0.0f;
        // Five buffers of one operand of one step each, P and Q of the steps in turn: those of step t and t + 1, and P of step t + 2.
        constexpr uint32_t kFifth = kPBytes, kAll = 5 * kFifth;
        auto after = [&](uint32_t buffer, uint32_t by) { return buffer + by * kFifth >= kAll ? buffer + by * kFifth - kAll : buffer + by * kFifth; };
        static_assert(BP == BQ && sq.kPieces == 8 && sp.kPieces == (kPDirect ? 8 : 4), "buffers of one size, a piece for every other product");
        fetch_p(0, lds0);
        sp.settle();
        put_p(lds);
        fetch_q(0, lds0 + kFifth);
        fetch_p(1, lds0 + 2 * kFifth);
        fetch_q(1, lds0 + 3 * kFifth);
        asm volatile("s_waitcnt vmcnt(%0)" ::"i"(kPDirect ? sp.kUnits + sq.kUnits : 0) : "memory");
        meet();
        sp.settle();
        u32x4 p[2][F], q[2][F];
#pragma unroll
        for (int i = 0; i < F; i++) {
            p[0][i] = fp.get(lds, 0, i);
            q[0][i] = fq.get(lds + kFifth, 0, i);
        }
        uint32_t at = 0;                                    // the buffer of P of step t
        for (int t = 0; t < steps; t++) {
            const uint32_t next = after(at, 2), third = after(at, 4);
            const int left = left_of(t + 2);
            // A wavefront issues an instruction in about four cycles and its product takes 32: what goes between two products is kept
            // short, and the reads come first, so that they are back when the products that need them are due.
#pragma unroll
            for (int h = 0; h < 4; h++) {
                if (h == 3) {
                    // this step's fragments are all in registers and so its buffers are free; the next step's operands have arrived,
                    // whose last pieces were asked for a step ago (P of step t + 2 may still be on its way; an 8-bit one has come into
                    // registers)
                    asm volatile("s_waitcnt vmcnt(%0)" ::"i"(kPDirect ? sp.kUnits : 0) : "memory");
                    meet();
                    sp.settle();
                }
                MQ_LDS char* fromp = lds + (h == 3 ? next : at);
                MQ_LDS char* fromq = lds + (h == 3 ? after(next, 1) : after(at, 1));
#pragma unroll
                for (int m = 0; m < F * F; m++) {
                    acc[m / F][m % F] = mfma<D>(p[h & 1][m / F], q[h & 1][m % F], acc[m / F][m % F]);
                    if (m < F) p[h & 1 ^ 1][m] = fp.get(fromp, h + 1 & 3, m);
                    else if (m < 2 * F) q[h & 1 ^ 1][m - F] = fq.get(fromq, h + 1 & 3, m - F);
                    else if (kPDirect && h < 2) {            // P of step t + 2, eight pieces in two parts of this step
                        if (m % 2 == 0) sp.fetch_piece((m - 8) / 2 + h * 4, lds0 + third, left);
                    } else if (h == 3) {
                        sq.fetch_piece(m - 8, lds0 + at, left);
                    }
                    // An 8-bit P: that of step t + 2 is asked for, and that of step t + 1 written out of its registers.
                    if (!kPDirect) {
                        if (h == 0 && m < 8 && m % 2 == 1) sp.fetch_piece(m / 2, 0, left);
                        if (h < 2 && m >= 8 && m % 2 == 0) sp.put_half((m - 8) / 4 + h * 2, m / 2 % 2, lds + next);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            sp.advance();
            sq.advance();
            at = next;
        }
        // nothing may reach this shared memory when it is another workgroup's
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        meet();
        MQ_LDS char* stage = lds + wave * (TQ * 256);
        const int row = lane & 31, four = lane >> 5;        // a lane has sixteen columns of a row, fours that are eight apart
        auto finish_half = [&](auto which) {               // (written out twice: the sums are registers, whose numbers are constants)
            constexpr int half = decltype(which)::value;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < F; j++)
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        const f32x16& c = acc[2 * half + i][j];
                        *(MQ_LDS f32x4*)(stage + stage_at(j * 32 + row, i * 8 + x * 2 + four)) = f32x4{c[4 * x], c[4 * x + 1], c[4 * x + 2], c[4 * x + 3]};
                    }
            lanes_meet();
            finish_block<D, EPILOGUE, TQ>(a, sums ? sums + half * 64 : nullptr, BP, q0 + wq * TQ, p0 + wp * TP + half * 64, stage);
        };
        finish_half(std::integral_constant<int, 0>{});
        lanes_meet();
        finish_half(std::integral_constant<int, 1>{});
    } else {
        Fragments<PM, BP, FP> fp;
        Fragments<QM, BQ, FQ> fq;
        fp.init(wp * TP);
        fq.init(wq * TQ);
        f32x4 acc[FP][FQ];
#pragma unroll
        for (int i = 0; i < FP; i++)
#pragma unroll
            for (int j = 0; j < FQ; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        // Several workgroups on a compute unit, two or three buffers each.  While step t is worked on, the next one or two are on their
        // way; what goes through registers was loaded a step earlier.
        static_assert(kPDirect || kRing == 2, "the registers hold the step after the next");
#pragma unroll
        for (int t = 0; t < kRing - 1; t++) {
            fetch_p(t, lds0 + t * kBuffer);
            fetch_q(t, lds0 + t * kBuffer + kPBytes);
        }
        if (!kPDirect) {
            sp.settle();
            put_p(lds);
            fetch_p(1, 0);
        }
        uint32_t at = 0;                                    // the buffer of step t
        for (int t = 0; t < steps; t++) {
            MQ_LDS char* from = lds + at;
            const uint32_t before = at == 0 ? (kRing - 1) * kBuffer : at - kBuffer;
            // this step has arrived, and everybody has read the one before, whose buffer is the next to be filled
            asm volatile("s_waitcnt vmcnt(%0)" ::"i"((kRing - 2) * (sp.kUnits + sq.kUnits)) : "memory");
            meet();
            sp.settle();
            fetch_q(t + kRing - 1, lds0 + before + kPBytes);
            if (kPDirect) fetch_p(t + kRing - 1, lds0 + before);
            else fetch_p(t + 2, 0);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                u32x4 p[FP], q[FQ];
#pragma unroll
                for (int i = 0; i < FP; i++) p[i] = fp.get(from, h, i);
#pragma unroll
                for (int j = 0; j < FQ; j++) q[j] = fq.get(from + kPBytes, h, j);
#pragma unroll
                for (int i = 0; i < FP; i++)
#pragma unroll
                    for (int j = 0; j < FQ; j++) acc[i][j] = mfma<D>(p[i], q[j], acc[i][j]);
            }
            if (!kPDirect) put_p(lds + before);             // (behind the reads, which would wait for the writes)
            at = at == (kRing - 1) * kBuffer ? 0 : at + kBuffer;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // (as above)
        meet();
        MQ_LDS char* stage = lds + wave * (TQ * 256);
        static_assert(TP == 64, "one block of columns");
#pragma unroll
        for (int i = 0; i < FP; i++)
#pragma unroll
            for (int j = 0; j < FQ; j++) *(MQ_LDS f32x4*)(stage + stage_at(j * 16 + (lane & 15), i * 4 + (lane >> 4))) = acc[i][j];
        lanes_meet();
        finish_block<D, EPILOGUE, TQ>(a, sums, BP, q0 + wq * TQ, p0 + wp * TP, stage);
    }
}

// ---- the host's side ---------------------------------------------------------------------------------------------------------
enum { kTileLarge = 0, kTileMiddle = 1, kTileLow = 2 };       // 256 x 256, 128 x 128, 128 (p) x 64 (q)
struct GemmPlan {
    int tile, tiles_p, tiles_q, whole, splits;
    int64_t k_split;
};
constexpr int kTileP[3] = {256, 128, 128}, kTileQ[3] = {256, 128, 64};

template <int D, int PM, int QM, bool EPILOGUE>
int gemm_launch(GemmArgs& a, const GemmPlan& plan, float* ws, hipStream_t st) {
    a.ws = ws;
    a.k_split = plan.k_split;
    a.tiles_p = plan.tiles_p;
    a.tiles_q = plan.tiles_q;
    a.whole = plan.whole;
    a.splits = plan.splits;
    const dim3 grid((unsigned)(plan.whole + (plan.tiles_p * plan.tiles_q - plan.whole) * plan.splits));
    if (plan.tile == kTileLarge) {
        hipLaunchKernelGGL((gemm_kernel<D, PM, QM, 256, 256, 2, 2, EPILOGUE>), grid, dim3(256), 0, st, a);
    } else if (plan.tile == kTileMiddle) {
        hipLaunchKernelGGL((gemm_kernel<D, PM, QM, 128, 128, 2, 2, EPILOGUE>), grid, dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL((gemm_kernel<D, PM, QM, 128, 64, 2, 2, EPILOGUE>), grid, dim3(256), 0, st, a);
    }
    return MQ_OK;
}

}  // namespace mq

// the three products, each in a file of its own: launched as planned, the partial sums of several splits left in ws
int mq_gemm_forward(int dtype, mq::GemmArgs& a, const mq::GemmPlan& plan, float* ws, hipStream_t st);
int mq_gemm_input_grad(int dtype, mq::GemmArgs& a, const mq::GemmPlan& plan, float* ws, hipStream_t st);
int mq_gemm_weight_grad(int dtype, mq::GemmArgs& a, const mq::GemmPlan& plan, float* ws, hipStream_t st);
