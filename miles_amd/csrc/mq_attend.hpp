// Attention of one token a sequence over a paged cache: softmax(scale q K^T) V with a running maximum and sum, on the matrix cores.
//
// A wavefront takes 32 tokens of a sequence's key head at a time, for up to 16 of the query heads that share it.  Everything goes from memory
// to the matrix instructions through registers, without shared memory and without a lane handing anything to another:
//   scores   S^T = K Q^T, 16 tokens x 16 heads: a lane's operand is eight elements of one token's key, which the cache's layout has beside those
//            of the neighbouring tokens, so that a load covers whole lines.  Lane (c, g) = (lane % 16, lane / 16) gets head c, tokens 4 g + r.
//   output   O^T += V^T P^T: the same lane needs, for element 8 c + e of the values, the weights and values of eight tokens.  Which
//            eight is free as long as both operands agree: 4 g + r of both halves of the 32, whose weights it has, and
//            whose values it reads as rows of 16 bytes; eight such rows are rearranged in its own registers, one instruction for two elements.
// Weights enter as sums of 16-bit numbers (one alone would be off by as much as the result's own rounding): three in bf16, which hold all their bits (two
// would leave 2 in 1000 results on the other side of a rounding, where these leave 4 in 10000), two in fp16, which hold 21, and whatever is above 2^-39 of the
// largest weight in the same tile.  The matrix cores have the time (7 % of the cycles in 16 bits, 13 in 8).  What bounds it is reading keys and values
// once: a tile's keys are asked for when the last tile's have been used, its values likewise, so that a wavefront always has one of the two on its way, and two wavefronts on a
// SIMD keep 64 KB a compute unit in flight.  32 query heads over 8 key heads of 128, bf16: 64 sequences of 8192 tokens 330 us, 6.5 TB/s; 64 of 1 to
// 8192 in 122, 5.9 TB/s (in 8 bits 125, 6.0 TB/s: half the bytes for twice the tokens); one of 131072 in fp16 in 94, 5.7 TB/s; one of 1024 in 12.5.
#pragma once
#include "mq_gemm.hpp"
#include "mq_paged.hpp"

namespace mq {

struct AttendArgs {
    const char *q, *keys, *values;
    const uint8_t *key_scales, *value_scales;
    const int32_t *table, *lengths;
    const float* sinks;
    char* out;
    float* parts;                  // partial results: a first and a last one of every worker
    uint32_t* starts;              // [batch + 1]: units before each sequence, and all of them
    int64_t q_batch, q_head, table_stride, capacity, window;
    uint32_t pages;
    uint32_t key_page, value_page, key_scale_page, value_scale_page;      // bytes of a page, below 2^31
    int batch, heads, kv_heads, group, key_dim, value_dim, page_shift;
    int blocks;                    // of query heads of a key head, block_heads each
    int head_waves;                // wavefronts that share tokens and have 16 different heads of a block each: 1 to 4
    int block_heads;
    uint32_t least;                // units that a worker takes at least
    float scale;                   // with log2(e), positive
    uint32_t flip;                 // signs of two elements of a query, where the scale was negative
};
// A row is a sequence's key head and a block of its query heads; rows are numbered by sequence, key head and block.  A row's units of work are
// its tiles of 32 tokens, behind kRowUnits that stand for what a row costs beside them: queries, the first tile's way from memory, the sums (without them
// 64 sequences of 1 to 8192 tokens in ascending order took 253 us where they take 150).
constexpr uint32_t kRowUnits = 4;
constexpr float kLowest = -3.0e38f;                      // the maximum of no scores: finite, so that differences are numbers
constexpr float kSlack = 8.0f;                           // powers of two by which weights may pass 1 before the sums are rescaled
constexpr int kAttendWaves = 4, kRowPad = 132;           // of a workgroup whose workers share rows out

// Workers of a workgroup that shares rows out: four, or one of several head waves, which go through their tiles in step
__host__ __device__ constexpr int attend_workers(int head_waves) { return head_waves > 1 ? 1 : kAttendWaves; }
// keys, values, queries and sums that fill the registers of one wavefront a SIMD
__host__ __device__ constexpr bool attend_is_wide(int nk, int nv) { return nv == 2 && nk > 4; }
// floats of a worker's partial result: 128 NV sums for each head of a block, then their maxima and totals
__host__ __device__ inline int64_t part_floats(int block_heads, int nv) { return (int64_t)block_heads * (128 * nv + 2); }
__host__ __device__ inline uint32_t units_of(int tiles) { return tiles ? (uint32_t)tiles + kRowUnits : 0u; }
__host__ __device__ inline uint32_t units_of_worker(uint32_t total, uint32_t workers, uint32_t least) {
    const uint32_t share = (total + workers - 1) / workers;
    return share > least ? share : least;
}

#define MQ_CONST __attribute__((address_space(4)))
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ Seen seen_by(const AttendArgs& a, int b) { return seen_of(a.lengths[b], a.capacity, a.window); }
__device__ __forceinline__ Seen seen_uniform(const AttendArgs& a, int b) {
    const Seen s = seen_by(a, b);
    return Seen{uniform(s.lo), uniform(s.hi)};
}

// over the four lanes that have the same head
__device__ __forceinline__ float max_of_head(float v) {
    const auto x = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    v = __builtin_fmaxf(u2f(x[0]), u2f(x[1]));
    const auto y = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
    return __builtin_fmaxf(u2f(y[0]), u2f(y[1]));
}
__device__ __forceinline__ float sum_of_head(float v) {
    const auto x = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    v = u2f(x[0]) + u2f(x[1]);
    const auto y = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
    return u2f(y[0]) + u2f(y[1]);
}

__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {           // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t up = __shfl_up(v, d);
        if (lane >= d) v += up;
    }
    return v;
}

template <int D>
__device__ __forceinline__ void store8(char* to, const float* f) {
    *(u32x4*)to = pack<D>(f);
}
// Two weights as sums of 16-bit numbers, all of them positive where the weight is: a value that is infinite times a part of 0, or times parts of both signs,
// would be a NaN, where its product with the weight is that infinity.  Each part but the last is what is left without its last bits, and where nothing is left
// the smallest number of the type, which the matrix instructions count like any other (bf16: 2^-133; fp16: 2^-24, of 2^15).
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t smaller2(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}
__device__ __forceinline__ uint32_t larger2(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}
template <int D>
constexpr int kWeightParts = D == MQ_F16 ? 2 : 3;
template <int D>
__device__ __forceinline__ void split_weights(float p, float q, u32x4* parts, int i) {
    if (D == MQ_F16) {
        const uint32_t big = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(p, q));
        parts[0][i] = big;
        parts[1][i] = larger2(pack2<D>(p - elem_lo<true>(big), q - elem_hi<true>(big)), smaller2(big, 0x00010001u));
        return;
    }
    uint32_t least = 0u;
#pragma unroll
    for (int part = 0; part < kWeightParts<D>; part++) {
        const uint32_t high = __builtin_amdgcn_perm(f2u(q), f2u(p), 0x07060302u);
        if (part == 0) least = smaller2(high, 0x00010001u);
        parts[part][i] = part == 0 ? high : larger2(high, least);
        p -= u2f(f2u(p) & 0xFFFF0000u);
        q -= u2f(f2u(q) & 0xFFFF0000u);
    }
}
// what a row of sums is multiplied with at the end, with the sink in its total; no weight at all: zeros
__device__ __forceinline__ float finish_factor(const AttendArgs& a, int head, float m, float l) {
    if (a.sinks) {
        const float sink = a.sinks[head] * 1.44269504088896f, top = __builtin_fmaxf(m, sink);
        const float f = __builtin_amdgcn_exp2f(m - top);
        l = l * f + __builtin_amdgcn_exp2f(sink - top);
        return l == 0.0f ? 0.0f : f / l;
    }
    return l == 0.0f ? 0.0f : 1.0f / l;
}

// Not DIRECT: workgroups of kAttendWaves wavefronts, head_waves of them a worker, whose share of all units it finds by itself and which nothing else
// waits for.  DIRECT: a workgroup has one row, its wavefronts every so manieth tile of it, and their sums meet in shared memory.
// SHARED: several head waves, whose accesses to the same lines meet in the compute unit's cache; else every line is read by one wavefront once, and
// the accesses say so (64 sequences of 8192: 6.2 TB/s instead of 5.7).
template <int D, bool KEPT, int NK, int NV, bool DIRECT, bool SHARED>
__global__ __launch_bounds__(kAttendWaves * kWave, attend_is_wide(NK, NV) ? 1 : 2) void attend_kernel(const AttendArgs a) {
    constexpr int kPolicy = SHARED ? 0 : 2;               // (2: non-temporal)
    constexpr int kLoads = KEPT ? NK / 2 : NK;            // of a tile's half's keys
    constexpr bool kOwnTop = D == MQ_F16;                 // a tile's weights are relative to its own maximum
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x / kWave), c = lane & 15, g = lane >> 4;
    const int rows = a.kv_heads * a.blocks;               // of a sequence
    const int head_wave = SHARED ? wave % a.head_waves : 0;

    // ---- which units
    int b;
    uint32_t rest, left, worker = 0;                      // first unit within its sequence, and how many
    bool first_of_worker = true;
    if (DIRECT) {
        const int row = (int)blockIdx.x % rows;
        b = (int)blockIdx.x / rows;
        const int tiles = tiles_of(seen_uniform(a, b));
        if (tiles == 0) {                                 // nothing to see
            const int n = a.group * a.value_dim / 8;
            if (row % a.blocks == 0) {
                char* to = a.out + ((int64_t)b * a.heads + (int64_t)(row / a.blocks) * a.group) * a.value_dim * 2;
                for (int i = threadIdx.x; i < n; i += (int)blockDim.x) *(u32x4*)(to + (int64_t)i * 16) = u32x4{0u, 0u, 0u, 0u};
            }
            return;
        }
        rest = (uint32_t)row * units_of(tiles);
        left = units_of(tiles);
    } else {
        const uint32_t workers = gridDim.x * (SHARED ? 1 : kAttendWaves);
        worker = SHARED ? blockIdx.x : blockIdx.x * kAttendWaves + wave;
        uint32_t total = 0, units = 0;
        for (int s = lane; s < a.batch; s += 64) total += (units = units_of(tiles_of(seen_by(a, s))) * rows);
        total = (uint32_t)uniform((int)wave_sum(total));
        const uint32_t per = units_of_worker(total, workers, a.least);
        const uint64_t u0 = (uint64_t)worker * per;
        // sequences without a token are shared out among all workers
        for (int e = (int)worker; e < a.batch; e += (int)workers) {
            if (tiles_of(seen_uniform(a, e)) != 0 || head_wave != 0) continue;
            char* to = a.out + (int64_t)e * a.heads * a.value_dim * 2;
            for (int i = lane; i < a.heads * a.value_dim / 8; i += 64) *(u32x4*)(to + (int64_t)i * 16) = u32x4{0u, 0u, 0u, 0u};
        }
        const bool notes = blockIdx.x == 0 && wave == 0;  // the sequences' first units, for the join
        if (notes && lane == 0) a.starts[a.batch] = total;
        if (u0 >= total && !notes) return;
        left = (uint32_t)uniform((int)(total - (uint32_t)u0 < per ? total - (uint32_t)u0 : per));
        // the sequence of unit u0: as many as end at or before it come first
        uint32_t before = 0;
        b = -1;
        rest = 0;
        for (int s0 = 0; s0 < a.batch && (b < 0 || notes); s0 += 64) {
            const int s = s0 + lane;
            if (a.batch > 64) units = s < a.batch ? units_of(tiles_of(seen_by(a, s))) * rows : 0u;
            const uint32_t inclusive = before + wave_scan(units);
            if (notes && s < a.batch) a.starts[s] = inclusive - units;
            const uint32_t end = (uint32_t)__builtin_amdgcn_readlane((int)inclusive, 63);
            if (b < 0 && end > (uint32_t)u0) {
                const int n = __builtin_popcountll(__ballot(inclusive <= (uint32_t)u0));
                b = s0 + n;
                rest = (uint32_t)u0 - (uint32_t)__builtin_amdgcn_readlane((int)(inclusive - units), n);
            }
            before = end;
        }
        if (u0 >= total || b < 0) return;
    }

    const int token_wave = DIRECT ? wave / a.head_waves : 0, token_waves = DIRECT ? (int)blockDim.x / kWave / a.head_waves : 1;
    const uint32_t k_lane = (uint32_t)(((g << a.page_shift) + c) * 16), k_step = (uint32_t)(4 << a.page_shift) * 16;
    const int key_row = a.key_dim * (KEPT ? 1 : 2), value_row = a.value_dim * (KEPT ? 1 : 2);
    const uint32_t v_lane = (uint32_t)(4 * g * value_row + c * (KEPT ? 8 : 16));

    for (;;) {                                            // a row, or the part of it that is this worker's
        const Seen seen = seen_uniform(a, b);
        const int tiles = tiles_of(seen);
        const uint32_t units = units_of(tiles);
        // (as the lengths were read above; should they change meanwhile, results are open, but nothing is read or written out of range)
        if (units == 0 || rest >= units * rows) return;
        const uint32_t row = rest / units, from = rest - row * units, to = units - from < left ? units : from + left;
        const int tile0 = from > kRowUnits ? (int)(from - kRowUnits) : 0, tile1 = to > kRowUnits ? (int)(to - kRowUnits) : 0;
        const int kv = (int)row / a.blocks, block = (int)row - kv * a.blocks, head0 = block * a.block_heads + head_wave * 16;      // within the group
        const int heads_here = a.group - head0 < 16 ? a.group - head0 : 16;
        const int t_base = seen.lo / kTile * kTile;
        left -= to - from;
        rest += to - from;
        if (tile0 < tile1) {
        u32x4 q[NK];
        {
            const char* from = a.q + ((int64_t)b * a.q_batch + (int64_t)(kv * a.group + head0 + c) * a.q_head) * 2;
#pragma unroll
            for (int j = 0; j < NK; j++) {
                const int at = KEPT ? (j / 2) * 64 + g * 16 + (j & 1) * 8 : j * 32 + g * 8;
                q[j] = c < heads_here && at < a.key_dim ? *(const u32x4*)(from + at * 2) ^ a.flip : u32x4{0u, 0u, 0u, 0u};
            }
        }
        f32x4 acc[NV * 8];
#pragma unroll
        for (int i = 0; i < NV * 8; i++) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        float top = kLowest, total = 0.0f;

        u32x4 k[2][kLoads];
        uint32_t ke[2][KEPT ? kLoads : 1];
        u32x4 v[KEPT ? 1 : NV][8];
        u32x2 v8[KEPT ? NV : 1][8];
        uint32_t ve[2][KEPT ? NV : 1];
        // of this workgroup's key head in page 0
        const char *keys = a.keys + (int64_t)kv * (key_row << a.page_shift), *values = a.values + (int64_t)kv * (value_row << a.page_shift);
        const uint8_t *key_scales = a.key_scales + (int64_t)kv * (a.key_dim / 32 << a.page_shift);
        const uint8_t *value_scales = a.value_scales + (int64_t)kv * (a.value_dim / 32 << a.page_shift);
        const MQ_CONST int32_t* table = (const MQ_CONST int32_t*)(uint64_t)(a.table + (int64_t)b * a.table_stride);

        // A tile's halves of 16 tokens: their pages, asked for two tiles ahead (behind the last token: its page), and whether there is
        // anything to read: a page of the cache's, a token that is seen, a tile of this workgroup's.  Accesses are bounds-checked against what a
        // half holds: 0 bytes where there is nothing, for which the memory is not touched and the lane has zeros.
        auto ask = [&](int t, uint32_t* ids) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int first = t_base + t * kTile + h * 16, last = seen.hi - 1;
                ids[h] = (uint32_t)table[(first < last ? first : last) >> a.page_shift];
            }
        };
        auto take = [&](int t, const uint32_t* ids, Half* to) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int first = t_base + t * kTile + h * 16;
                to[h] = half_of(ids[h], a.pages, first, seen, t < tile1);
            }
        };
        auto load_keys = [&](int t, const Half* at) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int place = (t_base + t * kTile + h * 16) & ((1 << a.page_shift) - 1);
                const auto from = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(keys) + (uint64_t)at[h].page * a.key_page + place * 16, 0,
                                                                    bytes_to_end(at[h], key_row, a.page_shift, place, 16), 0x00027000);
#pragma unroll
                for (int j = 0; j < kLoads; j++)          // (pieces behind the key's end: zeros)
                    k[h][j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, (int)(k_lane + j * k_step), 0, kPolicy));
                if (KEPT) {
                    const auto scales = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(key_scales) + (uint64_t)at[h].page * a.key_scale_page + place, 0,
                                                                          bytes_to_end(at[h], a.key_dim / 32, a.page_shift, place, 1), 0x00027000);
#pragma unroll
                    for (int j = 0; j < kLoads; j++) ke[h][j] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(scales, ((2 * j + (g >> 1)) << a.page_shift) + c, 0, 0);
                }
            }
        };
        auto load_values = [&](int t, const Half* at) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int first = t_base + t * kTile + h * 16, place = first & ((1 << a.page_shift) - 1);
                const auto from = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(values) + (uint64_t)at[h].page * a.value_page + place * value_row, 0,
                                                                    bytes_to_last(at[h], value_row, first, seen), 0x00027000);
#pragma unroll
                for (int nv = 0; nv < NV; nv++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t at_v = v_lane + i * value_row + nv * (KEPT ? 128 : 256);
                        if (KEPT) v8[nv][h * 4 + i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(from, (int)at_v, 0, kPolicy));
                        else v[nv][h * 4 + i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, (int)at_v, 0, kPolicy));
                    }
                if (KEPT) {
                    const auto scales = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(value_scales) + (uint64_t)at[h].page * a.value_scale_page + place, 0,
                                                                          bytes_to_end(at[h], a.value_dim / 32, a.page_shift, place, 1), 0x00027000);
#pragma unroll
                    for (int nv = 0; nv < NV; nv++)
                        ve[h][nv] = __builtin_amdgcn_raw_buffer_load_b32(scales, ((c / 4 + 4 * nv) << a.page_shift) + 4 * g, 0, 0);
                }
            }
        };

        int t = tile0 + token_wave;
        uint32_t ids[2];
        Half at[2], at_next[2];
        ask(t, ids);
        take(t, ids, at);
        // (the scheduler leaves the order of accesses as it is, which is what the waits count by)
        load_keys(t, at);
        __builtin_amdgcn_sched_barrier(0);
        load_values(t, at);
        ask(t + token_waves, ids);
        __builtin_amdgcn_sched_barrier(0);
        while (t < tile1) {
            const int next = t + token_waves;
            if (SHARED && !DIRECT) __builtin_amdgcn_s_barrier();
            // ---- scores
            f32x4 s[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int j = 0; j < kLoads; j++) {
                    if (KEPT) {
                        const u32x2 p0 = kept_pack4<D>(k[h][j].x, ke[h][j]), p1 = kept_pack4<D>(k[h][j].y, ke[h][j]);
                        const u32x2 p2 = kept_pack4<D>(k[h][j].z, ke[h][j]), p3 = kept_pack4<D>(k[h][j].w, ke[h][j]);
                        s[h] = mfma<D>(u32x4{p0.x, p0.y, p1.x, p1.y}, q[2 * j], s[h]);
                        s[h] = mfma<D>(u32x4{p2.x, p2.y, p3.x, p3.y}, q[2 * j + 1], s[h]);
                    } else s[h] = mfma<D>(k[h][j], q[j], s[h]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            take(next, ids, at_next);
            load_keys(next, at_next);
            __builtin_amdgcn_sched_barrier(0);
            // ---- weights
            const int first = t_base + t * kTile;
            const bool full = first >= seen.lo && first + kTile <= seen.hi && at[0].some && at[1].some;
            if (!full) {
                // what is not seen: no weight; values before a window as zeros (behind the last token they are), and in 8 bits the scales, which
                // may be any bytes there, a NaN's among them
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int token = first + (i / 4) * 16 + 4 * g + (i & 3);
                    const bool hidden = token < seen.lo || token >= seen.hi || !at[i / 4].some;
                    if (hidden) s[i / 4][i & 3] = -__builtin_inff();
#pragma unroll
                    for (int nv = 0; nv < NV; nv++) {
                        if (KEPT) {
                            if (token < seen.lo) v8[nv][i] = u32x2{0u, 0u};
                            if (hidden) ve[i / 4][nv] &= ~(0xFFu << (8 * (i & 3)));
                        } else if (token < seen.lo) v[nv][i] = u32x4{0u, 0u, 0u, 0u};
                    }
                }
            }
            // (times the scale before the maximum is taken from them: a fused operation would round one of the two and not the other, which beyond 2^24 is whole
            // powers of two, and a weight of 0 or an infinity for the largest score itself)
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; i++) p[i] = s[i / 4][i & 3] * a.scale;
            float most = p[0];
#pragma unroll
            for (int i = 1; i < 8; i++) most = __builtin_fmaxf(most, p[i]);
            // The running maximum need not be the largest: weights up to 2^kSlack of it are numbers as good.  Sums are rescaled when it is passed by
            // more, which after a row's first tile hardly ever is.
            const float higher = max_of_head(most);
            if (__any(higher > top + kSlack)) {
                const float now = __builtin_fmaxf(top, higher), f = __builtin_amdgcn_exp2f(top - now);
                total *= f;
#pragma unroll
                for (int i = 0; i < NV * 8; i++) acc[i] *= f;
                top = now;
            }
            // What the weights of this tile are relative to: fp16 ends at 2^-24, so that beside a weight of 1 all that is 2^25 times as small would be lost, which is the
            // result itself where the first token takes nearly all weight and its value is zero.  So fp16 weights are relative to their own tile's maximum, which
            // is 2^15 and its sums' factor makes up for; what is lost is below 2^-40 of that, of 32 tokens at most.
            const float of = kOwnTop ? __builtin_fmaxf(higher, kLowest) : top;
#pragma unroll
            for (int i = 0; i < 8; i++) p[i] = __builtin_amdgcn_exp2f(p[i] - of);
            float times = 1.0f;
            if (kOwnTop) {
                times = __builtin_amdgcn_exp2f(of - top);
                float here = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    here += p[i];
                    p[i] *= 0x1p15f;
                }
                total = __builtin_fmaf(here, times, total);
                times *= 0x1p-15f;
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) total += p[i];
            }
            u32x4 weights[kWeightParts<D>];
#pragma unroll
            for (int i = 0; i < 4; i++) split_weights<D>(p[2 * i], p[2 * i + 1], weights, i);
            // ---- values
#pragma unroll
            for (int nv = 0; nv < NV; nv++) {
                u32x4 x[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (KEPT) {
                        const uint32_t e = ve[i / 4][nv] >> (8 * (i & 3)) & 0xFFu;
                        const u32x2 lo = kept_pack4<D>(v8[nv][i].x, e), hi = kept_pack4<D>(v8[nv][i].y, e);
                        x[i] = u32x4{lo.x, lo.y, hi.x, hi.y};
                    } else x[i] = v[nv][i];
                }
                // products that do not wait for each other, while two wavefronts' registers suffice (one after the other: 33 sequences of up to 9001 tokens, 40 heads over one of 256: 39.9 us instead of
                // 38.5)
                constexpr int kAtOnce = kOwnTop && NV == 2 && !attend_is_wide(NK, NV) ? 2 : 4;
#pragma unroll
                for (int e0 = 0; e0 < 8; e0 += kAtOnce) {
                    u32x4 row8[kAtOnce];
                    f32x4 sum[kAtOnce];
#pragma unroll
                    for (int i = 0; i < kAtOnce; i++) {
                        const int e = e0 + i;
                        const uint32_t pick = e & 1 ? 0x07060302u : 0x05040100u;
                        row8[i] = u32x4{__builtin_amdgcn_perm(x[1][e / 2], x[0][e / 2], pick), __builtin_amdgcn_perm(x[3][e / 2], x[2][e / 2], pick),
                                        __builtin_amdgcn_perm(x[5][e / 2], x[4][e / 2], pick), __builtin_amdgcn_perm(x[7][e / 2], x[6][e / 2], pick)};
                        sum[i] = kOwnTop ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : acc[nv * 8 + e];
                    }
#pragma unroll
                    for (int part = 0; part < kWeightParts<D>; part++)
#pragma unroll
                        for (int i = 0; i < kAtOnce; i++) sum[i] = mfma<D>(row8[i], weights[part], sum[i]);
#pragma unroll
                    for (int i = 0; i < kAtOnce; i++) {
                        f32x4& all = acc[nv * 8 + e0 + i];
                        if (!kOwnTop) all = sum[i];
                        else
#pragma unroll
                            for (int r = 0; r < 4; r++) all[r] = __builtin_fmaf(sum[i][r], times, all[r]);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            load_values(next, at_next);
            ask(next + token_waves, ids);
            __builtin_amdgcn_sched_barrier(0);
            t = next;
            at[0] = at_next[0];
            at[1] = at_next[1];
        }

        // ---- where the sums go
        total = sum_of_head(total);
        if (!DIRECT) {
            const bool whole = tile0 == 0 && tile1 == tiles;
            // the lane's numbers anew, which keeps the addresses below from being computed before the rows and held in up to 30 registers
            int c1 = c, g1 = g;
            asm("" : "+v"(c1), "+v"(g1));
            const int in_block = head_wave * 16 + c1, head = kv * a.group + head0 + c1;
            float* part = a.parts + ((int64_t)worker * 2 + (first_of_worker ? 0 : 1)) * part_floats(a.block_heads, NV);
            if (c1 < heads_here) {
                const float times = whole ? finish_factor(a, head, top, total) : 1.0f;
                if (!whole && g1 == 0) *(f32x2*)(part + a.block_heads * (128 * NV) + in_block * 2) = f32x2{top, total};
#pragma unroll
                for (int nv = 0; nv < NV; nv++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int at_dim = nv * 128 + 8 * (4 * g1 + r);
                        if (at_dim >= a.value_dim) continue;
                        float f[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) f[e] = acc[nv * 8 + e][r] * times;
                        if (whole) store8<D>(a.out + (((int64_t)b * a.heads + head) * a.value_dim + at_dim) * 2, f);
                        else {
                            float* sums = part + in_block * (128 * NV) + at_dim;
                            *(f32x4*)sums = f32x4{f[0], f[1], f[2], f[3]};
                            *(f32x4*)(sums + 4) = f32x4{f[4], f[5], f[6], f[7]};
                        }
                    }
            }
        } else {
            // the wavefronts' sums together: those that have the same heads, in their order
            __shared__ __attribute__((aligned(16))) float sums[DIRECT ? kAttendWaves : 1][16 * kRowPad];
            __shared__ float tops[DIRECT ? kAttendWaves : 1][16], totals[DIRECT ? kAttendWaves : 1][16];
            if (g == 0) {
                tops[wave][c] = top;
                totals[wave][c] = total;
            }
#pragma unroll
            for (int nv = 0; nv < NV; nv++) {
                __syncthreads();
                float highest = kLowest;
                for (int w = 0; w < token_waves; w++) highest = __builtin_fmaxf(highest, tops[w * a.head_waves + head_wave][c]);
                const float mine = __builtin_amdgcn_exp2f(top - highest);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float* sum = &sums[wave][c * kRowPad + 8 * (4 * g + r)];
                    const f32x4* x = &acc[nv * 8];
                    *(f32x4*)sum = f32x4{x[0][r], x[1][r], x[2][r], x[3][r]} * mine;
                    *(f32x4*)(sum + 4) = f32x4{x[4][r], x[5][r], x[6][r], x[7][r]} * mine;
                }
                __syncthreads();
                for (int i = threadIdx.x; i < a.head_waves * 256; i += (int)blockDim.x) {
                    const int hw = i >> 8, h = i >> 4 & 15, at_dim = (i & 15) * 8, head = block * a.block_heads + hw * 16 + h;               // within the group
                    if (head >= a.group || nv * 128 + at_dim >= a.value_dim) continue;
                    float m = kLowest, l = 0.0f, f[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                    for (int w = 0; w < token_waves; w++) m = __builtin_fmaxf(m, tops[w * a.head_waves + hw][h]);
                    for (int w = 0; w < token_waves; w++) {
                        const int of = w * a.head_waves + hw;
                        l += totals[of][h] * __builtin_amdgcn_exp2f(tops[of][h] - m);
                        const f32x4 x = *(const f32x4*)&sums[of][h * kRowPad + at_dim], y = *(const f32x4*)&sums[of][h * kRowPad + at_dim + 4];
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            f[j] += x[j];
                            f[4 + j] += y[j];
                        }
                    }
                    const int64_t to_head = (int64_t)kv * a.group + head;
                    const float times = finish_factor(a, (int)to_head, m, l);
#pragma unroll
                    for (int j = 0; j < 8; j++) f[j] *= times;
                    store8<D>(a.out + (((int64_t)b * a.heads + to_head) * a.value_dim + nv * 128 + at_dim) * 2, f);
                }
            }
            return;
        }
        }
        // ---- what comes next
        if (left == 0) return;
        first_of_worker = false;
        if (rest == units * rows) {
            rest = 0;
            do
                if (++b == a.batch) return;
            while (tiles_of(seen_uniform(a, b)) == 0);
        }
    }
}

template <int D, bool KEPT, int NK, int NV, bool SHARED>
void attend_launch(const AttendArgs& a, bool direct, unsigned grid, hipStream_t st) {
    if (direct) attend_kernel<D, KEPT, NK, NV, true, SHARED><<<grid, kAttendWaves / a.head_waves * a.head_waves * kWave, 0, st>>>(a);
    else attend_kernel<D, KEPT, NK, NV, false, SHARED><<<grid, (SHARED ? a.head_waves : kAttendWaves) * kWave, 0, st>>>(a);
}
template <int D, bool KEPT, int NK, int NV>
void attend_launch(const AttendArgs& a, bool direct, unsigned grid, hipStream_t st) {
    a.head_waves > 1 ? attend_launch<D, KEPT, NK, NV, true>(a, direct, grid, st) : attend_launch<D, KEPT, NK, NV, false>(a, direct, grid, st);
}
template <int D, bool KEPT>
int attend_launch(const AttendArgs& a, int nk, int nv, bool direct, unsigned grid, hipStream_t st) {
#define MQ_ATTEND(NK, NV) \
    if (nk == NK && nv == NV) attend_launch<D, KEPT, NK, NV>(a, direct, grid, st)
    MQ_ATTEND(2, 1);
    MQ_ATTEND(4, 1);
    MQ_ATTEND(6, 1);
    MQ_ATTEND(8, 1);
    MQ_ATTEND(2, 2);
    MQ_ATTEND(4, 2);
    MQ_ATTEND(6, 2);
    MQ_ATTEND(8, 2);
#undef MQ_ATTEND
    return mq_check_launch("mq_paged_attention");
}

}  // namespace mq

int mq_attend_bf16(const mq::AttendArgs& a, int nk, int nv, bool direct, unsigned grid, hipStream_t st);
int mq_attend_bf16_kept(const mq::AttendArgs& a, int nk, int nv, bool direct, unsigned grid, hipStream_t st);
int mq_attend_f16(const mq::AttendArgs& a, int nk, int nv, bool direct, unsigned grid, hipStream_t st);
int mq_attend_f16_kept(const mq::AttendArgs& a, int nk, int nv, bool direct, unsigned grid, hipStream_t st);
