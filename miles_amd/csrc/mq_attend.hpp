// Attention of one token a sequence over a paged cache: softmax(scale q K^T) V with a running maximum and sum, on the matrix cores.
//
// A wavefront takes 32 tokens of a sequence's key head at a time, for up to 16 of the query heads that share it.  Everything goes from memory
// to the matrix instructions through registers, without shared memory and without a lane handing anything to another:
//   scores   S^T = K Q^T, 16 tokens x 16 heads: a lane's operand is eight elements of one token's key, which the cache's layout has beside those
//            of the neighbouring tokens, so that a load covers whole lines.  Lane (c, g) = (lane % 16, lane / 16) gets head c, tokens 4 g + r.
//   output   O^T += V^T P^T: the same lane needs, for element 8 c + e of the values, the weights and values of eight tokens.  Which
//            eight is free as long as both operands agree: 4 g + r of both halves of the 32, whose weights it has, and
//            whose values it reads as rows of 16 bytes; eight such rows are rearranged in its own registers, one instruction for two elements.
// Weights enter as the sum of two 16-bit numbers, so that they are as good as the 32-bit ones (one alone would be off by as much as the
// result's own rounding); the matrix cores have the time.  What bounds it is reading keys and values once.
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
    float* parts;                  // partial results, null: every workgroup has whole sequences (direct)
    uint32_t* starts;              // [batch + 1]: units before each sequence, and all of them
    int64_t q_batch, q_head, table_stride, capacity, window;
    uint32_t pages;
    uint32_t key_page, value_page, key_scale_page, value_scale_page;      // bytes of a page, below 2^31
    int batch, heads, kv_heads, group, key_dim, value_dim, page_shift;
    int blocks;                    // of heads of a key head: groups of 16 x head_waves
    int head_waves;                // wavefronts of a workgroup that share tokens and have different heads: 1, 2 or 4
    uint32_t least;                // units that a workgroup takes at least
    float scale;                   // with log2(e)
};
// A unit of work is a tile of 32 tokens of one key head for one block of query heads; units are numbered by sequence, key head, block
// and tile.
constexpr float kLowest = -3.0e38f;                      // the maximum of no scores: finite, so that differences are numbers
constexpr int kAttendThreads = 256, kAttendWaves = 4, kRowPad = 132;

// floats of a workgroup's partial result: 16 heads x 128 NV sums for each head wave, then their maxima and totals
__host__ __device__ inline int64_t part_floats(int head_waves, int nv) { return (int64_t)head_waves * 16 * (128 * nv + 2); }

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

// Sums of units over all sequences before this lane's (inclusive), 256 sequences at a time
__device__ __forceinline__ uint32_t scan_units(uint32_t v, uint32_t* waves, uint32_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t up = __shfl_up(v, d);
        if (lane >= d) v += up;
    }
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kAttendWaves; w++) {
        if (w < wave) before += waves[w];
        total += waves[w];
    }
    __syncthreads();
    return v + before;
}

template <int D>
__device__ __forceinline__ void store8(char* to, const float* f) {
    *(u32x4*)to = pack<D>(f);
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

template <int D, bool KEPT, int NK, int NV>
__global__ __launch_bounds__(kAttendThreads, NV == 2 && NK > 4 ? 1 : 2) void attend_kernel(const AttendArgs a) {
    constexpr int kLoads = KEPT ? NK / 2 : NK;            // of a tile's half's keys
    __shared__ __attribute__((aligned(16))) float sums[kAttendWaves][16 * kRowPad];
    __shared__ float tops[kAttendWaves][16], totals[kAttendWaves][16];
    __shared__ uint32_t scratch[2 * kAttendWaves + 1];
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x / kWave), c = lane & 15, g = lane >> 4;
    const int per_tile = a.kv_heads * a.blocks;           // units of a tile of tokens

    // ---- which units
    int b;
    uint32_t rest, left;                                  // first unit within its sequence, and how many
    bool first_of_workgroup = true;
    if (!a.parts) {
        const int inner = (int)blockIdx.x % per_tile;
        b = (int)blockIdx.x / per_tile;
        const int tiles = tiles_of(seen_uniform(a, b));
        rest = (uint32_t)inner * tiles;
        left = tiles;
        if (tiles == 0) {                                 // nothing to see
            const int n = a.group * a.value_dim / 8;
            if (inner % a.blocks == 0) {
                char* to = a.out + ((int64_t)b * a.heads + (int64_t)(inner / a.blocks) * a.group) * a.value_dim * 2;
                for (int i = threadIdx.x; i < n; i += kAttendThreads) *(u32x4*)(to + (int64_t)i * 16) = u32x4{0u, 0u, 0u, 0u};
            }
            return;
        }
    } else {
        uint32_t total = 0, inclusive = 0, chunk;
        for (int b0 = 0; b0 < a.batch; b0 += kAttendThreads) {
            const int mine = b0 + (int)threadIdx.x;
            const uint32_t units = mine < a.batch ? (uint32_t)tiles_of(seen_by(a, mine)) * per_tile : 0u;
            inclusive = total + scan_units(units, scratch, chunk);
            if (blockIdx.x == 0 && mine < a.batch) a.starts[mine] = inclusive - units;
            total += chunk;
        }
        if (blockIdx.x == 0 && threadIdx.x == 0) a.starts[a.batch] = total;
        const uint32_t share = (total + gridDim.x - 1) / gridDim.x, per = share > a.least ? share : a.least;
        const uint64_t u0 = (uint64_t)blockIdx.x * per;
        // sequences without a token are shared out among all workgroups
        for (int e = blockIdx.x; e < a.batch; e += gridDim.x) {
            if (tiles_of(seen_uniform(a, e)) != 0) continue;
            char* to = a.out + (int64_t)e * a.heads * a.value_dim * 2;
            for (int i = threadIdx.x; i < a.heads * a.value_dim / 8; i += kAttendThreads) *(u32x4*)(to + (int64_t)i * 16) = u32x4{0u, 0u, 0u, 0u};
        }
        if (u0 >= total) return;
        left = (uint32_t)uniform((int)(total - (uint32_t)u0 < per ? total - (uint32_t)u0 : per));
        // the sequence of unit u0: as many as end at or before it come first
        uint32_t running = 0;
        for (int b0 = 0;; b0 += kAttendThreads) {
            if (a.batch > kAttendThreads) {
                const int mine = b0 + (int)threadIdx.x;
                const uint32_t units = mine < a.batch ? (uint32_t)tiles_of(seen_by(a, mine)) * per_tile : 0u;
                inclusive = running + scan_units(units, scratch, chunk);
                running += chunk;
                if (running <= (uint32_t)u0) continue;
            }
            const bool before = b0 + (int)threadIdx.x < a.batch && inclusive <= (uint32_t)u0;
            const uint64_t votes = __ballot(before);
            if (lane == 0) scratch[kAttendWaves + wave] = (uint32_t)__builtin_popcountll(votes);
            __syncthreads();
            int n = 0;
            for (int w = 0; w < kAttendWaves; w++) n += (int)scratch[kAttendWaves + w];
            b = b0 + uniform(n);
            if ((int)threadIdx.x == n) {
                const int tiles = tiles_of(seen_by(a, b));
                scratch[2 * kAttendWaves] = (uint32_t)u0 - (inclusive - (uint32_t)tiles * per_tile);
            }
            __syncthreads();
            rest = (uint32_t)uniform((int)scratch[2 * kAttendWaves]);
            break;
        }
    }

    const int head_wave = wave & (a.head_waves - 1), token_wave = wave / a.head_waves, token_waves = kAttendWaves / a.head_waves;
    const uint32_t k_lane = (uint32_t)(((g << a.page_shift) + c) * 16), k_step = (uint32_t)(4 << a.page_shift) * 16;
    const int key_row = a.key_dim * (KEPT ? 1 : 2), value_row = a.value_dim * (KEPT ? 1 : 2);
    const uint32_t v_lane = (uint32_t)(4 * g * value_row + c * (KEPT ? 8 : 16));

    for (;;) {                                            // a sequence's key head and block of query heads, or the part of it that is this workgroup's
        const Seen seen = seen_uniform(a, b);
        const int tiles = tiles_of(seen), inner = (int)(rest / (uint32_t)tiles), tile0 = (int)(rest - (uint32_t)inner * tiles);
        const int tile1 = (uint32_t)(tiles - tile0) < left ? tiles : tile0 + (int)left;
        const int kv = inner / a.blocks, block = inner - kv * a.blocks, head0 = (block * a.head_waves + head_wave) * 16;      // within the group
        const int heads_here = a.group - head0 < 16 ? a.group - head0 : 16;
        const int t_base = seen.lo / kTile * kTile;
        const int64_t row = (int64_t)b * a.table_stride;

        u32x4 q[NK];
        {
            const char* from = a.q + ((int64_t)b * a.q_batch + (int64_t)(kv * a.group + head0 + c) * a.q_head) * 2;
#pragma unroll
            for (int j = 0; j < NK; j++) {
                const int at = KEPT ? (j / 2) * 64 + g * 16 + (j & 1) * 8 : j * 32 + g * 8;
                q[j] = c < heads_here && at < a.key_dim ? *(const u32x4*)(from + at * 2) : u32x4{0u, 0u, 0u, 0u};
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
                    k[h][j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, (int)(k_lane + j * k_step), 0, 0));
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
                const int before = seen.lo - first - 4 * g;       // tokens of this lane's that lie before a window
                const auto from = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(values) + (uint64_t)at[h].page * a.value_page + place * value_row, 0,
                                                                    bytes_to_last(at[h], value_row, first, seen), 0x00027000);
#pragma unroll
                for (int nv = 0; nv < NV; nv++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t at_v = i < before ? kNowhere : v_lane + i * value_row + nv * (KEPT ? 128 : 256);
                        if (KEPT) v8[nv][h * 4 + i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(from, (int)at_v, 0, 0));
                        else v[nv][h * 4 + i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, (int)at_v, 0, 0));
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
            // ---- scores
            f32x4 s[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                s[h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (KEPT) {
#pragma unroll
                    for (int j = 0; j < kLoads; j++) {
                        const u32x2 p0 = kept_pack4<D>(k[h][j].x, ke[h][j]), p1 = kept_pack4<D>(k[h][j].y, ke[h][j]);
                        const u32x2 p2 = kept_pack4<D>(k[h][j].z, ke[h][j]), p3 = kept_pack4<D>(k[h][j].w, ke[h][j]);
                        s[h] = mfma<D>(u32x4{p0.x, p0.y, p1.x, p1.y}, q[2 * j], s[h]);
                        s[h] = mfma<D>(u32x4{p2.x, p2.y, p3.x, p3.y}, q[2 * j + 1], s[h]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < kLoads; j++) s[h] = mfma<D>(k[h][j], q[j], s[h]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            take(next, ids, at_next);
            load_keys(next, at_next);
            __builtin_amdgcn_sched_barrier(0);
            // ---- weights
            const int first = t_base + t * kTile;
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; i++) p[i] = s[i / 4][i & 3] * a.scale;
            if (!(first >= seen.lo && first + kTile <= seen.hi && at[0].some && at[1].some)) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int token = first + (i / 4) * 16 + 4 * g + (i & 3);
                    if (token < seen.lo || token >= seen.hi || !at[i / 4].some) p[i] = -__builtin_inff();
                }
            }
            float most = p[0];
#pragma unroll
            for (int i = 1; i < 8; i++) most = __builtin_fmaxf(most, p[i]);
            const float higher = __builtin_fmaxf(top, max_of_head(most));
            if (__any(higher > top)) {
                const float f = __builtin_amdgcn_exp2f(top - higher);
                total *= f;
#pragma unroll
                for (int i = 0; i < NV * 8; i++) acc[i] *= f;
                top = higher;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) p[i] = __builtin_amdgcn_exp2f(p[i] - top);
#pragma unroll
            for (int i = 0; i < 8; i++) total += p[i];
            uint32_t big[4], small[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                big[i] = pack2<D>(p[2 * i], p[2 * i + 1]);
                small[i] = pack2<D>(p[2 * i] - elem_lo<D == MQ_F16>(big[i]), p[2 * i + 1] - elem_hi<D == MQ_F16>(big[i]));
            }
            const u32x4 weights = {big[0], big[1], big[2], big[3]}, remainders = {small[0], small[1], small[2], small[3]};
            // ---- values
            uint32_t scale_mask[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
            if (KEPT) {                                   // scales of tokens that are not seen: any bytes, a NaN's among them
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int end = seen.hi - (first + h * 16 + 4 * g), begin = seen.lo - (first + h * 16 + 4 * g);
                    if (end < 4) scale_mask[h] = end <= 0 ? 0u : 0xFFFFFFFFu >> (32 - 8 * end);
                    if (begin > 0) scale_mask[h] &= begin >= 4 ? 0u : 0xFFFFFFFFu << (8 * begin);
                }
            }
#pragma unroll
            for (int nv = 0; nv < NV; nv++) {
                u32x4 x[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (KEPT) {
                        const uint32_t e = (ve[i / 4][nv] & scale_mask[i / 4]) >> (8 * (i & 3)) & 0xFFu;
                        const u32x2 lo = kept_pack4<D>(v8[nv][i].x, e), hi = kept_pack4<D>(v8[nv][i].y, e);
                        x[i] = u32x4{lo.x, lo.y, hi.x, hi.y};
                    } else x[i] = v[nv][i];
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t pick = e & 1 ? 0x07060302u : 0x05040100u;
                    const u32x4 row8 = {__builtin_amdgcn_perm(x[1][e / 2], x[0][e / 2], pick), __builtin_amdgcn_perm(x[3][e / 2], x[2][e / 2], pick),
                                        __builtin_amdgcn_perm(x[5][e / 2], x[4][e / 2], pick), __builtin_amdgcn_perm(x[7][e / 2], x[6][e / 2], pick)};
                    acc[nv * 8 + e] = mfma<D>(row8, weights, acc[nv * 8 + e]);
                    acc[nv * 8 + e] = mfma<D>(row8, remainders, acc[nv * 8 + e]);
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

        // ---- the wavefronts' sums together: those that have the same heads, in their order
        total = sum_of_head(total);
        if (g == 0) {
            tops[wave][c] = top;
            totals[wave][c] = total;
        }
        __syncthreads();
        float highest = kLowest;
        for (int w = 0; w < token_waves; w++) highest = __builtin_fmaxf(highest, tops[w * a.head_waves + head_wave][c]);
        const float mine = __builtin_amdgcn_exp2f(top - highest);
        const bool whole = tile0 == 0 && tile1 == tiles;
        float* part = whole ? nullptr : a.parts + ((int64_t)blockIdx.x * 2 + (first_of_workgroup ? 0 : 1)) * part_floats(a.head_waves, NV);
#pragma unroll
        for (int nv = 0; nv < NV; nv++) {
            if (nv) __syncthreads();
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float* to = &sums[wave][c * kRowPad + 8 * (4 * g + r)];
                *(f32x4*)to = f32x4{acc[nv * 8 + 0][r], acc[nv * 8 + 1][r], acc[nv * 8 + 2][r], acc[nv * 8 + 3][r]} * mine;
                *(f32x4*)(to + 4) = f32x4{acc[nv * 8 + 4][r], acc[nv * 8 + 5][r], acc[nv * 8 + 6][r], acc[nv * 8 + 7][r]} * mine;
            }
            __syncthreads();
            const int h = (int)threadIdx.x >> 4, at = ((int)threadIdx.x & 15) * 8;
            for (int hw = 0; hw < a.head_waves; hw++) {
                const int head = (block * a.head_waves + hw) * 16 + h;               // within the group
                if (head >= a.group) continue;
                float m = kLowest, l = 0.0f, f[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                for (int w = 0; w < token_waves; w++) m = __builtin_fmaxf(m, tops[w * a.head_waves + hw][h]);
                for (int w = 0; w < token_waves; w++) {
                    const int from = w * a.head_waves + hw;
                    l += totals[from][h] * __builtin_amdgcn_exp2f(tops[from][h] - m);
                    const f32x4 x = *(const f32x4*)&sums[from][h * kRowPad + at], y = *(const f32x4*)&sums[from][h * kRowPad + at + 4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        f[i] += x[i];
                        f[4 + i] += y[i];
                    }
                }
                if (part) {
                    float* to = part + (hw * 16 + h) * (128 * NV) + nv * 128 + at;
                    *(f32x4*)to = f32x4{f[0], f[1], f[2], f[3]};
                    *(f32x4*)(to + 4) = f32x4{f[4], f[5], f[6], f[7]};
                    if (nv == 0 && at == 0) {
                        float* ml = part + a.head_waves * 16 * (128 * NV) + (hw * 16 + h) * 2;
                        ml[0] = m;
                        ml[1] = l;
                    }
                } else if (nv * 128 + at < a.value_dim) {
                    const int64_t to_head = (int64_t)kv * a.group + head;
                    const float times = finish_factor(a, (int)to_head, m, l);
#pragma unroll
                    for (int i = 0; i < 8; i++) f[i] *= times;
                    store8<D>(a.out + (((int64_t)b * a.heads + to_head) * a.value_dim + nv * 128 + at) * 2, f);
                }
            }
        }
        // ---- what comes next
        left -= (uint32_t)(tile1 - tile0);
        if (left == 0) return;
        first_of_workgroup = false;
        rest += (uint32_t)(tile1 - tile0);
        if (rest == (uint32_t)tiles * per_tile) {
            rest = 0;
            do b++;
            while (tiles_of(seen_uniform(a, b)) == 0);
        }
        __syncthreads();                                  // shared memory is free again
    }
}

template <int D, bool KEPT>
int attend_launch(const AttendArgs& a, int nk, int nv, unsigned grid, hipStream_t st) {
#define MQ_ATTEND(NK, NV) \
    if (nk == NK && nv == NV) attend_kernel<D, KEPT, NK, NV><<<grid, kAttendThreads, 0, st>>>(a)
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

int mq_attend_bf16(const mq::AttendArgs& a, int nk, int nv, unsigned grid, hipStream_t st);
int mq_attend_bf16_kept(const mq::AttendArgs& a, int nk, int nv, unsigned grid, hipStream_t st);
int mq_attend_f16(const mq::AttendArgs& a, int nk, int nv, unsigned grid, hipStream_t st);
int mq_attend_f16_kept(const mq::AttendArgs& a, int nk, int nv, unsigned grid, hipStream_t st);
