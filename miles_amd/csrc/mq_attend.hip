// Attention over a paged cache: how its work is shared out, and the join of sequences that several workgroups had a part of.
//
// The lengths are on the device and differ, so the launch cannot follow them.  A launch has as many wavefronts as the card holds; each (or, where
// more than 16 query heads share a key head, each group of two or four) adds the lengths up and takes an equal share of all work, which may begin and end
// inside a row: at most the sums of its first and its last row are partial.  Where no sequence can be long, every workgroup has one row
// instead, and there is no join.
#include <stdio.h>

#include "mq_attend.hpp"

namespace mq {

// Partial results of a head, in an order that their number decides.  WAVES wavefronts have a head; a wavefront has 64 parts at a time, whose maxima and
// totals its lanes hold, and goes through them four at once with 16 lanes of eight elements each.
constexpr int kJoinThreads = 256, kJoinWaves = 4;
template <int D, int NV, int WAVES>
__global__ __launch_bounds__(kJoinThreads) void attend_join_kernel(const AttendArgs a, uint32_t workers, int64_t first) {
    __shared__ float tops[kJoinWaves];
    __shared__ __attribute__((aligned(16))) float sums[kJoinWaves][16][12];
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x / kWave), piece = lane & 15, sub = lane >> 4, nth_wave = WAVES > 1 ? wave : 0;
    const int64_t nth = first + (WAVES > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * kJoinWaves + wave);
    if (nth >= (int64_t)a.batch * a.heads) return;        // (with WAVES > 1: never)
    const int b = (int)(nth / a.heads), head = (int)(nth - (int64_t)b * a.heads);
    const uint32_t before = a.starts[b], units = a.starts[b + 1] - before, total = a.starts[a.batch];
    if (units == 0) return;
    const int kv = head / a.group, in_group = head - kv * a.group, block = in_group / a.block_heads, in_block = in_group - block * a.block_heads;
    const uint32_t row = units / (uint32_t)(a.kv_heads * a.blocks), u0 = before + (uint32_t)(kv * a.blocks + block) * row, per = units_of_worker(total, workers, a.least);
    // workers that have tiles of the row, which begin behind its first units: the first may have the end of other rows before it
    const uint32_t w0 = (u0 + kRowUnits) / per, w1 = (u0 + row - 1) / per, parts = w1 - w0 + 1;
    if (parts == 1 || w1 >= workers) return;              // one worker had it all (or the lengths changed under the first kernel)
    const bool inside_first = u0 > w0 * per;              // the first part is the last of its worker's
    auto part = [&](uint32_t i) { return a.parts + ((int64_t)(w0 + i) * 2 + (i == 0 && inside_first ? 1 : 0)) * part_floats(a.block_heads, NV); };
    const int64_t ml = (int64_t)a.block_heads * (128 * NV) + in_block * 2, row_at = (int64_t)in_block * (128 * NV) + piece * 8;
    // this wavefront's: every so manieth, from its own number on
    const uint32_t mine = parts > (uint32_t)nth_wave ? (parts - nth_wave + WAVES - 1) / WAVES : 0;
    auto nth_part = [&](uint32_t i) { return part(nth_wave + i * WAVES); };
    float top = kLowest, m = kLowest, l = 0.0f;
    for (uint32_t i = lane; i < mine; i += 64) {
        const f32x2 x = *(const f32x2*)(nth_part(i) + ml);
        m = x.x;
        l = x.y;
        top = __builtin_fmaxf(top, m);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) top = __builtin_fmaxf(top, __shfl_xor(top, d));
    if (WAVES > 1) {
        if (lane == 0) tops[wave] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kJoinWaves; i++) top = __builtin_fmaxf(top, tops[i]);
    }
    float all = 0.0f, f[NV][8];
#pragma unroll
    for (int nv = 0; nv < NV; nv++)
#pragma unroll
        for (int i = 0; i < 8; i++) f[nv][i] = 0.0f;
    for (uint32_t i0 = 0; i0 < mine; i0 += 64) {
        if (mine > 64) {                                  // (else they are here already)
            m = kLowest;
            l = 0.0f;
            if (i0 + lane < mine) {
                const f32x2 x = *(const f32x2*)(nth_part(i0 + lane) + ml);
                m = x.x;
                l = x.y;
            }
        }
        const float times = i0 + lane < mine ? __builtin_amdgcn_exp2f(m - top) : 0.0f;
        all += l * times;
        const int here = mine - i0 < 64 ? (int)(mine - i0) : 64;
        constexpr int kAtOnce = (WAVES > 1 ? 4 : 3) / NV + 1;         // loads on their way
        for (int k0 = 0; k0 < here; k0 += 4 * kAtOnce) {
            f32x4 x[kAtOnce][NV], y[kAtOnce][NV];
            float w[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; u++) {
                const int k = k0 + 4 * u + sub, last = here - 1;
                w[u] = __shfl(times, k & 63);                         // (of all lanes)
                const float* from = nth_part(i0 + (k < here ? k : last)) + row_at;
#pragma unroll
                for (int nv = 0; nv < NV; nv++) {
                    x[u][nv] = *(const f32x4*)(from + nv * 128);
                    y[u][nv] = *(const f32x4*)(from + nv * 128 + 4);
                }
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; u++) {
                if (k0 + 4 * u + sub >= here) continue;               // (the last part again, whose sums may be infinite)
#pragma unroll
                for (int nv = 0; nv < NV; nv++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        f[nv][i] += x[u][nv][i] * w[u];
                        f[nv][4 + i] += y[u][nv][i] * w[u];
                    }
            }
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) all += __shfl_xor(all, d);
#pragma unroll
    for (int nv = 0; nv < NV; nv++) {
#pragma unroll
        for (int i = 0; i < 8; i++) f[nv][i] = sum_of_head(f[nv][i]);
        if (WAVES > 1) {
            if (lane < 16) {
#pragma unroll
                for (int i = 0; i < 8; i++) sums[wave][piece][i] = f[nv][i];
                sums[wave][piece][8] = all;
            }
            __syncthreads();
            if (nv == 0) all = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) f[nv][i] = 0.0f;
#pragma unroll
            for (int w = 0; w < kJoinWaves; w++) {
                if (nv == 0) all += sums[w][piece][8];
#pragma unroll
                for (int i = 0; i < 8; i++) f[nv][i] += sums[w][piece][i];
            }
            __syncthreads();
        }
        const int at = nv * 128 + piece * 8;
        if (lane < 16 && nth_wave == 0 && at < a.value_dim) {
            const float times = finish_factor(a, head, top, all);
#pragma unroll
            for (int i = 0; i < 8; i++) f[nv][i] *= times;
            store8<D>(a.out + (nth * a.value_dim + at) * 2, f[nv]);
        }
    }
}

struct AttendPlan {
    int nk, nv, blocks, head_waves;
    bool direct;               // every workgroup has a row of its own; else rows are shared out
    unsigned grid;
    uint32_t least;
    int64_t bytes, starts_bytes;
};
// Tiles that a wavefront goes through at most where every workgroup has a row of its own: half as many where there are few rows, of which a long one
// would keep the others waiting.  32 query heads over 8 of 128, random lengths up to the given number of tokens, in brackets all of it (us, rows of their own / shared out):
// 8 sequences to 1024 13.0 / 14.8 (15.0 / 15.8), to 2048 21.8 / 16.9 (25.2 / 25.1); 24 to 2048 29.6 / 31.4 (37 / 43), to 4096 55 / 47 (64 / 75); 64 to 1024
// 31 / 33 (46 / 51), to 2048 62 / 61 (89 / 92), to 4096 109 / 100 (173 / 177).
constexpr int64_t kDirectSteps = 16, kManyRows = 128, kMostGrid = 1 << 22;

// false: too large
bool attend_plan(const mq_paged_cache* c, int64_t batch, int64_t heads, int64_t width, int64_t window, AttendPlan& p) {
    const int64_t sixteens = (heads / c->kv_heads + 15) / 16;
    p.nk = (int)((c->key_dim + 63) / 64) * 2;
    p.nv = c->value_dim > 128 ? 2 : 1;
    if (width > (INT32_MAX - 4096) / c->page_size) return false;      // (a token behind the last has a number, too)
    const int64_t capacity = width * c->page_size;
    int64_t tiles = (capacity + kTile - 1) / kTile;
    if (window > 0 && window < capacity) tiles = tiles < (window + kTile - 1) / kTile + 1 ? tiles : (window + kTile - 1) / kTile + 1;
    p.head_waves = sixteens > 4 ? 4 : (int)sixteens;
    p.blocks = (int)((sixteens + p.head_waves - 1) / p.head_waves);
    const int64_t rows = batch * c->kv_heads * p.blocks;
    if (rows > INT32_MAX / (tiles + kRowUnits)) return false;
    p.bytes = p.starts_bytes = 0;
    const int64_t steps = (tiles + kAttendWaves / p.head_waves - 1) / (kAttendWaves / p.head_waves);
    p.direct = steps <= (rows < kManyRows ? kDirectSteps / 2 : kDirectSteps) && rows <= kMostGrid;
    p.least = kRowUnits;
    p.grid = (unsigned)rows;
    if (p.direct) return true;
    // Wavefronts on the card: two on every SIMD; one where registers allow no more, and where a worker's partial result, of many heads, is as long as
    // several tiles
    const int64_t waves = p.head_waves > 1 || attend_is_wide(p.nk, p.nv) ? 1024 : 2048;
    const int64_t workers = (rows * (tiles + kRowUnits) + p.least - 1) / p.least, per_group = attend_workers(p.head_waves);
    const int64_t most = (workers + per_group - 1) / per_group, resident = waves / (per_group * (p.head_waves == 3 ? 4 : p.head_waves));
    p.grid = (unsigned)(most < resident ? most : resident);
    p.starts_bytes = ((batch + 1) * 4 + 255) / 256 * 256;
    p.bytes = p.starts_bytes + (int64_t)p.grid * per_group * 2 * part_floats(16 * p.head_waves, p.nv) * 4;
    return true;
}

bool attend_sizes_ok(const mq_paged_cache* c, int64_t batch, int64_t heads, int64_t width, int64_t window, AttendPlan& p, const char* what) {
    char text[128];
    if (!cache_ok(c, what)) return false;
    const char* why = nullptr;
    if (batch < 0 || heads < 0 || width < 0 || window < 0) why = "bad argument";
    else if (heads % c->kv_heads) why = "query heads that the key heads divide";
    else if (batch > INT32_MAX || heads > 65535 || (batch && heads && batch > INT32_MAX / heads)) why = "tensor too large";
    else if (batch && heads && !attend_plan(c, batch, heads, width, window, p)) why = "tensor too large";
    if (!why) return true;
    snprintf(text, sizeof(text), "%s: %s", what, why);
    mq_fail(MQ_ERR_ARG, text);
    return false;
}

template <int D>
int join_launch(const AttendArgs& a, const AttendPlan& p, hipStream_t st) {
    const int64_t rows = (int64_t)a.batch * a.heads;
    const uint32_t workers = p.grid * attend_workers(p.head_waves);
    // few heads: many parts each, a workgroup for a head; else a wavefront
    if (rows <= 1024) {
        if (p.nv == 2) attend_join_kernel<D, 2, 4><<<(unsigned)rows, kJoinThreads, 0, st>>>(a, workers, 0);
        else attend_join_kernel<D, 1, 4><<<(unsigned)rows, kJoinThreads, 0, st>>>(a, workers, 0);
        return mq_check_launch("mq_paged_attention");
    }
    for (int64_t first = 0; first < rows; first += (int64_t)kMostGrid * kJoinWaves) {       // (a launch has fewer than 2^32 lanes)
        const int64_t groups = (rows - first + kJoinWaves - 1) / kJoinWaves;
        const unsigned grid = (unsigned)(groups < kMostGrid ? groups : kMostGrid);
        if (p.nv == 2) attend_join_kernel<D, 2, 1><<<grid, kJoinThreads, 0, st>>>(a, workers, first);
        else attend_join_kernel<D, 1, 1><<<grid, kJoinThreads, 0, st>>>(a, workers, first);
        const int rc = mq_check_launch("mq_paged_attention");
        if (rc != MQ_OK) return rc;
    }
    return MQ_OK;
}

}  // namespace mq

extern "C" int mq_paged_attention_workspace(const mq_paged_cache* cache, int64_t batch, int64_t heads, int64_t width, int64_t window, int64_t* bytes) {
    mq::AttendPlan p;
    if (!bytes) return mq_fail(MQ_ERR_ARG, "mq_paged_attention_workspace: null pointer");
    if (!mq::attend_sizes_ok(cache, batch, heads, width, window, p, "mq_paged_attention_workspace")) return MQ_ERR_ARG;
    *bytes = batch && heads ? p.bytes : 0;
    return MQ_OK;
}

extern "C" int mq_paged_attention(const mq_paged_cache* c, const void* q, int64_t q_batch_stride, int64_t q_head_stride, const int32_t* table,
                                  int64_t table_stride, int64_t width, const int32_t* lengths, const float* sinks, double scale, int64_t window,
                                  void* out, int64_t batch, int64_t heads, void* ws, void* stream) {
    using namespace mq;
    AttendPlan p;
    if (!attend_sizes_ok(c, batch, heads, width, window, p, "mq_paged_attention")) return MQ_ERR_ARG;
    if (batch == 0 || heads == 0) return MQ_OK;           // (without a plan)
    if (!q || !out || !lengths || (width && !table) || (p.bytes && !ws)) return mq_fail(MQ_ERR_ARG, "mq_paged_attention: null pointer");
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)ws) % 16 || (batch > 1 && q_batch_stride % 8) || (heads > 1 && q_head_stride % 8))
        return mq_fail(MQ_ERR_ARG, "mq_paged_attention: vectors that begin at multiples of 16 bytes");
    AttendArgs a = {};
    a.q = (const char*)q, a.keys = (const char*)c->keys, a.values = (const char*)c->values, a.key_scales = c->key_scales, a.value_scales = c->value_scales;
    a.table = table, a.lengths = lengths, a.sinks = sinks, a.out = (char*)out;
    a.parts = p.direct ? nullptr : (float*)((char*)ws + p.starts_bytes), a.starts = p.direct ? nullptr : (uint32_t*)ws;
    a.q_batch = q_batch_stride, a.q_head = q_head_stride, a.table_stride = table_stride;
    a.pages = (uint32_t)(c->pages < INT32_MAX ? c->pages : INT32_MAX);       // (as many as a table can name)
    const uint32_t places = (uint32_t)(c->kv_heads * c->page_size), bytes = c->key_scales ? 1 : 2;
    a.key_page = places * (uint32_t)c->key_dim * bytes, a.value_page = places * (uint32_t)c->value_dim * bytes;
    a.key_scale_page = places * (uint32_t)(c->key_dim / 32), a.value_scale_page = places * (uint32_t)(c->value_dim / 32);
    a.capacity = c->pages ? width * c->page_size : 0, a.window = window;
    a.batch = (int)batch, a.heads = (int)heads, a.kv_heads = (int)c->kv_heads, a.group = (int)(heads / c->kv_heads);
    a.key_dim = (int)c->key_dim, a.value_dim = (int)c->value_dim, a.page_shift = __builtin_ctzll(c->page_size);
    a.blocks = p.blocks, a.head_waves = p.head_waves, a.block_heads = 16 * p.head_waves, a.least = p.least, a.flip = scale < 0 ? 0x80008000u : 0u;
    a.scale = (float)(__builtin_fabs(scale) * 1.4426950408889634);
    if (a.scale < 1.2e-38f) a.scale = 1.2e-38f;           // (a score that is not seen is an infinity, which no product may make a NaN)
    const hipStream_t st = (hipStream_t)stream;
    const bool bf16 = c->dtype == MQ_BF16, kept = c->key_scales;
    const int rc = bf16 ? (kept ? mq_attend_bf16_kept : mq_attend_bf16)(a, p.nk, p.nv, p.direct, p.grid, st)
                        : (kept ? mq_attend_f16_kept : mq_attend_f16)(a, p.nk, p.nv, p.direct, p.grid, st);
    if (rc != MQ_OK || p.direct) return rc;
    return bf16 ? join_launch<MQ_BF16>(a, p, st) : join_launch<MQ_F16>(a, p, st);
}
