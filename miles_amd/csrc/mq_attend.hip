// Attention over a paged cache: how its work is shared out, and the join of sequences that several workgroups had a part of.
//
// The lengths are on the device and differ, so the launch cannot follow them.  A launch has as many workgroups as the card holds; each adds
// the lengths up and takes an equal share of all tiles, which may begin and end inside a sequence: at most its first and its last
// sequence's sums are partial.  Where no sequence can be long, every workgroup has one sequence's key head instead, and there is no join.
#include <stdio.h>

#include "mq_attend.hpp"

namespace mq {

// Partial results of a head, in the workgroups' order.  WAVES wavefronts have a head; a lane has eight elements of each 128 and every
// (4 WAVES)th part.
template <int D, int NV, int WAVES>
__global__ __launch_bounds__(kAttendThreads) void attend_join_kernel(const AttendArgs a, uint32_t workgroups) {
    __shared__ __attribute__((aligned(16))) float sums[kAttendWaves][16][12];
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x / kWave), piece = lane & 15, sub = (lane >> 4) + (WAVES > 1 ? wave * 4 : 0);
    const int64_t nth = WAVES > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * kAttendWaves + wave;
    if (nth >= (int64_t)a.batch * a.heads) return;        // (with WAVES > 1: never)
    const int b = (int)(nth / a.heads), head = (int)(nth - (int64_t)b * a.heads);
    const uint32_t before = a.starts[b], units = a.starts[b + 1] - before, total = a.starts[a.batch];
    if (units == 0) return;
    const int kv = head / a.group, in_group = head - kv * a.group, block = in_group / (16 * a.head_waves), in_block = in_group - block * 16 * a.head_waves;
    const uint32_t tiles = units / (uint32_t)(a.kv_heads * a.blocks), u0 = before + (uint32_t)(kv * a.blocks + block) * tiles;
    const uint32_t share = (total + workgroups - 1) / workgroups, per = share > a.least ? share : a.least;
    const uint32_t w0 = u0 / per, w1 = (u0 + tiles - 1) / per;
    if (w0 == w1) return;                                 // one workgroup had it all
    const bool inside_first = u0 != w0 * per;             // the first part is the last of its workgroup's
    auto part = [&](uint32_t w) { return a.parts + ((int64_t)w * 2 + (w == w0 && inside_first ? 1 : 0)) * part_floats(a.head_waves, NV); };
    const int64_t ml = (int64_t)a.head_waves * 16 * (128 * NV) + in_block * 2;
    float top = kLowest;
    for (uint32_t w = w0 + sub; w <= w1; w += 4 * WAVES) top = __builtin_fmaxf(top, part(w)[ml]);
    top = max_of_head(top);
    if (WAVES > 1) {
        if (lane == 0) sums[wave][0][0] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kAttendWaves; i++) top = __builtin_fmaxf(top, sums[i][0][0]);
        __syncthreads();
    }
#pragma unroll
    for (int nv = 0; nv < NV; nv++) {
        float l = 0.0f, f[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (uint32_t w = w0 + sub; w <= w1; w += 4 * WAVES) {
            const float* from = part(w);
            const float m = from[ml], lw = from[ml + 1], times = __builtin_amdgcn_exp2f(m - top);
            const f32x4 x = *(const f32x4*)(from + in_block * (128 * NV) + nv * 128 + piece * 8), y = *(const f32x4*)(from + in_block * (128 * NV) + nv * 128 + piece * 8 + 4);
            l += lw * times;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                f[i] += x[i] * times;
                f[4 + i] += y[i] * times;
            }
        }
        l = sum_of_head(l);
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = sum_of_head(f[i]);
        if (WAVES > 1) {
            if (lane < 16) {
#pragma unroll
                for (int i = 0; i < 8; i++) sums[wave][piece][i] = f[i];
                sums[wave][piece][8] = l;
            }
            __syncthreads();
            l = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = 0.0f;
#pragma unroll
            for (int w = 0; w < kAttendWaves; w++) {
                l += sums[w][piece][8];
#pragma unroll
                for (int i = 0; i < 8; i++) f[i] += sums[w][piece][i];
            }
            __syncthreads();
        }
        const int at = nv * 128 + piece * 8;
        if (lane < 16 && (WAVES == 1 || wave == 0) && at < a.value_dim) {
            const float times = finish_factor(a, head, top, l);
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] *= times;
            store8<D>(a.out + (nth * a.value_dim + at) * 2, f);
        }
    }
}

struct AttendPlan {
    int nk, nv, blocks, head_waves;
    bool direct;
    unsigned grid;
    uint32_t least;
    int64_t bytes, starts_bytes;
};
constexpr int64_t kDirectTiles = 16, kMostGrid = 1 << 23;

// false: too large
bool attend_plan(const mq_paged_cache* c, int64_t batch, int64_t heads, int64_t width, int64_t window, AttendPlan& p) {
    const int64_t group = heads / c->kv_heads, tiles16 = (group + 15) / 16;
    p.head_waves = tiles16 > 2 ? 4 : (int)tiles16;
    p.blocks = (int)((tiles16 + p.head_waves - 1) / p.head_waves);
    p.nk = (int)((c->key_dim + 63) / 64) * 2;
    p.nv = c->value_dim > 128 ? 2 : 1;
    if (width > (INT32_MAX - 4096) / c->page_size) return false;      // (a token behind the last has a number, too)
    const int64_t capacity = width * c->page_size;
    int64_t tiles = (capacity + kTile - 1) / kTile;
    if (window > 0 && window < capacity) tiles = tiles < (window + kTile - 1) / kTile + 1 ? tiles : (window + kTile - 1) / kTile + 1;
    const int64_t rows = batch * c->kv_heads * p.blocks;
    if (rows > INT32_MAX / (tiles ? tiles : 1)) return false;
    p.direct = tiles <= kDirectTiles && rows <= kMostGrid;
    p.bytes = p.starts_bytes = 0;
    p.least = (uint32_t)(kAttendWaves / p.head_waves);
    if (p.direct) {
        p.grid = (unsigned)rows;
        return true;
    }
    const int64_t most = (rows * tiles + p.least - 1) / p.least, resident = p.nv == 2 && p.nk > 4 ? 256 : 512;
    p.grid = (unsigned)(most < resident ? most : resident);
    p.starts_bytes = ((batch + 1) * 4 + 255) / 256 * 256;
    p.bytes = p.starts_bytes + (int64_t)p.grid * 2 * part_floats(p.head_waves, p.nv) * 4;
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
    // few heads: many parts each, a workgroup for a head; else a wavefront
    if (rows <= 1024) {
        if (p.nv == 2) attend_join_kernel<D, 2, 4><<<(unsigned)rows, kAttendThreads, 0, st>>>(a, p.grid);
        else attend_join_kernel<D, 1, 4><<<(unsigned)rows, kAttendThreads, 0, st>>>(a, p.grid);
        return mq_check_launch("mq_paged_attention");
    }
    const unsigned grid = (unsigned)((rows + kAttendWaves - 1) / kAttendWaves);
    if (p.nv == 2) attend_join_kernel<D, 2, 1><<<grid, kAttendThreads, 0, st>>>(a, p.grid);
    else attend_join_kernel<D, 1, 1><<<grid, kAttendThreads, 0, st>>>(a, p.grid);
    return mq_check_launch("mq_paged_attention");
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
    a.blocks = p.blocks, a.head_waves = p.head_waves, a.least = p.least, a.scale = (float)(scale * 1.4426950408889634);
    const hipStream_t st = (hipStream_t)stream;
    const bool bf16 = c->dtype == MQ_BF16, kept = c->key_scales;
    const int rc = bf16 ? (kept ? mq_attend_bf16_kept : mq_attend_bf16)(a, p.nk, p.nv, p.grid, st)
                        : (kept ? mq_attend_f16_kept : mq_attend_f16)(a, p.nk, p.nv, p.grid, st);
    if (rc != MQ_OK || p.direct) return rc;
    return bf16 ? join_launch<MQ_BF16>(a, p, st) : join_launch<MQ_F16>(a, p, st);
}
