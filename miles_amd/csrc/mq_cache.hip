// Keys and values appended to a paged cache, keys (and queries) rotated on the way.
//
// A workgroup has some tokens: cosines and sines into shared memory, then 16-byte accesses of the tokens' vectors (32 into 8 bits, of which a lane makes
// one access of 16).  What bounds many tokens is reading and writing every element once and, into 8 bits, the arithmetic; what bounds few is the launch.
// What depends on a token alone, its slot's address above all, one lane computes into shared memory (every lane for itself: 16384 tokens of 4 heads of
// 192 and 128 into 8 bits 28 us; this takes 23.5, 2.7 TB/s, and a wavefront to a token 26.7), and the first elements are asked for before the angles and the slots are there.  A
// key's pieces are written page_size x 16 bytes apart; neighbours of a prompt fill the lines between them, for which the workgroups of 16 tokens run on
// one of the card's eight dies, behind whose cache they meet (8191 tokens of 32 query and 8 key heads of 128: 45 us, 4.5 TB/s, and 47 as they come).
// Pieces gathered in shared memory and written side by side by workgroups of their own took 60.
#include <stdio.h>

#include "mq_paged.hpp"
#include "mq_rotary.hpp"

namespace mq {

struct AppendArgs {
    char *keys, *values;
    uint8_t *key_scales, *value_scales;
    const char *k, *v, *q;
    char* q_out;
    int64_t k_token, k_head, v_token, v_head, q_token, q_head;       // strides, elements
    const void* slots;
    int64_t slot_count, tokens, first;          // first: token of this launch
    RotaryTurn turn;
    int slots64, page_shift, kv_heads, q_heads, key_dim, value_dim, per;
    int keys_end, values_end, queries_end;      // of a token's units: keys, then values, then queries, then none up to a multiple of 2
    int together;                               // workgroups of 16 tokens, which run on one die; 0: as they come
    SmallDivisor by_token, by_key, by_value, by_query;
};
constexpr int kAppendThreads = 256, kAppendTurns = 2048, kAppendTokens = 16;

// Sixteen elements as e4m3 codes of their group of 32, which two neighbouring lanes hold: the arithmetic of the MXFP8 quantizer, of fp32 values
__device__ __forceinline__ u32x4 kept_codes16(const float* f, uint32_t& e) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) m = keep_larger(m, f[i]);
    const uint32_t top = group_max2(f2u(m));
    e = keep_exponent(top);
    const float inv = e8m0_inverse(e);
    const bool infinite = top == kInfinity;
    return u32x4{keep_codes4(f[0], f[1], f[2], f[3], inv, infinite), keep_codes4(f[4], f[5], f[6], f[7], inv, infinite),
                 keep_codes4(f[8], f[9], f[10], f[11], inv, infinite), keep_codes4(f[12], f[13], f[14], f[15], inv, infinite)};
}

// An access: eight elements of a vector and, where they are turned in the halves layout, their partners.  In 16 bits a lane has both and writes both; in 8
// bits it writes its own, beside which its group's other three lanes have theirs.
struct Access {
    const char* x;
    int at, partner;               // bytes; partner < 0: none
};
// unit: of a vector, of all its pieces (OWN) or of pairs of pieces and the pieces behind them
template <bool INTER, bool OWN>
__device__ __forceinline__ Access access_of(const char* x, int unit, int turned, int half) {
    if (INTER) return Access{x, unit * 16, -1};
    if (OWN) return Access{x, unit * 16, unit >= 2 * turned ? -1 : unit * 16 + (unit >= turned ? -half : half)};
    return unit < turned ? Access{x, unit * 16, half + unit * 16} : Access{x, half + unit * 16, -1};
}
// p and its partner r turned, for both to be written
template <int D, bool INTER>
__device__ __forceinline__ void turn_both(const Access& x, u32x4& p, u32x4& r, const f32x2_t* turn, int half) {
    if (INTER) {
        if (x.at < 2 * half) turn_neighbours<D>(p, turn + x.at / 4);
    } else if (x.partner >= 0) turn_halves<D>(p, r, turn + x.at / 2);
}
// the eight own elements, turned, as fp32
template <int D, bool INTER>
__device__ __forceinline__ void turn_own(const Access& x, u32x4 p, u32x4 r, const f32x2_t* turn, int half, float* f) {
    unpack<D>(p, f);
    if (INTER) {
        if (x.at >= 2 * half) return;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const f32x2_t w = turn[x.at / 4 + j / 2];
            const float a = f[j], b = f[j + 1];
            f[j] = a * w.x - b * w.y;
            f[j + 1] = b * w.x + a * w.y;
        }
    } else if (x.partner >= 0) {
        const bool second = x.partner < x.at;
        float g[8];
        unpack<D>(r, g);
        const f32x2_t* w = turn + (second ? x.partner : x.at) / 2;
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = f[j] * w[j].x - g[j] * (second ? -w[j].y : w[j].y);
    }
}

// PAST: queries and values go past the caches (keys stay, until their neighbours have come)
template <int D, bool INTER, bool KEPT, bool PAST>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(const AppendArgs a) {
    __shared__ __attribute__((aligned(16))) f32x2_t cs[kAppendTurns];
    __shared__ const char* from[3][kAppendTokens];        // a token's keys, values and queries,
    __shared__ char* to[3][kAppendTokens];                // its place in the first head's keys and values, and its turned queries
    __shared__ uint8_t* scales_to[2][KEPT ? kAppendTokens : 1];
    __shared__ bool stored[kAppendTokens];
    uint32_t nth = blockIdx.x;
    if (a.together) {                                     // consecutive workgroups run on the eight dies in turn
        const uint32_t all = 8 * a.together, set = nth / all, in = nth - set * all;
        if ((set + 1) * all <= gridDim.x) nth = (set * 8 + in % 8) * a.together + in / 8;
    }
    const int64_t token0 = a.first + (int64_t)nth * a.per;
    const int here = (int)(a.tokens - token0 < a.per ? a.tokens - token0 : a.per), pairs = a.turn.pairs, mine = threadIdx.x;
    const int half = pairs * 2, turned = INTER ? pairs / 4 : pairs / 8;           // bytes, units
    const int pieces = a.key_dim / (KEPT ? 16 : 8);
    const uint32_t key_head = (uint32_t)(pieces * 16) << a.page_shift, value_head = (uint32_t)(a.value_dim * (KEPT ? 1 : 2)) << a.page_shift;       // bytes
    const uint32_t key_groups = (uint32_t)(a.key_dim / 32) << a.page_shift, value_groups = (uint32_t)(a.value_dim / 32) << a.page_shift;
    int64_t slot = 0;
    const char *const k = a.k + token0 * a.k_token * 2, *const v = a.v + token0 * a.v_token * 2, *const q = a.q + token0 * a.q_token * 2;
    if (mine < here) {
        slot = index_at(a.slots, token0 + mine, a.slots64);
        from[0][mine] = k + mine * a.k_token * 2;
        from[1][mine] = v + mine * a.v_token * 2;
        from[2][mine] = q + mine * a.q_token * 2;
    }
    if (a.per > 1) __syncthreads();
    const uint32_t n = (uint32_t)here * a.by_token.d;
    for (uint32_t i = mine; i < n || i == (uint32_t)mine; i += kAppendThreads) {
        // the first access is on its way while the angles are computed and the slots are asked for
        const bool some = i < n;
        const uint32_t t = a.per > 1 && some ? divide(i, a.by_token) : 0u, in_token = i - t * a.by_token.d;
        const int kind = (int)in_token < a.keys_end ? 0 : (int)in_token < a.values_end ? 1 : 2;
        const SmallDivisor by = kind == 0 ? a.by_key : kind == 1 ? a.by_value : a.by_query;
        uint32_t unit = in_token - (kind == 0 ? 0 : kind == 1 ? a.keys_end : a.values_end);
        const uint32_t head = divide(unit, by);
        unit -= __umul24(head, by.d);
        const bool two = KEPT && kind < 2, read = some && (int)in_token < a.queries_end;
        const char* const x0 = (a.per > 1 ? from[kind][t] : kind == 0 ? k : kind == 1 ? v : q) + (int64_t)head * (kind == 0 ? a.k_head : kind == 1 ? a.v_head : a.q_head) * 2;
        Access x, x2;                                     // x2: the second eight of sixteen elements that go into 8 bits
        if (KEPT && kind == 0) {
            x = access_of<INTER, true>(x0, 2 * unit, turned, half);
            x2 = access_of<INTER, true>(x0, 2 * unit + 1, turned, half);
        } else if (KEPT && kind == 1) {
            x = Access{x0, (int)unit * 32, -1};
            x2 = Access{x0, (int)unit * 32 + 16, -1};
        } else x = kind == 1 ? Access{x0, (int)unit * 16, -1} : access_of<INTER, false>(x0, unit, turned, half);
        u32x4 p = {}, r = {}, p2 = {}, r2 = {};
        if (read) {
            p = ld16_keep(x.x + x.at);
            if (two) p2 = ld16_keep(x2.x + x2.at);
            if (x.partner >= 0) r = ld16_keep(x.x + x.partner);
            if (two && x2.partner >= 0) r2 = ld16_keep(x2.x + x2.partner);
        }
        if (i == (uint32_t)mine) {
            for (int j = mine; j < here * pairs; j += kAppendThreads) {
                const int tj = j / pairs;
                cs[j] = turn_of(a.turn, index_at(a.turn.positions, token0 + tj, a.turn.positions64), j - tj * pairs);
            }
            if (mine < here) {
                const bool ok = inside(slot, a.slot_count);
                const uint64_t page = (uint64_t)(ok ? slot : 0) >> a.page_shift;
                const uint32_t place = (uint32_t)slot & ((1u << a.page_shift) - 1);
                stored[mine] = ok;
                to[0][mine] = a.keys + page * ((uint64_t)key_head * a.kv_heads) + place * 16;
                to[1][mine] = a.values + page * ((uint64_t)value_head * a.kv_heads) + place * (uint32_t)(a.value_dim * (KEPT ? 1 : 2));
                to[2][mine] = a.q_out + (token0 + mine) * ((int64_t)a.q_heads * a.key_dim * 2);
                if (KEPT) {
                    scales_to[0][mine] = a.key_scales + page * ((uint64_t)key_groups * a.kv_heads) + place;
                    scales_to[1][mine] = a.value_scales + page * ((uint64_t)value_groups * a.kv_heads) + place;
                }
            }
            __syncthreads();
        }
        if (!read || (kind < 2 && !stored[t])) continue;  // (a token that is left out has its queries)
        const f32x2_t* turn = cs + t * pairs;
        char* const y = to[kind][t];
        if (two) {
            float f[16];
            uint32_t e;
            if (kind == 0) {
                turn_own<D, INTER>(x, p, r, turn, half, f);
                turn_own<D, INTER>(x2, p2, r2, turn, half, f + 8);
            } else {
                unpack<D>(p, f);
                unpack<D>(p2, f + 8);
            }
            const u32x4 codes = kept_codes16(f, e);
            *(u32x4*)(y + head * (kind == 0 ? key_head : value_head) + (kind == 0 ? (unit << a.page_shift) * 16 : unit * 16)) = codes;
            if (unit % 2 == 0) scales_to[kind][t][head * (kind == 0 ? key_groups : value_groups) + ((unit / 2) << a.page_shift)] = (uint8_t)e;
        } else if (kind == 1) store16<PAST>(y + head * value_head + unit * 16, p);
        else {
            turn_both<D, INTER>(x, p, r, turn, half);
            if (kind == 0) {
                char* const z = y + head * key_head;
                *(u32x4*)(z + ((uint32_t)x.at << a.page_shift)) = p;
                if (x.partner >= 0) *(u32x4*)(z + ((uint32_t)x.partner << a.page_shift)) = r;
            } else {
                char* const z = y + __umul24(head, (uint32_t)a.key_dim * 2);
                store16<PAST>(z + x.at, p);
                if (x.partner >= 0) store16<PAST>(z + x.partner, r);
            }
        }
    }
}

bool cache_ok(const mq_paged_cache* c, const char* what) {
    char text[160];
    const char* why = nullptr;
    const bool kept = c && c->key_scales;
    if (!c) why = "null pointer";
    else if (c->dtype != MQ_BF16 && c->dtype != MQ_F16) why = "a cache of bf16 or fp16 values";
    else if (c->pages < 0 || c->kv_heads < 1 || c->kv_heads > 65535) why = "bad argument";
    else if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1))) why = "pages of 16 to 1024 places, a power of two";
    else if (c->key_dim < 8 || c->key_dim > 256 || c->value_dim < 8 || c->value_dim > 256) why = "keys and values of 8 to 256 elements";
    else if ((c->key_dim | c->value_dim) % (kept ? 32 : 8)) why = kept ? "keys and values whose length is a multiple of 32" : "keys and values whose length is a multiple of 8";
    else if (!c->key_scales != !c->value_scales) why = "scales for both keys and values, or for neither";
    else if (c->kv_heads * c->page_size * 256 * 2 >= (1ll << 31) || c->pages > (INT64_MAX >> 20) / (c->page_size * c->kv_heads)) why = "tensor too large";
    else if (c->pages && (!c->keys || !c->values)) why = "null pointer";
    else if (((uintptr_t)c->keys | (uintptr_t)c->values | (uintptr_t)c->key_scales | (uintptr_t)c->value_scales) % 16) why = "a cache that begins at multiples of 16 bytes";
    if (!why) return true;
    snprintf(text, sizeof(text), "%s: %s", what, why);
    mq_fail(MQ_ERR_ARG, text);
    return false;
}

}  // namespace mq

extern "C" int mq_cache_append(const mq_paged_cache* c, const mq_heads* k, const mq_heads* v, const mq_heads* q, int64_t tokens, const void* slots, int slots64,
                               const void* positions, int positions64, const void* inv_freq, int freq64, int64_t pairs, int interleaved, double scale,
                               void* stream) {
    using namespace mq;
    if (!cache_ok(c, "mq_cache_append")) return MQ_ERR_ARG;
    if (!k || !v || tokens < 0 || pairs < 0 || 2 * pairs > c->key_dim) return mq_fail(MQ_ERR_ARG, "mq_cache_append: bad argument");
    if (pairs % 8) return mq_fail(MQ_ERR_ARG, "mq_cache_append: a multiple of 8 pairs");
    if (k->heads != c->kv_heads || v->heads != c->kv_heads || (q && (q->heads < 0 || q->heads > 65535)))
        return mq_fail(MQ_ERR_ARG, "mq_cache_append: as many heads as the cache has");
    if (tokens > INT32_MAX) return mq_fail(MQ_ERR_ARG, "mq_cache_append: tensor too large");
    if (tokens == 0) return MQ_OK;
    if (!k->in || !v->in || !slots || (pairs && (!positions || !inv_freq)) || (q && q->heads && (!q->in || !q->out)))
        return mq_fail(MQ_ERR_ARG, "mq_cache_append: null pointer");
    AppendArgs a = {};
    for (const mq_heads* x : {k, v, q}) {
        if (!x || !x->heads) continue;
        if (((uintptr_t)x->in | (x == q ? (uintptr_t)x->out : 0)) % 16 || (tokens > 1 && x->token_stride % 8) || (x->heads > 1 && x->head_stride % 8))
            return mq_fail(MQ_ERR_ARG, "mq_cache_append: vectors that begin at multiples of 16 bytes");
    }
    a.keys = (char*)c->keys, a.values = (char*)c->values, a.key_scales = c->key_scales, a.value_scales = c->value_scales;
    a.k = (const char*)k->in, a.v = (const char*)v->in, a.q = q ? (const char*)q->in : nullptr, a.q_out = q ? (char*)q->out : nullptr;
    a.k_token = k->token_stride, a.k_head = k->head_stride, a.v_token = v->token_stride, a.v_head = v->head_stride;
    a.q_token = q ? q->token_stride : 0, a.q_head = q ? q->head_stride : 0, a.q_heads = q ? (int)q->heads : 0;
    a.slots = slots, a.slots64 = slots64, a.slot_count = c->pages * c->page_size, a.tokens = tokens;
    a.page_shift = __builtin_ctzll(c->page_size);
    a.turn = RotaryTurn{positions, inv_freq, scale, (int)pairs, positions64, freq64, 0};
    a.kv_heads = (int)c->kv_heads, a.key_dim = (int)c->key_dim, a.value_dim = (int)c->value_dim;
    const bool kept = c->key_scales;
    const int query_units = (int)(interleaved ? c->key_dim / 8 : (c->key_dim - pairs) / 8), key_units = kept ? (int)c->key_dim / 16 : query_units;
    const int value_units = (int)c->value_dim / (kept ? 16 : 8);
    const int64_t keys = c->kv_heads * key_units, values = c->kv_heads * value_units, queries = a.q_heads * (int64_t)query_units, units = (keys + values + queries + 1) / 2 * 2;
    if (units > 65534) return mq_fail(MQ_ERR_ARG, "mq_cache_append: tensor too large");
    a.keys_end = (int)keys, a.values_end = (int)(keys + values), a.queries_end = (int)(keys + values + queries);
    a.by_token = small_divisor((uint32_t)units);
    a.by_key = small_divisor((uint32_t)key_units), a.by_value = small_divisor((uint32_t)value_units), a.by_query = small_divisor((uint32_t)query_units);
    // tokens of a workgroup: for few accesses a lane, while there are workgroups for every compute unit (the 8191 tokens above by one or two 45, by four
    // 54; the 16384 by one 49, by two 31, by four 25.5, by eight 23.5)
    int64_t per = 1;
    while (per < kAppendTokens && per * 2 * pairs <= kAppendTurns && tokens / (per * 2) >= 1024 && per * 2 * units <= 640) per *= 2;
    a.per = (int)per;
    a.together = tokens >= 1024 ? kAppendTokens / (int)per : 0;
    const bool past = tokens * (a.q_heads * c->key_dim + c->kv_heads * c->value_dim) * 2 >= kPastCaches;
    constexpr int64_t kMost = 1 << 22;                    // tokens of a launch, which has fewer than 2^32 lanes
    const hipStream_t st = (hipStream_t)stream;
    const int64_t end = tokens;
    for (; a.first < end; a.first += kMost) {
        const int64_t left = end - a.first < kMost ? end - a.first : kMost;
        a.tokens = a.first + left;
        const dim3 grid((unsigned)((left + per - 1) / per));
        auto launch = [&](auto type, auto inter, auto in8) {
            constexpr int D = decltype(type)::value;
            constexpr bool kInter = decltype(inter)::value, kKept = decltype(in8)::value;
            if (past) append_kernel<D, kInter, kKept, true><<<grid, kAppendThreads, 0, st>>>(a);
            else append_kernel<D, kInter, kKept, false><<<grid, kAppendThreads, 0, st>>>(a);
        };
        auto by_kept = [&](auto type, auto inter) { kept ? launch(type, inter, std::true_type{}) : launch(type, inter, std::false_type{}); };
        auto by_layout = [&](auto type) { interleaved ? by_kept(type, std::true_type{}) : by_kept(type, std::false_type{}); };
        c->dtype == MQ_BF16 ? by_layout(std::integral_constant<int, MQ_BF16>{}) : by_layout(std::integral_constant<int, MQ_F16>{});
        const int rc = mq_check_launch("mq_cache_append");
        if (rc != MQ_OK) return rc;
    }
    return MQ_OK;
}
