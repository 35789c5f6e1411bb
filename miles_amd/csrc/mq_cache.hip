// Keys and values appended to a paged cache, keys (and queries) rotated on the way.
//
// A workgroup has some tokens: cosines and sines into shared memory, then 16-byte accesses of the tokens' vectors (32 into 8 bits, of which a lane makes
// one access of 16).  What bounds many tokens is reading and writing every element once and, into 8 bits, the arithmetic; what bounds few is the launch.
// A key's pieces are written page_size x 16 bytes apart; neighbours of a prompt fill the lines between them, for which the workgroups of 64 tokens run on
// one of the card's eight dies, behind whose cache they meet, and everything that is read once is read past it.
// 8191 tokens of 32 query and 8 key heads of 128: 35.9 us, 5.6 TB/s (as they come 42.5, read through the cache 46, queries and values past it 38.3, two
// tokens to a workgroup 37, four 42; pieces gathered in shared memory and written side by side by workgroups of their own 60).  16384 tokens of 4 heads
// of 192 and 128 into 8 bits: 24.4 us, 2.6 TB/s (16 tokens on a die 25.6, and 36.2 above; 128 24.3 and 37.6).
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
    int64_t slot_count, tokens, first;
    RotaryTurn turn;
    int slots64, page_shift, kv_heads, q_heads, key_dim, value_dim, per;
    int keys_end, values_end, queries_end;      // of a token's units: keys, then values, then queries, then padding to a multiple of 2
    int together;                               // workgroups of kAppendTogether tokens, which run on one die; 0: as they come
    SmallDivisor by_token, by_key, by_value, by_query;
};
constexpr int kAppendThreads = 256, kAppendTurns = 2048, kAppendTokens = 16, kAppendTogether = 64;

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

// The eight elements of a key's piece, turned, as fp32: with their partners in the other half where pairs are i and i + pairs
template <int D, bool INTER>
__device__ __forceinline__ void turned8(const char* x, int piece, int turned, int half, const f32x2_t* turn, float* f) {
    const u32x4 own = ld16_keep(x + piece * 16);          // (two lanes read it)
    if (INTER) {
        unpack<D>(own, f);
        if (piece >= turned) return;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const f32x2_t w = turn[piece * 4 + j / 2];
            const float p = f[j], r = f[j + 1];
            f[j] = p * w.x - r * w.y;
            f[j + 1] = r * w.x + p * w.y;
        }
    } else if (piece >= 2 * turned) {
        unpack<D>(own, f);
    } else {
        const bool second = piece >= turned;
        const u32x4 other = ld16_keep(x + piece * 16 + (second ? -half : half));
        float g[8];
        unpack<D>(own, f);
        unpack<D>(other, g);
        const f32x2_t* w = turn + (second ? piece - turned : piece) * 8;
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = f[j] * w[j].x - g[j] * (second ? -w[j].y : w[j].y);
    }
}

template <int D, bool INTER, bool KEPT>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(const AppendArgs a) {
    __shared__ __attribute__((aligned(16))) f32x2_t cs[kAppendTurns];
    __shared__ int64_t slot[kAppendTokens];
    uint32_t nth = blockIdx.x;
    if (a.together) {                                     // consecutive workgroups run on the eight dies in turn
        const uint32_t all = 8 * a.together, set = nth / all, in = nth - set * all;
        if ((set + 1) * all <= gridDim.x) nth = (set * 8 + in % 8) * a.together + in / 8;
    }
    const int64_t token0 = a.first + (int64_t)nth * a.per;
    const int here = (int)(a.tokens - token0 < a.per ? a.tokens - token0 : a.per), pairs = a.turn.pairs;
    for (int i = threadIdx.x; i < here * pairs; i += kAppendThreads) {
        const int t = i / pairs;
        cs[i] = turn_of(a.turn, index_at(a.turn.positions, token0 + t, a.turn.positions64), i - t * pairs);
    }
    if ((int)threadIdx.x < here) {
        const int64_t s = index_at(a.slots, token0 + threadIdx.x, a.slots64);
        slot[threadIdx.x] = inside(s, a.slot_count) ? s : -1;
    }
    __syncthreads();
    const int page_size = 1 << a.page_shift, half = pairs * 2;           // (bytes)
    const int turned = INTER ? pairs / 4 : pairs / 8;                    // units
    for (uint32_t i = threadIdx.x, n = (uint32_t)here * a.by_token.d; i < n; i += kAppendThreads) {
        const uint32_t t = divide(i, a.by_token);
        int unit = (int)(i - t * a.by_token.d);
        const f32x2_t* turn = cs + t * pairs;
        const bool is_key = unit < a.keys_end;
        if (is_key || unit < a.values_end) {
            const int64_t s = slot[t];
            if (s < 0) continue;                                         // (of all lanes of a group alike)
            if (!is_key) unit -= a.keys_end;
            const int h = (int)divide(unit, is_key ? a.by_key : a.by_value);
            unit -= h * (int)(is_key ? a.by_key.d : a.by_value.d);
            const int64_t at = (s >> a.page_shift) * a.kv_heads + h;     // page and head
            const int place = (int)(s & (page_size - 1));
            if (KEPT) {                                                  // sixteen elements
                float f[16];
                uint32_t e;
                if (is_key) {
                    const char* x = a.k + ((token0 + t) * a.k_token + (int64_t)h * a.k_head) * 2;
                    turned8<D, INTER>(x, 2 * unit, turned, half, turn, f);
                    turned8<D, INTER>(x, 2 * unit + 1, turned, half, turn, f + 8);
                } else {
                    const char* x = a.v + ((token0 + t) * a.v_token + (int64_t)h * a.v_head + unit * 16) * 2;
                    unpack<D>(ld16(x), f);
                    unpack<D>(ld16(x + 16), f + 8);
                }
                const u32x4 codes = kept_codes16(f, e);
                if (is_key) *(u32x4*)(a.keys + (((at * (a.key_dim / 16) + unit) << a.page_shift) + place) * 16) = codes;
                else *(u32x4*)(a.values + ((at << a.page_shift) + place) * a.value_dim + unit * 16) = codes;
                if (unit % 2 == 0) {
                    uint8_t* const scales = is_key ? a.key_scales : a.value_scales;
                    scales[((at * ((is_key ? a.key_dim : a.value_dim) / 32) + unit / 2) << a.page_shift) + place] = (uint8_t)e;
                }
                continue;
            }
            if (!is_key) {
                *(u32x4*)(a.values + (((at << a.page_shift) + place) * a.value_dim + unit * 8) * 2) =
                    ld16(a.v + ((token0 + t) * a.v_token + (int64_t)h * a.v_head + unit * 8) * 2);
                continue;
            }
            const char* x = a.k + ((token0 + t) * a.k_token + (int64_t)h * a.k_head) * 2;
            char* y = a.keys + (((at * (a.key_dim / 8)) << a.page_shift) + place) * 16;         // its first piece
            if (unit >= turned) {
                const int piece = (INTER ? 0 : turned) + unit;
                *(u32x4*)(y + ((int64_t)piece << a.page_shift) * 16) = ld16(x + piece * 16);
            } else if (INTER) {
                u32x4 p = ld16(x + unit * 16);
                turn_neighbours<D>(p, turn + unit * 4);
                *(u32x4*)(y + ((int64_t)unit << a.page_shift) * 16) = p;
            } else {
                u32x4 p = ld16(x + unit * 16), r = ld16(x + half + unit * 16);
                turn_halves<D>(p, r, turn + unit * 8);
                *(u32x4*)(y + ((int64_t)unit << a.page_shift) * 16) = p;
                *(u32x4*)(y + ((int64_t)(unit + turned) << a.page_shift) * 16) = r;
            }
        } else if (unit < a.queries_end) {
            unit -= a.values_end;
            const int h = (int)divide(unit, a.by_query);
            unit -= h * (int)a.by_query.d;
            const char* x = a.q + ((token0 + t) * a.q_token + (int64_t)h * a.q_head) * 2;
            char* y = a.q_out + ((token0 + t) * a.q_heads + h) * (int64_t)a.key_dim * 2;
            if (unit >= turned) {
                const int piece = (INTER ? 0 : turned) + unit;
                *(u32x4*)(y + piece * 16) = ld16(x + piece * 16);
            } else if (INTER) {
                u32x4 p = ld16(x + unit * 16);
                turn_neighbours<D>(p, turn + unit * 4);
                *(u32x4*)(y + unit * 16) = p;
            } else {
                u32x4 p = ld16(x + unit * 16), r = ld16(x + half + unit * 16);
                turn_halves<D>(p, r, turn + unit * 8);
                *(u32x4*)(y + unit * 16) = p;
                *(u32x4*)(y + half + unit * 16) = r;
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
    // tokens of a workgroup: for an access or two a lane, while there are workgroups for every compute unit (the 16384 above, 16 on a die, by one 35, by two or four
    // 25.7, by eight 29.7)
    int64_t per = 1;
    while (per < kAppendTokens && per * 2 * pairs <= kAppendTurns && tokens / (per * 2) >= 1024 && per * 2 * units <= 384) per *= 2;
    a.per = (int)per;
    a.together = tokens >= 1024 ? kAppendTogether / (int)per : 0;
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
            append_kernel<D, kInter, kKept><<<grid, kAppendThreads, 0, st>>>(a);
        };
        auto by_kept = [&](auto type, auto inter) { kept ? launch(type, inter, std::true_type{}) : launch(type, inter, std::false_type{}); };
        auto by_layout = [&](auto type) { interleaved ? by_kept(type, std::true_type{}) : by_kept(type, std::false_type{}); };
        c->dtype == MQ_BF16 ? by_layout(std::integral_constant<int, MQ_BF16>{}) : by_layout(std::integral_constant<int, MQ_F16>{});
        const int rc = mq_check_launch("mq_cache_append");
        if (rc != MQ_OK) return rc;
    }
    return MQ_OK;
}
