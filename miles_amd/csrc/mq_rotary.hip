// Rotary positions, forward and backward (the backward pass turns by the negative angle).
//
// A workgroup has some tokens: its lanes compute the tokens' cosines and sines into shared memory and go through the heads' vectors in
// 16-byte accesses, of which those of the halves layout come in pairs.  What bounds it is reading and writing every element once.
#include "mq_rotary.hpp"

namespace mq {

// Results of this many bytes and more go past the caches (non-temporal stores: 16384 tokens of 40 heads of 128 in 56 us instead of 61, 4096 in 17.4 instead of
// 18.8); fewer may be there still when the next kernel reads them.  A template's argument of the kernel, since stores of both kinds behind one branch
// become one plain store.
constexpr int64_t kPastCaches = 16 << 20;
template <bool PAST>
__device__ __forceinline__ void store16(char* p, u32x4 v) {
    if (PAST) st16(p, v);
    else *(u32x4*)p = v;
}

struct RotaryArgs {
    const char* in[2];
    char* out[2];
    int64_t batch_stride[2], token_stride[2], head_stride[2];    // of the inputs, elements
    int heads[2];
    int64_t position_batch_stride;
    RotaryTurn turn;
    int64_t tokens, total;         // of a batch entry, and of all
    int64_t first;                 // token of this launch
    int dim, per;                  // elements of a vector; tokens of a workgroup
    SmallDivisor by_token, by_head;        // units of a token and of a vector: accesses (pairs of them in the halves layout), or single elements
};
constexpr int kRotaryThreads = 256, kRotaryTurns = 2048, kRotaryTokens = 16;

// VEC: every vector begins at a multiple of 16 bytes, and so does its second half; else element by element
// PAST: results go past the caches
template <int D, bool INTER, bool VEC, bool PAST>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(const RotaryArgs a) {
    constexpr int V = VEC ? kVec<D> : 1;
    __shared__ __attribute__((aligned(16))) f32x2_t cs[kRotaryTurns];
    const int64_t token0 = a.first + (int64_t)blockIdx.x * a.per;
    const int here = (int)(a.total - token0 < a.per ? a.total - token0 : a.per), pairs = a.turn.pairs;
    const uint32_t units = a.by_token.d, n = (uint32_t)here * units;
    const int turned = VEC ? (INTER ? 2 * pairs / V : pairs / V) : pairs, half = pairs * kElem<D>;
    auto batch_of = [&](uint32_t token) { return a.total == a.tokens ? 0u : token / (uint32_t)a.tokens; };       // (all of them: fewer than 2^31)
    struct Unit {
        const char* x;
        char* y;
        int at, token;                                    // number within the vector, and of the token within the workgroup
    };
    auto unit_of = [&](uint32_t i) {
        const uint32_t t = VEC ? divide(i, a.by_token) : i / units, in_token = i - t * units;
        uint32_t head = VEC ? divide(in_token, a.by_head) : in_token / a.by_head.d;
        const int at = (int)(in_token - head * a.by_head.d), w = head >= (uint32_t)a.heads[0];
        if (w) head -= a.heads[0];
        const uint32_t token = (uint32_t)token0 + t, b = batch_of(token);
        return Unit{a.in[w] + ((int64_t)b * a.batch_stride[w] + (int64_t)(token - b * (uint32_t)a.tokens) * a.token_stride[w] + (int64_t)head * a.head_stride[w]) * kElem<D>,
                    a.out[w] + ((int64_t)token * a.heads[w] + head) * a.dim * kElem<D>, at, (int)t};
    };
    auto angles = [&]() {
        for (int i = threadIdx.x; i < here * pairs; i += kRotaryThreads) {
            const int t = i / pairs;
            const uint32_t token = (uint32_t)token0 + t, b = batch_of(token);
            cs[i] = turn_of(a.turn, index_at(a.turn.positions, b * a.position_batch_stride + (token - b * (uint32_t)a.tokens), a.turn.positions64), i - t * pairs);
        }
        __syncthreads();
    };
    if (VEC) {
        // The first access is on its way while the angles are computed, one at a time: 16384 tokens of 40 heads of 128 in bf16 in 56 us, 6.0 TB/s (the
        // angles first 62; two accesses at a time were 2 us slower; a copy of as many bytes runs at 6.2 to 6.5).
        const bool any = threadIdx.x < n;
        for (uint32_t i = threadIdx.x; i < n || i == threadIdx.x; i += kRotaryThreads) {
            Unit unit = {};
            u32x4 p, q;
            int at = 0;
            if (any) {
                unit = unit_of(i);
                at = unit.at >= turned && !INTER ? 2 * half + (unit.at - turned) * 16 : unit.at * 16;
                p = ld16(unit.x + at);
                if (!INTER && unit.at < turned) q = ld16(unit.x + half + at);
            }
            if (i == threadIdx.x) angles();
            if (!any) return;
            if (unit.at < turned) {
                const f32x2_t* turn = cs + unit.token * pairs;
                if (INTER) turn_neighbours<D>(p, turn + unit.at * (V / 2));
                else {
                    turn_halves<D>(p, q, turn + unit.at * V);
                    store16<PAST>(unit.y + half + at, q);
                }
            }
            store16<PAST>(unit.y + at, p);
        }
    } else {
        angles();
        for (uint32_t i = threadIdx.x; i < n; i += kRotaryThreads) {
            const Unit unit = unit_of(i);
            if (unit.at >= turned) {                      // behind the part that is turned
                store_dtype(unit.y, pairs + unit.at, load_f32(unit.x, pairs + unit.at, D), D);
                continue;
            }
            const f32x2_t w = cs[unit.token * pairs + unit.at];
            const int i0 = INTER ? 2 * unit.at : unit.at, i1 = INTER ? i0 + 1 : unit.at + pairs;
            const float p = load_f32(unit.x, i0, D), q = load_f32(unit.x, i1, D);
            store_dtype(unit.y, i0, p * w.x - q * w.y, D);
            store_dtype(unit.y, i1, q * w.x + p * w.y, D);
        }
    }
}

template <int D>
int rotary_launch(RotaryArgs a, bool inter, bool vec, bool past, hipStream_t st) {
    constexpr int64_t kMost = 1 << 23;                    // workgroups of a launch, which has fewer than 2^32 lanes
    for (; a.first < a.total; a.first += kMost * a.per) {
        const int64_t left = (a.total - a.first + a.per - 1) / a.per;
        const dim3 grid((unsigned)(left < kMost ? left : kMost));
        auto launch = [&](auto kind, auto far) {
            constexpr bool kInter = decltype(kind)::value, kPast = decltype(far)::value;
            if (vec) rotary_kernel<D, kInter, true, kPast><<<grid, kRotaryThreads, 0, st>>>(a);
            else rotary_kernel<D, kInter, false, false><<<grid, kRotaryThreads, 0, st>>>(a);
        };
        auto by_past = [&](auto kind) { past ? launch(kind, std::true_type{}) : launch(kind, std::false_type{}); };
        inter ? by_past(std::true_type{}) : by_past(std::false_type{});
        const int rc = mq_check_launch("mq_rotary");
        if (rc != MQ_OK) return rc;
    }
    return MQ_OK;
}

}  // namespace mq

extern "C" int mq_rotary(const struct mq_heads* x, int n, int dtype, int64_t batch, int64_t tokens, int64_t dim, const void* positions, int positions64,
                         int64_t position_batch_stride, const void* inv_freq, int freq64, int64_t pairs, int interleaved, double scale, int back, void* stream) {
    using namespace mq;
    if (!x || n < 1 || n > 2 || dtype < MQ_BF16 || dtype > MQ_F32 || batch < 0 || tokens < 0 || dim < 0 || pairs < 0 || 2 * pairs > dim)
        return mq_fail(MQ_ERR_ARG, "mq_rotary: bad argument");
    if (dim > 1024) return mq_fail(MQ_ERR_ARG, "mq_rotary: vectors of at most 1024 elements");
    if (batch && tokens > INT32_MAX / batch) return mq_fail(MQ_ERR_ARG, "mq_rotary: tensor too large");
    int64_t heads = 0;
    for (int w = 0; w < n; w++) {
        if (x[w].heads < 0) return mq_fail(MQ_ERR_ARG, "mq_rotary: bad argument");
        if (x[w].heads > 65535) return mq_fail(MQ_ERR_ARG, "mq_rotary: tensor too large");
        heads += x[w].heads;
    }
    if (batch * tokens * dim * heads == 0) return MQ_OK;
    const int elem = dtype == MQ_F32 ? 4 : 2, v = 16 / elem;
    RotaryArgs a = {};
    bool vec = dim % v == 0 && pairs * (interleaved ? 2 : 1) % v == 0;
    if ((pairs && (!positions || !inv_freq))) return mq_fail(MQ_ERR_ARG, "mq_rotary: null pointer");
    for (int w = 0; w < n; w++) {
        if (x[w].heads && (!x[w].in || !x[w].out)) return mq_fail(MQ_ERR_ARG, "mq_rotary: null pointer");
        a.in[w] = (const char*)x[w].in;
        a.out[w] = (char*)x[w].out;
        a.batch_stride[w] = x[w].batch_stride;
        a.token_stride[w] = x[w].token_stride;
        a.head_stride[w] = x[w].head_stride;
        a.heads[w] = (int)x[w].heads;
        if (x[w].heads)
            vec = vec && ((uintptr_t)x[w].in | (uintptr_t)x[w].out) % 16 == 0 && (batch == 1 || x[w].batch_stride % v == 0) &&
                  (tokens == 1 || x[w].token_stride % v == 0) && (x[w].heads == 1 || x[w].head_stride % v == 0);
    }
    a.position_batch_stride = position_batch_stride;
    a.turn = RotaryTurn{positions, inv_freq, scale, (int)pairs, positions64, freq64, back};
    a.tokens = tokens;
    a.total = batch * tokens;
    a.dim = (int)dim;
    const int64_t units = vec ? (interleaved ? dim / v : (dim - pairs) / v) : dim - pairs;
    if (heads * units > 65535 * (vec ? 1 : 64)) return mq_fail(MQ_ERR_ARG, "mq_rotary: tensor too large");
    // Tokens of a workgroup: enough for all lanes to have an angle to compute and an access or two to make, while there are workgroups for every
    // compute unit (8192 tokens of 9 heads of 64 by eight at once 7.0 us, by one 12.9; of 40 heads of 128 by one or two 58, by four 61, by eight 70).
    int64_t per = 1;
    while (per < kRotaryTokens && per * 2 * pairs <= kRotaryTurns && per * pairs < kRotaryThreads && a.total / (per * 2) >= 1024 &&
           per * 2 * heads * units <= 512)
        per *= 2;
    a.per = (int)per;
    const bool past = a.total * heads * dim * elem >= kPastCaches;
    a.by_token = small_divisor((uint32_t)(heads * units));
    a.by_head = small_divisor((uint32_t)units);
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == MQ_BF16) return rotary_launch<MQ_BF16>(a, interleaved, vec, past, st);
    if (dtype == MQ_F16) return rotary_launch<MQ_F16>(a, interleaved, vec, past, st);
    return rotary_launch<MQ_F32>(a, interleaved, vec, past, st);
}
