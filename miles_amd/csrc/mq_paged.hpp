// The paged cache's arithmetic of places, the same on the host and on the device.
#pragma once
#include "mq_api_internal.hpp"

namespace mq {

constexpr int kTile = 32;             // tokens of a wavefront's step

// Whether a page or slot number that came from the device's memory names one of the cache's: everything that is read or written through
// such a number asks this first.
__host__ __device__ inline bool inside(int64_t number, int64_t count) { return number >= 0 && number < count; }

// The tokens that a query sees, [lo, hi), of a sequence of `length` (any number) whose pages hold `capacity`
struct Seen {
    int lo, hi;
};
__host__ __device__ inline Seen seen_of(int64_t length, int64_t capacity, int64_t window) {
    const int64_t hi = length < 0 ? 0 : length < capacity ? length : capacity;
    // (the window counts from the length itself, also where the table ends before it)
    int64_t lo = window > 0 && length > window ? length - window : 0;
    if (lo > hi) lo = hi;
    return Seen{(int)lo, (int)hi};
}
// Steps that cover them, from a multiple of kTile on
__host__ __device__ inline int tiles_of(const Seen& s) { return s.hi > s.lo ? (s.hi + kTile - 1) / kTile - s.lo / kTile : 0; }

// Sixteen tokens of a step, from token `first` on: the page with the number `id` that the table has for them, if there is anything to read there (a page
// of the cache's, a token that is seen, a step that is somebody's), else page 0 and nothing.
struct Half {
    uint32_t page;
    bool some;
};
__host__ __device__ inline Half half_of(uint32_t id, uint32_t pages, int first, const Seen& seen, bool live) {
    const bool some = (int)(id < pages) & (int)(first + 16 > seen.lo) & (int)(first < seen.hi) & (int)live;
    return Half{some ? id : 0u, some};
}
// Bytes that may be read from a half's first place on: to the end of the head's keys (or of anything that lies in units of a place's bytes), and
// the values up to the last token that is seen
__host__ __device__ inline int bytes_to_end(const Half& h, int row, int page_shift, int place, int unit) { return h.some ? (row << page_shift) - place * unit : 0; }
__host__ __device__ inline int bytes_to_last(const Half& h, int row, int first, const Seen& seen) {
    return h.some ? (seen.hi - first < 16 ? seen.hi - first : 16) * row : 0;
}

// false, with the reason said, for a cache that the kernels do not take
bool cache_ok(const mq_paged_cache* c, const char* what);

}  // namespace mq
