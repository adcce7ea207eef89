// Position buckets (eeggan_buckets) on the host and in kernels.
#pragma once
#include "common.h"

namespace eeggan {

inline __host__ __device__ int bucket_side(const eeggan_buckets& b) { return b.bidirectional ? b.count / 2 : b.count; }
// distance from which the bias is constant, on either side
inline __host__ __device__ int bucket_far(const eeggan_buckets& b) {
    const int last = b.edges[bucket_side(b) - 1];
    return last > 1 ? last : 1;
}

// a 32 x 32 tile of pairs with one within `far` holds distances up to this
inline __host__ __device__ int band_width(const eeggan_buckets& b) { return bucket_far(b) + 31 * b.step + 31; }

__device__ __forceinline__ int bucket_of(const eeggan_buckets& b, long long rel) {
    const int side = bucket_side(b);
    long long dist = rel < 0 ? -rel : rel;
    if (!b.bidirectional && rel > 0) dist = 0;
    int j = 0;
    for (int i = 1; i < side; ++i) j += dist >= b.edges[i];
    return j + (b.bidirectional && rel > 0 ? side : 0);
}

inline int check_buckets(const char* what, const eeggan_buckets* b) {
    EEGGAN_REQUIRE(b, "%s: buckets missing", what);
    EEGGAN_REQUIRE(b->count >= 2 && b->count <= 128 && (!b->bidirectional || b->count % 2 == 0),
                   "%s: %d buckets (2 .. 128, even when bidirectional)", what, b->count);
    EEGGAN_REQUIRE(b->bidirectional || b->count <= 64, "%s: %d buckets on one side (at most 64)", what, b->count);
    EEGGAN_REQUIRE(b->step >= 1 && b->step <= 16, "%s: step %d outside 1 .. 16", what, b->step);
    EEGGAN_REQUIRE(b->offset > -(1 << 30) && b->offset < (1 << 30), "%s: offset %d out of range", what, b->offset);
    const int side = bucket_side(*b);
    EEGGAN_REQUIRE(b->edges[0] == 0, "%s: the first bucket must start at distance 0", what);
    for (int i = 1; i < side; ++i)
        EEGGAN_REQUIRE(b->edges[i] > b->edges[i - 1], "%s: bucket edges must increase", what);
    EEGGAN_REQUIRE(b->edges[side - 1] <= 1024, "%s: distances up to 1024 have buckets of their own, got %d", what,
                   b->edges[side - 1]);
    return 0;
}

}  // namespace eeggan
