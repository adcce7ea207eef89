// Host side shared by the fused attention's entry points: argument checks, the choice of the tile class, the table of
// position biases by distance.
#pragma once
#include <atomic>

#include "attention_tiles.h"
#include "buckets.h"

namespace eeggan {
namespace attn {

// Opt-in to more than 64 KiB of dynamic LDS, once per kernel and device.
struct LdsReady {
    static constexpr int DEVICES = 64;
    std::atomic<bool> done[DEVICES] = {};
    int reserve(const char* what, const void* kernel, size_t bytes) {
        int dev = 0;
        if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= DEVICES) dev = 0;
        if (done[dev].load(std::memory_order_acquire)) return 0;
        const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        EEGGAN_REQUIRE(e == hipSuccess, "%s: cannot reserve %zu bytes of LDS: %s", what, bytes, hipGetErrorString(e));
        done[dev].store(true, std::memory_order_release);
        return 0;
    }
};

constexpr size_t MAX_BAND = 2 * (1024 + 31 * 16 + 31) + 1;  // 2 width + 1 at the widest buckets

// A few query columns per key head: the forward pass lets its waves share them and split the keys.
inline bool few_columns(const eeggan_attention& a) { return (long long)(a.H / a.KV) * a.Tq <= 32 && a.Tk > 64; }

// bfloat16: whether P and dS meet their products in two bf16 pieces (2^-18 of them is left) instead of one (2^-9).
//   * By the pairs of ONE sample (all its heads), so that a sample is rounded alike alone and in any batch.
//   * Up to 16 M of them: in calls of no more pairs than that the second pieces cost nothing that can be measured (8 x 8 heads
//     of 64 channels, 512 steps, 16 M pairs: training 133 us without, 131 with, forward 17 and 17), and they leave the results'
//     own rounding as the largest; in larger batches of such samples they cost up to 10% (1024 steps: 131 and 144 us).
//     Samples beyond have one piece: there the second would cost up to 30% (2048 steps: 387 and 496).  A few columns over
//     many keys are bound by reading those: two pieces up to 1 M pairs (8 samples x 16 heads of 128 over 16384 keys, 0.26 M
//     each: 57 us without, 63 with).
//   * The forward pass also with a table, and for up to 64 keys.  The backward pass takes delta = sum_c dO O for
//     sum_s P dP: with P rounded in O only, the two differ by 2^-9 / sqrt(keys) of dP, and every dS of the row with them.
//     That shows in the table's gradient, where thousands of dS of both signs cancel (0.0028 of its norm, against 3e-4),
//     and in rows of few keys.
inline double sample_pairs(const eeggan_attention& a) { return (double)a.H * a.Tq * a.Tk; }
inline bool fine_backward(const eeggan_attention& a) { return a.bf16 && sample_pairs(a) <= 16777216.0; }
inline bool fine_forward(const eeggan_attention& a) {
    return a.bf16 && (a.table || a.Tk <= 64 || sample_pairs(a) <= (few_columns(a) ? 1048576.0 : 16777216.0));
}

int check_attention(const char* what, const eeggan_attention* a);
// rel table of a call: entries per head, bytes (a multiple of 16), and the launch that fills it (nothing without a bias)
inline long long positions_entries(const eeggan_attention& a) {
    return a.table ? (long long)a.Tq + (long long)a.buckets->step * (a.Tk - 1) : 0;
}
inline size_t positions_bytes(const eeggan_attention& a) {
    return ((size_t)a.H * (size_t)positions_entries(a) * sizeof(float) + 15) / 16 * 16;
}
int positions(const eeggan_attention& a, float* rel, Positions* p, hipStream_t st);
// out[bucket, head] from histograms by distance: hist [H][rows][2 width + 3] (distances -width .. width, behind, ahead)
int bucket_sums(const float* hist, void* out, int out_bf16, const eeggan_buckets& bk, int H, long long rows, int width,
                hipStream_t st);

// The channel counts are rounded up to the first class that holds them; the classes are the layer's own shapes
// (Dk = C / 8, Dv = C / 2 for 64, 128 and 256 channels), equal halves, and what lies between where padding cost most
// (8 x 8 x 1024, forward + queries + keys: 32 + 64 channels in float32 495 us as 64 + 64, 318 in their own class; 96 in
// bfloat16 253 us as 128, 197).  bfloat16 has no eight-channel form: one instruction reduces over sixteen.
#define EEGGAN_ATTENTION_CLASS_T(TYPE, a, ...)                                                            \
    {                                                                                                     \
        typedef TYPE T;                                                                                   \
        if ((a).Dk <= 8 && (a).Dv <= 32) {                                                                \
            constexpr int DK = Elem<T>::NP == 3 ? 8 : 16, DV = 32;                                        \
            __VA_ARGS__;                                                                                  \
        } else if ((a).Dk <= 16 && (a).Dv <= 64) {                                                        \
            constexpr int DK = 16, DV = 64;                                                               \
            __VA_ARGS__;                                                                                  \
        } else if ((a).Dk <= 32 && (a).Dv <= 32) {                                                        \
            constexpr int DK = 32, DV = 32;                                                               \
            __VA_ARGS__;                                                                                  \
        } else if ((a).Dk <= 32 && (a).Dv <= 64) {                                                        \
            constexpr int DK = 32, DV = 64;                                                               \
            __VA_ARGS__;                                                                                  \
        } else if ((a).Dk <= 64 && (a).Dv <= 64) {                                                        \
            constexpr int DK = 64, DV = 64;                                                               \
            __VA_ARGS__;                                                                                  \
        } else if ((a).Dk <= 32) {                                                                        \
            constexpr int DK = 32, DV = 128;                                                              \
            __VA_ARGS__;                                                                                  \
        } else if ((a).Dk <= 96 && (a).Dv <= 96) {                                                        \
            constexpr int DK = 96, DV = 96;                                                               \
            __VA_ARGS__;                                                                                  \
        } else {                                                                                          \
            constexpr int DK = 128, DV = 128;                                                             \
            __VA_ARGS__;                                                                                  \
        }                                                                                                 \
    }
#define EEGGAN_ATTENTION_CLASS(a, ...)                                                                    \
    if ((a).bf16) EEGGAN_ATTENTION_CLASS_T(__bf16, a, __VA_ARGS__) else EEGGAN_ATTENTION_CLASS_T(float, a, __VA_ARGS__)

}  // namespace attn
}  // namespace eeggan
