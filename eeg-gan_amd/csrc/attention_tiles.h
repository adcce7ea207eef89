// Tiles, fragments and products shared by the fused attention kernels (attention_fwd.hip, attention_bwd.hip).
//
// Tensors are channels-first: a head's queries are a [Dk, Tq] matrix with time contiguous, keys [Dk, Tk], values
// [Dv, Tk].  All products run on v_mfma_f32_32x32x16_bf16 (operand A: row = lane & 31, eight reduction indices per
// lane half; result: column = lane & 31, row = (r & 3) + 8 (r >> 2) + 4 (lane >> 5)).  Float32 tensors are multiplied
// through three bf16 pieces per operand (v = p1 + p2 + p3 up to 2^-24 |v|, the six products down to 2^-16 of the
// leading one: the rounding of an fp32 product); bfloat16 tensors directly.
//
// A streamed operand lies in LDS as it lies in memory, channels in rows, and two products alternate on it:
//   * scores-like, rows x = a time axis, reduction over channels: read with the transposing LDS loads (16 lanes give the
//     addresses of four rows' neighbouring values, each lane gets one column of the block), the other operand stationary
//     in registers (SFrag);
//   * values-like, rows = channels, reduction over the time axis x: read as it lies, and the other operand is the result
//     registers of the first product as they are: lane half h holds rows x = 16 kk + 8 a + 4 h + c (kk, a in {0, 1}, c <
//     4) in registers 8 kk + 4 a + c, so a row stores x at position 16 kk + 8 h + 4 a + c and one 16-byte read yields the
//     matching operand.
// (A second, transposed copy of the tiles took a third of the backward kernels' time to write.)
#pragma once
#include "common.h"

namespace eeggan {
namespace attn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2u __attribute__((ext_vector_type(2), aligned(2)));  // four bfloat16 from any address

constexpr int THREADS = 256;
constexpr float LOG2E = 1.44269504088896340736f;

template <class T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int NP = 3;  // bf16 pieces per operand
    typedef f32x4 raw4;
};
template <>
struct Elem<__bf16> {
    static constexpr int NP = 1;
    typedef u32x2 raw4;
};

__device__ __forceinline__ f32x4 load4(const float* p) { return *reinterpret_cast<const f32x4u*>(p); }
__device__ __forceinline__ u32x2 load4(const __bf16* p) {
    const u32x2u v = *reinterpret_cast<const u32x2u*>(p);
    u32x2 o;
    o[0] = v[0];
    o[1] = v[1];
    return o;
}
__device__ __forceinline__ f32x4 gather4(const float* p, int i0, int i1, int i2, int i3) {
    const f32x4 v = {p[i0], p[i1], p[i2], p[i3]};
    return v;
}
__device__ __forceinline__ u32x2 gather4(const __bf16* q, int i0, int i1, int i2, int i3) {
    const unsigned short* p = reinterpret_cast<const unsigned short*>(q);
    const unsigned a = p[i0], b = p[i1], c = p[i2], d = p[i3];
    const u32x2 v = {a | b << 16, c | d << 16};
    return v;
}

__device__ __forceinline__ unsigned pack2(float a, float b) {
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    const f32x2_t v = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2_t));
}
__device__ __forceinline__ float lo_f(unsigned w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float hi_f(unsigned w) { return __builtin_bit_cast(float, w & 0xffff0000u); }

// The operand words of two neighbouring values: NP = 1 rounds to bfloat16, NP = 3 splits exactly (each remainder is
// formed exactly in float32; the third piece is rounded at 2^-24 of the value).
template <int NP>
__device__ __forceinline__ void pieces2(float a, float b, unsigned (&w)[NP]) {
    w[0] = pack2(a, b);
    if constexpr (NP == 3) {
        const float ra = a - lo_f(w[0]), rb = b - hi_f(w[0]);
        w[1] = pack2(ra, rb);
        w[2] = pack2(ra - lo_f(w[1]), rb - hi_f(w[1]));
    }
}

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bf16x8 lds8(const char* p) { return *reinterpret_cast<const bf16x8*>(p); }
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// The two lane halves' values combined: one exchange of register halves, no trip through LDS.  (The second operand is
// hidden from the compiler: given the same value twice, it takes both results for one.)
__device__ __forceinline__ void halves(float v, float& lo, float& hi) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    unsigned w = u;
    asm("" : "+v"(w));
    const auto r = __builtin_amdgcn_permlane32_swap(u, w, false, false);
    const unsigned a = r[0], b = r[1];
    lo = __builtin_bit_cast(float, a);
    hi = __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float half_max(float v) {
    float lo, hi;
    halves(v, lo, hi);
    return fmaxf(lo, hi);
}
__device__ __forceinline__ float half_sum(float v) {
    float lo, hi;
    halves(v, lo, hi);
    return lo + hi;
}

// ---- tiles --------------------------------------------------------------------------------------------------
// Eight channels in three pieces: the pieces share the reduction axis (see SFrag), one row holds all of them.
template <int NP, int D>
constexpr bool packed8() { return NP == 3 && D == 8; }

// Row strides are odd multiples of 16 bytes: the 16-byte reads of 32 consecutive rows spread over all banks.
template <int NP, int D, int XT>
struct Tile {
    static constexpr bool P8 = packed8<NP, D>();
    static constexpr int RS = 2 * XT + 16;
    static constexpr int ROWS = D < 32 ? 32 : D;  // the values-like products read whole groups of 32 rows
    static constexpr int PIECE = P8 ? 8 * RS : ROWS * RS;
    static constexpr int BYTES = P8 ? 32 * RS : NP * ROWS * RS;
    static constexpr int GROUPS = D < 32 ? 1 : D / 32;
};
// byte offset of time index x (a multiple of 4) in a row
__device__ __forceinline__ int n_off(int x) { return 2 * ((x & ~31) + (x & 16) + ((x & 4) << 1) + ((x & 8) >> 1)); }

// Which steps of a stage count, one bit each (the same in every lane).
template <int XT>
struct Steps {
    static_assert(XT <= 64, "one word");
    unsigned long long w;
    // steps [x0, x0 + XT) of `len`, less the masked ones: `raw` is what StepsAhead read for them
    __device__ __forceinline__ void find(int x0, int len, unsigned char raw, int lane) {
        w = __ballot(lane < XT && x0 + lane < len && raw != 0);
    }
    __device__ __forceinline__ bool all() const { return w == ~0ull >> (64 - XT); }
    __device__ __forceinline__ unsigned tile(int x0) const { return (unsigned)(w >> x0); }            // the 32 steps from x0
    __device__ __forceinline__ unsigned quad(int kq) const { return (unsigned)(w >> (4 * kq)) & 15u; }  // the four from 4 kq
};

// The mask bytes of a stage on their way: read with the stage's data and looked at only when that is stored (a vote right
// behind the loads would wait for all of them).
template <int XT>
struct StepsAhead {
    unsigned char raw;
    int x0;
    // mask: nonzero bytes count; null: all
    __device__ __forceinline__ void load(int first, int len, const unsigned char* mask, int lane) {
        x0 = first;
        raw = mask ? mask[min(first + lane, len - 1)] : 1;
    }
};

// The attended keys of [begin, end) lie in the range this leaves (end <= begin: none); all threads, ends in a barrier.
__device__ __forceinline__ void attended_range(const unsigned char* mask, int& begin, int& end, int* lds) {
    int lo = end, hi = begin;
    for (int x = begin + (int)threadIdx.x; x < end; x += THREADS)
        if (mask[x]) {
            lo = min(lo, x);
            hi = x + 1;
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        lo = min(lo, __shfl_xor(lo, o, 64));
        hi = max(hi, __shfl_xor(hi, o, 64));
    }
    if ((threadIdx.x & 63) == 0) {
        lds[2 * (threadIdx.x >> 6)] = lo;
        lds[2 * (threadIdx.x >> 6) + 1] = hi;
    }
    __syncthreads();
    begin = __builtin_amdgcn_readfirstlane(min(min(lds[0], lds[2]), min(lds[4], lds[6])));
    end = __builtin_amdgcn_readfirstlane(max(max(lds[1], lds[3]), max(lds[5], lds[7])));
    __syncthreads();
}

// A [D, XT] block of a channels-first matrix on its way from memory into LDS: 4 x 4 units (four channels, four time
// steps), neighbouring threads on neighbouring steps.  Loads never branch per value
// (the compiler would wait at every join): whatever lies past the matrix is read at its last row or step.  Such values and
// those of masked steps become zeros on their way into LDS, so what they hold (NaN included) never meets a product.
template <class T, int D, int XT>
struct Block {
    static constexpr int NP = Elem<T>::NP;
    static constexpr int XQ = XT / 4, DB = D / 4, UNITS = DB * XQ, U = (UNITS + THREADS - 1) / THREADS;
    typename Elem<T>::raw4 r[U][4];
    unsigned off[U][4];  // byte offsets of the unit's rows from (channel 0, first step of the stage)

    static __device__ __forceinline__ int unit_kq(int unit) { return unit % XQ; }
    static __device__ __forceinline__ int unit_db(int unit) { return unit / XQ; }

    // stride (channels, in elements) times 128 fits 32 bits in bytes: checked on the host
    __device__ __forceinline__ void init(long long stride, int channels, int tid) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int unit = tid + THREADS * u;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                off[u][i] = (unsigned)((min(4 * unit_db(unit) + i, channels - 1) * (unsigned)stride + 4 * unit_kq(unit)) * sizeof(T));
        }
    }

    // base: channel 0, step 0 of the head; steps [x0, x0 + XT) of `len`
    __device__ __forceinline__ void load(const T* base, int x0, int len, int tid) {
        if (x0 + XT <= len) {
            const char* p = reinterpret_cast<const char*>(base + x0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (UNITS % THREADS != 0 && tid + THREADS * u >= UNITS) continue;
#pragma unroll
                for (int i = 0; i < 4; ++i) r[u][i] = load4(reinterpret_cast<const T*>(p + off[u][i]));
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int unit = tid + THREADS * u;
                if (UNITS % THREADS != 0 && unit >= UNITS) continue;
                const int kq = unit_kq(unit), x = x0 + 4 * kq, last = len - 1;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    r[u][i] = gather4(reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + off[u][i]) - 4 * kq,
                                      min(x, last), min(x + 1, last), min(x + 2, last), min(x + 3, last));
            }
        }
    }

    // into the tile; steps: which count
    __device__ __forceinline__ void store(char* tile, int channels, const Steps<XT>& steps, int tid) {
        typedef Tile<NP, D, XT> TL;
        const bool clean = steps.all() && channels == D;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int unit = tid + THREADS * u;
            if (UNITS % THREADS != 0 && unit >= UNITS) continue;
            const int kq = unit_kq(unit), db = unit_db(unit);
            if (!clean) {
                const unsigned keep = steps.quad(kq);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned k = 4 * db + i < channels ? keep : 0u;
                    if constexpr (NP == 3) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) r[u][i][e] = (k >> e) & 1u ? r[u][i][e] : 0.f;
                    } else {
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            r[u][i][e] &= ((k >> (2 * e)) & 1u ? 0xffffu : 0u) | ((k >> (2 * e + 1)) & 1u ? 0xffff0000u : 0u);
                    }
                }
            }
            unsigned w[4][2][NP];  // [channel][pair of steps][piece]
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (NP == 3) {
                    pieces2<NP>(r[u][i][0], r[u][i][1], w[i][0]);
                    pieces2<NP>(r[u][i][2], r[u][i][3], w[i][1]);
                } else {
                    w[i][0][0] = r[u][i][0];
                    w[i][1][0] = r[u][i][1];
                }
            }
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                char* row = tile + p * TL::PIECE + (4 * db) * TL::RS + n_off(4 * kq);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const u32x2 o = {w[i][0][p], w[i][1][p]};
                    *reinterpret_cast<u32x2*>(row + i * TL::RS) = o;
                }
            }
        }
    }
};

template <int N, class F, int I = 0>
__device__ __forceinline__ void static_unroll(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_unroll<N, F, I + 1>(static_cast<F&&>(f));
    }
}

// ---- fragments ----------------------------------------------------------------------------------------------
// The stationary operand of a scores-like product: this lane's column (one time step) of a [D, T] matrix.  Eight
// channels in three pieces: two pieces of a term fill the sixteen reduction indices of one instruction, so the six
// products take three instructions and two fragments.
template <int NP, int D>
struct SFrag {
    static constexpr int N = packed8<NP, D>() ? 2 : NP * D / 16;
    bf16x8 f[N];

    static constexpr int VALUES = packed8<NP, D>() ? 8 : D / 2;  // channels of a lane (half)
    static __device__ __forceinline__ int channel(int i, int h) {
        return packed8<NP, D>() ? i : 16 * (i / 8) + 8 * h + i % 8;
    }
    // the lane's channels of column `at` of p, values [FIRST, FIRST + N) of them; past the matrix the last channel again, to be
    // zeroed.  (The rows' offsets are scalars, a lane picks its half's: two instructions a load.)
    template <int FIRST = 0, int N = VALUES, class T>
    static __device__ __forceinline__ void read(const T* p, unsigned at, long long stride, int channels, int h, float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const unsigned o0 = min(channel(FIRST + i, 0), channels - 1) * (unsigned)stride;
            const unsigned o1 = min(channel(FIRST + i, 1), channels - 1) * (unsigned)stride;
            v[i] = ld1(reinterpret_cast<const T*>(reinterpret_cast<const char*>(p) + (size_t)(unsigned)((at + (h ? o1 : o0)) * sizeof(T))));
        }
    }
    // v: the (already scaled) values, zero past the matrix
    __device__ __forceinline__ void fill(int h, const float (&v)[VALUES]) {
        if constexpr (packed8<NP, D>()) {
            u32x4 w0, w1, w2;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                unsigned w[3];
                pieces2<3>(v[2 * i], v[2 * i + 1], w);
                w0[i] = w[0];
                w1[i] = w[1];
                w2[i] = w[2];
            }
            f[0] = __builtin_bit_cast(bf16x8, h ? w1 : w0);
            f[1] = __builtin_bit_cast(bf16x8, h ? w0 : w2);
        } else {
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                u32x4 ws[NP];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    unsigned w[NP];
                    pieces2<NP>(v[8 * j + 2 * i], v[8 * j + 2 * i + 1], w);
#pragma unroll
                    for (int p = 0; p < NP; ++p) ws[p][i] = w[p];
                }
#pragma unroll
                for (int p = 0; p < NP; ++p) f[p * (D / 16) + j] = __builtin_bit_cast(bf16x8, ws[p]);
            }
        }
    }
};

// Eight channels of one step per lane, out of rows of neighbouring steps: lane s of a group of sixteen gives the address of
// four steps (quad s % 4) of channel s / 4, and lane i receives step i of the four channels.
__device__ __forceinline__ bf16x8 lds8_transposed(const char* p, int four_rows) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + four_rows));
    const s16x8 v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return __builtin_bit_cast(bf16x8, v);
}
// The operands of a scores-like product for 32 steps (rows of the result) from `tile` (+ 2 * first step).
template <int NP, int D, int XT>
struct SRead {
    static constexpr int N = packed8<NP, D>() ? 3 : NP * D / 16;
    typedef Tile<NP, D, XT> TL;
    bf16x8 a[N];
    // this lane's address in a tile
    static __device__ __forceinline__ int offset(int lane) {
        const int s = lane & 15, h = lane >> 5;
        return ((s >> 2) + (TL::P8 ? 0 : 8 * h)) * TL::RS + n_off(4 * (4 * ((lane >> 4) & 1) + (s & 3)));
    }
    // p: tile + 2 * first step + offset(lane)
    __device__ __forceinline__ void load(const char* p, int h) {
        if constexpr (TL::P8) {
            a[0] = lds8_transposed(p + (h ? 2 * TL::PIECE : 0), 4 * TL::RS);
            a[1] = lds8_transposed(p + TL::PIECE, 4 * TL::RS);
            a[2] = lds8_transposed(p, 4 * TL::RS);
        } else {
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
#pragma unroll
                for (int q = 0; q < NP; ++q)
                    a[NP * j + q] = lds8_transposed(p + 16 * j * TL::RS + q * TL::PIECE, 4 * TL::RS);
        }
    }
    // acc[b][x, column] += sum_d tile[x, d] frag[b][d, column] for CB column blocks: every operand serves all of them
    template <int CB>
    __device__ __forceinline__ void mma(const SFrag<NP, D> (&s)[CB], f32x16 (&acc)[CB]) const {
        if constexpr (TL::P8) {
#pragma unroll
            for (int b = 0; b < CB; ++b) acc[b] = mfma(a[0], s[b].f[1], acc[b]);  // p1 q3 | p3 q1
#pragma unroll
            for (int b = 0; b < CB; ++b) acc[b] = mfma(a[1], s[b].f[0], acc[b]);  // p2 q1 | p2 q2
#pragma unroll
            for (int b = 0; b < CB; ++b) acc[b] = mfma(a[2], s[b].f[0], acc[b]);  // p1 q1 | p1 q2
        } else {
            constexpr int J = D / 16;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                if constexpr (NP == 3) {
                    const bf16x8 &a0 = a[3 * j], &a1 = a[3 * j + 1], &a2 = a[3 * j + 2];
#pragma unroll
                    for (int b = 0; b < CB; ++b) acc[b] = mfma(a2, s[b].f[j], acc[b]);
#pragma unroll
                    for (int b = 0; b < CB; ++b) acc[b] = mfma(a0, s[b].f[2 * J + j], acc[b]);
#pragma unroll
                    for (int b = 0; b < CB; ++b) acc[b] = mfma(a1, s[b].f[J + j], acc[b]);
#pragma unroll
                    for (int b = 0; b < CB; ++b) acc[b] = mfma(a1, s[b].f[j], acc[b]);
#pragma unroll
                    for (int b = 0; b < CB; ++b) acc[b] = mfma(a0, s[b].f[J + j], acc[b]);
                }
#pragma unroll
                for (int b = 0; b < CB; ++b) acc[b] = mfma(a[NP * j], s[b].f[j], acc[b]);
            }
        }
    }
};
// Whether a tile's operands are all read before the first product: up to this many for one product, for scores and dP together
// (the compiler reads each one right before its product and waits for it; past that the registers do not hold them).
constexpr int READ_AHEAD = 6, READ_AHEAD_TWO = 9;

template <int NP, int D, int XT, int CB>
__device__ __forceinline__ void mma_scores(const char* p, int h, const SFrag<NP, D> (&s)[CB], f32x16 (&acc)[CB]) {
    SRead<NP, D, XT> r;
    r.load(p, h);
    if constexpr (SRead<NP, D, XT>::N <= READ_AHEAD) __builtin_amdgcn_sched_barrier(0);
    r.template mma<CB>(s, acc);
}
// scores and dP of a tile
template <int NP, int DK, int DV, int XT>
__device__ __forceinline__ void two_scores(const char* k, const SFrag<NP, DK> (&fk)[1], f32x16 (&s)[1], const char* v,
                                           const SFrag<NP, DV> (&fv)[1], f32x16 (&dp)[1], int h) {
    if constexpr (SRead<NP, DK, XT>::N + SRead<NP, DV, XT>::N <= READ_AHEAD_TWO) {
        SRead<NP, DK, XT> rk;
        SRead<NP, DV, XT> rv;
        rk.load(k, h);
        rv.load(v, h);
        __builtin_amdgcn_sched_barrier(0);
        rk.template mma<1>(fk, s);
        rv.template mma<1>(fv, dp);
    } else {
        mma_scores<NP, DK, XT, 1>(k, h, fk, s);
        mma_scores<NP, DV, XT, 1>(v, h, fv, dp);
    }
}

// The result registers of a scores-like product as the operand of a values-like one.
template <int NP>
struct PFrag {
    bf16x8 f[2][NP];  // [kk][piece]
    __device__ __forceinline__ void fill(const f32x16& v) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            u32x4 ws[NP];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                unsigned w[NP];
                pieces2<NP>(v[8 * kk + 2 * i], v[8 * kk + 2 * i + 1], w);
#pragma unroll
                for (int p = 0; p < NP; ++p) ws[p][i] = w[p];
            }
#pragma unroll
            for (int p = 0; p < NP; ++p) f[kk][p] = __builtin_bit_cast(bf16x8, ws[p]);
        }
    }
    // what fill() rounded away (NP = 1), rounded in turn: 2^-18 of the values is left
    __device__ __forceinline__ void fill_rest(const f32x16& v) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            u32x4 ws;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = v[8 * kk + 2 * i], y = v[8 * kk + 2 * i + 1];
                const unsigned w = pack2(x, y);
                ws[i] = pack2(x - lo_f(w), y - hi_f(w));
            }
            f[kk][0] = __builtin_bit_cast(bf16x8, ws);
        }
    }
};

// acc[b][g][row, column] += sum_x tile[32 g + row, x] frag[b][x, column] over the 32 steps from x0.
// Eight rows in three pieces: the pieces lie one after the other in the rows of ONE instruction (rows 8 p + d), three
// instructions instead of six; eight_rows() sums the pieces' results.
template <int NP, int D, int XT, int CB>
__device__ __forceinline__ void mma_values(const char* tile, int x0, int l31, int h, const PFrag<NP> (&f)[CB],
                                           f32x16 (&acc)[CB][Tile<NP, D, XT>::GROUPS]) {
    typedef Tile<NP, D, XT> NL;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
        for (int g = 0; g < NL::GROUPS; ++g) {
            const char* row = tile + (32 * g + l31) * NL::RS + 2 * x0 + 16 * h + 32 * kk;
            const bf16x8 a0 = lds8(row);
            bf16x8 a1 = a0, a2 = a0;
            if constexpr (NP == 3 && !NL::P8) {
                a1 = lds8(row + NL::PIECE);
                a2 = lds8(row + 2 * NL::PIECE);
            }
#pragma unroll
            for (int b = 0; b < CB; ++b) {
                f32x16 c = acc[b][g];
                if constexpr (NL::P8) {
                    c = mfma(a0, f[b].f[kk][2], c);
                    c = mfma(a0, f[b].f[kk][1], c);
                } else if constexpr (NP == 3) {
                    c = mfma(a2, f[b].f[kk][0], c);
                    c = mfma(a0, f[b].f[kk][2], c);
                    c = mfma(a1, f[b].f[kk][1], c);
                    c = mfma(a1, f[b].f[kk][0], c);
                    c = mfma(a0, f[b].f[kk][1], c);
                }
                acc[b][g] = mfma(a0, f[b].f[kk][0], c);
            }
        }
    }
}
// channel of result register r (of group 0) and whether the register holds one
template <int NP, int D>
__device__ __forceinline__ void eight_rows(f32x16& a) {
    if constexpr (packed8<NP, D>()) {
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = (a[8 + i] + a[4 + i]) + a[i];
    }
}
__device__ __forceinline__ int acc_row(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }

// Workgroup -> (head, part of it).  Workgroups are dealt to the eight XCDs in turn, each with an L2 of its own: the parts
// of a head go to one of them, so that what its parts share (keys and values, or queries) is read into one L2.
__device__ __forceinline__ void place(int blk, int heads, int parts, int& head, int& part) {
    const int spread = heads / 8 * 8 * parts;
    if (blk < spread) {
        const int i = blk >> 3;
        head = (blk & 7) + 8 * (i / parts);
        part = i % parts;
    } else {
        head = blk / parts;
        part = blk - head * parts;
    }
}

// ---- positions ----------------------------------------------------------------------------------------------
// Key s lies at position step * s + offset, query t at position t; the bias of the pair depends on their difference
// through its bucket, and is constant from `far` on, on either side.  rel[head][step * s + (Tq - 1) - t] holds it times
// log2(e) (attn_positions_kernel); -inf bars a pair.
struct Positions {
    const float* rel;  // null: no bias
    int nrel;          // entries per head
    int step, offset, far;
    int width;  // near tiles hold distances -width .. width: far + 31 step + 31
};

// -1 / +1: every pair of the 32 x 32 tile lies beyond `far` on that side; 0: near.  s: first key, t: first query.
__device__ __forceinline__ int tile_side(const Positions& p, int s, int t) {
    const long long base = (long long)p.step * s + p.offset - t;
    const long long lo = base - 31, hi = base + 31 * p.step;
    return lo >= p.far ? 1 : hi <= -p.far ? -1 : 0;
}
// entry of a head's table for a distance (clamped: a value past the table belongs to no pair)
__device__ __forceinline__ float rel_at(const Positions& p, const float* head, int tq, long long distance) {
    const long long i = distance - p.offset + (tq - 1);
    return head[i < 0 ? 0 : i >= p.nrel ? p.nrel - 1 : i];
}
// The near distances' values in LDS (2 width + 1 floats): read from memory inside the loop over the tiles they cost a
// trip to the L2 per tile, which nothing hides at two waves per SIMD.
__device__ __forceinline__ void fill_band(float* band, const Positions& p, const float* head, int tq, int first, int stride) {
    for (int i = first; i <= 2 * p.width; i += stride) band[i] = rel_at(p, head, tq, i - p.width);
}

}  // namespace attn
}  // namespace eeggan
