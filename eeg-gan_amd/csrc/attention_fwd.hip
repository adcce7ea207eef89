// Attention over time, channels first, without storing the probabilities:
//   S[s, t] = scale * sum_d K[d, s] Q[d, t] (+ the position bias of (s, t));  O[c, t] = sum_s V[c, s] softmax_s(S)[s, t]
// One pass over the keys per query column with a running reference m and sum l (P' = 2^(S log2e - m), O = sum V P' / l);
// what the backward pass needs besides its inputs and the output are two numbers per query, m and log2 l (as their sum, log2 l
// would be rounded at the magnitude of m, which is that of the position bias).
//
// A wave owns 32 query columns; the head's keys pass through LDS in stages shared by the workgroup's four waves.
// A lane holds one query's column of S, so the statistics are per-lane scalars: the maximum over its sixteen
// registers and one exchange between the lane halves, the sum without any exchange until the end.  The reference m
// moves only when a score exceeds it by 8 (a factor 256: the sums stay far inside float32's range and lose
// nothing), which after the first stages is rare, so the accumulators are hardly ever rescaled.  Where it moves far (scores
// of -10^4 or -10^9 from a position bias, then ordinary ones), the tile's scores are formed again against the new one: on
// top of the old one they were rounded at the distance's magnitude.
// Few query columns (a single new step): the waves share the columns and split each stage's keys (KW > 1), and the keys
// are split over workgroups; every part leaves (O unscaled, m, l) and attn_join_kernel combines them in a fixed order.
//
// Measured (calls one after the other): bfloat16, 8 samples x 8 heads of 64 channels over 2048 steps 107 us = 642 TFLOP/s (a
// large library product: 1330).  What bounds it: products, exponentials with their sums, and the tiles' way through LDS
// share a wave's issue slots, and two waves per SIMD do not overlap them fully (the exponentials left out save 20 us, the
// staging 35, the products 45).  Float32 (six products each, three pieces of P formed per pair): 8 x 8 x 1024 at 64 channels
// 106 us = 162 TFLOP/s, the rate of a large float32 library product.  One step over 16384 keys (8 x 4 key heads of 128,
// bfloat16, P in two pieces): 51 us = 5.3 TB/s, all of it reading keys and values.
#include "attention_host.h"

namespace eeggan {
namespace attn {

struct FwdArgs {
    const void *q, *k, *v;
    long long qsb, qsc, ksb, ksc, vsb, vsc;  // strides between samples and channels, in elements
    const unsigned char* mask;               // [B, Tk], nonzero = attended; null: all
    void* out;                               // [B, H Dv, Tq]
    void* rest;                              // what the rounding of out left over (bfloat16); null: not wanted
    float* lse;                              // [2, B, H, Tq]: m, log2 l; null: not wanted
    float* part;                             // parts of a split: O, then m, then l; null: not split
    Positions pos;
    int B, KV, G, Dk, Dv, Tq, Tk;
    int coltiles, nsplit, split_keys;
    float scale;
    bool fine;  // bfloat16: P meets V in two pieces (fine_forward)
};

// KW waves share the columns and split a stage's keys; CB: column blocks of a wave (its LDS operands serve all of them).
template <class T, int DK, int DV, int XT>
struct FwdCut {
    static constexpr int NP = Elem<T>::NP;
    static constexpr int STAGE = Tile<NP, DK, XT>::BYTES + Tile<NP, DV, XT>::BYTES;
    static constexpr int BUFS = 2 * STAGE <= 80 * 1024 ? 2 : 1;  // (two workgroups to a CU)
    static constexpr int LDS = BUFS * STAGE;
};
// A move of the reference by more than this has the tile's scores formed again: up to it they are rounded at 2^-16 at most.
// (Moves up by more than 150 leave nothing of the sums so far: 2^-256 of them is zero.)
constexpr float FAR_MOVE = 256.f;
// FINE: has the code for a.fine (where it is not taken its registers cost few columns 10%)
template <class T, int DK, int DV, int KW, int XT, int CB, bool BIAS, bool FINE>
__global__ __launch_bounds__(THREADS, 2) void attn_fwd_kernel(FwdArgs a) {
    typedef FwdCut<T, DK, DV, XT> Cut;
    constexpr int NP = Elem<T>::NP;
    constexpr int WC = 4 / KW;                  // waves along the columns
    constexpr int SUBS = XT / (32 * KW);        // key tiles a wave takes of a stage
    constexpr int J = CB == 1 && SUBS % 2 == 0 ? 2 : 1;  // ... of them at once: independent chains to overlap
    typedef Tile<NP, DK, XT> KT;
    typedef Tile<NP, DV, XT> VT;
    typedef SRead<NP, DK, XT> KR;
    extern __shared__ __attribute__((aligned(16))) char smem[];

    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ksub = wave % KW;
    int bkv, part;
    place(blockIdx.x, a.B * a.KV, a.coltiles * a.nsplit, bkv, part);
    const int tile = part % a.coltiles, split = part / a.coltiles;
    const int b = bkv / a.KV, kvh = bkv - b * a.KV;

    const int ncols = a.G * a.Tq;
    const int col0 = (tile * WC + wave / KW) * 32 * CB;
    const int k_off = KR::offset(lane);
    const float c = a.scale * LOG2E;
    // per column block: its lane's query and head
    bool live[CB];
    int t[CB], head[CB];
    SFrag<NP, DK> fq[CB];
    // position bias: beyond the last edge (behind, ahead) one value per lane; near tiles read band[distance + width] in LDS,
    // or, where the block's columns belong to several heads (which never count as far), rel[step * s] in memory
    float beyond[CB][2];
    const float* rel[CB];
    bool one_head[CB];
    float* const bands = reinterpret_cast<float*>(smem + Cut::LDS) + wave * CB * (2 * a.pos.width + 1);
#pragma unroll
    for (int i = 0; i < CB; ++i) {
        const int n0 = col0 + 32 * i, n = n0 + l31;
        live[i] = n < ncols;
        const int g = live[i] ? n / a.Tq : 0;
        t[i] = live[i] ? n - g * a.Tq : 0;
        head[i] = kvh * a.G + g;
        const T* q = reinterpret_cast<const T*>(a.q) + b * a.qsb + (long long)head[i] * a.Dk * a.qsc + t[i];
        // (float32: the scale goes into the split operand; bfloat16 operands stay exact and the scores are scaled)
        typedef SFrag<NP, DK> F;
        float x[F::VALUES];
        F::read(q, 0u, a.qsc, a.Dk, h, x);
#pragma unroll
        for (int e = 0; e < F::VALUES; ++e)
            x[e] = live[i] && F::channel(e, h) < a.Dk ? (NP == 3 ? x[e] * c : x[e]) : 0.f;
        fq[i].fill(h, x);
        if constexpr (BIAS) {
            const float* const mine = a.pos.rel + (long long)head[i] * a.pos.nrel;
            rel[i] = mine + (a.Tq - 1 - t[i]);
            one_head[i] = n0 < ncols && n0 / a.Tq == min(n0 + 31, ncols - 1) / a.Tq;
            beyond[i][0] = rel_at(a.pos, mine, a.Tq, -a.pos.far);
            beyond[i][1] = rel_at(a.pos, mine, a.Tq, a.pos.far);
            if (one_head[i])  // (the whole wave is of one head: lane 0's)
                fill_band(bands + i * (2 * a.pos.width + 1), a.pos,
                          a.pos.rel + (long long)(kvh * a.G + n0 / a.Tq) * a.pos.nrel, a.Tq, lane, 64);
        }
    }
    const T* const kb = reinterpret_cast<const T*>(a.k) + b * a.ksb + (long long)kvh * a.Dk * a.ksc;
    const T* const vb = reinterpret_cast<const T*>(a.v) + b * a.vsb + (long long)kvh * a.Dv * a.vsc;
    const unsigned char* const mask = a.mask ? a.mask + (long long)b * a.Tk : nullptr;

    int s_begin = split * a.split_keys;
    int s_end = min(a.Tk, s_begin + a.split_keys);
    if (mask && s_begin < s_end) attended_range(mask, s_begin, s_end, reinterpret_cast<int*>(smem));

    float m[CB], l[CB], threshold[CB];  // threshold -inf: no key seen yet
    f32x16 o[CB][VT::GROUPS];
#pragma unroll
    for (int i = 0; i < CB; ++i) {
        m[i] = l[i] = 0.f;
        threshold[i] = -INFINITY;
#pragma unroll
        for (int e = 0; e < VT::GROUPS; ++e) o[i][e] = zero16();
    }

    Block<T, DK, XT> kblk;
    Block<T, DV, XT> vblk;
    kblk.init(a.ksc, a.Dk, tid);
    vblk.init(a.vsc, a.Dv, tid);
    StepsAhead<XT> ahead;
    Steps<XT> now, next;  // which keys of the stage are attended
    auto fetch = [&](int s0) {
        ahead.load(s0, s_end, mask, lane);
        kblk.load(kb, s0, s_end, tid);
        vblk.load(vb, s0, s_end, tid);
    };
    auto put = [&](int buf) {
        char* const kt = smem + buf * Cut::STAGE;
        next.find(ahead.x0, s_end, ahead.raw, lane);
        kblk.store(kt, a.Dk, next, tid);
        vblk.store(kt + KT::BYTES, a.Dv, next, tid);
    };
    int buf = 0;
    if (s_begin < s_end) {
        fetch(s_begin);
        put(0);
        now = next;
        if (s_begin + XT < s_end) fetch(s_begin + XT);
        __syncthreads();
    }
    for (int s0 = s_begin; s0 < s_end; s0 += XT) {
        // two buffers: the next stage goes into the other one before this one is worked on
        if (Cut::BUFS == 2 && s0 + XT < s_end) {
            put(buf ^ 1);
            if (s0 + 2 * XT < s_end) fetch(s0 + 2 * XT);
        }
        const char* const kt = smem + buf * Cut::STAGE;
        const char* const vt = kt + KT::BYTES;
#pragma unroll
        for (int u = 0; u < SUBS; u += J) {
            unsigned word[J], any = 0;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                word[j] = now.tile(32 * (KW == 1 ? u + j : ksub));
                any |= word[j];
            }
            if (any == 0 || col0 >= ncols) continue;  // (the same for every lane of the wave)
            f32x16 acc[J][CB];
            auto form = [&](bool first) __attribute__((always_inline)) {
                int at = s0;
                if constexpr (BIAS) asm volatile("" : "+s"(at));  // (or the loop below keeps every address in registers)
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const int x0 = 32 * (KW == 1 ? u + j : ksub);
#pragma unroll
                    for (int i = 0; i < CB; ++i) acc[j][i] = zero16();
                    mma_scores<NP, DK, XT, CB>(kt + 2 * x0 + k_off, h, fq, acc[j]);
                }
                bool again = false;
#pragma unroll
                for (int i = 0; i < CB; ++i) {
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        const int x0 = 32 * (KW == 1 ? u + j : ksub);
                        if constexpr (BIAS) {
                            const int s = at + x0, n0 = col0 + 32 * i, t0 = n0 % a.Tq;
                            const int side = one_head[i] ? tile_side(a.pos, s, t0) : 0;
                            if (side != 0) {
                                const float base = (side < 0 ? beyond[i][0] : beyond[i][1]) - m[i];
#pragma unroll
                                for (int r = 0; r < 16; ++r)
                                    acc[j][i][r] = __builtin_fmaf(acc[j][i][r], NP == 3 ? 1.f : c, base);
                            } else if (one_head[i]) {
                                const float* const r0 = bands + i * (2 * a.pos.width + 1) +
                                                        (int)((long long)a.pos.step * s + a.pos.offset - t0 + a.pos.width) +
                                                        a.pos.step * 4 * h - l31;
#pragma unroll
                                for (int r = 0; r < 16; ++r)
                                    acc[j][i][r] = __builtin_fmaf(acc[j][i][r], NP == 3 ? 1.f : c,
                                                                  r0[a.pos.step * ((r & 3) + 8 * (r >> 2))] - m[i]);
                            } else {
                                const int first = min(s + 4 * h, a.Tk - 1), last = a.Tk - 1 - first;
                                const float* r0 = rel[i] + (long long)a.pos.step * first;
#pragma unroll
                                for (int r = 0; r < 16; ++r)
                                    acc[j][i][r] = __builtin_fmaf(acc[j][i][r], NP == 3 ? 1.f : c,
                                                                  r0[a.pos.step * min((r & 3) + 8 * (r >> 2), last)] - m[i]);
                            }
                        } else {
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                acc[j][i][r] = NP == 3 ? acc[j][i][r] - m[i] : __builtin_fmaf(acc[j][i][r], c, -m[i]);
                        }
                        if (word[j] != 0xffffffffu) {
                            const unsigned w = word[j] >> (4 * h);
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                acc[j][i][r] = (w >> ((r & 3) + 8 * (r >> 2))) & 1u ? acc[j][i][r] : -INFINITY;
                        }
                    }
                    float top = acc[0][i][0];
#pragma unroll
                    for (int j = 0; j < J; ++j)
#pragma unroll
                        for (int r = 0; r < 16; ++r) top = fmaxf(top, acc[j][i][r]);
                    top = half_max(top);
                    const bool move = top > threshold[i];
                    if (__any(move)) {
                        // (d: what m really moves by)
                        const float to = move ? m[i] + top : m[i], d = to - m[i];
                        const bool far = move && first && fabsf(top) > FAR_MOVE;
                        const float f = move && threshold[i] > 0.f ? __builtin_amdgcn_exp2f(-d) : 1.f;
                        // far: nothing is left of the sums (f = 0, or there were none), and the second time starts them
                        if (move) threshold[i] = far ? -INFINITY : 8.f;
                        again = again || far;
                        m[i] = to;
                        l[i] *= f;
#pragma unroll
                        for (int e = 0; e < VT::GROUPS; ++e)
#pragma unroll
                            for (int r = 0; r < 16; ++r) o[i][e][r] *= f;
#pragma unroll
                        for (int j = 0; j < J; ++j)
#pragma unroll
                            for (int r = 0; r < 16; ++r) acc[j][i][r] -= d;
                    }
                }
                return again;
            };
            // A second time where a reference moved far (see above): the scores are read again, not kept in registers for this.
            // With a bias one copy of the code in a loop, without one two of them (loop / copies: a ragged batch with positions
            // 258 / 285 us, one step over 16384 keys 66 / 59).
            if constexpr (BIAS) {
                for (bool first = true; __any(form(first)); first = false) asm volatile("" ::: "memory");
            } else if (__builtin_expect(__any(form(true)), 0)) {
                asm volatile("" ::: "memory");
                form(false);
            }
#pragma unroll
            for (int i = 0; i < CB; ++i) {
                float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        acc[j][i][r] = __builtin_amdgcn_exp2f(acc[j][i][r]);
                        s4[r & 3] += acc[j][i][r];
                    }
                l[i] += (s4[0] + s4[1]) + (s4[2] + s4[3]);
            }
#pragma unroll
            for (int j = 0; j < J; ++j) {
                PFrag<NP> p[CB];
#pragma unroll
                for (int i = 0; i < CB; ++i) p[i].fill(acc[j][i]);
                mma_values<NP, DV, XT, CB>(vt, 32 * (KW == 1 ? u + j : ksub), l31, h, p, o);
                if (FINE && a.fine) {
#pragma unroll
                    for (int i = 0; i < CB; ++i) p[i].fill_rest(acc[j][i]);
                    mma_values<NP, DV, XT, CB>(vt, 32 * (KW == 1 ? u + j : ksub), l31, h, p, o);
                }
            }
        }
        if (s0 + XT < s_end) {
            __syncthreads();
            if (Cut::BUFS == 1) {
                put(0);
                if (s0 + 2 * XT < s_end) fetch(s0 + 2 * XT);
                __syncthreads();
            } else {
                buf ^= 1;
            }
            now = next;
        }
    }

#pragma unroll
    for (int i = 0; i < CB; ++i) {
        const float sum = half_sum(l[i]);
        if (!live[i]) continue;
        if (a.part == nullptr) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;  // (no key: a column of zeros)
            const long long row = (long long)b * a.KV * a.G + head[i];
            if (a.lse && h == 0) {
                float* const stat = a.lse + row * a.Tq + t[i];
                stat[0] = m[i];
                stat[(long long)a.B * a.KV * a.G * a.Tq] = sum == 0.f ? INFINITY : __builtin_amdgcn_logf(sum);
            }
            T* out = reinterpret_cast<T*>(a.out) + row * a.Dv * a.Tq + t[i];
            T* rest = NP == 1 && a.rest ? reinterpret_cast<T*>(a.rest) + row * a.Dv * a.Tq + t[i] : nullptr;
#pragma unroll
            for (int e = 0; e < VT::GROUPS; ++e)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int d = 32 * e + acc_row(r, h);
                    if (d < a.Dv) {
                        const float v = o[i][e][r] * inv;
                        st1(out + (long long)d * a.Tq, v);
                        if (NP == 1 && rest) st1(rest + (long long)d * a.Tq, v - (float)(T)v);
                    }
                }
        } else {
            const long long nparts = (long long)a.nsplit * KW;
            const long long at = (long long)bkv * nparts + split * KW + ksub;
            float* po = a.part + at * a.Dv * ncols + col0 + 32 * i + l31;
#pragma unroll
            for (int e = 0; e < VT::GROUPS; ++e)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int d = 32 * e + acc_row(r, h);
                    if (d < a.Dv) po[(long long)d * ncols] = o[i][e][r];
                }
            if (h == 0) {
                const long long total = (long long)a.B * a.KV * nparts;
                float* pm = a.part + total * a.Dv * ncols + at * ncols + col0 + 32 * i + l31;
                pm[0] = m[i];
                pm[total * ncols] = sum;
            }
        }
    }
}

// Parts of a split over the keys -> output: M = max m, O = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i; parts that saw
// no key (l = 0) are left out.  `lanes` threads share an output's parts, joined in LDS in a
// fixed order: there are few outputs and up to hundreds of parts, and a thread that walked them alone would wait for one
// load after the other.
template <class T>
__global__ __launch_bounds__(THREADS) void attn_join_kernel(FwdArgs a, int nparts, int lanes, long long items) {
    __shared__ float red[3][THREADS];
    const int tid = threadIdx.x, per = THREADS / lanes;  // outputs of the workgroup
    const int lane = tid / per;
    const long long i = (long long)blockIdx.x * per + tid % per;
    const int ncols = a.G * a.Tq;
    float top = -INFINITY, l = 0.f, o = 0.f;
    if (i < items) {
        const int n = (int)(i % ncols);
        const long long j = i / ncols;
        const int d = (int)(j % a.Dv);
        const long long bkv = j / a.Dv;
        const long long total = (long long)a.B * a.KV * nparts;
        const float* po = a.part + (bkv * nparts * a.Dv + d) * ncols + n;
        const float* pm = a.part + total * a.Dv * ncols + bkv * nparts * ncols + n;
        const float* pl = pm + total * ncols;
        for (int p = lane; p < nparts; p += lanes) {
            const float lp = pl[(long long)p * ncols], mp = pm[(long long)p * ncols], op = po[(long long)p * a.Dv * ncols];
            if (lp != 0.f) {
                const float t = fmaxf(top, mp);
                const float f = __builtin_amdgcn_exp2f(top - t), e = __builtin_amdgcn_exp2f(mp - t);
                l = l * f + lp * e;
                o = o * f + op * e;
                top = t;
            }
        }
    }
    if (lanes > 1) {
        red[0][tid] = top, red[1][tid] = l, red[2][tid] = o;
        __syncthreads();
        if (lane != 0) return;
        for (int w = 1; w < lanes; ++w) {
            const float mp = red[0][tid + w * per], lp = red[1][tid + w * per], op = red[2][tid + w * per];
            if (lp != 0.f) {
                const float t = fmaxf(top, mp);
                const float f = __builtin_amdgcn_exp2f(top - t), e = __builtin_amdgcn_exp2f(mp - t);
                l = l * f + lp * e;
                o = o * f + op * e;
                top = t;
            }
        }
    }
    if (i >= items) return;
    const int n = (int)(i % ncols);
    const long long j = i / ncols;
    const int d = (int)(j % a.Dv);
    const long long bkv = j / a.Dv;
    const int g = n / a.Tq, t = n - g * a.Tq;
    const long long row = bkv * a.G + g;
    const float v = l == 0.f ? 0.f : o / l;
    const long long at = (row * a.Dv + d) * a.Tq + t;
    st1(reinterpret_cast<T*>(a.out) + at, v);
    if (Elem<T>::NP == 1 && a.rest) st1(reinterpret_cast<T*>(a.rest) + at, v - (float)(T)v);
    if (a.lse && d == 0) {
        float* const stat = a.lse + row * a.Tq + t;
        stat[0] = l == 0.f ? 0.f : top;
        stat[(long long)a.B * a.KV * a.G * a.Tq] = l == 0.f ? INFINITY : __builtin_amdgcn_logf(l);
    }
}

}  // namespace attn
}  // namespace eeggan

using namespace eeggan;
using namespace eeggan::attn;

namespace {

// How the forward pass is cut.  Up to 32 query columns per key head: the waves split every stage's keys.  Beyond that, and
// for a single stage of keys, each wave has columns of its own.  Keys are split over workgroups until there are `WANTED` of
// them.
struct FwdPlan {
    int kw, xt, cb, coltiles, nsplit, split_keys, nparts;
};
constexpr int WANTED = 512;

template <class T, int DK, int DV>
struct Cuts {
    static constexpr bool F32 = Elem<T>::NP == 3;
    static constexpr int FEW_XT = F32 && DK + DV > 160 ? 32 : 64;  // keys of a stage: few columns / many
    static constexpr int XT = F32 && DK + DV > 96 ? 32 : 64;
    // column blocks of a wave, where there are enough workgroups left (8 x 8 x 2048, 64 channels, bfloat16: 115 us with two;
    // with one, at three workgroups to a CU, 119)
    static constexpr int CB = DK + DV <= (F32 ? 64 : 128) ? 2 : 1;
};

template <class T, int DK, int DV>
FwdPlan plan_of(const eeggan_attention& a) {
    typedef Cuts<T, DK, DV> C;
    FwdPlan p;
    const long long ncols = (long long)(a.H / a.KV) * a.Tq, heads = (long long)a.B * a.KV;
    const bool few = few_columns(a);
    p.xt = few ? C::FEW_XT : C::XT;
    p.kw = few ? p.xt / 32 : 1;
    p.cb = !few && C::CB == 2 && heads * ((ncols + 255) / 256) >= WANTED ? 2 : 1;
    p.coltiles = few ? 1 : (int)((ncols + 128 * p.cb - 1) / (128 * p.cb));
    const long long blocks = heads * p.coltiles;
    const long long stages = (a.Tk + p.xt - 1) / p.xt;
    // (half a fill is left as it is: a ragged batch's 296 workgroups in two parts each, and joined: 224 us for 217 of the call)
    long long n = blocks >= WANTED / 2 ? 1 : (WANTED + blocks - 1) / blocks;
    const long long most = few ? stages : stages / 4 > 0 ? stages / 4 : 1;
    if (n > most) n = most;
    const long long per = (stages + n - 1) / n;
    p.split_keys = (int)(per * p.xt);
    p.nsplit = (int)((stages + per - 1) / per);
    p.nparts = p.nsplit * p.kw;
    return p;
}

constexpr size_t NEVER_NONE = 16;  // (a workspace of no bytes says that the descriptor was rejected)

size_t part_bytes(const eeggan_attention& a, const FwdPlan& p) {
    if (p.nparts == 1) return 0;
    const size_t ncols = (size_t)(a.H / a.KV) * a.Tq;
    return (size_t)a.B * a.KV * p.nparts * ncols * (a.Dv + 2) * sizeof(float);
}

template <class T, int DK, int DV, int KW, int XT, int CB, bool BIAS, bool FINE = Elem<T>::NP == 1>
int launch(const FwdArgs& f, const FwdPlan& p, hipStream_t st) {
    constexpr size_t tiles = FwdCut<T, DK, DV, XT>::LDS, most = tiles + (BIAS ? 4 * CB * MAX_BAND * sizeof(float) : 0);
    static_assert(most <= 160 * 1024, "LDS");
    const size_t lds = tiles + (BIAS ? 4 * CB * (2 * (size_t)f.pos.width + 1) * sizeof(float) : 0);
    auto kernel = &attn_fwd_kernel<T, DK, DV, KW, XT, CB, BIAS, FINE>;
    static LdsReady ready;
    if (ready.reserve("attention", reinterpret_cast<const void*>(kernel), most)) return 1;
    const long long grid = (long long)f.B * f.KV * p.nsplit * p.coltiles;
    EEGGAN_REQUIRE(grid < (1ll << 31), "attention: too many workgroups");
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(THREADS), lds, st, f);
    return check_launch("attention");
}

template <class T, int DK, int DV, bool BIAS>
int launch_cut(const FwdArgs& f, const FwdPlan& p, hipStream_t st) {
    typedef Cuts<T, DK, DV> C;
    if constexpr (C::FEW_XT == 64) {
        if (p.kw == 2) {
            if constexpr (!BIAS) {  // (with a table bfloat16 is always fine)
                if (!f.fine) return launch<T, DK, DV, 2, 64, 1, BIAS, false>(f, p, st);
            }
            return launch<T, DK, DV, 2, 64, 1, BIAS>(f, p, st);
        }
    }
    if constexpr (C::CB == 2) {
        if (p.cb == 2) return launch<T, DK, DV, 1, C::XT, 2, BIAS>(f, p, st);
    }
    return launch<T, DK, DV, 1, C::XT, 1, BIAS>(f, p, st);
}

template <class T, int DK, int DV>
int forward(const eeggan_attention& a, void* out, void* rest, float* lse, void* ws, size_t bytes, hipStream_t st) {
    const FwdPlan p = plan_of<T, DK, DV>(a);
    const size_t rel = positions_bytes(a);
    EEGGAN_REQUIRE(bytes >= rel + part_bytes(a, p) + NEVER_NONE, "attention: workspace too small");
    FwdArgs f;
    f.q = a.q, f.k = a.k, f.v = a.v;
    f.qsb = a.q_batch, f.qsc = a.q_channel, f.ksb = a.k_batch, f.ksc = a.k_channel, f.vsb = a.v_batch, f.vsc = a.v_channel;
    f.mask = a.mask, f.out = out, f.rest = rest, f.lse = lse;
    f.part = p.nparts > 1 ? reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + rel) : nullptr;
    f.B = a.B, f.KV = a.KV, f.G = a.H / a.KV, f.Dk = a.Dk, f.Dv = a.Dv, f.Tq = a.Tq, f.Tk = a.Tk;
    f.coltiles = p.coltiles, f.nsplit = p.nsplit, f.split_keys = p.split_keys, f.scale = a.scale;
    if (positions(a, reinterpret_cast<float*>(ws), &f.pos, st)) return 1;
    f.fine = fine_forward(a);
    if (a.table ? launch_cut<T, DK, DV, true>(f, p, st) : launch_cut<T, DK, DV, false>(f, p, st)) return 1;
    if (p.nparts == 1) return 0;
    const long long items = (long long)a.B * a.KV * a.Dv * f.G * a.Tq;
    int lanes = 1;  // threads that share an output's parts: at least four parts each
    while (lanes < 16 && lanes * 8 <= p.nparts) lanes *= 2;
    const long long blocks = (items * lanes + THREADS - 1) / THREADS;
    EEGGAN_REQUIRE(blocks < (1ll << 31), "attention: too many outputs");
    hipLaunchKernelGGL(attn_join_kernel<T>, dim3((unsigned)blocks), dim3(THREADS), 0, st, f, p.nparts, lanes, items);
    return check_launch("attention (join)");
}

}  // namespace

extern "C" size_t eeggan_attention_fwd_workspace(const eeggan_attention* a) {
    if (check_attention("attention", a)) return 0;
    size_t parts = 0;
    EEGGAN_ATTENTION_CLASS(*a, parts = part_bytes(*a, (plan_of<T, DK, DV>(*a))))
    return positions_bytes(*a) + parts + NEVER_NONE;
}

extern "C" int eeggan_attention_fwd(const eeggan_attention* a, void* out, void* rest, float* lse, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    if (check_attention("attention", a)) return 1;
    EEGGAN_REQUIRE(out && workspace, "attention: null pointer");
    int rc = 1;
    EEGGAN_ATTENTION_CLASS(*a, rc = (forward<T, DK, DV>(*a, out, rest, lse, workspace, workspace_bytes, as_stream(stream))))
    return rc;
}
