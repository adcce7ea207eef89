// Attention over time, channels first, without storing the probabilities:
//   S[s, t] = scale * sum_d K[d, s] Q[d, t] (+ the position bias of (s, t));  O[c, t] = sum_s V[c, s] softmax_s(S)[s, t]
// One pass over the keys per query column with a running reference m and sum l (P' = 2^(S log2e - m), O = sum V P' / l);
// what the backward pass needs besides its inputs is one number per query, lse = m + log2 l.
//
// A wave owns 32 query columns; the head's keys pass through LDS in stages shared by the workgroup's four waves.
// A lane holds one query's column of S, so the statistics are per-lane scalars: the maximum over its sixteen
// registers and one exchange between the lane halves, the sum without any exchange until the end.  The reference m
// moves only when a score exceeds it by 8 (a factor 256: the sums stay far inside float32's range and lose
// nothing), which after the first stages is rare, so the accumulators are hardly ever rescaled.
// Few query columns (a single new step): the waves share the columns and split each stage's keys (KW > 1), and the keys
// are split over workgroups; every part leaves (O unscaled, m, l) and attn_join_kernel combines them in a fixed order.
#include "attention_host.h"

namespace eeggan {
namespace attn {

struct FwdArgs {
    const void *q, *k, *v;
    long long qsb, qsc, ksb, ksc, vsb, vsc;  // strides between samples and channels, in elements
    const unsigned char* mask;               // [B, Tk], nonzero = attended; null: all
    void* out;                               // [B, H Dv, Tq]
    void* rest;                              // what the rounding of out left over (bfloat16); null: not wanted
    float* lse;                              // [B, H, Tq]; null: not wanted
    float* part;                             // parts of a split: O, then m, then l; null: not split
    Positions pos;
    int B, KV, G, Dk, Dv, Tq, Tk;
    int coltiles, nsplit, split_keys;
    float scale;
};

template <class T, int DK, int DV, int KW, int XT, bool BIAS>
__global__ __launch_bounds__(THREADS, 2) void attn_fwd_kernel(FwdArgs a) {
    constexpr int NP = Elem<T>::NP;
    constexpr int WC = 4 / KW;                 // column tiles of a workgroup
    constexpr int SUBS = XT / (32 * KW);       // key tiles a wave takes of a stage
    typedef TTile<NP, DK, XT> KT;
    typedef NTile<NP, DV, XT> VT;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char* const kt = smem;
    char* const vt = smem + KT::BYTES;

    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ksub = wave % KW;
    int blk = blockIdx.x;
    const int tile = blk % a.coltiles;
    blk /= a.coltiles;
    const int split = blk % a.nsplit;
    const int bkv = blk / a.nsplit;
    const int b = bkv / a.KV, kvh = bkv - b * a.KV;

    const int ncols = a.G * a.Tq;
    const int col0 = (tile * WC + wave / KW) * 32;
    const int n = col0 + l31;
    const bool live = n < ncols;
    const int g = live ? n / a.Tq : 0, t = live ? n - g * a.Tq : 0;
    const int head = kvh * a.G + g;

    const float c = a.scale * LOG2E;
    SFrag<NP, DK> fq;
    {
        const T* q = reinterpret_cast<const T*>(a.q) + b * a.qsb + (long long)head * a.Dk * a.qsc + t;
        // (float32: the scale goes into the split operand; bfloat16 operands stay exact and the scores are scaled)
        typedef SFrag<NP, DK> F;
        float x[F::VALUES];
        F::read(q, a.qsc, a.Dk, h, x);
#pragma unroll
        for (int i = 0; i < F::VALUES; ++i) x[i] = live && F::channel(i, h) < a.Dk ? (NP == 3 ? x[i] * c : x[i]) : 0.f;
        fq.fill(h, x);
    }
    const T* const kb = reinterpret_cast<const T*>(a.k) + b * a.ksb + (long long)kvh * a.Dk * a.ksc;
    const T* const vb = reinterpret_cast<const T*>(a.v) + b * a.vsb + (long long)kvh * a.Dv * a.vsc;
    const unsigned char* const mask = a.mask ? a.mask + (long long)b * a.Tk : nullptr;
    // position bias: rel[step * s] relative to this lane's query
    const float* const rel = BIAS ? a.pos.rel + (long long)head * a.pos.nrel + (a.Tq - 1 - t) : nullptr;
    // (a tile of columns of several heads is always near)
    const bool one_head = col0 / a.Tq == min(col0 + 31, ncols - 1) / a.Tq;
    const int t_tile = col0 % a.Tq;

    const int s_begin = split * a.split_keys;
    const int s_end = min(a.Tk, s_begin + a.split_keys);

    float m = 0.f, l = 0.f, threshold = -INFINITY;  // threshold -inf: no key seen yet
    f32x16 cinit = zero16();                        // -m in every register: the scores accumulate on top of it
    f32x16 o[VT::GROUPS];
#pragma unroll
    for (int i = 0; i < VT::GROUPS; ++i) o[i] = zero16();

    Block<T, DK, XT> kblk;
    Block<T, DV, XT> vblk;
    Steps<XT> ahead;  // which keys of the stage are attended
    auto fetch = [&](int s0) {
        kblk.load(kb, a.ksc, a.Dk, s0, s_end, tid);
        vblk.load(vb, a.vsc, a.Dv, s0, s_end, tid);
        ahead.find(s0, s_end, mask, lane);
    };
    if (s_begin < s_end) fetch(s_begin);
    for (int s0 = s_begin; s0 < s_end; s0 += XT) {
        __syncthreads();
        const Steps<XT> now = ahead;
        kblk.template store<true, false>(kt, nullptr, a.Dk, now, tid);
        vblk.template store<false, true>(nullptr, vt, a.Dv, now, tid);
        __syncthreads();
        if (s0 + XT < s_end) fetch(s0 + XT);
#pragma unroll
        for (int u = 0; u < SUBS; ++u) {
            const int sub = KW == 1 ? u : ksub;
            const int x0 = 32 * sub;
            const unsigned word = now.tile(x0);
            if (word == 0) continue;  // (the same for every lane of the wave)
            f32x16 acc;
            if constexpr (BIAS) {
                const long long s = s0 + x0;
                if (one_head && tile_side(a.pos, s, t_tile) != 0) {
                    const float bias = rel[a.pos.step * s];
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[r] = cinit[r] + bias;
                } else {
                    const int first = min((int)s + 4 * h, a.Tk - 1), last = a.Tk - 1 - first;
                    const float* r0 = rel + (long long)a.pos.step * first;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int i = (r & 3) + 8 * (r >> 2);
                        acc[r] = cinit[r] + r0[a.pos.step * min(i, last)];
                    }
                }
            } else {
                acc = cinit;
            }
            if constexpr (NP == 3) {
                acc = mma_scores<NP, DK, XT>(kt + (x0 + l31) * KT::RS, h, fq, acc);
            } else {
                const f32x16 raw = mma_scores<NP, DK, XT>(kt + (x0 + l31) * KT::RS, h, fq, zero16());
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[r] = __builtin_fmaf(raw[r], c, acc[r]);
            }
            if (word != 0xffffffffu) {
                const unsigned w = word >> (4 * h);
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[r] = (w >> ((r & 3) + 8 * (r >> 2))) & 1u ? acc[r] : -INFINITY;
            }
            float top = acc[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) top = fmaxf(top, acc[r]);
            top = half_max(top);
            const bool move = top > threshold;
            if (__any(move)) {
                const float d = move ? top : 0.f;
                const float f = move && threshold > 0.f ? __builtin_amdgcn_exp2f(-d) : 1.f;
                if (move) threshold = 8.f;
                m += d;
                l *= f;
#pragma unroll
                for (int i = 0; i < VT::GROUPS; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[i][r] *= f;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    acc[r] -= d;
                    cinit[r] = -m;
                }
            }
            float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                acc[r] = __builtin_amdgcn_exp2f(acc[r]);
                s4[r & 3] += acc[r];
            }
            l += (s4[0] + s4[1]) + (s4[2] + s4[3]);
            PFrag<NP> p;
            p.fill(acc);
            mma_values<NP, DV, XT>(vt, x0, l31, h, p, o);
        }
    }

    l = half_sum(l);
    if (!live) return;
    if (a.part == nullptr) {
        const float inv = l == 0.f ? 0.f : 1.f / l;  // (no key: a column of zeros)
        const long long row = (long long)b * a.KV * a.G + head;
        if (a.lse && h == 0) a.lse[row * a.Tq + t] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
        T* out = reinterpret_cast<T*>(a.out) + row * a.Dv * a.Tq + t;
#pragma unroll
        for (int i = 0; i < VT::GROUPS; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = 32 * i + acc_row(r, h);
                if (d < a.Dv) {
                    const float v = o[i][r] * inv;
                    st1(out + (long long)d * a.Tq, v);
                    if (NP == 1 && a.rest) {
                        T* rest = reinterpret_cast<T*>(a.rest) + row * a.Dv * a.Tq + t;
                        st1(rest + (long long)d * a.Tq, v - (float)(T)v);
                    }
                }
            }
    } else {
        const long long nparts = (long long)a.nsplit * KW;
        const long long part = ((long long)bkv * nparts + split * KW + ksub);
        float* po = a.part + part * a.Dv * ncols + n;
#pragma unroll
        for (int i = 0; i < VT::GROUPS; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = 32 * i + acc_row(r, h);
                if (d < a.Dv) po[(long long)d * ncols] = o[i][r];
            }
        if (h == 0) {
            const long long total = (long long)a.B * a.KV * nparts;
            float* pm = a.part + total * a.Dv * ncols + part * ncols + n;
            pm[0] = m;
            pm[total * ncols] = l;
        }
    }
}

// Parts of a split over the keys -> output: M = max m, O = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i; parts that saw
// no key (l = 0) are left out.
template <class T>
__global__ __launch_bounds__(THREADS) void attn_join_kernel(FwdArgs a, int nparts, long long items) {
    const long long i = (long long)blockIdx.x * THREADS + threadIdx.x;
    if (i >= items) return;
    const int ncols = a.G * a.Tq;
    const int n = (int)(i % ncols);
    const long long j = i / ncols;
    const int d = (int)(j % a.Dv);
    const long long bkv = j / a.Dv;
    const long long total = (long long)a.B * a.KV * nparts;
    const float* po = a.part + (bkv * nparts * a.Dv + d) * ncols + n;
    const float* pm = a.part + total * a.Dv * ncols + bkv * nparts * ncols + n;
    const float* pl = pm + total * ncols;
    float top = -INFINITY;
    for (int p = 0; p < nparts; ++p)
        if (pl[(long long)p * ncols] != 0.f) top = fmaxf(top, pm[(long long)p * ncols]);
    float l = 0.f, o = 0.f;
    for (int p = 0; p < nparts; ++p) {
        const float lp = pl[(long long)p * ncols];
        if (lp != 0.f) {
            const float f = __builtin_amdgcn_exp2f(pm[(long long)p * ncols] - top);
            l += f * lp;
            o += f * po[(long long)p * a.Dv * ncols];
        }
    }
    const int g = n / a.Tq, t = n - g * a.Tq;
    const long long row = bkv * a.G + g;
    const float v = l == 0.f ? 0.f : o / l;
    const long long at = (row * a.Dv + d) * a.Tq + t;
    st1(reinterpret_cast<T*>(a.out) + at, v);
    if (Elem<T>::NP == 1 && a.rest) st1(reinterpret_cast<T*>(a.rest) + at, v - (float)(T)v);
    if (a.lse && d == 0) a.lse[row * a.Tq + t] = l == 0.f ? INFINITY : top + __builtin_amdgcn_logf(l);
}

}  // namespace attn
}  // namespace eeggan

using namespace eeggan;
using namespace eeggan::attn;

namespace {

// How the forward pass is cut.  Up to 32 query columns per key head: the waves split every stage's keys.  Beyond that
// each wave has columns of its own.  Keys are split over workgroups until there are `WANTED` of them.
struct FwdPlan {
    int kw, xt, coltiles, nsplit, split_keys, nparts;
};
constexpr int WANTED = 512;

template <class T, int DK, int DV>
constexpr int stage_keys(bool few) {
    constexpr bool f32 = Elem<T>::NP == 3;
    return few ? (f32 && DK + DV > 128 ? 64 : 128) : (f32 && DK + DV > 160 ? 32 : 64);
}

template <class T, int DK, int DV>
FwdPlan plan_of(const eeggan_attention& a) {
    FwdPlan p;
    const long long ncols = (long long)(a.H / a.KV) * a.Tq;
    const bool few = ncols <= 32;
    p.xt = stage_keys<T, DK, DV>(few);
    p.kw = few ? p.xt / 32 : 1;
    p.coltiles = few ? 1 : (int)((ncols + 127) / 128);
    const long long blocks = (long long)a.B * a.KV * p.coltiles;
    const long long stages = (a.Tk + p.xt - 1) / p.xt;
    long long n = blocks >= WANTED ? 1 : (WANTED + blocks - 1) / blocks;
    const long long most = few ? stages : stages / 4 > 0 ? stages / 4 : 1;
    if (n > most) n = most;
    const long long per = (stages + n - 1) / n;
    p.split_keys = (int)(per * p.xt);
    p.nsplit = (int)((stages + per - 1) / per);
    p.nparts = p.nsplit * p.kw;
    return p;
}

size_t part_bytes(const eeggan_attention& a, const FwdPlan& p) {
    if (p.nparts == 1) return 0;
    const size_t ncols = (size_t)(a.H / a.KV) * a.Tq;
    return (size_t)a.B * a.KV * p.nparts * ncols * (a.Dv + 2) * sizeof(float);
}

template <class T, int DK, int DV, int KW, int XT, bool BIAS>
int launch(const FwdArgs& f, const FwdPlan& p, hipStream_t st) {
    constexpr int NP = Elem<T>::NP;
    constexpr size_t lds = TTile<NP, DK, XT>::BYTES + NTile<NP, DV, XT>::BYTES;
    static_assert(lds <= 160 * 1024, "LDS");
    auto kernel = &attn_fwd_kernel<T, DK, DV, KW, XT, BIAS>;
    static LdsReady ready;
    if (ready.reserve("attention", reinterpret_cast<const void*>(kernel), lds)) return 1;
    const long long grid = (long long)f.B * f.KV * p.nsplit * p.coltiles;
    EEGGAN_REQUIRE(grid < (1ll << 31), "attention: too many workgroups");
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(THREADS), lds, st, f);
    return check_launch("attention");
}

template <class T, int DK, int DV>
int forward(const eeggan_attention& a, void* out, void* rest, float* lse, void* ws, size_t bytes, hipStream_t st) {
    const FwdPlan p = plan_of<T, DK, DV>(a);
    const size_t rel = positions_bytes(a);
    EEGGAN_REQUIRE(bytes >= rel + part_bytes(a, p), "attention: workspace too small");
    FwdArgs f;
    f.q = a.q, f.k = a.k, f.v = a.v;
    f.qsb = a.q_batch, f.qsc = a.q_channel, f.ksb = a.k_batch, f.ksc = a.k_channel, f.vsb = a.v_batch, f.vsc = a.v_channel;
    f.mask = a.mask, f.out = out, f.rest = rest, f.lse = lse;
    f.part = p.nparts > 1 ? reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + rel) : nullptr;
    f.B = a.B, f.KV = a.KV, f.G = a.H / a.KV, f.Dk = a.Dk, f.Dv = a.Dv, f.Tq = a.Tq, f.Tk = a.Tk;
    f.coltiles = p.coltiles, f.nsplit = p.nsplit, f.split_keys = p.split_keys, f.scale = a.scale;
    if (positions(a, reinterpret_cast<float*>(ws), &f.pos, st)) return 1;
    int rc;
    constexpr int XF = stage_keys<T, DK, DV>(true), XN = stage_keys<T, DK, DV>(false);
    if (p.kw > 1)
        rc = a.table ? launch<T, DK, DV, XF / 32, XF, true>(f, p, st) : launch<T, DK, DV, XF / 32, XF, false>(f, p, st);
    else
        rc = a.table ? launch<T, DK, DV, 1, XN, true>(f, p, st) : launch<T, DK, DV, 1, XN, false>(f, p, st);
    if (rc || p.nparts == 1) return rc;
    const long long items = (long long)a.B * a.KV * a.Dv * f.G * a.Tq;
    EEGGAN_REQUIRE((items + THREADS - 1) / THREADS < (1ll << 31), "attention: too many outputs");
    hipLaunchKernelGGL(attn_join_kernel<T>, dim3((unsigned)((items + THREADS - 1) / THREADS)), dim3(THREADS), 0, st, f,
                       p.nparts, items);
    return check_launch("attention (join)");
}

}  // namespace

extern "C" size_t eeggan_attention_fwd_workspace(const eeggan_attention* a) {
    if (check_attention("attention", a)) return 0;
    size_t parts = 0;
    EEGGAN_ATTENTION_CLASS(*a, parts = part_bytes(*a, (plan_of<T, DK, DV>(*a))))
    return positions_bytes(*a) + parts + 16;
}

extern "C" int eeggan_attention_fwd(const eeggan_attention* a, void* out, void* rest, float* lse, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    if (check_attention("attention", a)) return 1;
    EEGGAN_REQUIRE(out && workspace, "attention: null pointer");
    int rc = 1;
    EEGGAN_ATTENTION_CLASS(*a, rc = (forward<T, DK, DV>(*a, out, rest, lse, workspace, workspace_bytes, as_stream(stream))))
    return rc;
}
