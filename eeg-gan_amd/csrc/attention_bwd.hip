// Backward pass of the fused attention: the probabilities are formed again from q, k and the forward's m and log2 l.
//   P[s,t] = 2^((S log2e - m[t]) - log2 l[t]);  delta[t] = sum_c O dO;  dP = V^T dO;  dS = P (dP - delta)
//   dQ[d,t] = scale sum_s K[d,s] dS[s,t]          (attn_dq_kernel: a wave owns 32 queries, the keys stream through LDS)
//   dV[c,s] = sum_t dO[c,t] P[s,t],  dK[d,s] = scale sum_t Q[d,t] dS[s,t]
//                                                 (attn_dkv_kernel: a wave owns 32 keys, q and dO stream)
// Two kernels, each forming S and dP (seven products where one kernel would need five): a sum over keys and a sum over
// queries cannot both stay in one wave's registers, and one of them through atomics would make the result depend on
// their order.  Both orientations have their result registers where the next product wants its operand
// (attention_tiles.h), so nothing crosses lanes.  -delta is the initial accumulator of dP.
//
// The position table's gradient rides on attn_dq_kernel: tiles whose distances all lie beyond the last bucket's edge
// add to one register; a near tile goes through LDS, every lane adds up the pairs of one distance, and the sums go to a
// histogram by distance that belongs to the wave: a fixed order, no races.  (LDS float atomics in the place of that took
// ~300 cycles per instruction: 73 us of 167 at 4 x 6 heads over 1537 steps.)
//
// Measured (calls one after the other, both kernels together): bfloat16, 8 samples x 8 heads of 64 channels over 2048 steps
// 273 us = 881 TFLOP/s over the seven products (a large library product: 1330), the keys' kernel 1.3 times as long as the
// queries'; float32, 8 x 8 x 1024: 342 us = 176 TFLOP/s (library: 154).  Bound as the forward pass is: the products fill two
// thirds of the time, exponentials and staging the rest.
#include "attention_host.h"

namespace eeggan {
namespace attn {

struct BwdArgs {
    const void *q, *k, *v;
    long long qsb, qsc, ksb, ksc, vsb, vsc;
    const unsigned char* mask;
    const void *out, *rest, *g;  // [B, H Dv, Tq]; out + rest: the output before its rounding (float32: rest null)
    const float* lse;  // [2, B, H, Tq]: m, log2 l (infinite: no key)
    float* delta;  // [B, H, Tq]: written by attn_dq_kernel, read by attn_dkv_kernel
    void *gq, *gk, *gv;
    float* part;  // dK, dV of a split over the queries; null: not split
    float* hist;  // [H, B * coltiles, nhist + 2] sums of dS by distance (then: beyond it, behind / ahead); null: not wanted
    Positions pos;
    int B, KV, G, Dk, Dv, Tq, Tk;
    int coltiles, nsplit, nhist;
    float scale;
    bool fine;  // bfloat16: P and dS meet their products in two pieces (fine_backward)
};

template <class T, int DK, int DV, int XT>
struct DqCut {
    static constexpr int NP = Elem<T>::NP;
    static constexpr int STAGE = Tile<NP, DK, XT>::BYTES + Tile<NP, DV, XT>::BYTES;
    static constexpr int BUFS = 2 * STAGE <= 64 * 1024 ? 2 : 1;  // (two workgroups to a CU, with room for histograms)
    static constexpr int LDS = BUFS * STAGE;
};
constexpr int SQUARE = 32 * 33;  // a wave's tile of dS on its way into the histogram by distance
// Two workgroups to a CU (256 registers a wave) but for float32 past 160 channels: 8 x 8 x 1024 at 128 channels 300 us with
// one and 530 with two, at 32 + 128 channels 191 and 159.
template <class T, int DK, int DV, int XT, bool BIAS>
__global__ __launch_bounds__(THREADS, DK + DV > 160 && Elem<T>::NP == 3 ? 1 : 2) void attn_dq_kernel(BwdArgs a) {
    typedef DqCut<T, DK, DV, XT> Cut;
    constexpr int NP = Elem<T>::NP;
    typedef Tile<NP, DK, XT> KT;
    extern __shared__ __attribute__((aligned(16))) char smem[];

    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int H = a.KV * a.G;
    int group, part_of;
    place(blockIdx.x, a.B * a.KV, a.G * a.coltiles, group, part_of);
    const int b = group / a.KV, kvh = group - b * a.KV;
    const int tile = part_of % a.coltiles, head = kvh * a.G + part_of / a.coltiles;

    const int k_off = SRead<NP, DK, XT>::offset(lane), v_off = SRead<NP, DV, XT>::offset(lane);
    const int t0 = (tile * 4 + wave) * 32;
    const bool inside = t0 + l31 < a.Tq;
    const int t = inside ? t0 + l31 : 0;
    const long long row = (long long)b * H + head;
    const long long queries = (long long)a.B * H * a.Tq;
    float ref = a.lse[row * a.Tq + t], lsum = a.lse[queries + row * a.Tq + t];
    const bool live = inside && lsum != INFINITY;  // (a query without keys takes no part)
    if (!live) ref = 0.f, lsum = INFINITY;

    const float c = a.scale * LOG2E;
    SFrag<NP, DK> fq[1];
    SFrag<NP, DV> fg[1];
    // (delta in double: where a query's keys all share a bucket, its error is all that the query leaves in the table's gradient)
    float delta = 0.f;
    // Every other tile of queries works on -dS: the matrix instruction rounds an accumulator towards minus infinity where it
    // aligns it with larger products, a bias of 6e-9 of dP that the table's sums over all rows would add up
    // (float32: error 2.4e-6 of the gradient's norm with one sign, 4e-7 with both).
    const float sign = wave & 1 ? -1.f : 1.f;
    {
        const T* q = reinterpret_cast<const T*>(a.q) + b * a.qsb + (long long)head * a.Dk * a.qsc;
        const T* g = reinterpret_cast<const T*>(a.g) + row * a.Dv * a.Tq;
        const T* o = reinterpret_cast<const T*>(a.out) + row * a.Dv * a.Tq;
        const T* w = reinterpret_cast<const T*>(NP == 1 ? a.rest : a.out) + row * a.Dv * a.Tq;
        typedef SFrag<NP, DK> FK;
        typedef SFrag<NP, DV> FV;
        float x[FK::VALUES], y[FV::VALUES];
        FK::read(q, t, a.qsc, a.Dk, h, x);
#pragma unroll
        for (int i = 0; i < FK::VALUES; ++i) x[i] = live && FK::channel(i, h) < a.Dk ? (NP == 3 ? x[i] * c : x[i]) : 0.f;
        fq[0].fill(h, x);
        typename std::conditional<NP == 3, double, float>::type sum = 0;
        // (sixteen values of a lane at a time: all loads of 128 channels in flight spill registers)
        constexpr int SOME = FV::VALUES < 16 ? FV::VALUES : 16;
        static_unroll<FV::VALUES / SOME>([&](auto part) {
            constexpr int FIRST = decltype(part)::value * SOME;
            float yy[SOME], z[SOME], zz[SOME];
            if constexpr (FIRST != 0) __builtin_amdgcn_sched_barrier(0);
            FV::template read<FIRST>(g, t, a.Tq, a.Dv, h, yy);
            FV::template read<FIRST>(o, t, a.Tq, a.Dv, h, z);
            if constexpr (NP == 1) FV::template read<FIRST>(w, t, a.Tq, a.Dv, h, zz);
#pragma unroll
            for (int i = 0; i < SOME; ++i) {
                const bool ok = live && FV::channel(FIRST + i, h) < a.Dv;
                const float v = ok ? yy[i] : 0.f;
                if constexpr (NP == 3)
                    sum = ok ? __builtin_fma((double)v, (double)z[i], sum) : sum;
                else
                    sum = ok ? __builtin_fmaf(v, z[i] + zz[i], sum) : sum;
                y[FIRST + i] = sign * v;
            }
        });
        fg[0].fill(h, y);
        if constexpr (NP == 3)
            delta = (float)(sum + __shfl_xor(sum, 32, 64));
        else
            delta = half_sum(sum);
        if (inside && h == 0) a.delta[row * a.Tq + t] = delta;
    }
    const T* const kb = reinterpret_cast<const T*>(a.k) + b * a.ksb + (long long)kvh * a.Dk * a.ksc;
    const T* const vb = reinterpret_cast<const T*>(a.v) + b * a.vsb + (long long)kvh * a.Dv * a.vsc;
    const unsigned char* const mask = a.mask ? a.mask + (long long)b * a.Tk : nullptr;
    // position bias: one value per side beyond the last edge, near tiles from LDS
    const float* const rel = BIAS ? a.pos.rel + (long long)head * a.pos.nrel : nullptr;
    float* const band = reinterpret_cast<float*>(smem + Cut::LDS);
    float side_bias[2] = {0.f, 0.f};
    if constexpr (BIAS) {
        side_bias[0] = (rel_at(a.pos, rel, a.Tq, -a.pos.far) - ref) - lsum;
        side_bias[1] = (rel_at(a.pos, rel, a.Tq, a.pos.far) - ref) - lsum;
        fill_band(band, a.pos, rel, a.Tq, tid, THREADS);
    }

    f32x16 dinit;
#pragma unroll
    for (int r = 0; r < 16; ++r) dinit[r] = -sign * delta;
    f32x16 dq[1][KT::GROUPS];
#pragma unroll
    for (int i = 0; i < KT::GROUPS; ++i) dq[0][i] = zero16();

    double beyond[2] = {0.0, 0.0};  // sums of dS over far tiles, behind / ahead of the query (thousands of terms)
    float* const hist = BIAS ? band + (2 * a.pos.width + 1) + wave * a.nhist : nullptr;
    const bool want = BIAS && a.hist != nullptr;
    float* const square = band + (2 * a.pos.width + 1) + 4 * a.nhist + wave * SQUARE;
    const int width = a.nhist / 2;  // (distances -width .. width)
    if (want)
        for (int i = lane; i < a.nhist; i += 64) hist[i] = 0.f;

    Block<T, DK, XT> kblk;
    Block<T, DV, XT> vblk;
    kblk.init(a.ksc, a.Dk, tid);
    vblk.init(a.vsc, a.Dv, tid);
    int s_begin = 0, s_end = a.Tk;
    if (mask) attended_range(mask, s_begin, s_end, reinterpret_cast<int*>(smem));
    StepsAhead<XT> ahead;
    Steps<XT> now, next;
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
    }
    __syncthreads();
    for (int s0 = s_begin; s0 < s_end; s0 += XT) {
        if (Cut::BUFS == 2 && s0 + XT < s_end) {
            put(buf ^ 1);
            if (s0 + 2 * XT < s_end) fetch(s0 + 2 * XT);
        }
        const char* const kt = smem + buf * Cut::STAGE;
        const char* const vt = kt + KT::BYTES;
#pragma unroll
        for (int u = 0; u < XT / 32; ++u) {
            const int x0 = 32 * u;
            const unsigned word = now.tile(x0);
            if (word == 0) continue;
            const int s = s0 + x0;
            // (the scores accumulate from zero and meet m and log2 l once: on top of them every partial sum would be rounded
            // at their magnitude)
            f32x16 raw[1] = {zero16()}, dsv[1] = {dinit};
            two_scores<NP, DK, DV, XT>(kt + 2 * x0 + k_off, fq, raw, vt + 2 * x0 + v_off, fg, dsv, h);
            f32x16 &acc = raw[0], &ds = dsv[0];
            const float k1 = NP == 3 ? 1.f : c;
            int side = 0;
            if constexpr (BIAS) side = tile_side(a.pos, s, t0);
            if (BIAS && side == 0) {
                const float* const r0 = band + (int)((long long)a.pos.step * s + a.pos.offset - t0 + a.pos.width) +
                                        a.pos.step * 4 * h - l31;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    acc[r] = __builtin_fmaf(acc[r], k1, (r0[a.pos.step * ((r & 3) + 8 * (r >> 2))] - ref) - lsum);
            } else {
                const float base = !BIAS ? -(ref + lsum) : side < 0 ? side_bias[0] : side_bias[1];
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[r] = __builtin_fmaf(acc[r], k1, base);
            }
            if (word != 0xffffffffu) {
                const unsigned w = word >> (4 * h);
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[r] = (w >> ((r & 3) + 8 * (r >> 2))) & 1u ? acc[r] : -INFINITY;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) ds[r] *= __builtin_amdgcn_exp2f(acc[r]);
            if constexpr (BIAS) {
                if (want) {
                    if (side != 0) {
                        float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int r = 0; r < 16; ++r) s4[r & 3] += ds[r];
                        beyond[side > 0] += (double)((s4[0] + s4[1]) + (s4[2] + s4[3]));
                    } else {
                        // the tile goes through LDS and every lane adds up one distance's pairs (row i, column
                        // step i - distance, of the tile), 64 distances at a time
                        wave_exchange();  // (the last tile's values are read, its histogram entries written)
#pragma unroll
                        for (int r = 0; r < 16; ++r) square[acc_row(r, h) * 33 + l31] = ds[r];
                        wave_exchange();
                        const int step = a.pos.step, span = 31 * step + 32, most = (32 + step - 1) / step;
                        float* const hp = hist + (int)((long long)step * s + a.pos.offset - t0 + width) - 31;
                        for (int d0 = 0; d0 < span; d0 += 64) {
                            const int e = d0 + lane - 31;          // distance relative to the tile's first pair
                            const int i0 = e <= 0 ? 0 : (e + step - 1) / step;  // first row with a column >= 0
                            float sum = 0.f;
#pragma unroll 8
                            for (int i = 0; i < most; ++i) {
                                const int row = i0 + i, col = step * row - e;
                                const bool ok = row < 32 && col >= 0 && col < 32;
                                const float v = square[ok ? row * 33 + col : 0];
                                sum += ok ? v : 0.f;
                            }
                            if (d0 + lane < span) hp[d0 + lane] += sum;
                        }
                    }
                }
            }
            PFrag<NP> p[1];
            p[0].fill(ds);
            mma_values<NP, DK, XT, 1>(kt, x0, l31, h, p, dq);
            if (NP == 1 && a.fine) {
                p[0].fill_rest(ds);
                mma_values<NP, DK, XT, 1>(kt, x0, l31, h, p, dq);
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
    if (inside) {
        eight_rows<NP, DK>(dq[0][0]);
        T* out = reinterpret_cast<T*>(a.gq) + row * a.Dk * a.Tq + t;
#pragma unroll
        for (int i = 0; i < KT::GROUPS; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = 32 * i + acc_row(r, h);
                if (d < a.Dk && (!KT::P8 || r < 4)) st1(out + (long long)d * a.Tq, live ? dq[0][i][r] * (sign * a.scale) : 0.f);
            }
    }
    if constexpr (BIAS) {
        if (want) {
            float* const part = a.hist + ((long long)head * a.B * a.coltiles + (long long)b * a.coltiles + tile) * (a.nhist + 2);
            __syncthreads();
            const float* const all = band + (2 * a.pos.width + 1);
            for (int i = tid; i < a.nhist; i += THREADS)
                part[i] = (all[i] - all[a.nhist + i]) + (all[2 * a.nhist + i] - all[3 * a.nhist + i]);  // (their signs)
            float* const sums = reinterpret_cast<float*>(smem);
            const float s0 = wave_sum((float)beyond[0]), s1 = wave_sum((float)beyond[1]);
            if (lane == 0) {
                sums[wave] = s0;
                sums[4 + wave] = s1;
            }
            __syncthreads();
            if (tid < 2) part[a.nhist + tid] = (sums[4 * tid] - sums[4 * tid + 1]) + (sums[4 * tid + 2] - sums[4 * tid + 3]);
        }
    }
}

// WK waves along the keys, WT = 4 / WK along the queries of a stage (their sums are joined through LDS at the end).
template <class T, int DK, int DV, int WK, int XT, bool BIAS>
struct DkvCut {
    static constexpr int NP = Elem<T>::NP;
    static constexpr int STATS = BIAS ? 3 : 2;  // numbers per query
    static constexpr int STAGE = Tile<NP, DK, XT>::BYTES + Tile<NP, DV, XT>::BYTES + STATS * XT * (int)sizeof(float);
    static constexpr int BUFS = 2 * STAGE <= 80 * 1024 ? 2 : 1;
    static constexpr int WORDS = (Tile<NP, DK, XT>::GROUPS + Tile<NP, DV, XT>::GROUPS) * 16 * 64;  // a wave's sums
    static constexpr int JOIN = (4 / WK - 1) * WK * WORDS * (int)sizeof(float);
    static constexpr int LDS = BUFS * STAGE > JOIN ? BUFS * STAGE : JOIN;
};
// Two workgroups to a CU as long as a wave's columns and sums leave room in 256 registers (8 x 8 x 1024, one / two: bfloat16
// at 32 + 128 channels 78 / 54 us, at 96 94 / 111, at 128 107 / 279; float32 at 64 259 / 228, at 32 + 128 287 / 409).
template <class T, int DK, int DV, int WK, int XT, bool BIAS>
__global__ __launch_bounds__(THREADS, DK + DV > (Elem<T>::NP == 3 ? 128 : 160) ? 1 : 2) void attn_dkv_kernel(BwdArgs a) {
    typedef DkvCut<T, DK, DV, WK, XT, BIAS> Cut;
    constexpr int NP = Elem<T>::NP;
    constexpr int WT = 4 / WK, SUBS = XT / (32 * WT);
    typedef Tile<NP, DK, XT> QT;
    typedef Tile<NP, DV, XT> GT;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    // a stage: q, dO, then of its queries -delta and -(m + log2 l), with a bias -delta, -log2 l and -m

    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wk = wave % WK, wt = wave / WK;
    int bkv, part;
    place(blockIdx.x, a.B * a.KV, a.coltiles * a.nsplit, bkv, part);
    const int tile = part % a.coltiles, split = part / a.coltiles;
    const int b = bkv / a.KV, kvh = bkv - b * a.KV;
    const int H = a.KV * a.G;

    const int q_off = SRead<NP, DK, XT>::offset(lane), g_off = SRead<NP, DV, XT>::offset(lane);
    const int s_tile = (tile * WK + wk) * 32;
    const int s = s_tile + l31;
    const bool inside = s < a.Tk;
    const bool live = inside && (!a.mask || a.mask[(long long)b * a.Tk + s]);

    const bool any_live = __any(live);

    const float c = a.scale * LOG2E;
    SFrag<NP, DK> fk[1];
    SFrag<NP, DV> fv[1];
    {
        const T* k = reinterpret_cast<const T*>(a.k) + b * a.ksb + (long long)kvh * a.Dk * a.ksc;
        const T* v = reinterpret_cast<const T*>(a.v) + b * a.vsb + (long long)kvh * a.Dv * a.vsc;
        const unsigned at = live ? s : 0;
        typedef SFrag<NP, DK> FK;
        typedef SFrag<NP, DV> FV;
        float x[FK::VALUES], y[FV::VALUES];
        FK::read(k, at, a.ksc, a.Dk, h, x);
#pragma unroll
        for (int i = 0; i < FK::VALUES; ++i) x[i] = live && FK::channel(i, h) < a.Dk ? (NP == 3 ? x[i] * c : x[i]) : 0.f;
        fk[0].fill(h, x);
        FV::read(v, at, a.vsc, a.Dv, h, y);
#pragma unroll
        for (int i = 0; i < FV::VALUES; ++i) y[i] = live && FV::channel(i, h) < a.Dv ? y[i] : 0.f;
        fv[0].fill(h, y);
    }
    f32x16 dk[1][QT::GROUPS], dv[1][GT::GROUPS];
#pragma unroll
    for (int i = 0; i < QT::GROUPS; ++i) dk[0][i] = zero16();
#pragma unroll
    for (int i = 0; i < GT::GROUPS; ++i) dv[0][i] = zero16();

    const int per_head = (a.Tq + XT - 1) / XT;
    const int stages = a.G * per_head;
    const int first = (int)((long long)stages * split / a.nsplit), last = (int)((long long)stages * (split + 1) / a.nsplit);

    Block<T, DK, XT> qblk;
    Block<T, DV, XT> gblk;
    qblk.init(a.qsc, a.Dk, tid);
    gblk.init(a.Tq, a.Dv, tid);
    const long long queries = (long long)a.B * H * a.Tq;
    float stat = 0.f;
    int ahead = 0;  // first query of the stage that is on its way
    auto fetch = [&](int stage) {
        const int g = stage / per_head, t0 = (stage - g * per_head) * XT;
        const int head = kvh * a.G + g;
        const long long row = (long long)b * H + head;
        qblk.load(reinterpret_cast<const T*>(a.q) + b * a.qsb + (long long)head * a.Dk * a.qsc, t0, a.Tq, tid);
        gblk.load(reinterpret_cast<const T*>(a.g) + row * a.Dv * a.Tq, t0, a.Tq, tid);
        ahead = t0;
        if (tid < Cut::STATS * XT) {
            const int t = t0 + tid % XT, which = tid / XT;
            const long long at = row * a.Tq + min(t, a.Tq - 1);
            float x = (which == 0 ? a.delta : which == 1 ? a.lse + queries : a.lse)[at];
            if (!BIAS && which == 1) x += a.lse[at];
            stat = t < a.Tq ? -x : which == 1 ? -INFINITY : 0.f;
        }
    };
    auto put = [&](int buf) {
        char* const qt = smem + buf * Cut::STAGE;
        char* const gt = qt + QT::BYTES;
        Steps<XT> steps;
        steps.find(ahead, a.Tq, 1, lane);
        qblk.store(qt, a.Dk, steps, tid);
        gblk.store(gt, a.Dv, steps, tid);
        if (tid < Cut::STATS * XT) reinterpret_cast<float*>(gt + GT::BYTES)[tid] = stat;
    };
    // position bias: near tiles read the stage's head's band in LDS, two of them so that the next head's can be filled
    // while the last one's is in use
    float* const bands = reinterpret_cast<float*>(smem + Cut::LDS);
    float side_bias[2] = {0.f, 0.f};
    auto band_of = [&](int g) { return bands + (g & 1) * (2 * a.pos.width + 1); };
    auto put_band = [&](int g) {
        fill_band(band_of(g), a.pos, a.pos.rel + (long long)(kvh * a.G + g) * a.pos.nrel, a.Tq, tid, THREADS);
    };
    int head_now = -1;
    int buf = 0;
    if (first < last) {
        fetch(first);
        put(0);
        if (BIAS) put_band(first / per_head);
        if (first + 1 < last) fetch(first + 1);
        __syncthreads();
    }
    for (int stage = first; stage < last; ++stage) {
        if (Cut::BUFS == 2 && stage + 1 < last) {
            put(buf ^ 1);
            if (stage + 2 < last) fetch(stage + 2);
        }
        if (BIAS && stage + 1 < last && (stage + 1) / per_head != stage / per_head) put_band((stage + 1) / per_head);
        const char* const qt = smem + buf * Cut::STAGE;
        const char* const gt = qt + QT::BYTES;
        const float* const stats = reinterpret_cast<const float*>(gt + GT::BYTES);
        const int g = stage / per_head, t0 = (stage - g * per_head) * XT;
        if (BIAS && g != head_now) {
            head_now = g;
            const float* const rel = a.pos.rel + (long long)(kvh * a.G + g) * a.pos.nrel;
            side_bias[0] = rel_at(a.pos, rel, a.Tq, -a.pos.far);
            side_bias[1] = rel_at(a.pos, rel, a.Tq, a.pos.far);
        }
#pragma unroll
        for (int u = 0; u < SUBS; ++u) {
            const int x0 = 32 * (u * WT + wt);
            if (t0 + x0 >= a.Tq || !any_live) continue;  // (the same for every lane of the wave)
            f32x16 acc, raw[1] = {zero16()}, dsv[1];
            f32x16& ds = dsv[0];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 e = *reinterpret_cast<const f32x4*>(stats + x0 + 8 * i + 4 * h);
                const f32x4 f = *reinterpret_cast<const f32x4*>(stats + (BIAS ? 2 : 1) * XT + x0 + 8 * i + 4 * h);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    ds[4 * i + j] = e[j];
                    acc[4 * i + j] = f[j];
                }
            }
            if constexpr (BIAS) {
                const int t = t0 + x0, side = tile_side(a.pos, s_tile, t);
                if (side != 0) {
                    const float bias = side < 0 ? side_bias[0] : side_bias[1];
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[r] += bias;
                } else {
                    const float* const r0 = band_of(g) +
                                            (int)((long long)a.pos.step * s_tile + a.pos.offset - t + a.pos.width) +
                                            a.pos.step * l31;
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[r] += r0[-acc_row(r, h)];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 e = *reinterpret_cast<const f32x4*>(stats + XT + x0 + 8 * i + 4 * h);
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[4 * i + j] += e[j];
                }
            }
            two_scores<NP, DK, DV, XT>(qt + 2 * x0 + q_off, fk, raw, gt + 2 * x0 + g_off, fv, dsv, h);
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[r] = NP == 3 ? raw[0][r] + acc[r] : __builtin_fmaf(raw[0][r], c, acc[r]);
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[r] = __builtin_amdgcn_exp2f(acc[r]);
            PFrag<NP> p[1];
            p[0].fill(acc);
            mma_values<NP, DV, XT, 1>(gt, x0, l31, h, p, dv);
            if (NP == 1 && a.fine) {
                p[0].fill_rest(acc);
                mma_values<NP, DV, XT, 1>(gt, x0, l31, h, p, dv);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) ds[r] *= acc[r];
            p[0].fill(ds);
            mma_values<NP, DK, XT, 1>(qt, x0, l31, h, p, dk);
            if (NP == 1 && a.fine) {
                p[0].fill_rest(ds);
                mma_values<NP, DK, XT, 1>(qt, x0, l31, h, p, dk);
            }
        }
        if (stage + 1 < last) {
            __syncthreads();
            if (Cut::BUFS == 1) {
                put(0);
                if (stage + 2 < last) fetch(stage + 2);
                __syncthreads();
            } else {
                buf ^= 1;
            }
        }
    }
    if constexpr (WT > 1) {
        // the sums of the waves wt = 1 .. WT - 1 are added to those of wave wt = 0, in that order
        constexpr int WORDS = Cut::WORDS;
        float* const buf = reinterpret_cast<float*>(smem);
        __syncthreads();
        if (wt > 0) {
            float* const mine = buf + ((wt - 1) * WK + wk) * WORDS + lane;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
#pragma unroll
                for (int i = 0; i < QT::GROUPS; ++i) mine[(16 * i + r) * 64] = dk[0][i][r];
#pragma unroll
                for (int i = 0; i < GT::GROUPS; ++i) mine[(16 * (QT::GROUPS + i) + r) * 64] = dv[0][i][r];
            }
        }
        __syncthreads();
        if (wt > 0) return;
        for (int w = 1; w < WT; ++w) {
            const float* const other = buf + ((w - 1) * WK + wk) * WORDS + lane;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
#pragma unroll
                for (int i = 0; i < QT::GROUPS; ++i) dk[0][i][r] += other[(16 * i + r) * 64];
#pragma unroll
                for (int i = 0; i < GT::GROUPS; ++i) dv[0][i][r] += other[(16 * (QT::GROUPS + i) + r) * 64];
            }
        }
    }
    if (!inside) return;
    eight_rows<NP, DK>(dk[0][0]);
    auto each = [&](auto&& put_k, auto&& put_v) {
#pragma unroll
        for (int i = 0; i < QT::GROUPS; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = 32 * i + acc_row(r, h);
                if (d < a.Dk && (!QT::P8 || r < 4)) put_k(d, live ? dk[0][i][r] * a.scale : 0.f);
            }
#pragma unroll
        for (int i = 0; i < GT::GROUPS; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = 32 * i + acc_row(r, h);
                if (d < a.Dv) put_v(d, live ? dv[0][i][r] : 0.f);
            }
    };
    if (a.part == nullptr) {
        T* const gk = reinterpret_cast<T*>(a.gk) + (long long)bkv * a.Dk * a.Tk + s;
        T* const gv = reinterpret_cast<T*>(a.gv) + (long long)bkv * a.Dv * a.Tk + s;
        each([&](int d, float x) { st1(gk + (long long)d * a.Tk, x); }, [&](int d, float x) { st1(gv + (long long)d * a.Tk, x); });
    } else {
        const long long heads = (long long)a.B * a.KV;
        float* const pk = a.part + ((long long)split * heads + bkv) * a.Dk * a.Tk + s;
        float* const pv = a.part + (long long)a.nsplit * heads * a.Dk * a.Tk + ((long long)split * heads + bkv) * a.Dv * a.Tk + s;
        each([&](int d, float x) { pk[(long long)d * a.Tk] = x; }, [&](int d, float x) { pv[(long long)d * a.Tk] = x; });
    }
}

// dK and dV of a split over the queries: the parts' sums, in order.
template <class T>
__global__ __launch_bounds__(THREADS) void attn_sum_kernel(const float* part, T* gk, T* gv, long long nk, long long nv,
                                                           int nsplit) {
    const long long i = (long long)blockIdx.x * THREADS + threadIdx.x;
    if (i >= nk + nv) return;
    const bool is_k = i < nk;
    const float* p = is_k ? part + i : part + nsplit * nk + (i - nk);
    const long long n = is_k ? nk : nv;
    float s = 0.f;
    for (int j = 0; j < nsplit; ++j) s += p[j * n];
    st1(is_k ? gk + i : gv + (i - nk), s);
}

}  // namespace attn
}  // namespace eeggan

using namespace eeggan;
using namespace eeggan::attn;

namespace {

template <class T, int DK, int DV>
struct Cut {
    static constexpr bool F32 = Elem<T>::NP == 3;
    // keys of a stage (bfloat16 at 128 channels: 32 at two workgroups to a CU 105 us, 64 at one 127)
    static constexpr int DQ_XT = DK + DV > (F32 ? 96 : 128) ? 32 : 64;
    static constexpr int WIDE_XT = F32 && DK + DV > 96 ? 32 : 64;
    static constexpr bool NARROW = !(F32 && DK + DV > 96);  // has a form whose waves share keys
};
constexpr int WANTED = 512;

struct BwdPlan {
    bool narrow;
    int qtiles, ktiles, nsplit, nhist;
    size_t rel, delta, part, hist, total;
};

template <class T, int DK, int DV>
BwdPlan plan_of(const eeggan_attention& a, bool want_table) {
    typedef Cut<T, DK, DV> C;
    BwdPlan p;
    p.qtiles = (a.Tq + 127) / 128;
    const long long heads = (long long)a.B * a.KV;
    p.narrow = C::NARROW && a.Tk <= 64;
    const int keys = p.narrow ? 64 : 128, xt = p.narrow ? 64 : C::WIDE_XT;
    p.ktiles = (a.Tk + keys - 1) / keys;
    const long long blocks = heads * p.ktiles, stages = (long long)(a.H / a.KV) * ((a.Tq + xt - 1) / xt);
    long long n = blocks >= WANTED ? 1 : WANTED / blocks;
    if (n > stages / 2) n = stages / 2 > 0 ? stages / 2 : 1;
    p.nsplit = (int)n;
    p.nhist = a.table && want_table ? 2 * band_width(*a.buckets) + 1 : 0;
    auto up = [](size_t x) { return (x + 15) / 16 * 16; };
    p.rel = positions_bytes(a);
    p.delta = up((size_t)a.B * a.H * a.Tq * sizeof(float));
    p.part = n > 1 ? up((size_t)n * heads * (a.Dk + a.Dv) * a.Tk * sizeof(float)) : 0;
    p.hist = p.nhist ? up((size_t)a.H * a.B * p.qtiles * (p.nhist + 2) * sizeof(float)) : 0;
    p.total = p.rel + p.delta + p.part + p.hist;
    return p;
}

template <class T, int DK, int DV, bool BIAS>
int launch_dq(const BwdArgs& f, const BwdPlan& p, hipStream_t st) {
    constexpr int XT = Cut<T, DK, DV>::DQ_XT;
    constexpr size_t tiles = DqCut<T, DK, DV, XT>::LDS;
    constexpr size_t most = tiles + (BIAS ? (5 * MAX_BAND + 4 * SQUARE) * sizeof(float) : 0);
    static_assert(most <= 160 * 1024, "LDS");
    auto kernel = &attn_dq_kernel<T, DK, DV, XT, BIAS>;
    static LdsReady ready;
    if (ready.reserve("attention backward", reinterpret_cast<const void*>(kernel), most)) return 1;
    const long long grid = (long long)f.B * f.KV * f.G * p.qtiles;
    EEGGAN_REQUIRE(grid < (1ll << 31), "attention backward: too many workgroups");
    BwdArgs a = f;
    a.coltiles = p.qtiles;
    a.nhist = p.nhist;
    const size_t lds = tiles + (BIAS ? (2 * (size_t)f.pos.width + 1 + (p.nhist ? 4 * (size_t)(p.nhist + SQUARE) : 0)) * sizeof(float) : 0);
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(THREADS), lds, st, a);
    return check_launch("attention backward (queries)");
}

template <class T, int DK, int DV, int WK, int XT, bool BIAS>
int launch_dkv(const BwdArgs& f, const BwdPlan& p, hipStream_t st) {
    constexpr size_t tiles = DkvCut<T, DK, DV, WK, XT, BIAS>::LDS, most = tiles + (BIAS ? 2 * MAX_BAND * sizeof(float) : 0);
    const size_t lds = tiles + (BIAS ? 2 * (2 * (size_t)f.pos.width + 1) * sizeof(float) : 0);
    static_assert(most <= 160 * 1024 && 3 * XT <= THREADS, "LDS");
    auto kernel = &attn_dkv_kernel<T, DK, DV, WK, XT, BIAS>;
    static LdsReady ready;
    if (ready.reserve("attention backward", reinterpret_cast<const void*>(kernel), most)) return 1;
    const long long grid = (long long)f.B * f.KV * p.ktiles * p.nsplit;
    EEGGAN_REQUIRE(grid < (1ll << 31), "attention backward: too many workgroups");
    BwdArgs a = f;
    a.coltiles = p.ktiles;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(THREADS), lds, st, a);
    return check_launch("attention backward (keys)");
}

template <class T, int DK, int DV, bool BIAS>
int backward(const BwdArgs& f, const BwdPlan& p, hipStream_t st) {
    typedef Cut<T, DK, DV> C;
    if (launch_dq<T, DK, DV, BIAS>(f, p, st)) return 1;
    if (!f.gk) return 0;
    if constexpr (C::NARROW) {
        if (p.narrow) return launch_dkv<T, DK, DV, 2, 64, BIAS>(f, p, st);
    }
    return launch_dkv<T, DK, DV, 4, C::WIDE_XT, BIAS>(f, p, st);
}

template <class T, int DK, int DV>
int backward_all(const eeggan_attention& a, const void* out, const void* rest, const float* lse, const void* g, void* gq, void* gk, void* gv,
                 void* g_table, char* ws, size_t bytes, hipStream_t st) {
    const BwdPlan p = plan_of<T, DK, DV>(a, g_table != nullptr);
    EEGGAN_REQUIRE(bytes >= p.total, "attention backward: workspace too small");
    BwdArgs f;
    f.q = a.q, f.k = a.k, f.v = a.v;
    f.qsb = a.q_batch, f.qsc = a.q_channel, f.ksb = a.k_batch, f.ksc = a.k_channel, f.vsb = a.v_batch, f.vsc = a.v_channel;
    f.mask = a.mask, f.out = out, f.rest = rest, f.g = g, f.lse = lse, f.gq = gq, f.gk = gk, f.gv = gv;
    f.delta = reinterpret_cast<float*>(ws + p.rel);
    f.part = p.nsplit > 1 ? reinterpret_cast<float*>(ws + p.rel + p.delta) : nullptr;
    f.hist = p.nhist ? reinterpret_cast<float*>(ws + p.rel + p.delta + p.part) : nullptr;
    f.B = a.B, f.KV = a.KV, f.G = a.H / a.KV, f.Dk = a.Dk, f.Dv = a.Dv, f.Tq = a.Tq, f.Tk = a.Tk;
    f.coltiles = 0, f.nsplit = p.nsplit, f.nhist = 0, f.scale = a.scale, f.fine = fine_backward(a);
    if (positions(a, reinterpret_cast<float*>(ws), &f.pos, st)) return 1;
    if (a.table ? backward<T, DK, DV, true>(f, p, st) : backward<T, DK, DV, false>(f, p, st)) return 1;
    if (p.nsplit > 1 && gk) {
        const long long nk = (long long)a.B * a.KV * a.Dk * a.Tk, nv = (long long)a.B * a.KV * a.Dv * a.Tk;
        const long long blocks = (nk + nv + THREADS - 1) / THREADS;
        EEGGAN_REQUIRE(blocks < (1ll << 31), "attention backward: too many outputs");
        hipLaunchKernelGGL(attn_sum_kernel<T>, dim3((unsigned)blocks), dim3(THREADS), 0, st, f.part, reinterpret_cast<T*>(gk),
                           reinterpret_cast<T*>(gv), nk, nv, p.nsplit);
        if (check_launch("attention backward (sums)")) return 1;
    }
    if (p.nhist) {
        return bucket_sums(f.hist, g_table, a.table_bf16, *a.buckets, a.H, (long long)a.B * p.qtiles, p.nhist / 2, st);
    }
    return 0;
}

}  // namespace

extern "C" size_t eeggan_attention_bwd_workspace(const eeggan_attention* a, int want_table) {
    if (check_attention("attention backward", a)) return 0;
    size_t n = 0;
    EEGGAN_ATTENTION_CLASS(*a, n = (plan_of<T, DK, DV>(*a, want_table != 0).total))
    return n;
}

extern "C" int eeggan_attention_bwd(const eeggan_attention* a, const void* out, const void* rest, const float* lse,
                                    const void* g, void* gq, void* gk, void* gv, void* g_table, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    if (check_attention("attention backward", a)) return 1;
    EEGGAN_REQUIRE(out && lse && g && gq && !gk == !gv && workspace, "attention backward: null pointer");
    EEGGAN_REQUIRE(!a->bf16 || rest, "attention backward: bfloat16 needs the rest of the output");
    EEGGAN_REQUIRE(!g_table || a->table, "attention backward: a table gradient without a table");
    int rc = 1;
    EEGGAN_ATTENTION_CLASS(*a, rc = (backward_all<T, DK, DV>(*a, out, rest, lse, g, gq, gk, gv, g_table,
                                                             reinterpret_cast<char*>(workspace), workspace_bytes,
                                                             as_stream(stream))))
    return rc;
}
