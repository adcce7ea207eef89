// Learned relative position bias by buckets: on stored scores, its gradient, and the per-distance table the fused
// attention reads.  (bucket, head) sums run in a fixed order.
#include "attention_host.h"

namespace eeggan {
namespace attn {
namespace {

constexpr int MAX_T = 1 << 27;  // time steps of one call

// the first n (1 .. 3) of four values, the rest zero
__device__ __forceinline__ f32x4 load_few(const float* p, int n) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    v[0] = p[0];
    if (n > 1) v[1] = p[1];
    if (n > 2) v[2] = p[2];
    return v;
}

// rel[head][i] = log2(e) * table[bucket(first + i)][head]; entries at or below -1e30 (a mask written into the table, the
// type's lowest value among them) bar the pair.
template <class T>
__global__ __launch_bounds__(256) void positions_kernel(const T* __restrict__ table, float* __restrict__ rel,
                                                        eeggan_buckets bk, int heads, int nrel, int first) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= nrel) return;
    const int head = blockIdx.y;
    const float v = ld1(table + (long long)bucket_of(bk, (long long)first + i) * heads + head);
    rel[(long long)head * nrel + i] = v <= -1e30f ? -INFINITY : v * LOG2E;
}

// The bias of one head by distance, -far .. far, in LDS: what lies beyond has the value at the border.
__device__ __forceinline__ void fill_lut(float* lut, const float* table, const eeggan_buckets& bk, int H, int h, int far) {
    for (int i = threadIdx.x; i <= 2 * far; i += 256) lut[i] = table[(long long)bucket_of(bk, far - i) * H + h];
}

// out[n, s, t] = scores[n, s, t] + table[bucket(step s + offset - t), n % H].  A pure stream: a workgroup takes `rows`
// consecutive rows (n, s) of one n, its threads neighbouring groups of four steps; the value comes from LDS (one read
// per element, a tenth of what LDS can deliver at the rate the memory can).
// NT: streaming accesses; HAVE: with scores.  Measured at 64 maps of 1920 x 1920: 357 us, 5.3 TB/s read and written.
template <bool NT, bool HAVE>
__global__ __launch_bounds__(256) void relbias_kernel(const float* __restrict__ scores, const float* __restrict__ table,
                                                      float* __restrict__ out, eeggan_buckets bk, int H, int Tk, int Tq,
                                                      int rows, int chunks) {
    extern __shared__ float lut[];
    const int far = bucket_far(bk);
    const long long n = blockIdx.x / chunks;
    const int s0 = (int)(blockIdx.x % chunks) * rows;
    const int s1 = min(Tk, s0 + rows);
    fill_lut(lut, table, bk, H, (int)(n % H), far);
    __syncthreads();
    if (Tq < 4) {
        for (int i = threadIdx.x; i < (s1 - s0) * Tq; i += 256) {
            const int s = s0 + i / Tq, t = i % Tq;
            const long long at = (n * Tk + s) * Tq + t, d = (long long)t - (long long)bk.step * s - bk.offset + far;
            out[at] = (scores ? scores[at] : 0.f) + lut[d < 0 ? 0 : d > 2 * far ? 2 * far : (int)d];
        }
        return;
    }
    // a row's last quad starts at Tq - 4: where it overlaps its neighbour both store the same values
    const int quads = (Tq + 3) / 4;
    const int drow = 256 / quads, dq = 256 % quads;  // (a thread's next item, without a division per item)
    int s = s0 + (int)threadIdx.x / quads, q = (int)threadIdx.x % quads;
    const long long first = n * Tk * Tq;
    constexpr int U = 4;  // items in flight per thread (past the end: the last row again, not stored)
    while (s < s1) {
        int is[U], it[U];
        f32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            is[u] = s, it[u] = min(4 * q, Tq - 4);
            const f32x4u* p = reinterpret_cast<const f32x4u*>(scores + first + (long long)min(s, s1 - 1) * Tq + it[u]);
            const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
            v[u] = HAVE ? (f32x4)(NT ? __builtin_nontemporal_load(p) : *p) : zero;
            q += dq;
            s += drow;
            if (q >= quads) {
                q -= quads;
                ++s;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // lut index of the quad's first step (far outside: just outside)
            const long long wide = (long long)it[u] - (long long)bk.step * is[u] - bk.offset + far;
            const int i0 = (int)(wide < -4 ? -4 : wide > 2 * far ? 2 * far : wide);
            f32x4u o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = v[u][e] + lut[min(max(i0 + e, 0), 2 * far)];
            f32x4u* p = reinterpret_cast<f32x4u*>(out + first + (long long)is[u] * Tq + it[u]);
            if (is[u] < s1) {
                if (NT) __builtin_nontemporal_store(o, p);
                else *p = o;
            }
        }
    }
}

// Sums of g by distance.  A wave takes every fourth of its workgroup's rows, 2048 values of a row at a time with all
// loads in flight.  Four neighbouring values beyond the last edge on one side (most of a long row) go to one sum; the
// others to a histogram by distance in LDS that belongs to the wave (within an instruction no two lanes share a
// distance): a fixed order, and in double (the near entries of a long recording sum millions of terms) but for
// those four, which are added in float32.
// 64 maps of 1920 x 1920: 168 us, 5.6 TB/s.  hist: [H][rows of partial sums][2 far + 1]: distances -(far - 1) .. far - 1,
// then everything behind, then everything ahead.
__global__ __launch_bounds__(256) void relbias_sums_kernel(const float* __restrict__ g, double* __restrict__ hist,
                                                           eeggan_buckets bk, int B, int H, int Tk, int Tq, int rows,
                                                           int chunks) {
    extern __shared__ double band[];
    const int far = bucket_far(bk), width = far - 1, n = 2 * width + 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double* const mine = band + wave * (n + 2);
    for (int i = lane; i < n + 2; i += 64) mine[i] = 0.0;
    wave_exchange();
    const long long bh = blockIdx.x / chunks;
    const int chunk = (int)(blockIdx.x % chunks);
    const int s0 = chunk * rows, s1 = min(Tk, s0 + rows);
    double behind = 0.0, ahead = 0.0;
    constexpr int U = 8;
    for (int s = s0 + wave; s < s1; s += 4) {
        const float* row = g + (bh * Tk + s) * Tq;
        const long long key = (long long)bk.step * s + bk.offset;  // distance of step t: key - t
        // steps [0, a): ahead of them by `far` or more; [a, b): the band; [b, Tq): behind
        const int a = (int)min((long long)Tq, max(0ll, key - far + 1)), b = (int)min((long long)Tq, max(0ll, key + far));
        const int at_a = (int)(key - a + width);  // histogram entry of step a (meaningful where the band has steps)
        for (int t0 = 0; t0 < Tq; t0 += 256 * U) {
            f32x4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                // (a row's last values are read in the quad that starts at Tq - 4 and moved to their places below)
                const int t = t0 + 256 * u + 4 * lane;
                v[u] = Tq >= 4 ? load4(row + min(t, Tq - 4)) : load_few(row, Tq);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int t = t0 + 256 * u + 4 * lane, over = Tq >= 4 ? t - min(t, Tq - 4) : t;
                if (over > 0) {
                    const f32x4 w = v[u];
                    v[u][0] = over == 1 ? w[1] : over == 2 ? w[2] : over == 3 ? w[3] : 0.f;
                    v[u][1] = over == 1 ? w[2] : over == 2 ? w[3] : 0.f;
                    v[u][2] = over == 1 ? w[3] : 0.f;
                    v[u][3] = 0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int t = t0 + 256 * u + 4 * lane;
                if (t + 4 <= a) {
                    ahead += (double)((v[u][0] + v[u][1]) + (v[u][2] + v[u][3]));
                } else if (t >= b) {
                    behind += (double)((v[u][0] + v[u][1]) + (v[u][2] + v[u][3]));  // (zeros past the row)
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (t + e < a) ahead += (double)v[u][e];
                        else if (t + e >= b) behind += (double)v[u][e];
                        else
                            __hip_atomic_fetch_add(mine + (at_a - (t + e - a)), (double)v[u][e], __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_WORKGROUP);
                    }
                }
            }
        }
    }
    for (int o = 32; o > 0; o >>= 1) {
        behind += __shfl_xor(behind, o, 64);
        ahead += __shfl_xor(ahead, o, 64);
    }
    if (lane == 0) {
        mine[n] = behind;
        mine[n + 1] = ahead;
    }
    __syncthreads();
    const long long b = bh / H, h = bh % H;
    double* const out = hist + ((h * B + b) * chunks + chunk) * (n + 2);
    for (int i = threadIdx.x; i < n + 2; i += 256)
        out[i] = (band[i] + band[n + 2 + i]) + (band[2 * (n + 2) + i] + band[3 * (n + 2) + i]);
}

// Bucket sums from histograms by distance (-width .. width, behind, ahead): one workgroup per (bucket, head); a bucket
// is a stretch of the histogram.
template <class TH, class TO>
__global__ __launch_bounds__(256) void bucket_sums_kernel(const TH* __restrict__ hist, TO* __restrict__ out, eeggan_buckets bk,
                                                          int H, long long rows, int width) {
    __shared__ double red[256];
    const int j = blockIdx.x, head = blockIdx.y, side = bucket_side(bk);
    const bool ahead = j >= side;
    const int e = ahead ? j - side : j;
    const bool last = e == side - 1;
    const int near = bk.edges[e], beyond = last ? width : min(width, bk.edges[last ? e : e + 1] - 1);
    int lo, hi;
    if (ahead) {
        lo = width + max(near, 1);
        hi = width + beyond;
    } else {
        lo = width - beyond;
        hi = !bk.bidirectional && e == 0 ? 2 * width : width - near;
    }
    const int behind_at = last && !ahead ? 2 * width + 1 : -1;
    const int ahead_at = (ahead && last) || (!bk.bidirectional && e == 0) ? 2 * width + 2 : -1;
    const int n = max(0, hi - lo + 1), stride = 2 * width + 3;
    const TH* const h0 = hist + (long long)head * rows * stride;
    double sum = 0.0;
    if (n > 0) {
        // neighbouring threads on neighbouring entries, as many rows at a time as fit, eight loads in flight
        const int w = min(n, 256), at = (int)threadIdx.x % w, step = 256 / w, r0 = (int)threadIdx.x / w;
        if (r0 < step)
            for (int i = at; i < n; i += w) {
                const TH* p = h0 + lo + i;
#pragma unroll 8
                for (int r = r0; r < (int)rows; r += step) sum += (double)p[(long long)r * stride];
            }
    }
    for (long long r = threadIdx.x; r < rows; r += 256) {
        if (behind_at >= 0) sum += (double)h0[r * stride + behind_at];
        if (ahead_at >= 0) sum += (double)h0[r * stride + ahead_at];
    }
    red[threadIdx.x] = sum;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) st1(out + (long long)j * H + head, (float)red[0]);
}

}  // namespace

int check_attention(const char* what, const eeggan_attention* a) {
    EEGGAN_REQUIRE(a && a->q && a->k && a->v, "%s: null pointer", what);
    EEGGAN_REQUIRE(a->B > 0 && a->H > 0 && a->KV > 0 && a->Tq > 0 && a->Tk > 0 && a->Dk > 0 && a->Dv > 0,
                   "%s: bad shape (B=%d H=%d KV=%d Dk=%d Dv=%d Tq=%d Tk=%d)", what, a->B, a->H, a->KV, a->Dk, a->Dv, a->Tq,
                   a->Tk);
    EEGGAN_REQUIRE(a->H % a->KV == 0, "%s: %d query heads cannot share %d key heads", what, a->H, a->KV);
    EEGGAN_REQUIRE(a->Dk <= 128 && a->Dv <= 128, "%s: heads of up to 128 channels, got %d and %d", what, a->Dk, a->Dv);
    EEGGAN_REQUIRE(a->Tq <= MAX_T && a->Tk <= MAX_T && (long long)(a->H / a->KV) * a->Tq <= MAX_T,
                   "%s: more than %d time steps", what, MAX_T);
    EEGGAN_REQUIRE(a->q_batch >= 0 && a->q_channel >= 0 && a->k_batch >= 0 && a->k_channel >= 0 && a->v_batch >= 0 &&
                       a->v_channel >= 0,
                   "%s: negative stride", what);
    // (a head's rows are addressed with 32-bit byte offsets)
    const int64_t reach = (1ll << 31) / (128 * (a->bf16 ? 2 : 4));
    EEGGAN_REQUIRE(a->q_channel <= reach && a->k_channel <= reach && a->v_channel <= reach && a->Tq <= reach,
                   "%s: channel strides beyond %lld elements", what, (long long)reach);
    const uintptr_t odd = a->bf16 ? 1 : 3;
    EEGGAN_REQUIRE(((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) |
                     reinterpret_cast<uintptr_t>(a->v)) & odd) == 0, "%s: misaligned tensor", what);
    if (a->table) {
        if (check_buckets(what, a->buckets)) return 1;
        EEGGAN_REQUIRE(positions_entries(*a) < (1ll << 30), "%s: positions out of range", what);
        EEGGAN_REQUIRE(a->H <= 65535, "%s: too many heads", what);
    }
    return 0;
}

int positions(const eeggan_attention& a, float* rel, Positions* p, hipStream_t st) {
    if (!a.table) {
        *p = Positions{nullptr, 0, 1, 0, 1, 0};
        return 0;
    }
    const eeggan_buckets bk = *a.buckets;
    const int nrel = (int)positions_entries(a);
    *p = Positions{rel, nrel, bk.step, bk.offset, bucket_far(bk), band_width(bk)};
    const dim3 grid((unsigned)((nrel + 255) / 256), (unsigned)a.H);
    const int first = bk.offset - (a.Tq - 1);
    if (a.table_bf16)
        hipLaunchKernelGGL(positions_kernel<__bf16>, grid, dim3(256), 0, st, reinterpret_cast<const __bf16*>(a.table), rel,
                           bk, a.H, nrel, first);
    else
        hipLaunchKernelGGL(positions_kernel<float>, grid, dim3(256), 0, st, reinterpret_cast<const float*>(a.table), rel, bk,
                           a.H, nrel, first);
    return check_launch("attention (positions)");
}

int bucket_sums(const float* hist, void* out, int out_bf16, const eeggan_buckets& bk, int H, long long rows, int width,
                hipStream_t st) {
    const dim3 grid((unsigned)bk.count, (unsigned)H);
    if (out_bf16)
        hipLaunchKernelGGL((bucket_sums_kernel<float, __bf16>), grid, dim3(256), 0, st, hist, reinterpret_cast<__bf16*>(out),
                           bk, H, rows, width);
    else
        hipLaunchKernelGGL((bucket_sums_kernel<float, float>), grid, dim3(256), 0, st, hist, reinterpret_cast<float*>(out),
                           bk, H, rows, width);
    return check_launch("attention backward (table)");
}

}  // namespace attn
}  // namespace eeggan

using namespace eeggan;
using namespace eeggan::attn;

static int check_relbias(const char* what, const eeggan_buckets* b, int B, int H, int Tk, int Tq) {
    EEGGAN_REQUIRE(B > 0 && H > 0 && Tk > 0 && Tq > 0 && Tk <= MAX_T && Tq <= MAX_T && H <= 65535,
                   "%s: bad shape (B=%d H=%d Tk=%d Tq=%d)", what, B, H, Tk, Tq);
    return check_buckets(what, b);
}

namespace {
struct Rows {
    int rows, chunks;
    long long blocks;
};
// rows (n, s) of one n per workgroup, for about `elements` elements, and the number of workgroups
Rows rows_of(long long n, int Tk, int Tq, long long elements) {
    long long rows = elements / Tq;
    rows = rows < 4 ? 4 : rows;
    if (rows > Tk) rows = Tk;
    Rows r;
    r.rows = (int)rows;
    r.chunks = (int)((Tk + rows - 1) / rows);
    r.blocks = n * r.chunks;
    return r;
}
// sums: at most ~2048 workgroups (their partial sums are read again), at least 4 rows each
Rows sum_rows_of(long long n, int Tk, int Tq) {
    const long long total = n * Tk * (long long)Tq;
    return rows_of(n, Tk, Tq, total / 2048 > 32768 ? total / 2048 : 32768);
}
}  // namespace

extern "C" int eeggan_relative_bias(const float* scores, const float* table, const eeggan_buckets* buckets, float* out,
                                    int B, int H, int Tk, int Tq, void* stream) {
    EEGGAN_REQUIRE(table && out, "relative_bias: null pointer");
    if (check_relbias("relative_bias", buckets, B, H, Tk, Tq)) return 1;
    // 16 K elements to a workgroup: enough to hide its start (the table in LDS), few enough to fill the chip
    const Rows r = rows_of((long long)B * H, Tk, Tq, 16384);
    EEGGAN_REQUIRE(r.blocks < (1ll << 31), "relative_bias: too many rows");
    const size_t lds = (2 * (size_t)bucket_far(*buckets) + 1) * sizeof(float);
    const dim3 grid((unsigned)r.blocks);
    const bool nt = streams_past_caches((size_t)B * H * Tk * Tq * sizeof(float) * (scores ? 2 : 1));
    auto kernel = nt ? (scores ? &relbias_kernel<true, true> : &relbias_kernel<true, false>)
                     : (scores ? &relbias_kernel<false, true> : &relbias_kernel<false, false>);
    hipLaunchKernelGGL(kernel, grid, dim3(256), lds, as_stream(stream), scores, table, out, *buckets, H, Tk, Tq, r.rows, r.chunks);
    return check_launch("relative_bias");
}

extern "C" size_t eeggan_relative_bias_grad_workspace(const eeggan_buckets* buckets, int B, int H, int Tk, int Tq) {
    if (check_relbias("relative_bias_grad", buckets, B, H, Tk, Tq)) return 0;
    return (size_t)sum_rows_of((long long)B * H, Tk, Tq).blocks * (2 * (size_t)bucket_far(*buckets) + 1) * sizeof(double);
}

extern "C" int eeggan_relative_bias_grad(const float* g, const eeggan_buckets* buckets, float* g_table, int B, int H,
                                         int Tk, int Tq, void* workspace, size_t workspace_bytes, void* stream) {
    EEGGAN_REQUIRE(g && g_table && workspace, "relative_bias_grad: null pointer");
    if (check_relbias("relative_bias_grad", buckets, B, H, Tk, Tq)) return 1;
    EEGGAN_REQUIRE(workspace_bytes >= eeggan_relative_bias_grad_workspace(buckets, B, H, Tk, Tq) &&
                       (reinterpret_cast<uintptr_t>(workspace) & 7) == 0,
                   "relative_bias_grad: workspace too small or misaligned");
    const Rows r = sum_rows_of((long long)B * H, Tk, Tq);
    EEGGAN_REQUIRE(r.blocks < (1ll << 31), "relative_bias_grad: too many rows");
    const int far = bucket_far(*buckets);
    const size_t lds = 4 * (2 * (size_t)far + 1) * sizeof(double);
    static LdsReady ready;
    if (ready.reserve("relative_bias_grad", reinterpret_cast<const void*>(&relbias_sums_kernel), 4 * 2049 * sizeof(double)))
        return 1;
    double* const hist = reinterpret_cast<double*>(workspace);
    hipStream_t st = as_stream(stream);
    hipLaunchKernelGGL(relbias_sums_kernel, dim3((unsigned)r.blocks), dim3(256), lds, st, g, hist, *buckets, B, H, Tk, Tq,
                       r.rows, r.chunks);
    if (check_launch("relative_bias_grad")) return 1;
    hipLaunchKernelGGL((bucket_sums_kernel<double, float>), dim3((unsigned)buckets->count, (unsigned)H), dim3(256), 0, st, hist,
                       g_table, *buckets, H, (long long)B * r.chunks, far - 1);
    return check_launch("relative_bias_grad (buckets)");
}
