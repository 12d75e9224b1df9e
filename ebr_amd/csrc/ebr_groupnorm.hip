// Group norm with an activation over channels-last tensors [B, L, C] on gfx950, with its first and second derivatives (C
// ABI: include/ebr_block.h).
//
// A group is L cells of cg = C / groups channels, m = L cg elements. With its mean mu and r = (variance + eps)^-1/2:
//   h = (x - mu) r,  a = w h + b,  y = f(a);   P(v) = r (v - mean v - h mean(v h)) carries a gradient of h back to x
//   backward:    da = dy f'(a),  k = w da,  dx = P(k),  dw = sum da h,  db = sum da
//   backward2 (cotangents u of dx, uw of dw, ub of db):  q = w P(u) + uw h + ub,  t = dy f''(a) q
//     gdy = f'(a) q,  gw = sum (da P(u) + t h),  gb = sum t
//     gx = P(v) - r^2 h (mean(k u) - mean k mean u - mean(u h) mean(k h)),  v = w t + uw da - r (u mean(k h) + k mean(u h))
//
// Every mean above is a weighted sum over channels of per-channel sums of u, u h, da, da h, da u and, as q is linear in 1,
// h and u with factors that are constant in a channel and group, of s, s h, s h^2, s u, s u h with s = dy f''(a): one pass
// over the tensors gives them all, a second writes the outputs. A thread keeps the same channels over all its cells, so the
// sums need no exchange until the end, and the parameters' gradients come out of the same sums.
//
// Variances are never taken as a difference of squares: eight cells at a time give a mean and the squares about it, and
// these go together by the rule for the variance of a union.
#include <type_traits>

#include "rowwise.hpp"

namespace ebr_gn {

using namespace ebr_row;

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int SUMS[3] = {2, 2, 10};   // of a mode; mode 0: the mean and the squares about it
constexpr int MEANS[3] = {2, 2, 6};   // kept of a group: mode 0: mu, r; 1: mean k, mean(k h); 2: see Group2

struct Args {
    const void *x, *dy, *u;
    const void *w, *b, *uw, *ub;  // of the accumulation type, or null
    void *y, *gdy;                // y: also dx and gx
    void *stats;                  // [B][G][2]: mu, r
    void *part;                   // [B][splits][sums][C]
    void *means;                  // [B][G][MEANS]
    void *chan;                   // [B][2][C]: a sample's share of dw and db (gw and gb)
    void *dw, *db;
    int64_t B, L;
    int C, G, cg;
    int tx, tiles, splits;  // threads across the channels, workgroups across them, parts of L
    int64_t rows;           // of a part
    double eps;
};

__device__ __forceinline__ float pow_e(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896f); }
__device__ __forceinline__ double pow_e(double x) { return exp(x); }
__device__ __forceinline__ float inverse(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ double inverse(double x) { return 1.0 / x; }

// The activation's value, or its first two derivatives. ACT 0: none, 1: silu.
template <int ACT, typename A> __device__ __forceinline__ A act(A a) {
    if constexpr (ACT == 0) return a;
    return a * inverse((A)1 + pow_e(-a));
}
template <int ACT, typename A> __device__ __forceinline__ void slopes(A a, A& f1, A& f2) {
    if constexpr (ACT == 0) {
        f1 = 1;
        f2 = 0;
    } else {
        const A s = inverse((A)1 + pow_e(-a));
        f1 = s * ((A)1 + a * ((A)1 - s));
        f2 = s * ((A)1 - s) * ((A)2 + a * ((A)1 - (A)2 * s));
    }
}

// n values' mean and squares about it, together with those of others.
template <typename A> struct Spread {
    A n, mean, m2;
    __device__ __forceinline__ void merge(A on, A omean, A om2) {
        const A all = n + on;
        if (all == (A)0) return;
        const A d = omean - mean, f = on / all;
        mean += d * f;
        m2 += om2 + d * d * n * f;
        n = all;
    }
};

template <typename A> __device__ __forceinline__ A param(const void* p, int c, A none) {
    return p ? reinterpret_cast<const A*>(p)[c] : none;
}

// What a thread knows of its channels.
template <typename A, int VEC> struct Channels {
    A mu[VEC], r[VEC], w[VEC], b[VEC];
    __device__ __forceinline__ void load(const Args& a, int64_t n, int c) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const A* s = reinterpret_cast<const A*>(a.stats) + (n * a.G + (c + e) / a.cg) * 2;
            mu[e] = s[0];
            r[e] = s[1];
            w[e] = param<A>(a.w, c + e, (A)1);
            b[e] = param<A>(a.b, c + e, (A)0);
        }
    }
};

// A workgroup's place: sample, part of L, channels of this thread, and its first and last cell.
struct Place {
    int64_t n, from, to;
    int split, c, ty, step;
    bool on;
};
template <int VEC> __device__ __forceinline__ Place place(const Args& a) {
    Place p;
    int64_t i = blockIdx.x;
    const int tile = (int)(i % a.tiles);
    i /= a.tiles;
    p.split = (int)(i % a.splits);
    p.n = i / a.splits;
    p.c = (tile * a.tx + threadIdx.x % a.tx) * VEC;
    p.ty = threadIdx.x / a.tx;
    p.step = THREADS / a.tx;
    p.on = p.c < a.C;
    p.from = p.split * a.rows;
    p.to = p.from + a.rows < a.L ? p.from + a.rows : a.L;
    return p;
}

// Per-channel sums of a part of L.
template <typename T, int VEC, int MODE, int ACT> __global__ __launch_bounds__(THREADS) void k_sums(Args a) {
    using A = typename Acc<T>::type;
    constexpr int NS = MODE == 0 ? 2 : MODE == 1 ? 2 : ACT ? 10 : 5, NL = MODE == 0 ? 3 : NS;
    __shared__ A lds[WAVES][64 * VEC];
    const Place p = place<VEC>(a);
    const int64_t base = p.n * a.L * a.C + p.c;
    A s[NL][VEC];
#pragma unroll
    for (int i = 0; i < NL; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[i][e] = 0;
    if (p.on) {
        if constexpr (MODE == 0) {
            for (int64_t l = p.from + p.ty; l < p.to; l += 8 * (int64_t)p.step) {
                Pack<T, VEC> x[8];
                int n = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int64_t row = l + (int64_t)i * p.step;
                    if (row < p.to) {
                        x[i] = ldp<T, VEC>(reinterpret_cast<const T*>(a.x) + base + row * a.C);
                        ++n;
                    }
                }
                const A f = (A)1 / (A)n;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    A mean = 0, m2 = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i < n) mean += (A)x[i].e[e];
                    mean *= f;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i < n) m2 += ((A)x[i].e[e] - mean) * ((A)x[i].e[e] - mean);
                    Spread<A> v = {s[2][e], s[0][e], s[1][e]};
                    v.merge((A)n, mean, m2);
                    s[2][e] = v.n;
                    s[0][e] = v.mean;
                    s[1][e] = v.m2;
                }
            }
        } else {
            Channels<A, VEC> ch;
            ch.load(a, p.n, p.c);
            for (int64_t l = p.from + p.ty; l < p.to; l += p.step) {
                const int64_t at = base + l * a.C;
                const Pack<T, VEC> x = ldp<T, VEC>(reinterpret_cast<const T*>(a.x) + at);
                const Pack<T, VEC> dy = ldp<T, VEC>(reinterpret_cast<const T*>(a.dy) + at);
                Pack<T, VEC> u;
                if constexpr (MODE == 2) u = ldp<T, VEC>(reinterpret_cast<const T*>(a.u) + at);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const A h = ((A)x.e[e] - ch.mu[e]) * ch.r[e];
                    A f1, f2;
                    slopes<ACT, A>(ch.w[e] * h + ch.b[e], f1, f2);
                    const A da = (A)dy.e[e] * f1;
                    if constexpr (MODE == 1) {
                        s[0][e] += da;
                        s[1][e] += da * h;
                    } else {
                        const A uv = (A)u.e[e];
                        s[0][e] += uv;
                        s[1][e] += uv * h;
                        s[2][e] += da;
                        s[3][e] += da * h;
                        s[4][e] += da * uv;
                        if constexpr (ACT != 0) {
                            const A t = (A)dy.e[e] * f2;
                            s[5][e] += t;
                            s[6][e] += t * h;
                            s[7][e] += t * h * h;
                            s[8][e] += t * uv;
                            s[9][e] += t * uv * h;
                        }
                    }
                }
            }
        }
    }
    // over the threads of the same channels: in a wave, then over the waves
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if constexpr (MODE == 0) {
        for (int d = a.tx; d < 64; d <<= 1)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                Spread<A> v = {s[2][e], s[0][e], s[1][e]};
                v.merge(__shfl_xor(v.n, d, 64), __shfl_xor(v.mean, d, 64), __shfl_xor(v.m2, d, 64));
                s[2][e] = v.n;
                s[0][e] = v.mean;
                s[1][e] = v.m2;
            }
    } else {
        for (int d = a.tx; d < 64; d <<= 1)
#pragma unroll
            for (int i = 0; i < NL; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) s[i][e] += __shfl_xor(s[i][e], d, 64);
    }
    A* part = reinterpret_cast<A*>(a.part) + (p.n * a.splits + p.split) * NS * a.C + p.c;
    A got[WAVES][NL][VEC];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        __syncthreads();
        if (lane < a.tx)
#pragma unroll
            for (int e = 0; e < VEC; ++e) lds[wave][lane * VEC + e] = s[i][e];
        __syncthreads();
        if ((int)threadIdx.x < a.tx)
#pragma unroll
            for (int w = 0; w < WAVES; ++w)
#pragma unroll
                for (int e = 0; e < VEC; ++e) got[w][i][e] = lds[w][lane * VEC + e];
    }
    if ((int)threadIdx.x >= a.tx || !p.on) return;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        if constexpr (MODE == 0) {
            Spread<A> v = {got[0][2][e], got[0][0][e], got[0][1][e]};
#pragma unroll
            for (int w = 1; w < WAVES; ++w) v.merge(got[w][2][e], got[w][0][e], got[w][1][e]);
            part[e] = v.mean;
            part[a.C + e] = v.m2;
        } else {
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                A v = got[0][i][e];
#pragma unroll
                for (int w = 1; w < WAVES; ++w) v += got[w][i][e];
                part[i * a.C + e] = v;
            }
        }
    }
}

// A sum over a workgroup of doubles, for everyone.
__device__ __forceinline__ double all_sum(double v, double* lds) {
    v = lanes_sum<64>(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v += lds[w];
    return v;
}

// One group of one sample: its means from the per-channel sums, and its channels' share of the parameters' gradients.
// These few sums are taken in 64 bits: differences of means follow.
template <typename A, int MODE, int ACT> __global__ __launch_bounds__(THREADS) void k_means(Args a) {
    constexpr int NS = MODE == 0 ? 2 : MODE == 1 ? 2 : ACT ? 10 : 5;
    __shared__ double lds[WAVES];
    const int64_t n = blockIdx.x / a.G;
    const int g = (int)(blockIdx.x % a.G), c0 = g * a.cg, c1 = c0 + a.cg;
    const double m = (double)a.L * a.cg;
    const A* part = reinterpret_cast<const A*>(a.part) + n * a.splits * NS * a.C;
    const auto total = [&](int i, int c) {
        double v = 0;
        for (int s = 0; s < a.splits; ++s) v += (double)part[((int64_t)s * NS + i) * a.C + c];
        return v;
    };
    const auto cells = [&](int s) { return (double)(s + 1 < a.splits ? a.rows : a.L - s * a.rows); };
    A* stats = reinterpret_cast<A*>(a.stats) + (n * a.G + g) * 2;
    if constexpr (MODE == 0) {
        double v = 0;
        for (int c = c0 + threadIdx.x; c < c1; c += blockDim.x)
            for (int s = 0; s < a.splits; ++s) v += cells(s) * (double)part[(int64_t)s * 2 * a.C + c];
        const double mu = all_sum(v, lds) / m;
        v = 0;
        for (int c = c0 + threadIdx.x; c < c1; c += blockDim.x)
            for (int s = 0; s < a.splits; ++s) {
                const double d = (double)part[(int64_t)s * 2 * a.C + c] - mu;
                v += (double)part[((int64_t)s * 2 + 1) * a.C + c] + cells(s) * d * d;
            }
        const double var = all_sum(v, lds) / m;
        if (threadIdx.x == 0) {
            stats[0] = (A)mu;
            stats[1] = (A)(1.0 / sqrt(var + a.eps));
        }
        return;
    }
    const double r = (double)stats[1];
    A* out = reinterpret_cast<A*>(a.means) + (n * a.G + g) * MEANS[MODE];
    A* chan = reinterpret_cast<A*>(a.chan) + n * 2 * a.C;
    if constexpr (MODE == 1) {
        double k1 = 0, k2 = 0;
        for (int c = c0 + threadIdx.x; c < c1; c += blockDim.x) {
            const double w = (double)param<A>(a.w, c, (A)1), da = total(0, c), dah = total(1, c);
            k1 += w * da;
            k2 += w * dah;
            if (a.chan) {
                chan[c] = (A)dah;
                chan[a.C + c] = (A)da;
            }
        }
        k1 = all_sum(k1, lds);
        k2 = all_sum(k2, lds);
        if (threadIdx.x == 0) {
            out[0] = (A)(k1 / m);
            out[1] = (A)(k2 / m);
        }
    }
    if constexpr (MODE == 2) {
        double u1 = 0, u2 = 0, k1 = 0, k2 = 0, ku = 0;
        for (int c = c0 + threadIdx.x; c < c1; c += blockDim.x) {
            const double w = (double)param<A>(a.w, c, (A)1);
            u1 += total(0, c);
            u2 += total(1, c);
            k1 += w * total(2, c);
            k2 += w * total(3, c);
            ku += w * total(4, c);
        }
        u1 = all_sum(u1, lds) / m;
        u2 = all_sum(u2, lds) / m;
        k1 = all_sum(k1, lds) / m;
        k2 = all_sum(k2, lds) / m;
        ku = all_sum(ku, lds) / m;
        double v1 = 0, v2 = 0;
        for (int c = c0 + threadIdx.x; c < c1; c += blockDim.x) {
            const double w = (double)param<A>(a.w, c, (A)1), uw = (double)param<A>(a.uw, c, (A)0);
            const double da = total(2, c), dah = total(3, c);
            double t = 0, th = 0;
            if constexpr (ACT != 0) {  // q = cu u + ch h + cc
                const double cu = w * r, ch = uw - cu * u2, cc = (double)param<A>(a.ub, c, (A)0) - cu * u1;
                const double s0 = total(5, c), s1 = total(6, c);
                t = cu * total(8, c) + ch * s1 + cc * s0;
                th = cu * total(9, c) + ch * total(7, c) + cc * s1;
            }
            v1 += w * t + uw * da;
            v2 += w * th + uw * dah;
            if (a.chan) {
                chan[c] = (A)(r * (total(4, c) - u1 * da - u2 * dah) + th);
                chan[a.C + c] = (A)t;
            }
        }
        v1 = all_sum(v1, lds) / m - r * (u1 * k2 + k1 * u2);
        v2 = all_sum(v2, lds) / m - 2.0 * r * u2 * k2;
        if (threadIdx.x == 0) {
            out[0] = (A)u1;
            out[1] = (A)u2;
            out[2] = (A)k2;
            out[3] = (A)v1;
            out[4] = (A)v2;
            out[5] = (A)(ku - k1 * u1 - u2 * k2);
        }
    }
}

// The samples' shares of the parameters' gradients together, in order.
template <typename A> __global__ __launch_bounds__(1024) void k_params(Args a) {
    __shared__ double lds[16][64];
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + tx;
    const A* chan = reinterpret_cast<const A*>(a.chan) + (int64_t)blockIdx.y * a.C + c;
    double v = 0;
    if (c < a.C)
        for (int64_t n = ty; n < a.B; n += 16) v += (double)chan[n * 2 * a.C];
    lds[ty][tx] = v;
    __syncthreads();
    if (ty || c >= a.C) return;
    for (int i = 1; i < 16; ++i) v += lds[i][tx];
    A* out = reinterpret_cast<A*>(blockIdx.y ? a.db : a.dw);
    if (out) out[c] = (A)v;
}

// The outputs of a part of L.
template <typename T, int VEC, int MODE, int ACT> __global__ __launch_bounds__(THREADS) void k_apply(Args a) {
    using A = typename Acc<T>::type;
    const Place p = place<VEC>(a);
    if (!p.on) return;
    const int64_t base = p.n * a.L * a.C + p.c;
    Channels<A, VEC> ch;
    ch.load(a, p.n, p.c);
    A g[6][VEC], uw[VEC], ub[VEC];
    if constexpr (MODE != 0)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const A* s = reinterpret_cast<const A*>(a.means) + (p.n * a.G + (p.c + e) / a.cg) * MEANS[MODE];
#pragma unroll
            for (int i = 0; i < MEANS[MODE]; ++i) g[i][e] = s[i];
            uw[e] = MODE == 2 ? param<A>(a.uw, p.c + e, (A)0) : (A)0;
            ub[e] = MODE == 2 ? param<A>(a.ub, p.c + e, (A)0) : (A)0;
        }
    for (int64_t l = p.from + p.ty; l < p.to; l += p.step) {
        const int64_t at = base + l * a.C;
        const Pack<T, VEC> x = ldp<T, VEC>(reinterpret_cast<const T*>(a.x) + at);
        Pack<T, VEC> dy, u, o, o2;
        if constexpr (MODE != 0) dy = ldp<T, VEC>(reinterpret_cast<const T*>(a.dy) + at);
        if constexpr (MODE == 2) u = ldp<T, VEC>(reinterpret_cast<const T*>(a.u) + at);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const A r = ch.r[e], w = ch.w[e], h = ((A)x.e[e] - ch.mu[e]) * r, av = w * h + ch.b[e];
            if constexpr (MODE == 0) {
                o.e[e] = (T)act<ACT, A>(av);
            } else {
                A f1, f2;
                slopes<ACT, A>(av, f1, f2);
                const A da = (A)dy.e[e] * f1, k = w * da;
                if constexpr (MODE == 1) {
                    o.e[e] = (T)(r * (k - g[0][e] - h * g[1][e]));
                } else {
                    const A uv = (A)u.e[e], u1 = g[0][e], u2 = g[1][e], k2 = g[2][e];
                    const A q = w * r * (uv - u1 - h * u2) + uw[e] * h + ub[e];
                    const A v = w * (A)dy.e[e] * f2 * q + uw[e] * da - r * (uv * k2 + k * u2);
                    o.e[e] = (T)(r * (v - g[3][e] - h * g[4][e]) - r * r * h * g[5][e]);
                    o2.e[e] = (T)(f1 * q);
                }
            }
        }
        stp<T, VEC>(reinterpret_cast<T*>(a.y) + at, o);
        if constexpr (MODE == 2) stp<T, VEC>(reinterpret_cast<T*>(a.gdy) + at, o2);
    }
}

// -- launches ----------------------------------------------------------------------------------------------------------

static int check(int dtype, int64_t B, int64_t L, int C, int groups, int act) {
    if (dtype != EBR_DTYPE_F32 && dtype != EBR_DTYPE_BF16 && dtype != EBR_DTYPE_F16 && dtype != EBR_DTYPE_F64)
        return EBR_ERR_DTYPE;
    if (B < 1 || L < 1 || C < 1 || C > (1 << 20) || groups < 1 || C % groups || B >= ((int64_t)1 << 31) ||
        L >= ((int64_t)1 << 40) || B * L >= ((int64_t)1 << 40) || B * L * C >= ((int64_t)1 << 40) ||
        (act != EBR_ACT_NONE && act != EBR_ACT_SILU) || B * groups > MAX_BLOCKS)
        return EBR_ERR_SHAPE;
    return EBR_OK;
}

static int vector_of(int dtype, int C) {
    const int v = dtype == EBR_DTYPE_F64 ? 2 : dtype == EBR_DTYPE_F32 ? 4 : 8;
    return C % v == 0 ? v : 1;
}

// How the work is laid out, from the sizes alone: 16 threads of 16 bytes take 256 bytes of each cell; parts of L as many
// as give the card about eight workgroups for each of its 256 compute units, with at least 8 cells for each thread.
struct Plan {
    int vec, tx, tiles, splits;
    int64_t rows;
    Plan(int dtype, int64_t B, int64_t L, int C, bool vector) {
        vec = vector ? vector_of(dtype, C) : 1;
        tx = 1;
        while (tx < (vec > 1 ? 16 : 64) && tx * vec < C) tx *= 2;
        tiles = (C + tx * vec - 1) / (tx * vec);
        const int64_t step = THREADS / tx, least = 8 * step;
        int64_t s = 2048 / (B * tiles);
        if (s > (L + least - 1) / least) s = (L + least - 1) / least;
        if (s < 1) s = 1;
        rows = (L + s - 1) / s;
        splits = (int)((L + rows - 1) / rows);
    }
};

static int64_t acc_bytes(int dtype) { return dtype == EBR_DTYPE_F64 ? 8 : 4; }

template <typename F> static void by_kind(int dtype, bool vector, int act, F f) {
    const auto with = [&](auto v, auto n) {
        if (act == EBR_ACT_SILU) f(v, n, std::integral_constant<int, 1>());
        else f(v, n, std::integral_constant<int, 0>());
    };
    const auto one = [&](auto v) {
        using T = decltype(v);
        if (vector) with(v, std::integral_constant<int, 16 / (int)sizeof(T)>());
        else with(v, std::integral_constant<int, 1>());
    };
    switch (dtype) {
        case EBR_DTYPE_F32: one(float()); break;
        case EBR_DTYPE_BF16: one(__bf16()); break;
        case EBR_DTYPE_F16: one(_Float16()); break;
        default: one(double()); break;
    }
}

static bool all_aligned(std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if (!aligned(p, 16)) return false;
    return true;
}

// Bytes of scratch of a mode, laid out: part, means, chan.
struct Scratch {
    int64_t part, means, chan;
    Scratch(const Plan& p, int mode, int64_t B, int C, int groups, int64_t es) {
        const auto up = [](int64_t n) { return (n + 15) / 16 * 16; };
        part = up(B * p.splits * SUMS[mode] * C * es);
        means = up(B * groups * MEANS[mode] * es);
        chan = mode == 0 ? 0 : up(B * 2 * C * es);
    }
    int64_t all() const { return part + means + chan; }
};

template <int MODE> static int run(int dtype, int act, Args a, void* scratch, void* stream) {
    const bool vector = vector_of(dtype, a.C) > 1 && all_aligned({a.x, a.dy, a.u, a.y, a.gdy});
    const Plan p(dtype, a.B, a.L, a.C, vector);
    const Scratch sc(p, MODE, a.B, a.C, a.G, acc_bytes(dtype));
    char* at = reinterpret_cast<char*>(scratch);
    a.part = at;
    a.means = at + sc.part;
    a.chan = MODE != 0 && (a.dw || a.db) ? at + sc.part + sc.means : nullptr;
    a.cg = a.C / a.G;
    a.tx = p.tx;
    a.tiles = p.tiles;
    a.splits = p.splits;
    a.rows = p.rows;
    const int64_t blocks = a.B * p.splits * p.tiles;
    if (blocks > MAX_BLOCKS) return EBR_ERR_SHAPE;
    hipStream_t s = (hipStream_t)stream;
    by_kind(dtype, vector, act, [&](auto v, auto n, auto f) {
        using T = decltype(v);
        using A = typename Acc<T>::type;
        constexpr int VEC = decltype(n)::value, ACT = decltype(f)::value;
        hipLaunchKernelGGL((k_sums<T, VEC, MODE, ACT>), dim3((unsigned)blocks), dim3(THREADS), 0, s, a);
        hipLaunchKernelGGL((k_means<A, MODE, ACT>), dim3((unsigned)(a.B * a.G)), dim3(a.cg > 64 ? THREADS : 64), 0, s, a);
        hipLaunchKernelGGL((k_apply<T, VEC, MODE, ACT>), dim3((unsigned)blocks), dim3(THREADS), 0, s, a);
        if (MODE != 0 && a.chan) hipLaunchKernelGGL((k_params<A>), dim3((a.C + 63) / 64, 2), dim3(1024), 0, s, a);
    });
    return launched();
}

}  // namespace ebr_gn

using namespace ebr_gn;

extern "C" {

int64_t ebr_block_groupnorm_scratch(int dtype, int order, int64_t B, int64_t L, int C, int groups) {
    if (check(dtype, B, L, C, groups, 0) || order < 0 || order > 2) return -1;
    int64_t most = 0;
    for (const bool vector : {true, false}) {  // tensors off 16-byte alignment take another plan
        const Plan p(dtype, B, L, C, vector);
        const int64_t n = Scratch(p, order, B, C, groups, acc_bytes(dtype)).all();
        most = n > most ? n : most;
    }
    return most;
}

int ebr_block_groupnorm(int dtype, int act, int64_t B, int64_t L, int C, int groups, double eps, const void* x, const void* w,
                        const void* b, void* y, void* stats, void* scratch, void* stream) {
    const int rc = check(dtype, B, L, C, groups, act);
    if (rc) return rc;
    if (!x || !y || !stats) return EBR_ERR_NULL;
    if (!scratch) return EBR_ERR_SCRATCH;
    if (!aligned(scratch, 16)) return EBR_ERR_ALIGN;
    Args a = {};
    a.x = x, a.w = w, a.b = b, a.y = y, a.stats = stats, a.B = B, a.L = L, a.C = C, a.G = groups, a.eps = eps;
    return run<0>(dtype, act, a, scratch, stream);
}

int ebr_block_groupnorm_bwd(int dtype, int act, int64_t B, int64_t L, int C, int groups, const void* x, const void* w,
                            const void* b, const void* stats, const void* dy, void* dx, void* dw, void* db, void* scratch,
                            void* stream) {
    const int rc = check(dtype, B, L, C, groups, act);
    if (rc) return rc;
    if (!x || !dy || !dx || !stats) return EBR_ERR_NULL;
    if (!scratch) return EBR_ERR_SCRATCH;
    if (!aligned(scratch, 16)) return EBR_ERR_ALIGN;
    Args a = {};
    a.x = x, a.w = w, a.b = b, a.dy = dy, a.y = dx, a.dw = dw, a.db = db, a.stats = const_cast<void*>(stats);
    a.B = B, a.L = L, a.C = C, a.G = groups;
    return run<1>(dtype, act, a, scratch, stream);
}

int ebr_block_groupnorm_bwd2(int dtype, int act, int64_t B, int64_t L, int C, int groups, const void* x, const void* w,
                             const void* b, const void* stats, const void* dy, const void* u, const void* uw, const void* ub,
                             void* gx, void* gdy, void* gw, void* gb, void* scratch, void* stream) {
    const int rc = check(dtype, B, L, C, groups, act);
    if (rc) return rc;
    if (!x || !dy || !u || !gx || !gdy || !stats) return EBR_ERR_NULL;
    if (!scratch) return EBR_ERR_SCRATCH;
    if (!aligned(scratch, 16)) return EBR_ERR_ALIGN;
    Args a = {};
    a.x = x, a.w = w, a.b = b, a.dy = dy, a.u = u, a.uw = uw, a.ub = ub, a.y = gx, a.gdy = gdy, a.dw = gw, a.db = gb;
    a.stats = const_cast<void*>(stats), a.B = B, a.L = L, a.C = C, a.G = groups;
    return run<2>(dtype, act, a, scratch, stream);
}

}  // extern "C"
