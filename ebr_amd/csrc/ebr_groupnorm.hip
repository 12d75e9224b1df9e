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
// Variances are not taken as a difference of squares about zero or a first cell, which a group far from it would lose: they
// are about the mean, or of eight cells at a time about theirs, which go together by the rule for the variance of a union.
//
// Bound by memory as far as the arithmetic (some 20, 30 and 75 operations an element) leaves it. 768 boards of 81 x 512 bf16
// (64 MB a tensor), groups of 16 channels: 29 us (4.4 TB/s), 42 (4.5), 88 (3.6) for the norm, its gradient and the second
// derivative; 64 boards of 900 x 512 (59 MB): 34 and 50 to 57 us, and 134 for the second derivative, read twice and at one
// wave a SIMD in k_sums. Two grids of 128 x 128 x 320 fp32 (42 MB a tensor, read twice, the second time from the last-level
// cache): 35, 47 and 77 us in three launches each.
#include <type_traits>

#include "rowwise.hpp"

namespace ebr_gn {

using namespace ebr_row;

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int SUMS[3] = {2, 2, 10};   // of a mode; mode 0: the mean and the squares about it
// kept of a group: mode 0: mu, r; 1: mean k, mean(k h); 2: u, u h, k h, v, v h, and Group2's along
constexpr int MEANS[3] = {2, 2, 6};

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
    int tile;               // channels of a workgroup that holds whole groups
    int64_t rows;           // of a part
    double eps;
    double inv;          // 1 / (L cg)
    double unit, units;  // the power of two that is 1 / (L cg) or the next below, and 1 / unit
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
        m2 += om2 + d * (d * (n * f));  // n f is 0 where a side has nothing: d is a mean then, its square perhaps infinite
        n = all;
    }
};

template <typename A> __device__ __forceinline__ A param(const void* p, int c, A none) {
    return p ? reinterpret_cast<const A*>(p)[c] : none;
}

template <typename A, int VEC> __device__ __forceinline__ void params(const void* p, int c, A none, A (&v)[VEC]) {
    if (p)
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = reinterpret_cast<const A*>(p)[c + e];
    else
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = none;
}

// What a thread knows of its channels. Elements enter as d = x - mu, not through x r - mu r in one step: of a group of
// (nearly) one value the difference is exact, where mu r would be rounded at the size of mu / sqrt(eps). The factor r of
// h = d r goes into the weights and, after the last cell, into the sums.
template <typename A, int VEC> struct Channels {
    A mu[VEC], r[VEC], w[VEC], b[VEC];
    __device__ __forceinline__ void load(const Args& a, int64_t n, int c) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const A* s = reinterpret_cast<const A*>(a.stats) + (n * a.G + (c + e) / a.cg) * 2;
            mu[e] = s[0];
            r[e] = s[1];
        }
        params<A, VEC>(a.w, c, (A)1, w);
        params<A, VEC>(a.b, c, (A)0, b);
    }
};

// An element's part of the sums of modes 1 and 2, with d in h's place; wr = w r. Returns da.
template <int ACT, int MODE, typename A, int NS, int VEC>
__device__ __forceinline__ A add_sums(A (&s)[NS][VEC], int e, A x, A dy, A u, A mu, A wr, A b) {
    const A d = x - mu;
    A f1, f2;
    slopes<ACT, A>(wr * d + b, f1, f2);
    const A da = dy * f1;
    if constexpr (MODE == 1) {
        s[0][e] += da;
        s[1][e] += da * d;
    } else {
        s[0][e] += u;
        s[1][e] += u * d;
        s[2][e] += da;
        s[3][e] += da * d;
        s[4][e] += da * u;
        if constexpr (ACT != 0) {
            const A t = dy * f2, td = t * d, tu = t * u;
            s[5][e] += t;
            s[6][e] += td;
            s[7][e] += td * d;
            s[8][e] += tu;
            s[9][e] += tu * d;
        }
    }
    return da;
}

// Their factors of r.
template <int MODE, typename A, int NS, int VEC> __device__ __forceinline__ void scale_sums(A (&s)[NS][VEC], int e, A r) {
    s[1][e] *= r;
    if constexpr (MODE == 2) {
        s[3][e] *= r;
        if constexpr (NS > 5) {
            s[6][e] *= r;
            s[7][e] *= r * r;
            s[9][e] *= r;
        }
    }
}

// A group's constants of gx = r (v - v1 - h (v2 + r along)) and gdy, the factor r in all that it takes: of the weights
// wr = w r and uwr = uw r alone are left.
template <typename A> struct Group2 {
    A u1, ru2, rrk2, rv1, e2;
    __device__ __forceinline__ Group2() {}
    // from the means of u, u h, and r times those of k h, v, v h and along
    __device__ __forceinline__ Group2(A r, A u1_, A u2, A rk2, A rv1_, A rv2, A ralong)
        : u1(u1_), ru2(r * u2), rrk2(r * rk2), rv1(rv1_), e2(r * (rv2 + r * ralong)) {}
};
template <int ACT, typename A>
__device__ __forceinline__ void second_out(const Group2<A>& g, A x, A dy, A u, A mu, A wr, A b, A uwr, A ub, A& gx, A& gdy) {
    const A d = x - mu;
    A f1, f2;
    slopes<ACT, A>(wr * d + b, f1, f2);
    const A da = dy * f1, rk = wr * da;
    const A q = wr * (u - g.u1 - d * g.ru2) + uwr * d + ub;
    gx = wr * (dy * f2 * q) + uwr * da - u * g.rrk2 - rk * g.ru2 - g.rv1 - d * g.e2;
    gdy = f1 * q;
}

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

// Per-channel sums of a part of L. Three tensors of 42 MB in 29 us (4.3 TB/s).
template <typename T, int VEC, int MODE, int ACT> __global__ __launch_bounds__(THREADS) void k_sums(Args a) {
    using A = typename Acc<T>::type;
    using Raw = typename Words<VEC * (int)sizeof(T)>::type;
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
                Raw x[8];  // (past the end the last cell again)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int64_t row = l + (int64_t)i * p.step;
                    x[i] = *reinterpret_cast<const Raw*>(reinterpret_cast<const T*>(a.x) + base +
                                                         (row < p.to ? row : p.to - 1) * a.C);
                }
                const int64_t left = (p.to - 1 - l) / p.step + 1;
                const int n = left < 8 ? (int)left : 8;
                const A f = (A)1 / (A)n;
                Pack<T, VEC> xv[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) xv[i] = unpacked<T, VEC>(x[i]);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    A mean = 0, m2 = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i < n) mean += (A)xv[i].e[e] - (A)xv[0].e[e];  // 0 of cells of one value
                    mean = (A)xv[0].e[e] + mean * f;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i < n) m2 += ((A)xv[i].e[e] - mean) * ((A)xv[i].e[e] - mean);
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
                for (int e = 0; e < VEC; ++e)
                    add_sums<ACT, MODE, A>(s, e, (A)x.e[e], (A)dy.e[e], MODE == 2 ? (A)u.e[e] : (A)0, ch.mu[e],
                                           ch.w[e] * ch.r[e], ch.b[e]);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) scale_sums<MODE, A>(s, e, ch.r[e]);
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

// A sum over a workgroup's threads of every sum, for everyone.
template <int K> __device__ __forceinline__ void all_sums(double (&v)[K], double* lds) {
#pragma unroll
    for (int i = 0; i < K; ++i) v[i] = lanes_sum<64>(v[i]);
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < K; ++i) lds[(threadIdx.x >> 6) * K + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < K; ++i) {
        v[i] = lds[i];
        for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v[i] += lds[w * K + i];
    }
}

// What follows from a channel's sums in a group of given means: a share of dw and db (gw, gb), and of the means of v and v h.
struct Second {
    double t, th, v1, v2, gw;
};
template <int ACT> __device__ __forceinline__ Second second(const double* s, double w, double uw, double ub, double r,
                                                            double u1, double u2) {
    Second o = {0, 0, 0, 0, 0};
    if constexpr (ACT != 0) {  // q = cu u + ch h + cc
        const double cu = w * r, ch = uw - cu * u2, cc = ub - cu * u1;
        o.t = cu * s[8] + ch * s[6] + cc * s[5];
        o.th = cu * s[9] + ch * s[7] + cc * s[6];
    }
    o.v1 = w * o.t + uw * s[2];
    o.v2 = w * o.th + uw * s[3];
    o.gw = r * (s[4] - u1 * s[2] - u2 * s[3]) + o.th;
    return o;
}

// One group of one sample: its means from the per-channel sums of all parts, and its channels' share of the parameters'
// gradients. Threads go over the channels and, as many as are left, over the parts. These few sums are taken in 64 bits:
// differences of means follow.
template <typename A, int MODE, int ACT> __global__ __launch_bounds__(THREADS) void k_means(Args a) {
    constexpr int NS = MODE == 0 ? 2 : MODE == 1 ? 2 : ACT ? 10 : 5;
    __shared__ double lds[WAVES * 5];
    __shared__ double tot[NS][THREADS];
    const int64_t n = blockIdx.x / a.G;
    const int g = (int)(blockIdx.x % a.G), c0 = g * a.cg;
    const double inv = a.inv;
    int cols = 1;
    while (cols < a.cg && cols < (int)blockDim.x) cols *= 2;
    const int tc = threadIdx.x % cols, ts = threadIdx.x / cols, lanes = (int)blockDim.x / cols;
    const A* part = reinterpret_cast<const A*>(a.part) + n * a.splits * NS * a.C;
    const auto cells = [&](int s) { return (double)(s + 1 < a.splits ? a.rows : a.L - s * a.rows); };
    A* stats = reinterpret_cast<A*>(a.stats) + (n * a.G + g) * 2;
    if constexpr (MODE == 0) {
        // about the first part's first mean, in 64 bits: one pass over the parts
        const double about = (double)part[c0];
        double v[2] = {0, 0};
        for (int c = tc; c < a.cg; c += cols)
#pragma unroll 4
            for (int s = ts; s < a.splits; s += lanes) {
                const double d = (double)part[(int64_t)s * 2 * a.C + c0 + c] - about;
                v[0] += cells(s) * d;
                v[1] += (double)part[((int64_t)s * 2 + 1) * a.C + c0 + c] + cells(s) * d * d;
            }
        all_sums<2>(v, lds);
        const double off = v[0] * inv, mu = about + off, var = v[1] * inv - off * off;
        if (threadIdx.x == 0) {
            stats[0] = (A)mu;
            stats[1] = (A)(1.0 / sqrt((var > 0 ? var : var == var ? 0.0 : var) + a.eps));
        }
        return;
    }
    // a channel's sums over all parts, for its first thread
    const auto channel = [&](int c, double (&s)[NS]) {
#pragma unroll
        for (int i = 0; i < NS; ++i) s[i] = 0;
        if (c < a.cg)
#pragma unroll 4
            for (int p = ts; p < a.splits; p += lanes)
#pragma unroll
                for (int i = 0; i < NS; ++i) s[i] += (double)part[((int64_t)p * NS + i) * a.C + c0 + c];
        for (int d = cols; d < 64; d <<= 1)
#pragma unroll
            for (int i = 0; i < NS; ++i) s[i] += __shfl_xor(s[i], d, 64);
        const int wide = cols < 64 ? 64 : cols;  // threads that hold the same sums, or parts of others
        if (wide == (int)blockDim.x) return;
        __syncthreads();
        if ((int)threadIdx.x % wide < cols)
#pragma unroll
            for (int i = 0; i < NS; ++i) tot[i][threadIdx.x / wide * cols + tc] = s[i];
        __syncthreads();
        if (ts == 0)
            for (int l = 1; l < (int)blockDim.x / wide; ++l)
#pragma unroll
                for (int i = 0; i < NS; ++i) s[i] += tot[i][l * cols + tc];
    };
    const double r = (double)stats[1];
    A* out = reinterpret_cast<A*>(a.means) + (n * a.G + g) * MEANS[MODE];
    A* chan = reinterpret_cast<A*>(a.chan) + n * 2 * a.C + c0;
    if constexpr (MODE == 1) {
        double k[2] = {0, 0};
        for (int c = tc; c < (a.cg + cols - 1) / cols * cols; c += cols) {
            double s[NS];
            channel(c, s);
            if (ts || c >= a.cg) continue;
            const double w = (double)param<A>(a.w, c0 + c, (A)1);
            k[0] += w * s[0];
            k[1] += w * s[1];
            if (a.chan) {
                chan[c] = (A)s[1];
                chan[a.C + c] = (A)s[0];
            }
        }
        all_sums<2>(k, lds);
        if (threadIdx.x == 0) {
            out[0] = (A)(k[0] * inv);
            out[1] = (A)(k[1] * inv);
        }
    }
    if constexpr (MODE == 2) {
        const int rounds = (a.cg + cols - 1) / cols;
        double k[5] = {0, 0, 0, 0, 0}, s[NS];
        for (int i = 0; i < rounds; ++i) {
            const int c = tc + i * cols;
            channel(c, s);
            if (ts || c >= a.cg) continue;
            const double w = (double)param<A>(a.w, c0 + c, (A)1);
            k[0] += s[0];
            k[1] += s[1];
            k[2] += w * s[2];
            k[3] += w * s[3];
            k[4] += w * s[4];
        }
        all_sums<5>(k, lds);
        const double u1 = k[0] * inv, u2 = k[1] * inv, k1 = k[2] * inv, k2 = k[3] * inv, ku = k[4] * inv;
        double v[2] = {0, 0};
        for (int i = 0; i < rounds; ++i) {
            const int c = tc + i * cols;
            if (rounds > 1) channel(c, s);  // one round leaves them
            if (ts || c >= a.cg) continue;
            const Second o = second<ACT>(s, (double)param<A>(a.w, c0 + c, (A)1), (double)param<A>(a.uw, c0 + c, (A)0),
                                         (double)param<A>(a.ub, c0 + c, (A)0), r, u1, u2);
            v[0] += o.v1;
            v[1] += o.v2;
            if (a.chan) {
                chan[c] = (A)o.gw;
                chan[a.C + c] = (A)o.t;
            }
        }
        all_sums<2>(v, lds);
        if (threadIdx.x == 0) {
            out[0] = (A)u1;
            out[1] = (A)u2;
            out[2] = (A)k2;
            out[3] = (A)(v[0] * inv - r * (u1 * k2 + k1 * u2));
            out[4] = (A)(v[1] * inv - 2.0 * r * u2 * k2);
            out[5] = (A)(ku - k1 * u1 - u2 * k2);
        }
    }
}

// The samples' shares of the parameters' gradients together, in a fixed order.
template <typename A> __global__ __launch_bounds__(1024) void k_params(Args a) {
    __shared__ double lds[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + tx;
    const A* chan = reinterpret_cast<const A*>(a.chan) + (int64_t)blockIdx.y * a.C + c;
    double v = 0;
    if (c < a.C)
#pragma unroll 8
        for (int64_t n = ty; n < a.B; n += 32) v += (double)chan[n * 2 * a.C];
    lds[ty][tx] = v;
    __syncthreads();
    if (ty || c >= a.C) return;
    for (int i = 1; i < 32; ++i) v += lds[i][tx];
    A* out = reinterpret_cast<A*>(blockIdx.y ? a.db : a.dw);
    if (out) out[c] = (A)v;
}

// The outputs of a part of L, past the caches, which hold what is read here for the second time: a graded step of 64 boards
// of 900 x 512 bf16, whose second derivative comes here, takes 224 us through the caches and 214 past them, of 16 of 4,400 x
// 512, which comes here in all three orders, 289 and 264 (with a reader of each output 314 and 305, 397 and 381).
template <typename T, int VEC, int MODE, int ACT> __global__ __launch_bounds__(THREADS) void k_apply(Args a) {
    using A = typename Acc<T>::type;
    const Place p = place<VEC>(a);
    if (!p.on) return;
    const int64_t base = p.n * a.L * a.C + p.c;
    Channels<A, VEC> ch;
    ch.load(a, p.n, p.c);
    A g[2][VEC], uw[VEC], ub[VEC];
    Group2<A> g2[MODE == 2 ? VEC : 1];
    if constexpr (MODE == 2) {
        params<A, VEC>(a.uw, p.c, (A)0, uw);
        params<A, VEC>(a.ub, p.c, (A)0, ub);
    }
    if constexpr (MODE != 0)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const A* s = reinterpret_cast<const A*>(a.means) + (p.n * a.G + (p.c + e) / a.cg) * MEANS[MODE];
            if constexpr (MODE == 1) {
                g[0][e] = s[0] * ch.r[e];
                g[1][e] = s[1] * ch.r[e] * ch.r[e];
            } else {
                const A r = ch.r[e];
                g2[e] = Group2<A>(r, s[0], s[1], r * s[2], r * s[3], r * s[4], r * s[5]);
                uw[e] *= r;
            }
        }
    for (int64_t l = p.from + p.ty; l < p.to; l += p.step) {
        const int64_t at = base + l * a.C;
        const Pack<T, VEC> x = ldp<T, VEC>(reinterpret_cast<const T*>(a.x) + at);
        Pack<T, VEC> dy, u, o, o2;
        if constexpr (MODE != 0) dy = ldp<T, VEC>(reinterpret_cast<const T*>(a.dy) + at);
        if constexpr (MODE == 2) u = ldp<T, VEC>(reinterpret_cast<const T*>(a.u) + at);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const A wr = ch.w[e] * ch.r[e], b = ch.b[e];
            if constexpr (MODE == 2) {
                A gx, gdy;
                second_out<ACT, A>(g2[e], (A)x.e[e], (A)dy.e[e], (A)u.e[e], ch.mu[e], wr, b, uw[e], ub[e], gx, gdy);
                o.e[e] = (T)gx;
                o2.e[e] = (T)gdy;
            } else {
                const A d = (A)x.e[e] - ch.mu[e], av = wr * d + b;
                if constexpr (MODE == 0) {
                    o.e[e] = (T)act<ACT, A>(av);
                } else {
                    A f1, f2;
                    slopes<ACT, A>(av, f1, f2);
                    o.e[e] = (T)(wr * ((A)dy.e[e] * f1) - g[0][e] - d * g[1][e]);
                }
            }
        }
        store_past<T, VEC>(reinterpret_cast<T*>(a.y) + at, o.e);
        if constexpr (MODE == 2) store_past<T, VEC>(reinterpret_cast<T*>(a.gdy) + at, o2.e);
    }
}

// -- groups that a workgroup holds ---------------------------------------------------------------------------------------

__device__ __forceinline__ void opaque(uint4& w) { asm volatile("" : "+v"(w.x), "+v"(w.y), "+v"(w.z), "+v"(w.w)); }
__device__ __forceinline__ void opaque(uint32_t& w) { asm volatile("" : "+v"(w)); }
__device__ __forceinline__ void opaque(uint2& w) { asm volatile("" : "+v"(w.x), "+v"(w.y)); }

// The next cell's arithmetic after this one's: side by side they take registers that hold other waves' elements.
__device__ __forceinline__ void one_by_one() { __builtin_amdgcn_sched_barrier(0); }

// The elements of a sample's tile of whole groups stay in registers between the sums and the outputs: one launch, every
// tensor read once. R cells a thread, W waves; a thread's VEC channels lie in one group.
//
// A thread sums its own cells by channel. All that follows is linear in these sums, so a thread takes them to its group's
// means by itself, and what goes through shared memory is one number a thread for each mean (five and then two of the second
// derivative, in place of ten for each channel), and for the parameters' gradients, where they are wanted, two a channel.
// Every channel's sums through shared memory doubled the second derivative (224 and 113 us for 768 boards of 81 x 512). A wave
// for each group, without barriers, is slower (32 bytes of a cell at a time: 134 and 102 us), and so are wider cells (256
// bytes, eight waves: 107 and 102).
template <typename T, int VEC, int MODE, int ACT, int R, int W>
__global__ __launch_bounds__(64 * W, MODE == 2 && R == 12 ? 5 : 1) void k_whole(Args a) {
    using A = typename Acc<T>::type;
    using Raw = typename Words<VEC * (int)sizeof(T)>::type;
    constexpr int NS = MODE == 0 ? 1 : MODE == 1 ? 2 : ACT ? 10 : 5, NG = MODE == 2 ? 5 : NS;
    extern __shared__ __attribute__((aligned(16))) char shared[];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, tc = a.tx * VEC;
    // what lanes of the same channels have not added up between them: rows of a wave's each, or of the threads of a cell
    // where these are several waves
    const int rows = a.tx < 64 ? W : 64 * W / a.tx, row = a.tx < 64 ? wave : t / a.tx;
    const bool first = a.tx >= 64 || lane < a.tx;
    constexpr int SLOTS = 2 * VEC > 5 ? 2 * VEC : 5;
    A* waves = reinterpret_cast<A*>(shared);  // [rows][NG][tx], and [rows][2][tc]
    A* cols = waves + rows * SLOTS * a.tx;    // [NG][tx]
    const int tile = (int)(blockIdx.x % a.tiles);
    const int64_t n = blockIdx.x / a.tiles;
    const int c0 = tile * a.tile, have = a.C - c0 < a.tile ? a.C - c0 : a.tile;
    const int at = (t % a.tx) * VEC, ty = t / a.tx, step = 64 * W / a.tx;
    const bool on = at < have;
    const int c = on ? c0 + at : c0, g = c / a.cg, gcols = a.cg / VEC, gfrom = (c - c0) / a.cg * gcols;
    const int L = (int)a.L;
    const int64_t base = n * a.L * a.C + c;

    // no load depends on the thread: one without channels reads the tile's first, and a cell past the end is the last
    Raw x[R], dy[MODE >= 1 ? R : 1], u[MODE == 2 ? R : 1];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (MODE == 2 && i * step >= L) break;  // (in the others this costs registers)
        const int l = ty + i * step;
        const int64_t off = base + (int64_t)(l < L ? l : L - 1) * a.C;
        x[i] = *reinterpret_cast<const Raw*>(reinterpret_cast<const T*>(a.x) + off);
        if constexpr (MODE >= 1) dy[i] = *reinterpret_cast<const Raw*>(reinterpret_cast<const T*>(a.dy) + off);
        if constexpr (MODE == 2) u[i] = *reinterpret_cast<const Raw*>(reinterpret_cast<const T*>(a.u) + off);
    }
    A w[VEC], b[VEC], mu = 0, r = 0;
    params<A, VEC>(a.w, c, (A)1, w);
    params<A, VEC>(a.b, c, (A)0, b);
    if constexpr (MODE >= 1) {
        const A* st = reinterpret_cast<const A*>(a.stats) + (n * a.G + g) * 2;
        mu = st[0];
        r = st[1];
    }
    // Between the sums and the outputs the elements stay packed as they came, or they take twice the registers.
    const auto pack_again = [&]() {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            opaque(x[i]);
            if constexpr (MODE >= 1) opaque(dy[i]);
            if constexpr (MODE == 2) opaque(u[i]);
        }
    };
    // p's means over this thread's group: over the wave's threads of the same channels, over the waves, over the channels. The
    // sums stay in 32 bits, as the cells' are, and only the mean is taken in 64, by a product: with divisions, and the channels
    // added in 64 bits, the three orders of 768 boards of 81 x 512 bf16 take 31, 43 and 95 us in place of 28, 41 and 87.
    const auto means = [&](auto& p, double* out) {
        constexpr int K = sizeof(p) / sizeof(p[0]);
        for (int d = a.tx; d < 64; d <<= 1)
#pragma unroll
            for (int k = 0; k < K; ++k) p[k] += __shfl_xor(p[k], d, 64);
        if (first)
#pragma unroll
            for (int k = 0; k < K; ++k) waves[(row * K + k) * a.tx + t % a.tx] = p[k];
        __syncthreads();
        for (int i = t; i < K * a.tx; i += 64 * W) {
            A v = waves[i];
            for (int q = 1; q < rows; ++q) v += waves[q * K * a.tx + i];
            cols[i] = v;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            A v = 0;
            for (int i = 0; i < gcols; ++i) v += cols[k * a.tx + gfrom + i];
            out[k] = (double)v * a.inv;
        }
    };
    // the sample's share of the parameters' gradients
    const auto shares = [&](A (&pw)[VEC], A (&pb)[VEC]) {
        for (int d = a.tx; d < 64; d <<= 1)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                pw[e] += __shfl_xor(pw[e], d, 64);
                pb[e] += __shfl_xor(pb[e], d, 64);
            }
        if (first) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                waves[row * 2 * tc + at + e] = pw[e];
                waves[(row * 2 + 1) * tc + at + e] = pb[e];
            }
        }
        __syncthreads();
        // one sample's share is the gradient
        A* share = reinterpret_cast<A*>(a.chan) + n * 2 * a.C;
        A* of[2] = {a.B == 1 ? reinterpret_cast<A*>(a.dw) : share, a.B == 1 ? reinterpret_cast<A*>(a.db) : share + a.C};
        for (int i = t; i < 2 * tc; i += 64 * W) {
            A* out = of[i >= tc];
            const int at_ = i >= tc ? i - tc : i;
            if (at_ >= have || !out) continue;
            A v = waves[i];
            for (int q = 1; q < rows; ++q) v += waves[q * 2 * tc + i];
            out[c0 + at_] = v;
        }
    };

    if constexpr (MODE == 0) {
        // in units in which the sum of the largest values does not overflow; a power of two: nothing else changes
        const A unit = (A)a.unit;
        double v[1], v2[2];
        A p[1] = {0}, p2[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (on && ty + i * step < L) {
                const Pack<T, VEC> xv = unpacked<T, VEC>(x[i]);
#pragma unroll
                for (int e = 0; e < VEC; ++e) p[0] += (A)xv.e[e] * unit;
            }
        pack_again();
        means(p, v);
        // about that mean, which the sum's rounding has left a little off (and may have left past the largest value): the mean
        // of what is left makes it up
        mu = (A)fmin(fmax(v[0] * a.units, -(double)__FLT_MAX__), (double)__FLT_MAX__);
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (on && ty + i * step < L) {
                const Pack<T, VEC> xv = unpacked<T, VEC>(x[i]);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const A d = (A)xv.e[e] - mu;
                    p2[0] += d;
                    p2[1] += d * d;
                }
            }
        pack_again();
        means(p2, v2);
        mu = (A)((double)mu + v2[0]);
        const double var = v2[1] - v2[0] * v2[0];
        r = (A)(1.0 / sqrt((var > 0 ? var : var == var ? 0.0 : var) + a.eps));
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[e] *= r;
        if (on && at % a.cg == 0 && ty == 0) {
            A* st = reinterpret_cast<A*>(a.stats) + (n * a.G + g) * 2;
            st[0] = mu;
            st[1] = r;
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int l = ty + i * step;
            one_by_one();
            if (!on || l >= L) continue;
            const Pack<T, VEC> xv = unpacked<T, VEC>(x[i]);
            Pack<T, VEC> o;
#pragma unroll
            for (int e = 0; e < VEC; ++e) o.e[e] = (T)act<ACT, A>(w[e] * ((A)xv.e[e] - mu) + b[e]);
            stp<T, VEC>(reinterpret_cast<T*>(a.y) + base + (int64_t)l * a.C, o);
        }
    } else {
        // The gradient of up to four cells keeps da, and its second half has neither dy nor the activation to take again, which
        // is as long as the memory traffic (768 boards of 81 x 512 bf16 take 42 us, and 50 with both taken again). In the second
        // derivative, sigmoids that are kept would gain 2 us of 87 there, for 116 registers and a wave less on each SIMD.
        constexpr bool KEEP = MODE == 1 && ACT != 0 && R <= 4;
        A kept[KEEP ? R : 1][KEEP ? VEC : 1];
        A s[NS][VEC] = {};
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[e] *= r;  // from here on
#pragma unroll
        for (int i = 0; i < R; ++i) {
            one_by_one();
            if (!on || ty + i * step >= L) continue;
            const Pack<T, VEC> xv = unpacked<T, VEC>(x[i]), dv = unpacked<T, VEC>(dy[i]);
            const Pack<T, VEC> uv = unpacked<T, VEC>(u[MODE == 2 ? i : 0]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const A da =
                    add_sums<ACT, MODE, A>(s, e, (A)xv.e[e], (A)dv.e[e], MODE == 2 ? (A)uv.e[e] : (A)0, mu, w[e], b[e]);
                if constexpr (KEEP) kept[i][e] = da;
            }
        }
        pack_again();
#pragma unroll
        for (int e = 0; e < VEC; ++e) scale_sums<MODE, A>(s, e, r);
        A p[NG] = {};
#pragma unroll
        for (int e = 0; e < VEC; ++e)
#pragma unroll
            for (int k = 0; k < NG; ++k) p[k] += MODE == 1 || k >= 2 ? w[e] * s[k][e] : s[k][e];
        double v[NG];
        means(p, v);
        if constexpr (MODE == 1) {
            if (a.chan) shares(s[1], s[0]);
            const A rk1 = (A)v[0], rrk2 = r * (A)v[1];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int l = ty + i * step;
                one_by_one();
                if (!on || l >= L) continue;
                const Pack<T, VEC> xv = unpacked<T, VEC>(x[i]), dv = unpacked<T, VEC>(dy[i]);
                Pack<T, VEC> o;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const A d = (A)xv.e[e] - mu;
                    A da;
                    if constexpr (KEEP) {
                        da = kept[i][e];
                    } else {
                        A f1, f2;
                        slopes<ACT, A>(w[e] * d + b[e], f1, f2);
                        da = (A)dv.e[e] * f1;
                    }
                    o.e[e] = (T)(w[e] * da - rk1 - d * rrk2);
                }
                stp<T, VEC>(reinterpret_cast<T*>(a.y) + base + (int64_t)l * a.C, o);
            }
        } else {
            const double u1d = v[0], u2d = v[1], rk1 = v[2], rk2 = v[3], rd = (double)r;
            const A u1 = (A)u1d, u2 = (A)u2d;
            A uw[VEC], ub[VEC], gw[VEC], gb[VEC], q[2] = {0, 0};
            params<A, VEC>(a.uw, c, (A)0, uw);
            params<A, VEC>(a.ub, c, (A)0, ub);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                A th = 0;
                gb[e] = 0;
                if constexpr (ACT != 0) {  // q = cu u + ch h + cc
                    const A cu = w[e], ch = uw[e] - cu * u2, cc = ub[e] - cu * u1;
                    gb[e] = cu * s[8][e] + ch * s[6][e] + cc * s[5][e];
                    th = cu * s[9][e] + ch * s[7][e] + cc * s[6][e];
                }
                gw[e] = r * (s[4][e] - u1 * s[2][e] - u2 * s[3][e]) + th;
                uw[e] *= r;
                q[0] += w[e] * gb[e] + uw[e] * s[2][e];
                q[1] += w[e] * th + uw[e] * s[3][e];
            }
            double z[2];
            means(q, z);
            if (a.chan) shares(gw, gb);
            const Group2<A> gc(r, u1, u2, (A)rk2, (A)(z[0] - rd * (u1d * rk2 + rk1 * u2d)), (A)(z[1] - 2.0 * rd * u2d * rk2),
                               (A)(v[4] - rk1 * u1d - u2d * rk2));
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int l = ty + i * step;
                one_by_one();
                if (!on || l >= L) continue;
                const Pack<T, VEC> xv = unpacked<T, VEC>(x[i]), dv = unpacked<T, VEC>(dy[i]), uv = unpacked<T, VEC>(u[i]);
                Pack<T, VEC> o, o2;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    A gx, gdy;
                    second_out<ACT, A>(gc, (A)xv.e[e], (A)dv.e[e], (A)uv.e[e], mu, w[e], b[e], uw[e], ub[e], gx, gdy);
                    o.e[e] = (T)gx;
                    o2.e[e] = (T)gdy;
                }
                stp<T, VEC>(reinterpret_cast<T*>(a.y) + base + (int64_t)l * a.C, o);
                stp<T, VEC>(reinterpret_cast<T*>(a.gdy) + base + (int64_t)l * a.C, o2);
            }
        }
    }
}

// -- launches ----------------------------------------------------------------------------------------------------------

static int check(int dtype, int64_t B, int64_t L, int C, int groups, int act) {
    if (dtype != EBR_DTYPE_F32 && dtype != EBR_DTYPE_BF16 && dtype != EBR_DTYPE_F16 && dtype != EBR_DTYPE_F64)
        return EBR_ERR_DTYPE;
    if (B < 1 || L < 1 || C < 1 || C > (1 << 20) || groups < 1 || C % groups || B >= ((int64_t)1 << 31) ||
        L >= ((int64_t)1 << 40) || B > (((int64_t)1 << 40) - 1) / L || B * L * C >= ((int64_t)1 << 40) ||  // (no product wraps)
        (act != EBR_ACT_NONE && act != EBR_ACT_SILU))
        return EBR_ERR_SHAPE;
    return EBR_OK;
}

static int vector_of(int dtype, int C) {
    const int v = dtype == EBR_DTYPE_F64 ? 2 : dtype == EBR_DTYPE_F32 ? 4 : 8;
    return C % v == 0 ? v : 1;
}

// How the work is laid out, from the sizes alone: 16 threads of 16 bytes take 256 bytes of each cell; parts of L as many
// as give the card about four workgroups for each of its 256 compute units, with at least 8 cells for each thread.
struct Plan {
    int vec, tx, tiles, splits;
    int64_t rows;
    Plan(int dtype, int64_t B, int64_t L, int C, bool vector) {
        vec = vector ? vector_of(dtype, C) : 1;
        tx = 1;
        while (tx < (vec > 1 ? 16 : 64) && tx * vec < C) tx *= 2;
        tiles = (C + tx * vec - 1) / (tx * vec);
        const int64_t step = THREADS / tx, least = 8 * step;
        int64_t s = 1024 / (B * tiles);
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

// Whether a workgroup holds a sample's tile of groups, and how: W waves of some cells a thread, tx threads across the tile's
// channels. A thread's vector has to lie in one group, and a tile of whole groups to fill three quarters of the threads
// across, which take 128 bytes of a cell or more: more where a sample has fewer cells than the rest of the workgroup holds (a
// graded step of 1,000 samples of 4 cells of 1,024 bf16 channels takes 169 us with 28 of 32 threads idle, 118 across) or
// where a group is wider (one group of 16 such cells: 427 us through k_sums and k_apply, 132 held). Above 256 cells at 128
// bytes for the second derivative, 1,024 for the others, groups go through those, which read everything twice.
//
// The vector is 16 bytes, but 2 channels of 16 bits in the second derivative, whose ten sums a channel and three tensors
// fill the registers: 768 boards of 81 x 512 bf16 take 88 us so (five waves a SIMD), 132 at 4 channels. Of groups too wide for
// 2, 4. Kernels hold 12 or 32 cells a thread then: boards of 81 cells need 11, and of 100 13, which take 119 us at 768 boards
// (three waves a SIMD).
struct Whole {
    int waves = 0, cells = 0, vec = 0, tx = 0, tile = 0, tiles = 0;
    // the two numbers of cells that there are kernels for
    static constexpr int few(int mode, bool wide, int vec) { return mode != 2 ? 4 : wide ? 3 : vec == 2 ? 12 : 16; }
    static constexpr int many(int mode, bool wide, int vec) { return mode != 2 || wide ? 8 : vec == 2 ? 32 : 16; }
    Whole(int mode, int dtype, int64_t L, int C, int groups, bool vector) {
        const int full = vector_of(dtype, C);
        const bool wide = dtype == EBR_DTYPE_F32;
        if (!vector || dtype == EBR_DTYPE_F64 || full == 1 || L > 4096) return;
        if (mode == 2 && !wide) {
            if (!fit(mode, wide, 2, L, C, groups)) fit(mode, wide, 4, L, C, groups);
        } else {
            fit(mode, wide, full, L, C, groups);
        }
    }
    bool fit(int mode, bool wide, int v, int64_t L, int C, int groups) {
        const int cg = C / groups;
        if (cg % v) return false;
        for (int x = 128 / (v * (wide ? 4 : 2)); x <= 256; x *= 2) {
            const int t = x * v / cg * cg;
            if (t == 0 || (t * 4 < x * v * 3 && t < C)) continue;
            if (x < 256 && t < C && L * 2 * x <= 256) continue;  // half of the cells of a workgroup would be none
            for (const int w : {4, 16}) {
                if (w == 16 && (mode == 2 || x > 32)) continue;  // (registers; shared memory)
                const int64_t step = 64 * w / x;
                const int r = (int)((L + step - 1) / step);
                if (r > many(mode, wide, v) || (w == 4 && r > 4 && mode != 2 && x <= 32)) continue;
                waves = w;
                cells = r <= few(mode, wide, v) ? few(mode, wide, v) : many(mode, wide, v);
                vec = v;
                tx = x;
                tile = t < C ? t : C;
                tiles = (C + tile - 1) / tile;
                return true;
            }
        }
        return false;
    }
};

// The workgroups of a mode, or -1 where a launch does not hold them (or one for each group of the samples).
static int64_t blocks_of(const Plan& p, const Whole& h, int64_t B, int groups) {
    const int64_t n = h.waves ? B * h.tiles * (h.waves / 4) : B * p.splits * p.tiles;
    return n > MAX_BLOCKS || (!h.waves && B * groups > MAX_BLOCKS) ? -1 : n;
}

template <typename T, int VEC, int MODE, int ACT> static void launch_vec(hipStream_t s, const Whole& h, const Args& a) {
    using A = typename Acc<T>::type;
    constexpr bool WIDE = sizeof(T) == 4;
    constexpr int FEW = Whole::few(MODE, WIDE, VEC), MANY = Whole::many(MODE, WIDE, VEC);
    const int rows = h.tx < 64 ? h.waves : 64 * h.waves / h.tx;
    const size_t lds = ((size_t)rows * (2 * VEC > 5 ? 2 * VEC : 5) * h.tx + 5 * h.tx) * sizeof(A);
    const dim3 grid((unsigned)(a.B * h.tiles)), block(64 * h.waves);
    if (h.waves == 4 && h.cells == FEW) hipLaunchKernelGGL((k_whole<T, VEC, MODE, ACT, FEW, 4>), grid, block, lds, s, a);
    else if (h.waves == 4) hipLaunchKernelGGL((k_whole<T, VEC, MODE, ACT, MANY, 4>), grid, block, lds, s, a);
    else if constexpr (MODE != 2) {
        if (h.cells == FEW) hipLaunchKernelGGL((k_whole<T, VEC, MODE, ACT, FEW, 16>), grid, block, lds, s, a);
        else hipLaunchKernelGGL((k_whole<T, VEC, MODE, ACT, MANY, 16>), grid, block, lds, s, a);
    }
}

template <typename T, int MODE, int ACT> static void launch_whole(hipStream_t s, const Whole& h, const Args& a) {
    if constexpr (MODE == 2 && sizeof(T) == 2) {
        if (h.vec == 2) launch_vec<T, 2, MODE, ACT>(s, h, a);
        else launch_vec<T, 4, MODE, ACT>(s, h, a);
    } else {
        launch_vec<T, 16 / (int)sizeof(T), MODE, ACT>(s, h, a);
    }
}

template <int MODE> static int run(int dtype, int act, Args a, void* scratch, void* stream) {
    const bool vector = vector_of(dtype, a.C) > 1 && all_aligned({a.x, a.dy, a.u, a.y, a.gdy});
    const Plan p(dtype, a.B, a.L, a.C, vector);
    const Scratch sc(p, MODE, a.B, a.C, a.G, acc_bytes(dtype));
    char* at = reinterpret_cast<char*>(scratch);
    a.part = at;
    a.means = at + sc.part;
    a.chan = MODE != 0 && (a.dw || a.db) ? at + sc.part + sc.means : nullptr;
    a.cg = a.C / a.G;
    a.inv = 1.0 / ((double)a.L * a.cg);
    a.units = 1.0;
    while (a.units < (double)a.L * a.cg) a.units *= 2;
    a.unit = 1.0 / a.units;
    a.tx = p.tx;
    a.tiles = p.tiles;
    a.splits = p.splits;
    a.rows = p.rows;
    const Whole h(MODE, dtype, a.L, a.C, a.G, vector);
    const int64_t blocks = blocks_of(p, h, a.B, a.G);
    if (blocks < 0) return EBR_ERR_SHAPE;
    hipStream_t s = (hipStream_t)stream;
    by_kind(dtype, vector, act, [&](auto v, auto n, auto f) {
        using T = decltype(v);
        using A = typename Acc<T>::type;
        constexpr int VEC = decltype(n)::value, ACT = decltype(f)::value;
        if (h.waves) {
            if constexpr (VEC > 1 && sizeof(T) < 8) {
                a.tx = h.tx;
                a.tile = h.tile;
                a.tiles = h.tiles;
                launch_whole<T, MODE, ACT>(s, h, a);
            }
            if (MODE != 0 && a.chan && a.B > 1)
                hipLaunchKernelGGL((k_params<A>), dim3((a.C + 31) / 32, 2), dim3(1024), 0, s, a);
            return;
        }
        hipLaunchKernelGGL((k_sums<T, VEC, MODE, ACT>), dim3((unsigned)blocks), dim3(THREADS), 0, s, a);
        hipLaunchKernelGGL((k_means<A, MODE, ACT>), dim3((unsigned)(a.B * a.G)),
                           dim3(a.cg * (int64_t)a.splits > 64 ? THREADS : 64), 0, s, a);
        hipLaunchKernelGGL((k_apply<T, VEC, MODE, ACT>), dim3((unsigned)blocks), dim3(THREADS), 0, s, a);
        if (MODE != 0 && a.chan) hipLaunchKernelGGL((k_params<A>), dim3((a.C + 31) / 32, 2), dim3(1024), 0, s, a);
    });
    return launched();
}

}  // namespace ebr_gn

using namespace ebr_gn;

extern "C" {

int64_t ebr_block_groupnorm_scratch(int dtype, int order, int64_t B, int64_t L, int C, int groups) {
    if (check(dtype, B, L, C, groups, 0) || order < 0 || order > 2) return -1;
    int64_t most = -1;
    for (const bool aligned : {true, false}) {  // tensors off 16-byte alignment take another plan
        const bool vector = aligned && vector_of(dtype, C) > 1;
        const Plan p(dtype, B, L, C, vector);
        if (blocks_of(p, Whole(order, dtype, L, C, groups, vector), B, groups) < 0) continue;
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
