// Layer norm over the last dimension with a weight and a bias on gfx950, with its first and second derivatives and the
// reduction of the parameters' gradients (C ABI: include/ebr_block.h).
//
// A row of C has the mean mu and r = (variance + eps)^-1/2; h = (x - mu) r, y = w h + b. P(v) = r (v - mean v - h mean(v h))
// carries a gradient of h back to x.
//   backward:    k = w dy,  dx = P(k),  dw = sum over rows of dy h,  db = sum of dy
//   backward2 (cotangents u of dx, uw of dw, ub of db):  gdy = w P(u) + uw h + ub,  gw = sum of dy P(u),
//     gx = P(uw dy) + r^2 (h (3 mean(uh) mean(kh) - mean(ku) + mean k mean u) - mean(kh) (u - mean u) - mean(uh) (k - mean k))
//
// The mean is taken twice: mu = m + c, m the rounded mean and c the mean of the differences x - m, so that a row of (nearly)
// one value far from zero keeps what there is of its differences. Both come out of two sums over the row, the second of which
// gives the squares as well. Backwards read m, c and r back.
//
// Bound by memory: 62,208 rows of 256 in bf16 take 13.3 us forward, 17.8 backward and 31 in the second (4.8, 5.4 and 5.1 TB/s),
// 16,384 of 2048 23.5 and 42 (5.7 and 4.8 TB/s; a copy of this size goes at 5 to 7). A row stays in the registers of TPR threads
// between its sums and its outputs, so every tensor is read once; rows too wide for a workgroup, and fp64, go through k_rows and
// k_apply, which read them twice (1000 x 40000: 68 us forward and 84 backward in bf16, 102 and 167 in fp32). The parameters' sums stay in the registers of the threads that hold the columns, over all rows
// of a workgroup, then go through one partial a workgroup to k_params: always in the same order.
#include <type_traits>

#include "rowwise.hpp"

namespace ebr_ln {

using namespace ebr_row;

constexpr int ROW_SUMS = 8;  // kept of a row by k_rows for k_apply

struct Args {
    const void *x, *dy, *u;
    const void *w, *b, *uw, *ub;  // of wtype, or null
    void *y, *gdy;                // y: also dx and gx
    void *stats;                  // [rows][4]: m, c, r, 0
    void *rowc;                   // [rows][ROW_SUMS]
    void *part;                   // [parts][2][C], or null: no sums for the parameters
    int64_t rows, chunk;          // chunk: rows of a workgroup in k_apply
    int C, wtype;
    double eps, inv;
    double unit, mean;  // the sum's elements go in times the power of two from 1 / C down, the sum then times 1 / (C unit)
};

template <typename A> __device__ __forceinline__ A root(A x);
template <> __device__ __forceinline__ float root(float x) { return __builtin_sqrtf(x); }
template <> __device__ __forceinline__ double root(double x) { return sqrt(x); }

// The rounded mean of finite elements, which is one of them or between two, where the rounding left the range. (What an
// infinity or a NaN makes of the row shows in its differences.)
__device__ __forceinline__ float within(float m) { return fminf(fmaxf(m, -3.40282347e38f), 3.40282347e38f); }
__device__ __forceinline__ double within(double m) { return fmin(fmax(m, -1.7976931348623157e308), 1.7976931348623157e308); }

// From the mean square about the rounded mean, and the mean's rest: never below 0; squares past the range make it infinite (and
// h 0, where a difference of infinities would be none); a NaN stays one.
template <typename A> __device__ __forceinline__ A variance(A square, A c) {
    const A v = square - c * c;
    return square == (A)INFINITY ? square : v < (A)0 ? (A)0 : v;
}

// A row's vectors: where its width is no multiple of VEC, the last one ends with the row and shares its first ``skip`` elements
// with the one before, which alone counts them in sums (both write them, the same). VEC and more: a vector past the row.
template <int VEC> __device__ __forceinline__ int place(int col, int C) { return col < C - VEC ? col : C - VEC; }
template <int VEC, typename F> __device__ __forceinline__ void each(int skip, F f) {
    if (skip <= 0) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f(e);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (e >= skip) f(e);
    }
}
// In one access, whatever the alignment.
template <typename T, int VEC> __device__ __forceinline__ Pack<T, VEC> fetch(const T* p) {
    Pack<T, VEC> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}
template <typename T, int VEC> __device__ __forceinline__ void put(T* p, const Pack<T, VEC>& v) { __builtin_memcpy(p, &v, sizeof(v)); }

// Consecutive parameters of any type.
template <typename A, int VEC> __device__ __forceinline__ void params(const void* p, int type, int c, A none, A (&v)[VEC]) {
    const auto take = [&](auto zero) {
        using W = decltype(zero);
        W x[VEC];
        __builtin_memcpy(x, reinterpret_cast<const W*>(p) + c, sizeof(x));
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = (A)x[e];
    };
    if (!p) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = none;
    } else if (type == EBR_DTYPE_F32) take(float());
    else if (type == EBR_DTYPE_BF16) take(__bf16());
    else if (type == EBR_DTYPE_F16) take(_Float16());
    else take(double());
}

// The sum over aligned parts of W lanes, the same in all of them: in fp32 by rotations of rows of 16 lanes and swaps of rows.
template <int W> __device__ __forceinline__ float total(float v) {
    if constexpr (W < 16) {
        return lanes_sum<W>(v);
    } else {
        const auto turned = [](float x, auto how) {
            const int u = __float_as_int(x);
            return __int_as_float(__builtin_amdgcn_update_dpp(u, u, decltype(how)::value, 0xF, 0xF, false));
        };
        v += turned(v, std::integral_constant<int, 0x128>());
        v += turned(v, std::integral_constant<int, 0x124>());
        v += turned(v, std::integral_constant<int, 0x122>());
        v += turned(v, std::integral_constant<int, 0x121>());
        if constexpr (W >= 32) {
            const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
            v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        }
        if constexpr (W == 64) {
            const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
            v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        }
        return v;
    }
}
template <int W> __device__ __forceinline__ double total(double v) { return lanes_sum<W>(v); }

// Sums over the TPR threads of a row, for all of them.
template <int TPR, int K, typename A> __device__ __forceinline__ void row_sums(A (&v)[K], A* lds) {
#pragma unroll
    for (int i = 0; i < K; ++i) v[i] = total<(TPR < 64 ? TPR : 64)>(v[i]);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        __syncthreads();  // (the last sums have been read)
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < K; ++i) lds[i * W + wave] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < K; ++i) {
            v[i] = lane < W ? lds[i * W + lane] : (A)0;
            v[i] = lanes_sum<W>(v[i]);
            v[i] = __shfl(v[i], 0, 64);
        }
    }
}

// A row's constants in the first derivative, and in the second.
template <typename A> struct Row {
    A m, c, r;
    A k, kh, u, uh, ku, t, th;  // means; t = uw dy
    A along;
    __device__ __forceinline__ A h(A x) const { return ((x - m) - c) * r; }
    __device__ __forceinline__ A dx(A kv, A h) const { return r * (kv - k - h * kh); }
    __device__ __forceinline__ A pu(A uv, A h) const { return r * (uv - u - h * uh); }
    __device__ __forceinline__ void second() { along = (A)3 * uh * kh - ku + k * u; }
    __device__ __forceinline__ A gx(A kv, A uv, A h) const {
        return r * r * (h * along - kh * (uv - u) - uh * (kv - k));
    }
    __device__ __forceinline__ A ptx(A tv, A h) const { return r * (tv - t - h * th); }
};

template <typename A> __device__ __forceinline__ void load_stats(const Args& a, int64_t row, Row<A>& q) {
    A s[4];
    __builtin_memcpy(s, reinterpret_cast<const A*>(a.stats) + row * 4, sizeof(s));
    q.m = s[0];
    q.c = s[1];
    q.r = s[2];
}

// What an element adds to the sums of its row: mode 1: k, k h; mode 2: also u, u h, k u, t, t h.
template <int MODE, typename A, int K>
__device__ __forceinline__ void add_row(A (&s)[K], A h, A k, A u, A t) {
    s[0] += k;
    s[1] += k * h;
    if constexpr (MODE == 2) {
        s[2] += u;
        s[3] += u * h;
        s[4] += k * u;
        s[5] += t;
        s[6] += t * h;
    }
}
template <int MODE, typename A, int K> __device__ __forceinline__ void take_row(Row<A>& q, const A (&s)[K], A inv) {
    q.k = s[0] * inv;
    q.kh = s[1] * inv;
    if constexpr (MODE == 2) {
        q.u = s[2] * inv;
        q.uh = s[3] * inv;
        q.ku = s[4] * inv;
        q.t = s[5] * inv;
        q.th = s[6] * inv;
        q.second();
    }
}

// Rows held in registers: TPR threads of NV vectors each take a row, all threads of a workgroup the rows of one step.
template <typename T, int VEC, int MODE, int TPR, int NV>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_held(Args a) {
    using A = typename Acc<T>::type;
    using Raw = typename Words<VEC * (int)sizeof(T)>::type;
    static_assert(sizeof(Raw) == VEC * sizeof(T), "the words of a pack");
    constexpr int THREADS = TPR > 256 ? TPR : 256, SLOTS = THREADS / TPR, K = MODE == 2 ? 7 : 2;
    __shared__ A lds[THREADS * VEC];
    const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    const A inv = (A)a.inv, unit = (A)a.unit;
    A w[NV][VEC], sw[NV][VEC], sb[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int col = place<VEC>((j * TPR + lane) * VEC, a.C);
        params<A, VEC>(a.w, a.wtype, col, (A)1, w[j]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) sw[j][e] = sb[j][e] = 0;
        if (MODE == 0) params<A, VEC>(a.b, a.wtype, col, (A)0, sb[j]);
    }
    for (int64_t first = (int64_t)blockIdx.x * SLOTS; first < a.rows; first += (int64_t)gridDim.x * SLOTS) {
        const int64_t row = first + slot;
        if (SLOTS > 1 && row >= a.rows) break;  // (whole parts of waves; no barrier below where there are several rows)
        const int64_t base = row * a.C;
        Raw rx[NV], rd[NV], ru[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t at = base + place<VEC>((j * TPR + lane) * VEC, a.C);
            const auto words = [&](const void* p) {
                Raw r;
                __builtin_memcpy(&r, reinterpret_cast<const T*>(p) + at, sizeof(r));
                return r;
            };
            rx[j] = words(a.x);
            if constexpr (MODE != 0) rd[j] = words(a.dy);
            if constexpr (MODE == 2) ru[j] = words(a.u);
        }
        if constexpr (MODE == 0) {
            A s1[1] = {0};
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const Pack<T, VEC> x = unpacked<T, VEC>(rx[j]);
                each<VEC>((j * TPR + lane) * VEC - (a.C - VEC), [&](int e) { s1[0] += (A)x.e[e] * unit; });
            }
            row_sums<TPR>(s1, lds);
            const A m = within(s1[0] * (A)a.mean);
            A s2[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const Pack<T, VEC> x = unpacked<T, VEC>(rx[j]);
                each<VEC>((j * TPR + lane) * VEC - (a.C - VEC), [&](int e) {
                    const A d = (A)x.e[e] - m;
                    s2[0] += d;
                    s2[1] += d * d;
                });
            }
            row_sums<TPR>(s2, lds);
            const A c = s2[0] * inv;
            const A r = (A)1 / root(variance(s2[1] * inv, c) + (A)a.eps);
            if (lane == 0) {
                A* st = reinterpret_cast<A*>(a.stats) + row * 4;
                st[0] = m;
                st[1] = c;
                st[2] = r;
                st[3] = 0;
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int col = (j * TPR + lane) * VEC;
                if (col >= a.C) continue;
                const Pack<T, VEC> x = unpacked<T, VEC>(rx[j]);
                Pack<T, VEC> o;
#pragma unroll
                for (int e = 0; e < VEC; ++e) o.e[e] = (T)((((A)x.e[e] - m) - c) * r * w[j][e] + sb[j][e]);
                put<T, VEC>(reinterpret_cast<T*>(a.y) + base + place<VEC>(col, a.C), o);
            }
        } else {
            Row<A> q;
            load_stats(a, row, q);
            A s[K];
#pragma unroll
            for (int i = 0; i < K; ++i) s[i] = 0;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int col = (j * TPR + lane) * VEC;
                if (col >= a.C) continue;
                const Pack<T, VEC> x = unpacked<T, VEC>(rx[j]), d = unpacked<T, VEC>(rd[j]);
                Pack<T, VEC> u = x;
                if constexpr (MODE == 2) u = unpacked<T, VEC>(ru[j]);
                A uw[VEC];
                if (MODE == 2 && a.uw) params<A, VEC>(a.uw, a.wtype, place<VEC>(col, a.C), (A)0, uw);
                each<VEC>(col - (a.C - VEC), [&](int e) {
                    add_row<MODE>(s, q.h((A)x.e[e]), w[j][e] * (A)d.e[e], (A)u.e[e],
                                  MODE == 2 && a.uw ? uw[e] * (A)d.e[e] : (A)0);
                });
            }
            row_sums<TPR>(s, lds);
            take_row<MODE>(q, s, inv);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int col = (j * TPR + lane) * VEC;
                if (col >= a.C) continue;
                const Pack<T, VEC> x = unpacked<T, VEC>(rx[j]), d = unpacked<T, VEC>(rd[j]);
                Pack<T, VEC> u = x, o, o2;
                if constexpr (MODE == 2) u = unpacked<T, VEC>(ru[j]);
                A uw[VEC], ub[VEC];
                if (MODE == 2 && a.uw) params<A, VEC>(a.uw, a.wtype, place<VEC>(col, a.C), (A)0, uw);
                if (MODE == 2 && a.ub) params<A, VEC>(a.ub, a.wtype, place<VEC>(col, a.C), (A)0, ub);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const A h = q.h((A)x.e[e]), dv = (A)d.e[e], k = w[j][e] * dv;
                    if constexpr (MODE == 1) {
                        o.e[e] = (T)q.dx(k, h);
                        sw[j][e] += dv * h;
                        sb[j][e] += dv;
                    } else {
                        const A pu = q.pu((A)u.e[e], h);
                        A gx = q.gx(k, (A)u.e[e], h), gdy = w[j][e] * pu;
                        if (a.uw) {
                            gx += q.ptx(uw[e] * dv, h);
                            gdy += uw[e] * h;
                        }
                        if (a.ub) gdy += ub[e];
                        o.e[e] = (T)gx;
                        o2.e[e] = (T)gdy;
                        sw[j][e] += dv * pu;
                    }
                }
                put<T, VEC>(reinterpret_cast<T*>(a.y) + base + place<VEC>(col, a.C), o);
                if constexpr (MODE == 2) put<T, VEC>(reinterpret_cast<T*>(a.gdy) + base + place<VEC>(col, a.C), o2);
            }
        }
    }
    if (MODE == 0 || !a.part) return;
    A* part = reinterpret_cast<A*>(a.part) + (int64_t)blockIdx.x * 2 * a.C;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int col = (j * TPR + lane) * VEC;
#pragma unroll
        for (int i = 0; i < (MODE == 1 ? 2 : 1); ++i) {
            A v[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = i == 0 ? sw[j][e] : sb[j][e];
            if constexpr (SLOTS > 1) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < VEC; ++e) lds[threadIdx.x * VEC + e] = v[e];
                __syncthreads();
                if (slot == 0)
#pragma unroll
                    for (int o = 1; o < SLOTS; ++o)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) v[e] += lds[(o * TPR + lane) * VEC + e];
            }
            if (slot == 0 && col < a.C)
#pragma unroll
                for (int e = 0; e < VEC; ++e) part[(int64_t)i * a.C + place<VEC>(col, a.C) + e] = v[e];
        }
    }
}

constexpr int WIDE = 1024;  // threads of a row in k_rows

// The sums of rows of any width: a workgroup reads its row twice in mode 0, once in the others.
template <typename T, int VEC, int MODE> __global__ __launch_bounds__(WIDE) void k_rows(Args a) {
    using A = typename Acc<T>::type;
    constexpr int K = MODE == 2 ? 7 : 2;
    __shared__ A lds[8 * WIDE / 64];
    const A inv = (A)a.inv, unit = (A)a.unit;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(a.x) + row * a.C;
        if constexpr (MODE == 0) {
            A s1[1] = {0};
            for (int col = threadIdx.x * VEC; col < a.C; col += WIDE * VEC) {
                const int c = place<VEC>(col, a.C);
                const Pack<T, VEC> v = fetch<T, VEC>(x + c);
                each<VEC>(col - c, [&](int e) { s1[0] += (A)v.e[e] * unit; });
            }
            row_sums<WIDE>(s1, lds);
            const A m = within(s1[0] * (A)a.mean);
            A s2[2] = {0, 0};
            for (int col = threadIdx.x * VEC; col < a.C; col += WIDE * VEC) {
                const int c = place<VEC>(col, a.C);
                const Pack<T, VEC> v = fetch<T, VEC>(x + c);
                each<VEC>(col - c, [&](int e) {
                    const A d = (A)v.e[e] - m;
                    s2[0] += d;
                    s2[1] += d * d;
                });
            }
            row_sums<WIDE>(s2, lds);
            const A c = s2[0] * inv;
            if (threadIdx.x == 0) {
                A* st = reinterpret_cast<A*>(a.stats) + row * 4;
                st[0] = m;
                st[1] = c;
                st[2] = (A)1 / root(variance(s2[1] * inv, c) + (A)a.eps);
                st[3] = 0;
            }
        } else {
            const T* dy = reinterpret_cast<const T*>(a.dy) + row * a.C;
            const T* u = reinterpret_cast<const T*>(a.u) + row * a.C;
            Row<A> q;
            load_stats(a, row, q);
            A s[K];
#pragma unroll
            for (int i = 0; i < K; ++i) s[i] = 0;
            for (int col = threadIdx.x * VEC; col < a.C; col += WIDE * VEC) {
                const int c = place<VEC>(col, a.C);
                const Pack<T, VEC> xv = fetch<T, VEC>(x + c), dv = fetch<T, VEC>(dy + c);
                Pack<T, VEC> uv = xv;
                if constexpr (MODE == 2) uv = fetch<T, VEC>(u + c);
                A w[VEC], uw[VEC];
                params<A, VEC>(a.w, a.wtype, c, (A)1, w);
                params<A, VEC>(MODE == 2 ? a.uw : nullptr, a.wtype, c, (A)0, uw);
                each<VEC>(col - c, [&](int e) {
                    add_row<MODE>(s, q.h((A)xv.e[e]), w[e] * (A)dv.e[e], (A)uv.e[e], uw[e] * (A)dv.e[e]);
                });
            }
            row_sums<WIDE>(s, lds);
            if (threadIdx.x == 0)
#pragma unroll
                for (int i = 0; i < K; ++i) reinterpret_cast<A*>(a.rowc)[row * ROW_SUMS + i] = s[i];
        }
    }
}

// The outputs, and the parameters' sums over a chunk of rows, from what k_rows found: a thread keeps its columns.
template <typename T, int VEC, int MODE> __global__ __launch_bounds__(256) void k_apply(Args a) {
    using A = typename Acc<T>::type;
    constexpr int K = MODE == 2 ? 7 : 2;
    const int tiles = (a.C + 256 * VEC - 1) / (256 * VEC);
    const int from_col = ((int)(blockIdx.x % tiles) * 256 + threadIdx.x) * VEC, col = place<VEC>(from_col, a.C);
    const int64_t chunk = blockIdx.x / tiles, from = chunk * a.chunk;
    const int64_t to = from + a.chunk < a.rows ? from + a.chunk : a.rows;
    if (from_col >= a.C) return;
    const A inv = (A)a.inv;
    A w[VEC], b[VEC], uw[VEC], ub[VEC], sw[VEC], sb[VEC];
    params<A, VEC>(a.w, a.wtype, col, (A)1, w);
    params<A, VEC>(a.b, a.wtype, col, (A)0, b);
    params<A, VEC>(a.uw, a.wtype, col, (A)0, uw);
    params<A, VEC>(a.ub, a.wtype, col, (A)0, ub);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sw[e] = sb[e] = 0;
    for (int64_t row = from; row < to; ++row) {
        const int64_t at = row * a.C + col;
        const Pack<T, VEC> x = fetch<T, VEC>(reinterpret_cast<const T*>(a.x) + at);
        Pack<T, VEC> d = x, u = x, o, o2;
        if constexpr (MODE != 0) d = fetch<T, VEC>(reinterpret_cast<const T*>(a.dy) + at);
        if constexpr (MODE == 2) u = fetch<T, VEC>(reinterpret_cast<const T*>(a.u) + at);
        Row<A> q;
        load_stats(a, row, q);
        if constexpr (MODE != 0) {
            A s[K];
#pragma unroll
            for (int i = 0; i < K; ++i) s[i] = reinterpret_cast<const A*>(a.rowc)[row * ROW_SUMS + i];
            take_row<MODE>(q, s, inv);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const A h = q.h((A)x.e[e]), dv = (A)d.e[e], k = w[e] * dv;
            if constexpr (MODE == 0) {
                o.e[e] = (T)(h * w[e] + b[e]);
            } else if constexpr (MODE == 1) {
                o.e[e] = (T)q.dx(k, h);
                sw[e] += dv * h;
                sb[e] += dv;
            } else {
                const A pu = q.pu((A)u.e[e], h);
                A gx = q.gx(k, (A)u.e[e], h);
                if (a.uw) gx += q.ptx(uw[e] * dv, h);
                o.e[e] = (T)gx;
                o2.e[e] = (T)(w[e] * pu + uw[e] * h + ub[e]);
                sw[e] += dv * pu;
            }
        }
        put<T, VEC>(reinterpret_cast<T*>(a.y) + at, o);
        if constexpr (MODE == 2) put<T, VEC>(reinterpret_cast<T*>(a.gdy) + at, o2);
    }
    if (MODE == 0 || !a.part) return;
    A* part = reinterpret_cast<A*>(a.part) + chunk * 2 * a.C + col;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        part[e] = sw[e];
        if constexpr (MODE == 1) part[(int64_t)a.C + e] = sb[e];
    }
}

// The workgroups' sums added up, PCOLS columns a workgroup.
template <typename A, int PCOLS, int PROWS = 1024 / PCOLS>
__global__ __launch_bounds__(PCOLS * PROWS) void k_params(const void* part_, int64_t parts, int C, int wtype, void* dw, void* db) {
    __shared__ A lds[PROWS][PCOLS + 1];
    void* const out = blockIdx.y == 0 ? dw : db;
    if (!out) return;
    const int x = threadIdx.x % PCOLS, y = threadIdx.x / PCOLS, col = blockIdx.x * PCOLS + x;
    const A* part = reinterpret_cast<const A*>(part_) + (int64_t)blockIdx.y * C + col;
    A s = 0;
    if (col < C) {
        int64_t i = y;
        for (; i + 3 * PROWS < parts; i += 4 * PROWS) {
            A v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = part[(i + j * PROWS) * 2 * C];
            s += (v[0] + v[1]) + (v[2] + v[3]);
        }
        for (; i < parts; i += PROWS) s += part[i * 2 * C];
    }
    lds[y][x] = s;
    __syncthreads();
    for (int n = PROWS / 2; n > 0; n >>= 1) {
        if (y < n) lds[y][x] += lds[y + n][x];
        __syncthreads();
    }
    if (y != 0 || col >= C) return;
    const A v = lds[0][x];
    if (wtype == EBR_DTYPE_F32) reinterpret_cast<float*>(out)[col] = (float)v;
    else if (wtype == EBR_DTYPE_BF16) reinterpret_cast<__bf16*>(out)[col] = (__bf16)v;
    else if (wtype == EBR_DTYPE_F16) reinterpret_cast<_Float16*>(out)[col] = (_Float16)v;
    else reinterpret_cast<double*>(out)[col] = (double)v;
}

// -- launches ----------------------------------------------------------------------------------------------------------

static bool known(int dtype) {
    return dtype == EBR_DTYPE_F32 || dtype == EBR_DTYPE_BF16 || dtype == EBR_DTYPE_F16 || dtype == EBR_DTYPE_F64;
}

static int check(int dtype, int wtype, int64_t rows, int C) {
    if (!known(dtype) || !known(wtype)) return EBR_ERR_DTYPE;
    if (rows < 1 || C < 1 || C > (1 << 24) || rows >= ((int64_t)1 << 40) / C) return EBR_ERR_SHAPE;
    return EBR_OK;
}

static int64_t acc_bytes(int dtype) { return dtype == EBR_DTYPE_F64 ? 8 : 4; }

// How rows are laid out over threads, from the sizes alone: 8 to 32 elements a thread. A wave takes rows of up to 2048, without a
// barrier (16384 x 2048 bf16: forward 23.5 us; 26.8 by four waves of 8 elements a thread, backward the same 42), a workgroup of 256
// threads rows of up to 8192 (1000 x 5003 fp32: forward 10.0 us, backward 16.3; 12.5 and 18.2 with 1024 threads), one of 1024
// rows of up to 16384, as more elements a thread would not fit its registers.
struct Plan {
    int vec, tpr = 0, each = 0;  // tpr 0: through k_rows and k_apply
    int64_t parts, chunk = 0;
    Plan(int mode, int dtype, int64_t rows, int C) {
        vec = dtype == EBR_DTYPE_F64 ? 2 : dtype == EBR_DTYPE_F32 ? 4 : 8;
        if (C < vec) vec = 1;
        if (dtype != EBR_DTYPE_F64) {
            for (const int t : {16, 32, 64, 256, 1024})
                if (tpr == 0 && C <= (t < 64 ? 8 : t < 1024 ? 32 : 16) * t) tpr = t;
            if (tpr) each = vec == 1 ? 1 : (C + tpr * 8 - 1) / (tpr * 8) * 8;
        }
        if (tpr) {
            const int slots = tpr < 256 ? 256 / tpr : 1;
            // as many as the card holds at once where they keep sums (16384 x 2048 bf16 backward: 42 us with 512, 49 with 1024)
            const int64_t groups = (rows + slots - 1) / slots;
            const int64_t most = (mode == 0 ? 2048 : each > 16 ? 512 : 1024) / (tpr == 1024 ? 2 : 1);
            parts = groups < most ? groups : most;
        } else {
            const int64_t tiles = (C + 256 * vec - 1) / (256 * vec);
            int64_t n = 2048 / tiles;
            if (n < 1) n = 1;
            if (n > rows) n = rows;
            chunk = (rows + n - 1) / n;
            parts = (rows + chunk - 1) / chunk;
        }
    }
};

struct Scratch {
    int64_t part, rowc;
    Scratch(const Plan& p, int mode, int dtype, int64_t rows, int C) {
        const auto up = [](int64_t n) { return (n + 15) / 16 * 16; };
        part = mode == 0 ? 0 : up(p.parts * 2 * C * acc_bytes(dtype));
        rowc = mode == 0 || p.tpr ? 0 : up(rows * ROW_SUMS * acc_bytes(dtype));
    }
    int64_t all() const { return part + rowc + 16; }
};

template <typename T, int VEC, int MODE> static void launch(hipStream_t s, const Plan& p, const Args& a) {
    const dim3 grid((unsigned)p.parts);
#define EBR_HELD(TPR, EACH)                                                                                          \
    if (p.tpr == TPR && p.each == EACH) {                                                                            \
        hipLaunchKernelGGL((k_held<T, VEC, MODE, TPR, EACH / VEC>), grid, dim3(TPR > 256 ? TPR : 256), 0, s, a);     \
        return;                                                                                                      \
    }
    if constexpr (sizeof(T) < 8 && VEC == 1) {
        EBR_HELD(16, 1)  // (rows of fewer elements than a vector)
    } else {
        if constexpr (sizeof(T) < 8) {
            EBR_HELD(16, 8) EBR_HELD(32, 8) EBR_HELD(64, 8) EBR_HELD(64, 16) EBR_HELD(64, 24) EBR_HELD(64, 32)
            EBR_HELD(256, 16) EBR_HELD(256, 24) EBR_HELD(256, 32) EBR_HELD(1024, 16)
        }
        const int64_t tiles = (a.C + 256 * VEC - 1) / (256 * VEC);
        const int64_t most = MAX_BLOCKS / (WIDE / 256);  // (it goes on to the rows beyond)
        hipLaunchKernelGGL((k_rows<T, VEC, MODE>), dim3((unsigned)(a.rows < most ? a.rows : most)), dim3(WIDE), 0, s, a);
        hipLaunchKernelGGL((k_apply<T, VEC, MODE>), dim3((unsigned)(tiles * p.parts)), dim3(256), 0, s, a);
    }
#undef EBR_HELD
}

template <int MODE> static int run(int dtype, Args a, void* dw, void* db, void* scratch, void* stream) {
    const Plan p(MODE, dtype, a.rows, a.C);
    const Scratch sc(p, MODE, dtype, a.rows, a.C);
    a.part = dw || db ? scratch : nullptr;
    a.rowc = reinterpret_cast<char*>(scratch) + sc.part;
    a.chunk = p.chunk;
    a.inv = 1.0 / a.C;
    for (a.unit = 1.0; a.unit * a.C > 1.0;) a.unit /= 2;
    a.mean = a.inv / a.unit;
    hipStream_t s = (hipStream_t)stream;
    const auto with = [&](auto v) {
        using T = decltype(v);
        if (p.vec > 1) launch<T, 16 / (int)sizeof(T), MODE>(s, p, a);
        else launch<T, 1, MODE>(s, p, a);
        if (MODE == 0 || !a.part) return;
        using A = typename Acc<T>::type;
        const int pcols = a.C >= 4096 ? 64 : 16;  // (500 sums of 5003 in 64 columns each: 6.0 us, in 16: 10.0)
        const dim3 grid((a.C + pcols - 1) / pcols, MODE == 1 ? 2 : 1);
        const auto add = [&](auto k) { hipLaunchKernelGGL(k, grid, dim3(1024), 0, s, a.part, p.parts, a.C, a.wtype, dw, db); };
        if (pcols == 64) add(k_params<A, 64>);
        else add(k_params<A, 16>);
    };
    switch (dtype) {
        case EBR_DTYPE_F32: with(float()); break;
        case EBR_DTYPE_BF16: with(__bf16()); break;
        case EBR_DTYPE_F16: with(_Float16()); break;
        default: with(double()); break;
    }
    return launched();
}

}  // namespace ebr_ln

using namespace ebr_ln;

extern "C" {

int64_t ebr_block_layernorm_scratch(int dtype, int order, int64_t rows, int C) {
    if (check(dtype, dtype, rows, C) || order < 0 || order > 2) return -1;
    return Scratch(Plan(order, dtype, rows, C), order, dtype, rows, C).all();
}

int ebr_block_layernorm(int dtype, int wtype, int64_t rows, int C, double eps, const void* x, const void* w, const void* b,
                        void* y, void* stats, void* stream) {
    const int rc = check(dtype, wtype, rows, C);
    if (rc) return rc;
    if (!x || !y || !stats) return EBR_ERR_NULL;
    Args a = {};
    a.x = x, a.w = w, a.b = b, a.wtype = wtype, a.y = y, a.stats = stats, a.rows = rows, a.C = C, a.eps = eps;
    return run<0>(dtype, a, nullptr, nullptr, nullptr, stream);
}

int ebr_block_layernorm_bwd(int dtype, int wtype, int64_t rows, int C, const void* x, const void* w, const void* stats,
                            const void* dy, void* dx, void* dw, void* db, void* scratch, void* stream) {
    const int rc = check(dtype, wtype, rows, C);
    if (rc) return rc;
    if (!x || !dy || !dx || !stats) return EBR_ERR_NULL;
    if (!scratch) return EBR_ERR_SCRATCH;
    if (!aligned(scratch, 16)) return EBR_ERR_ALIGN;
    Args a = {};
    a.x = x, a.w = w, a.wtype = wtype, a.dy = dy, a.y = dx, a.stats = const_cast<void*>(stats), a.rows = rows, a.C = C;
    return run<1>(dtype, a, dw, db, scratch, stream);
}

int ebr_block_layernorm_bwd2(int dtype, int wtype, int64_t rows, int C, const void* x, const void* w, const void* stats,
                             const void* dy, const void* u, const void* uw, const void* ub, void* gx, void* gdy, void* gw,
                             void* scratch, void* stream) {
    const int rc = check(dtype, wtype, rows, C);
    if (rc) return rc;
    if (!x || !dy || !u || !gx || !gdy || !stats) return EBR_ERR_NULL;
    if (!scratch) return EBR_ERR_SCRATCH;
    if (!aligned(scratch, 16)) return EBR_ERR_ALIGN;
    Args a = {};
    a.x = x, a.w = w, a.uw = uw, a.ub = ub, a.wtype = wtype, a.dy = dy, a.u = u, a.y = gx, a.gdy = gdy;
    a.stats = const_cast<void*>(stats), a.rows = rows, a.C = C;
    return run<2>(dtype, a, gw, nullptr, scratch, stream);
}

}  // extern "C"
