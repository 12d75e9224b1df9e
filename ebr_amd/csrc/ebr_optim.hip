// AdamW over many tensors and the global norm of their gradients on gfx950 (C ABI and the formulas: include/ebr_optim.h).
//
// The tensors' addresses travel in the kernels' arguments, up to TENSORS (GRADS) a launch, so nothing is copied to the device
// and nothing kept: a workgroup finds its tensor by its own number in a table of the tensors' first workgroups.
//
// Bound by memory: 28 bytes an element with fp32 parameters, gradients and moments, 16 with moments in 8 bits, and the
// gradients once more for the norm. The step's factors (powers of the betas, the clipping) are taken once a tensor by
// k_factors, which also counts the step.
//
// Moments in 8 bits are what fp64 makes of them: a moment next to the border between two numbers goes to the same side in any
// order of operations. A wave takes the 256 elements of one scale, four a lane, in fp32, with a bound on how far each is off,
// and again in fp64 where that reaches over a border.
#include <algorithm>
#include <cmath>
#include <new>
#include <utility>
#include <vector>

#include "../../include/ebr_optim.h"
#include "rowwise.hpp"

namespace ebr_opt {

using namespace ebr_row;

constexpr int THREADS = 256, BLOCK = 256, TENSORS = 48, GRADS = 144;
constexpr int AT_ONCE = 4;                                                 // vectors under way in the norm
constexpr int64_t STEP = 1024, STEP8 = 4096, LEAST = 4096, MOST = 16384;   // elements of a workgroup: of a step, and of the norm

// What a step multiplies by, for one tensor.
struct alignas(16) Factors {
    double clip, step, root, decay;  // of the gradient; lr / (1 - beta1^t); 1 / sqrt(1 - beta2^t); 1 - lr decay
    uint32_t dither, zero[3];        // t * 0x9E3779B1
};

struct Table {
    ebr_optim_tensor t[TENSORS];
    int first[TENSORS + 1];  // the first workgroup of each, and of what would be next
    int count, per;          // per: elements of a workgroup
    const Factors* factors;
    double beta1, beta2, rest1, rest2, root2, eps;  // 1 - beta, and the second one's root
};

struct Prepare {
    int64_t* step[TENSORS];
    int count;
    Factors* factors;
    const float* lr_dev;
    const double* norm;
    double lr, beta1, beta2, decay, max_norm;
};

struct Sums {
    const void* g[GRADS];
    int64_t n[GRADS];
    int first[GRADS + 1], dtype[GRADS];
    int count, per;
    double* part;
};

__global__ __launch_bounds__(64) void k_factors(Prepare a) {
    const int i = threadIdx.x;
    if (i >= a.count) return;
    const int64_t t = *a.step[i] + 1;
    *a.step[i] = t;
    const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
    Factors f = {};
    f.clip = 1.0;
    if (a.norm) {
        const double c = a.max_norm / (*a.norm + 1e-6);
        f.clip = c > 1.0 ? 1.0 : c;  // (a norm that is NaN gives NaN)
    }
    f.step = lr / (1.0 - pow(a.beta1, (double)t));
    f.root = 1.0 / sqrt(1.0 - pow(a.beta2, (double)t));
    f.decay = 1.0 - lr * a.decay;
    f.dither = (uint32_t)t * 0x9E3779B1u;
    a.factors[i] = f;
}

// The tensor of this workgroup: the last one that begins at or before it.
template <typename Tab> __device__ __forceinline__ int tensor_of(const Tab& a) {
    int lo = 0, hi = a.count;
    const int b = blockIdx.x;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.first[mid] <= b) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Four elements from i on: ``full`` (for a whole wave) in one access whatever their alignment (which the hardware takes: the lanes'
// elements lie side by side, so most lines are whole all the same), else those of them that are below n.
template <typename T, typename A> __device__ __forceinline__ void load4(const T* p, int64_t i, int64_t n, bool full, A (&v)[4]) {
    if (full) {
        T x[4];
        __builtin_memcpy(x, p + i, sizeof(x));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (A)x[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = i + e < n ? (A)p[i + e] : (A)0;
    }
}
template <typename T, typename A> __device__ __forceinline__ void store4(T* p, int64_t i, int64_t n, bool full, const A (&v)[4]) {
    if (full) {
        T x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (T)v[e];
        __builtin_memcpy(p + i, x, sizeof(x));
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < n) p[i + e] = (T)v[e];
    }
}

template <typename A> __device__ __forceinline__ A root(A x);
template <> __device__ __forceinline__ float root(float x) { return __builtin_sqrtf(x); }
template <> __device__ __forceinline__ double root(double x) { return sqrt(x); }

template <typename P, typename G> __global__ __launch_bounds__(THREADS) void k_adamw(Table a) {
    using A = typename Acc<P>::type;
    const int which = tensor_of(a);
    const ebr_optim_tensor t = a.t[which];
    const Factors f = a.factors[which];
    const A clip = (A)f.clip, step = (A)f.step, rt = (A)f.root, decay = (A)f.decay, eps = (A)a.eps;
    const A b1 = (A)a.beta1, b2 = (A)a.beta2, c1 = (A)a.rest1, c2 = (A)a.rest2;
    P* const p = reinterpret_cast<P*>(t.p);
    const G* const g = reinterpret_cast<const G*>(t.g);
    A *const m = reinterpret_cast<A*>(t.m), *const v = reinterpret_cast<A*>(t.v);
    const int64_t from = (int64_t)(blockIdx.x - a.first[which]) * a.per;
    const int64_t to = from + a.per < t.n ? from + a.per : t.n;
    for (int64_t at = from; at < to; at += THREADS * 4) {
        const int64_t i = at + threadIdx.x * 4;
        const bool full = at + THREADS * 4 <= to;
        A pv[4], gv[4], mv[4], vv[4];
        load4(p, i, to, full, pv);
        load4(g, i, to, full, gv);
        load4(m, i, to, full, mv);
        load4(v, i, to, full, vv);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const A ge = gv[e] * clip;
            mv[e] = b1 * mv[e] + c1 * ge;
            vv[e] = b2 * vv[e] + c2 * (ge * ge);
            pv[e] = pv[e] * decay - step * mv[e] / (root(vv[e]) * rt + eps);
        }
        store4(p, i, to, full, pv);
        store4(m, i, to, full, mv);
        store4(v, i, to, full, vv);
    }
}

// The e4m3 number of y = |moment| / scale, as its seven bits: floor(y / s + t) steps s of its binade.
__device__ __forceinline__ uint32_t e4m3(double y, double t) {
    int e = __builtin_amdgcn_frexp_exp(y) - 1;
    if (e < -6 || y == 0.0) e = -6;
    const int code = ((e + 6) << 3) + (int)(__builtin_ldexp(y, 3 - e) + t);
    return y != y ? 0x7Fu : (uint32_t)(code > 0x7E ? 0x7E : code);
}

__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v = fmax(v, __shfl_xor(v, m, 64));
    return v;
}

// What a wave knows of its 256 elements: four a lane, the moments' numbers a byte each.
struct Eight {
    float p[4], g[4];
    uint32_t m, v;
    float ms, vs;
    uint32_t at;  // the first one's number, times the dither's factor, plus the step's part
};
__device__ __forceinline__ double dither(uint32_t w) { return (double)(w >> 8) * 0x1p-24; }
template <int E> __device__ __forceinline__ float number(uint32_t codes) { return __builtin_amdgcn_cvt_f32_fp8((int)codes, E); }
__device__ __forceinline__ void numbers(uint32_t codes, float (&x)[4]) {
    x[0] = number<0>(codes), x[1] = number<1>(codes), x[2] = number<2>(codes), x[3] = number<3>(codes);
}
// The low bytes of four words, and their high bytes.
__device__ __forceinline__ uint32_t low_bytes(const uint32_t (&x)[4]) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(x[3], x[2], 0x0C0C0400), __builtin_amdgcn_perm(x[1], x[0], 0x0C0C0400), 0x05040100);
}
__device__ __forceinline__ uint32_t high_bytes(const uint32_t (&x)[4]) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(x[3], x[2], 0x0C0C0703), __builtin_amdgcn_perm(x[1], x[0], 0x0C0C0703), 0x05040100);
}

// The step in fp64; the parameters of ``done`` (a bit each) have theirs.
__device__ __forceinline__ void step64(Eight& x, const Table& a, const Factors& f, int done) {
    const float step = (float)f.step, rt = (float)f.root, decay = (float)f.decay, eps = (float)a.eps;
    double mv[4], rv[4], mt = 0, vt = 0;
    float qm[4], qv[4];
    numbers(x.m, qm);
    numbers(x.v, qv);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const double ge = (double)x.g[e] * f.clip, r = (double)qv[e] * (double)x.vs;
        mv[e] = a.beta1 * ((double)qm[e] * (double)x.ms) + a.rest1 * ge;
        rv[e] = sqrt(a.beta2 * (r * r) + a.rest2 * (ge * ge));
        mt = fmax(mt, fabs(mv[e]));
        vt = fmax(vt, rv[e]);
        if (!(done >> e & 1)) x.p[e] = x.p[e] * decay - step * (float)mv[e] / ((float)rv[e] * rt + eps);
    }
    mt = wave_max(mt) / 448.0;
    vt = wave_max(vt) / 448.0;
    const bool some_m = !(mt < 0x1p-126), some_v = !(vt < 0x1p-126);
    const double im = some_m ? 1.0 / mt : 0.0, iv = some_v ? 1.0 / vt : 0.0;
    uint32_t cm[4], cv[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t w = x.at + (uint32_t)e * 0x85EBCA77u;
        cm[e] = e4m3(fabs(mv[e]) * im, dither(w)) | (__builtin_signbit(mv[e]) ? 0x80u : 0u);
        cv[e] = e4m3(rv[e] * iv, dither(w + 0x80000000u));
        if (some_v && rv[e] > 0 && cv[e] == 0) cv[e] = 1;
    }
    x.m = low_bytes(cm);
    x.v = low_bytes(cv);
    x.ms = some_m ? (float)mt : 0.f;
    x.vs = some_v ? (float)vt : 0.f;
}

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t umin(uint32_t a, uint32_t b) { return a < b ? a : b; }
__device__ __forceinline__ uint32_t bits(float x) { return __float_as_uint(x); }

// The largest of a wave's numbers, for all lanes: by rotations of rows of 16 lanes, then swaps of rows.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = umax(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x128, 0xF, 0xF, false));  // row_ror:8
    v = umax(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x124, 0xF, 0xF, false));
    v = umax(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x122, 0xF, 0xF, false));
    v = umax(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x121, 0xF, 0xF, false));
    auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = umax(r[0], r[1]);
    r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return __builtin_amdgcn_readfirstlane(umax(r[0], r[1]));
}

// The e4m3 number of y >= 0, in fp32 and integers. fp32's bits of y, read as a number of steps of 2^-20, are 8 (e + 127) + 8 f for
// y = 2^e (1 + f): an e4m3 number's code, and its 20 bits of fraction. Below 2^-6, where e4m3's steps stay 2^-9, they are those of
// y + 2^-6 less 8; the larger of the two is the right one on each side. The sum with t, of as many bits, is exact; what its
// fraction lacks to 0 or 1 is what y may be off by. ``line``: the bits, ``sum``: with t, and 64 for bytes to begin at 1024.
struct Code {
    uint32_t line, sum;
    __device__ __forceinline__ Code(float y, uint32_t t) : line(umax(bits(y), bits(y + 0x1p-6f) - (8u << 20))), sum(line + t + (64u << 20)) {}
    // in the low byte
    __device__ __forceinline__ uint32_t value(uint32_t least) const { return umax(umin(sum >> 20, 1024 + 0x7E), 1024 + least); }
    // below 2^19 where y is off by less than ``room``
    __device__ __forceinline__ uint32_t doubt(uint32_t room) const {
        const uint32_t d = sum & 0xFFFFF, mid = 1u << 19;
        return (d > mid ? d - mid : mid - d) + room;
    }
};

// The same in fp32, where it comes to the same numbers; where that is not sure, false, and ``done``'s parameters alone are new: how a
// parameter is taken depends on its own numbers, not on whether a neighbour's is in doubt. (But where the scale of a block is far out
// the first test sends all of it to fp64, and a parameter's last bit may be another one: step64 divides.) Parameters take the
// hardware's reciprocal and root, each within a step of fp32; they are 7.1e-8 off in the mean square.
//
// With u = 2^-24, the uniform factors being rounded once: a first moment's terms are off by 2 u each, so it by 3 u of their size S;
// the largest, and with it the scale, by no more than that of any S, at most 3 u (1 + 2 beta1 old largest / largest). A number of
// e4m3 is exact when squared; a root, and the largest root, are off by 4.5 u (a sum by 5 u, then the root's own 2 u). A scale's
// inverse and the products with it add 4 u. In steps of 2^-20 of the code, whose binade is 8 to 16 steps of e4m3, u of a number is
// 1 at most: 13 for a root, 7 + 6 beta1 old / new scale + 3 u S 2^(3 - e) / scale for a first moment, and 2 for what y + 2^-6 and t
// were cut by. About one wave in sixty has to go to fp64. Roots are taken of values scaled by a power of two near the old largest,
// so that squares stay in range. The largest numbers are compared as bits, where infinities and NaN are above all others.
__device__ __forceinline__ bool step32(Eight& x, const Table& a, const Factors& f, int& done) {
    done = 0;
    const int shift = x.vs > 0.f ? __builtin_amdgcn_frexp_expf(x.vs) + 9 : 0;
    const float unit = __builtin_ldexpf(1.f, -shift), back = __builtin_ldexpf(1.f, shift), vs = x.vs * unit;
    const float b1 = (float)(a.beta1 * x.ms), c1 = (float)(a.rest1 * f.clip), b2 = (float)(a.beta2 * ((double)vs * vs)),
                c2 = (float)(a.root2 * f.clip) * unit;
    const float step = (float)f.step, rt = (float)f.root * back, decay = (float)f.decay, eps = (float)a.eps;
    // what makes reciprocals and small squares safe: with it, a root of at least LEAST has both, and one of 0 has no part in it
    constexpr float LEAST_ROOT = 0x1p-55f, MOST_ROOT = 0x1p60f, MOST_MOMENT = 0x1p100f;
    if (!(rt >= 0x1p-60f && rt <= 0x1p55f && eps >= 0x1p-120f && eps <= 0x1p60f && (b2 == 0.f ? a.beta2 == 0.0 || x.vs == 0.f : b2 >= 0x1p-60f)))
        return false;
    float qm[4], qv[4], mv[4], rv[4], size[4], p[4];
    numbers(x.m, qm);
    numbers(x.v, qv);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float t1 = b1 * qm[e], t2 = c1 * x.g[e], gs = c2 * x.g[e];
        mv[e] = t1 + t2;
        size[e] = fabsf(t1) + fabsf(t2);
        rv[e] = __builtin_amdgcn_sqrtf(__builtin_fmaf(gs, gs, qv[e] * qv[e] * b2));
        p[e] = x.p[e] * decay - step * mv[e] * __builtin_amdgcn_rcpf(rv[e] * rt + eps);
    }
    const uint32_t mt = wave_max(umax(umax(bits(fabsf(mv[0])), bits(fabsf(mv[1]))), umax(bits(fabsf(mv[2])), bits(fabsf(mv[3])))));
    const uint32_t vt = wave_max(umax(umax(bits(rv[0]), bits(rv[1])), umax(bits(rv[2]), bits(rv[3]))));
    const bool small = __ballot(fminf(fminf(rv[0], rv[1]), fminf(rv[2], rv[3])) < LEAST_ROOT) != 0;
    bool sure = mt <= bits(MOST_MOMENT) && vt <= bits(MOST_ROOT);
    bool any_m = true, any_v = true;
    if (!sure || small || mt < bits(0x1p-90f) || vt < bits(0x1p-30f)) {
        // a root below LEAST_ROOT is one of zeros alone, or not done here; the largest are of zeros alone, or well inside fp32's range
        bool some_m = false, some_v = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool there = x.g[e] != 0.f || (qv[e] != 0.f && b2 != 0.f);
            some_m = some_m || x.g[e] != 0.f || qm[e] != 0.f;
            some_v = some_v || there;
            if ((rv[e] >= LEAST_ROOT || !there) && rv[e] <= MOST_ROOT && fabsf(mv[e]) <= MOST_MOMENT) {
                x.p[e] = p[e];
                done |= 1 << e;
            }
        }
        any_m = __ballot(some_m) != 0, any_v = __ballot(some_v) != 0;
        if (__ballot(done != 15) != 0 || (any_m && mt < bits(0x1p-90f)) || (any_v && vt < bits(0x1p-30f))) return false;
    } else {
        done = 15;
#pragma unroll
        for (int e = 0; e < 4; ++e) x.p[e] = p[e];
    }
    const float top_m = __uint_as_float(mt), top_v = __uint_as_float(vt);
    const float im = any_m ? 448.f * __builtin_amdgcn_rcpf(top_m) : 0.f, iv = any_v ? 448.f * __builtin_amdgcn_rcpf(top_v) : 0.f;
    const float ms = top_m * (1.f / 448.f), vs_new = top_v * (1.f / 448.f) * back;
    if ((any_v && !(vs_new >= 0x1p-100f)) || !(b1 * im <= 0x1p10f)) return false;  // (a room fits an integer)
    constexpr uint32_t room_v = 15;
    const float room_m = 10.f + 6.1f * b1 * im, more = 1.55f * im;  // 3.1 u 2^(3 + 20) / scale, to be times S 2^-e
    uint32_t cm[4], cv[4], doubt = 0, signs[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t t = (x.at + (uint32_t)e * 0x85EBCA77u) >> 12;
        const Code m(fabsf(mv[e]) * im, t), v(rv[e] * iv, t ^ 0x80000u);
        const float scale = __uint_as_float(0x7F000000u - (m.line & 0x7F800000u));  // 2^-e, or twice 2^6
        doubt = umax(doubt, umax(m.doubt((uint32_t)__builtin_fmaf(size[e] * more, scale, room_m)), v.doubt(room_v)));
        cm[e] = m.value(0);
        cv[e] = v.value(umin(bits(rv[e]), 1));
        signs[e] = bits(mv[e]);
    }
    if (__ballot(doubt >= 1u << 19) != 0) return false;
    x.m = low_bytes(cm) | (high_bytes(signs) & 0x80808080u);
    x.v = low_bytes(cv);
    x.ms = ms;
    x.vs = vs_new;
    return true;
}

// A word of four bytes, from i on.
__device__ __forceinline__ uint32_t load_word(const uint8_t* p, int64_t i, int64_t n, bool full) {
    uint32_t x = 0;
    if (full) {
        __builtin_memcpy(&x, p + i, 4);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < n) x |= (uint32_t)p[i + e] << 8 * e;
    }
    return x;
}
__device__ __forceinline__ void store_word(uint8_t* p, int64_t i, int64_t n, bool full, uint32_t x) {
    if (full) {
        __builtin_memcpy(p + i, &x, 4);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < n) p[i + e] = (uint8_t)(x >> 8 * e);
    }
}

template <typename P, typename G> __global__ __launch_bounds__(THREADS) void k_adamw8(Table a) {
    const int which = tensor_of(a);
    const ebr_optim_tensor t = a.t[which];
    const Factors f = a.factors[which];
    P* const p = reinterpret_cast<P*>(t.p);
    const G* const g = reinterpret_cast<const G*>(t.g);
    uint8_t *const m = reinterpret_cast<uint8_t*>(t.m), *const v = reinterpret_cast<uint8_t*>(t.v);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t from = (int64_t)(blockIdx.x - a.first[which]) * a.per;
    const int64_t to = from + a.per < t.n ? from + a.per : t.n;
    for (int64_t b = from + wave * BLOCK; b < to; b += THREADS / 64 * BLOCK) {
        const int64_t i = b + lane * 4;
        const bool full = b + BLOCK <= to;
        Eight x;
        load4(p, i, to, full, x.p);
        load4(g, i, to, full, x.g);
        x.m = load_word(m, i, to, full);
        x.v = load_word(v, i, to, full);
        x.ms = t.ms[b / BLOCK];
        x.vs = t.vs[b / BLOCK];
        x.at = (uint32_t)i * 0x85EBCA77u + f.dither;
        int done;
        if (!step32(x, a, f, done)) step64(x, a, f, done);
        store4(p, i, to, full, x.p);
        store_word(m, i, to, full, x.m);
        store_word(v, i, to, full, x.v);
        if (lane == 0) {
            t.ms[b / BLOCK] = x.ms;
            t.vs[b / BLOCK] = x.vs;
        }
    }
}

// The size of x in fp64, from its bits: fp32's fraction and exponent, moved (the conversion takes four times a sum's time). What is
// 0 or below the normal numbers comes out between 2^-127 and 2^-126, what is not finite above all that is.
__device__ __forceinline__ double moved(uint32_t hi, uint32_t lo) { return __hiloint2double((int)(hi + (896u << 20)), (int)lo); }
__device__ __forceinline__ double size_of(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
    return moved(b >> 3, b << 29);
}
__device__ __forceinline__ double size_of(_Float16 x) { return size_of((float)x); }
__device__ __forceinline__ double size_of(__bf16 x) {
    uint16_t b;
    __builtin_memcpy(&b, &x, 2);
    return moved((uint32_t)(b & 0x7FFF) << 13, 0);
}

// The sum of squares of g[from, to), a thread's share of it, in fp64. FAST: of sizes as above.
template <typename G, bool FAST> __device__ __forceinline__ double squares(const void* g_, int64_t from, int64_t to) {
    const G* const g = reinterpret_cast<const G*>(g_);
    constexpr int N = 16 / (int)sizeof(G);
    double sum[AT_ONCE] = {};
    const auto add = [&](int k, G x) {
        double v;
        if constexpr (FAST) v = size_of(x);
        else v = (double)x;
        sum[k] = __builtin_fma(v, v, sum[k]);
    };
    int64_t i = from + threadIdx.x * N;
    G x[AT_ONCE][N];
    for (; i + ((AT_ONCE - 1) * THREADS + 1) * N <= to; i += AT_ONCE * THREADS * N) {
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) __builtin_memcpy(x[k], g + i + k * THREADS * N, 16);  // whatever their alignment
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
            for (int e = 0; e < N; ++e) add(k, x[k][e]);
    }
    for (; i + N <= to; i += THREADS * N) {
        __builtin_memcpy(x[0], g + i, 16);
#pragma unroll
        for (int e = 0; e < N; ++e) add(0, x[0][e]);
    }
    for (; i < to; ++i) add(0, g[i]);  // (the last thread's: less than a vector)
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

__device__ __forceinline__ double block_sum(double s, double* lds) {
    s = lanes_sum<64>(s);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    double all = 0;
    for (int w = 0; w < (int)blockDim.x / 64; ++w) all += lds[w];
    return all;
}

__global__ __launch_bounds__(THREADS) void k_squares(Sums a) {
    __shared__ double lds[THREADS / 64];
    const int which = tensor_of(a);
    const int64_t from = (int64_t)(blockIdx.x - a.first[which]) * a.per;
    const int64_t to = from + a.per < a.n[which] ? from + a.per : a.n[which];
    const void* g = a.g[which];
    const int dtype = a.dtype[which];
    double s = 0;
    if (dtype == EBR_DTYPE_F32) s = squares<float, true>(g, from, to);
    else if (dtype == EBR_DTYPE_BF16) s = squares<__bf16, true>(g, from, to);
    else if (dtype == EBR_DTYPE_F16) s = squares<_Float16, true>(g, from, to);
    s = block_sum(s, lds);
    // an fp64 gradient, one that is not finite, and sums that a size's 2^-126 counts in
    if (!(s >= 0x1p-120 && s <= 0x1p255)) {
        if (dtype == EBR_DTYPE_F32) s = squares<float, false>(g, from, to);
        else if (dtype == EBR_DTYPE_BF16) s = squares<__bf16, false>(g, from, to);
        else if (dtype == EBR_DTYPE_F16) s = squares<_Float16, false>(g, from, to);
        else s = squares<double, false>(g, from, to);
        __syncthreads();
        s = block_sum(s, lds);
    }
    if (threadIdx.x == 0) a.part[blockIdx.x] = s;
}

__global__ __launch_bounds__(1024) void k_norm(const double* part, int64_t parts, double* norm, float* single) {
    __shared__ double lds[16];
    double s = 0;
    for (int64_t i = threadIdx.x; i < parts; i += 1024) s += part[i];
    s = sqrt(block_sum(s, lds));
    if (threadIdx.x != 0) return;
    *norm = s;
    if (single) *single = (float)s;
}

// -- launches ----------------------------------------------------------------------------------------------------------

static bool known(int d) { return d == EBR_DTYPE_F32 || d == EBR_DTYPE_BF16 || d == EBR_DTYPE_F16 || d == EBR_DTYPE_F64; }

// Elements of a workgroup of the norm, a multiple of LEAST: eight workgroups for each of the 256 compute units where there is
// enough, and no more than MOST (with 65,536 the last workgroups leave the card half empty: a quarter longer at 160 million).
static int64_t per_group(int64_t total) {
    const int64_t want = (total / 2048 + LEAST - 1) / LEAST * LEAST;
    return std::min(std::max(want, LEAST), MOST);
}

// Elements of a workgroup of a step. With 32-bit moments one vector a thread (80 million fp32 elements: 412 us, 417 with 4; a
// workgroup of 64 vectors a thread is a stream of its own through four arrays, and took a quarter longer). With 8-bit ones, where
// a workgroup's start counts against few bytes, up to four where that leaves eight workgroups for every compute unit: 80 million
// elements 343 us (one vector: 372), 900,001 in 60 tensors 7.9 us with one (four: 13.8).
static int64_t per_step(int64_t total, int bits) {
    const int64_t want = total / 2048 / STEP * STEP;
    return bits == 8 ? std::min(std::max(want, STEP), STEP8) : STEP;
}
static int64_t groups(int64_t n, int64_t per) { return (n + per - 1) / per; }

constexpr int64_t TOO_MANY = (int64_t)1 << 40;  // elements

static int64_t total_of(int64_t count, const ebr_optim_grad* g) {
    int64_t total = 0;
    for (int64_t i = 0; i < count; ++i) {
        if (g[i].n < 0 || g[i].n >= TOO_MANY || (total += g[i].n) >= TOO_MANY) return -1;
    }
    return total;
}

template <typename P, typename G> static void step(hipStream_t s, int bits, unsigned blocks, const Table& a) {
    if constexpr (sizeof(P) < 8) {
        if (bits == 8) {
            hipLaunchKernelGGL((k_adamw8<P, G>), dim3(blocks), dim3(THREADS), 0, s, a);
            return;
        }
    }
    hipLaunchKernelGGL((k_adamw<P, G>), dim3(blocks), dim3(THREADS), 0, s, a);
}

using Ranges = std::vector<std::pair<uintptr_t, uintptr_t>>;  // of addresses, the end past the last

// The memory that a step writes, in order of address.
static Ranges written(int64_t count, const ebr_optim_tensor* t, int64_t pbytes, int bits) {
    Ranges at;
    at.reserve(count * (bits == 8 ? 6 : 4));
    const auto add = [&](const void* p, int64_t bytes) {
        if (bytes > 0) at.emplace_back((uintptr_t)p, (uintptr_t)p + bytes);
    };
    for (int64_t i = 0; i < count; ++i) {
        const int64_t n = t[i].n, held = bits == 8 ? n : n * (pbytes == 8 ? 8 : 4), scales = bits == 8 ? (n + BLOCK - 1) / BLOCK * 4 : 0;
        add(t[i].p, n * pbytes), add(t[i].m, held), add(t[i].v, held), add(t[i].ms, scales), add(t[i].vs, scales), add(t[i].step, 8);
    }
    std::sort(at.begin(), at.end());
    return at;
}
// Whether any two of them share memory.
static bool twice(const Ranges& at) {
    for (size_t i = 1; i < at.size(); ++i)
        if (at[i].first < at[i - 1].second) return true;
    return false;
}
// Whether ``bytes`` from p on do with one of them, no two of which do.
static bool meets(const Ranges& at, const void* p, int64_t bytes) {
    const auto next = std::lower_bound(at.begin(), at.end(), std::pair<uintptr_t, uintptr_t>((uintptr_t)p + bytes, 0));
    return p && bytes > 0 && next != at.begin() && (next - 1)->second > (uintptr_t)p;
}

static int64_t bytes_of(int dtype) { return dtype == EBR_DTYPE_F64 ? 8 : dtype == EBR_DTYPE_F32 ? 4 : 2; }

}  // namespace ebr_opt

using namespace ebr_opt;

extern "C" {

int64_t ebr_block_grad_norm_scratch(int64_t count, const ebr_optim_grad* grads) {
    if (count < 1 || !grads) return -1;
    const int64_t total = total_of(count, grads);
    if (total < 0) return -1;
    const int64_t per = per_group(total);
    int64_t parts = 0;
    for (int64_t i = 0; i < count; ++i) parts += ebr_opt::groups(grads[i].n, per);
    return parts > MAX_BLOCKS ? -1 : 8 * parts + 16;
}

int ebr_block_grad_norm(int64_t count, const ebr_optim_grad* grads, double* norm, float* single, void* scratch,
                        void* stream) {
    if (count < 1) return EBR_ERR_SHAPE;
    if (!grads || !norm) return EBR_ERR_NULL;
    for (int64_t i = 0; i < count; ++i) {
        if (!known(grads[i].dtype)) return EBR_ERR_DTYPE;
        if (grads[i].n > 0 && !grads[i].g) return EBR_ERR_NULL;
    }
    if (ebr_block_grad_norm_scratch(count, grads) < 0) return EBR_ERR_SHAPE;
    if (!scratch) return EBR_ERR_SCRATCH;
    if (!aligned(scratch, 16)) return EBR_ERR_ALIGN;
    hipStream_t s = (hipStream_t)stream;
    const int64_t per = per_group(total_of(count, grads));
    int64_t parts = 0;
    for (int64_t i = 0; i < count;) {
        Sums a;
        int blocks = 0;
        for (a.count = 0; i < count && a.count < GRADS; ++i) {
            if (grads[i].n == 0) continue;
            a.g[a.count] = grads[i].g;
            a.n[a.count] = grads[i].n;
            a.dtype[a.count] = grads[i].dtype;
            a.first[a.count++] = blocks;
            blocks += (int)ebr_opt::groups(grads[i].n, per);
        }
        if (blocks == 0) break;
        a.first[a.count] = blocks;
        a.per = (int)per;
        a.part = reinterpret_cast<double*>(scratch) + parts;
        hipLaunchKernelGGL(k_squares, dim3(blocks), dim3(THREADS), 0, s, a);
        parts += blocks;
    }
    hipLaunchKernelGGL(k_norm, dim3(1), dim3(1024), 0, s, reinterpret_cast<const double*>(scratch), parts, norm, single);
    return launched();
}

int64_t ebr_block_adamw_scratch(int64_t count) {
    return count < 0 || count > MAX_BLOCKS ? -1 : count * (int64_t)sizeof(Factors) + 16;
}

int ebr_block_adamw(int ptype, int gtype, int bits, int64_t count, const ebr_optim_tensor* tensors, double lr,
                    const float* lr_dev, double beta1, double beta2, double eps, double decay, const double* norm,
                    double max_norm, void* scratch, void* stream) {
    const bool half = gtype == EBR_DTYPE_BF16 || gtype == EBR_DTYPE_F16;
    if (!known(ptype) || !known(gtype) || (gtype != ptype && !(ptype == EBR_DTYPE_F32 && half)) ||
        (bits != 32 && bits != 8) || (bits == 8 && ptype == EBR_DTYPE_F64))
        return EBR_ERR_DTYPE;
    if (ebr_block_adamw_scratch(count) < 0 || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0))
        return EBR_ERR_SHAPE;
    if (count == 0) return EBR_OK;
    if (!tensors) return EBR_ERR_NULL;
    int64_t total = 0;
    for (int64_t i = 0; i < count; ++i) {
        const ebr_optim_tensor& t = tensors[i];
        if (t.n < 0 || t.n >= TOO_MANY || (total += t.n) >= TOO_MANY) return EBR_ERR_SHAPE;
        if (!t.step || (t.n > 0 && (!t.p || !t.g || !t.m || !t.v || (bits == 8 && (!t.ms || !t.vs))))) return EBR_ERR_NULL;
    }
    Ranges at;
    try {
        at = written(count, tensors, bytes_of(ptype), bits);
    } catch (const std::bad_alloc&) {
        return EBR_ERR_HIP_BASE + (int)hipErrorOutOfMemory;
    }
    if (twice(at)) return EBR_ERR_SHAPE;
    if (!scratch) return EBR_ERR_SCRATCH;
    if (!aligned(scratch, 16)) return EBR_ERR_ALIGN;
    // what is read: a gradient may be its parameter, element by element
    bool met = meets(at, lr_dev, 4) || meets(at, norm, 8) || meets(at, scratch, ebr_block_adamw_scratch(count));
    for (int64_t i = 0; i < count && !met; ++i)
        met = !(tensors[i].g == tensors[i].p && gtype == ptype) && meets(at, tensors[i].g, tensors[i].n * bytes_of(gtype));
    if (met) return EBR_ERR_SHAPE;
    hipStream_t s = (hipStream_t)stream;
    Factors* factors = reinterpret_cast<Factors*>(scratch);
    int64_t per = per_step(total, bits);
    while (total / per + TENSORS > MAX_BLOCKS) per *= 2;  // (of a launch)
    for (int64_t i = 0; i < count; i += TENSORS, factors += TENSORS) {
        Table a = {};
        Prepare pre = {};
        a.count = pre.count = (int)std::min<int64_t>(TENSORS, count - i);
        a.factors = pre.factors = factors;
        a.per = (int)per;
        a.beta1 = pre.beta1 = beta1, a.beta2 = pre.beta2 = beta2;
        a.rest1 = 1.0 - beta1, a.rest2 = 1.0 - beta2, a.root2 = std::sqrt(a.rest2), a.eps = eps;
        pre.lr = lr, pre.lr_dev = lr_dev, pre.decay = decay, pre.norm = norm, pre.max_norm = max_norm;
        int blocks = 0;
        for (int k = 0; k < a.count; ++k) {
            a.t[k] = tensors[i + k];
            pre.step[k] = a.t[k].step;
            a.first[k] = blocks;
            blocks += (int)ebr_opt::groups(a.t[k].n, per);
        }
        a.first[a.count] = blocks;
        hipLaunchKernelGGL(k_factors, dim3(1), dim3(64), 0, s, pre);
        if (blocks == 0) continue;
        if (ptype == EBR_DTYPE_F64) step<double, double>(s, bits, blocks, a);
        else if (ptype == EBR_DTYPE_BF16) step<__bf16, __bf16>(s, bits, blocks, a);
        else if (ptype == EBR_DTYPE_F16) step<_Float16, _Float16>(s, bits, blocks, a);
        else if (gtype == EBR_DTYPE_BF16) step<float, __bf16>(s, bits, blocks, a);
        else if (gtype == EBR_DTYPE_F16) step<float, _Float16>(s, bits, blocks, a);
        else step<float, float>(s, bits, blocks, a);
    }
    return launched();
}

}  // extern "C"
