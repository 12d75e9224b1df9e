// Distillation from a teacher's top logits on gfx950, with its gradient (C ABI: include/ebr_block.h).
//
// A row has V logits x of the student and K entries (id, t) of the teacher; an entry counts where id is in [0, V).
//   p = softmax of the counted t / T,  q = softmax of x / T
//   loss = T^2 sum_k p_k (log p_k - log q_id_k),   dx_j = g T (q_j - sum over { k : id_k = j } of p_k)
// A row without an entry of positive probability has loss 0 and gradient 0 and is not counted in the mean.
//
// Bound by memory: the forward reads the logits once (running maximum and sum), the backward reads them again and writes
// the gradient; between them a row keeps four numbers. Exponents are taken of (x - max) (log2 e) / T: the difference of
// raw logits is exact or nearly so, where x / T would be rounded at the size of x, and x (log2 e) / T could pass the
// largest float where a mask has left nothing but the type's lowest value.
//
// Rows of any width start at any element. A row's first elements up to a 16-byte boundary go by themselves, and whole
// vectors follow: global memory takes them at the type's own alignment too, but a read of 4,096 rows of 50,021 bf16 logits
// that way reached 4.2 TB/s, of 50,048 5.1.
#include <type_traits>

#include "rowwise.hpp"

namespace ebr_distill {

using namespace ebr_row;

constexpr int K_MAX = 1024;  // a row's entries, held in shared memory by the backward
constexpr double LN2 = 0.6931471805599453, LOG2E = 1.4426950408889634;

__device__ __forceinline__ float pow2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ double pow2(double x) { return exp2(x); }
__device__ __forceinline__ float lg2(float x) { return log2f(x); }
__device__ __forceinline__ double lg2(double x) { return log2(x); }
// Leaves a NaN aside: the sum keeps it.
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }
template <typename A> __device__ __forceinline__ A lowest() { return (A)-__builtin_inff(); }

struct Args {
    const void *x, *teacher, *ids;
    int64_t N, row;  // row: elements from one row of x to the next
    int V, K, teacher_type, wide;
    double k;  // log2 e / T
    float k_low;  // what k lacks in 32 bits
    double weight;  // forward: T^2 ln 2; backward: T
    int reduction;
    void *stats, *loss, *scale, *part;
    const void* grad;
    int64_t grad_step;
    void* dx;
    int splits, width;  // parts of a row where there are few, and their columns
    int seen;           // words of k_grad's bits for a row's columns, a power of two
    void* soft;         // [N][splits]: a part's maximum and sum
};

// What a row's softmaxes need: its largest logit and the sum above it, the teacher's alike. ts is 0 for a row that is not
// counted.
template <typename A> struct alignas(4 * sizeof(A)) Stats { A m, s, tm, ts; };

// The factor of exponents: d times it in base 2. At 32 bits its own rounding would be a relative error of every exponent,
// 3e-8 of up to some 30 in a small probability; FINE adds what it lacks. 16-bit outputs do without.
template <typename A, bool FINE> struct Base {
    A k, low;
    __device__ __forceinline__ explicit Base(const Args& a) : k((A)a.k), low((A)a.k_low) {}
    __device__ __forceinline__ A times(A d) const {
        if constexpr (FINE && sizeof(A) == 4) return __builtin_fmaf(d, k, fmaxf(d, -1e30f) * low);  // -inf stays -inf
        return d * k;
    }
    __device__ __forceinline__ A power(A d) const { return pow2(times(d)); }
};
template <typename T> using BaseOf = Base<typename Acc<T>::type, sizeof(T) >= 4>;
template <typename A> struct alignas(16) Partial { double loss, rows; };

template <typename A> __device__ __forceinline__ A teacher_at(const Args& a, int64_t i) {
    switch (a.teacher_type) {
        case EBR_DTYPE_F32: return (A)reinterpret_cast<const float*>(a.teacher)[i];
        case EBR_DTYPE_BF16: return (A)(float)reinterpret_cast<const __bf16*>(a.teacher)[i];
        case EBR_DTYPE_F16: return (A)(float)reinterpret_cast<const _Float16*>(a.teacher)[i];
        default: return (A)reinterpret_cast<const double*>(a.teacher)[i];
    }
}

// An entry's column, -1 for one that does not count.
__device__ __forceinline__ int column(const Args& a, int64_t i) {
    const int64_t v = a.wide ? reinterpret_cast<const int64_t*>(a.ids)[i] : reinterpret_cast<const int*>(a.ids)[i];
    return v >= 0 && v < a.V ? (int)v : -1;
}

// A maximum and the sum of 2^((x - m) k) above it, of parts of a row.
template <typename A> struct Soft {
    A m, s;
    template <typename B> __device__ __forceinline__ void add(A x, const B& k) {
        if (x > m) {
            s *= k.power(m - x);  // 0 from nothing: s is 0 then
            m = x;
        }
        s += m == lowest<A>() ? (x == m ? (A)0 : x) : k.power(x - m);  // nothing but -inf so far: 0, or a NaN
    }
    template <typename B> __device__ __forceinline__ void merge(A om, A os, const B& k) {
        const A top = larger(m, om);
        const A base = top == lowest<A>() ? (A)0 : top;
        s = s * k.power(m - base) + os * k.power(om - base);
        m = top;
    }
};

template <typename T, int VEC> struct __attribute__((packed, aligned(sizeof(T)))) Loose { T e[VEC]; };

template <typename T, int VEC> __device__ __forceinline__ void store_past(T* p, const Loose<T, VEC>& v) {
    using W = uint32_t __attribute__((ext_vector_type(4)));
    typedef W __attribute__((aligned(2))) LooseW;
    W w;
    __builtin_memcpy(&w, &v, 16);
    __builtin_nontemporal_store(w, reinterpret_cast<LooseW*>(p));
}

// Elements before the next 16-byte boundary.
template <typename T> __device__ __forceinline__ int before_vectors(const T* p) {
    return (int)(((16 - ((uintptr_t)p & 15)) & 15) / sizeof(T));
}

// Columns [from, to) of a row by TEAM threads, several vectors at a time: one step of the running maximum for all of them.
template <typename T, int TEAM, typename A>
__device__ __forceinline__ Soft<A> soft_row(const T* x, int from, int to, int t, const BaseOf<T>& k) {
    constexpr int VEC = 16 / (int)sizeof(T), AT_ONCE = 4;
    using V = Loose<T, VEC>;
    Soft<A> v = {lowest<A>(), 0};
    const int head = before_vectors(x + from);
    if (t < head && from + t < to) v.add((A)x[from + t], k);
    int j = from + head + t * VEC;
    const auto step = [&](const A* e, int n) {
        A top = v.m;
#pragma unroll
        for (int i = 0; i < n; ++i) top = larger(e[i], top);
        const A base = top == lowest<A>() ? (A)0 : top;
        A sum = 0;
#pragma unroll
        for (int i = 0; i < n; ++i) sum += k.power(e[i] - base);
        v.s = v.s * k.power(v.m - base) + sum;
        v.m = top;
    };
    for (; j + (AT_ONCE - 1) * TEAM * VEC + VEC <= to; j += AT_ONCE * TEAM * VEC) {
        V p[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) p[i] = *reinterpret_cast<const V*>(x + j + i * TEAM * VEC);
        A e[AT_ONCE * VEC];
#pragma unroll
        for (int i = 0; i < AT_ONCE * VEC; ++i) e[i] = (A)p[i / VEC].e[i % VEC];
        step(e, AT_ONCE * VEC);
    }
    for (; j + VEC <= to; j += TEAM * VEC) {
        const V p = *reinterpret_cast<const V*>(x + j);
        A e[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) e[i] = (A)p.e[i];
        step(e, VEC);
    }
    for (; j < to; ++j) v.add((A)x[j], k);  // the thread whose vector the row's end cuts
    return v;
}

// Over the TEAM threads of a row: aligned lanes of a wave, or the whole workgroup.
template <int TEAM, typename A, typename B> __device__ __forceinline__ void soft_all(Soft<A>& v, const B& k, A* lds) {
    constexpr int W = TEAM < 64 ? TEAM : 64;
#pragma unroll
    for (int d = W / 2; d >= 1; d >>= 1) {
        const A om = __shfl_xor(v.m, d, 64), os = __shfl_xor(v.s, d, 64);
        v.merge(om, os, k);
    }
    if constexpr (TEAM > 64) {
        constexpr int WAVES = TEAM / 64;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            lds[threadIdx.x >> 6] = v.m;
            lds[WAVES + (threadIdx.x >> 6)] = v.s;
        }
        __syncthreads();
        v.m = lds[0];
        v.s = lds[WAVES];
        for (int w = 1; w < WAVES; ++w) v.merge(lds[w], lds[WAVES + w], k);
    }
}
template <int TEAM, typename A> __device__ __forceinline__ A sum_all(A v, A* lds) {
    v = lanes_sum<(TEAM < 64 ? TEAM : 64)>(v);
    if constexpr (TEAM > 64) {
        constexpr int WAVES = TEAM / 64;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0];
        for (int w = 1; w < WAVES; ++w) v += lds[w];
    }
    return v;
}

// The teacher's part of a row, once its student statistics are known: its statistics and the row's loss in units of
// weight. These few terms are taken in 64 bits: a logit that a mask has set to the type's lowest value has a logarithm
// that 32 bits hold in the end, but not in base 2 nor below T = 1.
template <typename T, int TEAM, typename A>
__device__ __forceinline__ double teach(const Args& a, int64_t n, Stats<A>& st, int t, bool on, A* lds, double* sums) {
    const Base<A, true> k(a);
    Soft<A> v = {lowest<A>(), 0};
    if (on)
        for (int i = t; i < a.K; i += TEAM)
            if (column(a, n * a.K + i) >= 0) v.add(teacher_at<A>(a, n * a.K + i), k);
    soft_all<TEAM, A>(v, k, lds);
    st.tm = v.m;
    st.ts = v.s;
    double sum = 0;
    if (on && v.s != (A)0) {
        const double ts2 = lg2(v.s), s2 = lg2(st.s);
        const T* x = reinterpret_cast<const T*>(a.x) + n * a.row;
        for (int i = t; i < a.K; i += TEAM) {
            const int c = column(a, n * a.K + i);
            if (c < 0) continue;
            const A e = k.times(teacher_at<A>(a, n * a.K + i) - v.m), p = pow2(e) / v.s;
            if (p == (A)0) continue;
            sum += p * ((e - ts2) - (((double)x[c] - st.m) * a.k - s2));
        }
    }
    return sum_all<TEAM, double>(sum, sums);
}

// The loss and the factor of its rows from their sum and number.
template <typename A> __device__ __forceinline__ void finish(const Args& a, const Partial<A>& v) {
    const double f = a.reduction == EBR_REDUCE_SUM ? 1.0 : 1.0 / (v.rows > 0 ? v.rows : 1.0);
    *reinterpret_cast<A*>(a.loss) = (A)(v.loss * f);
    *reinterpret_cast<A*>(a.scale) = (A)f;
}

// A part of a row, where there are too few rows to fill the card: 24 rows of 131,072 fp32 logits take 95 us a workgroup each,
// in 32 parts 5 us and 6 to join them (their gradient 108 and 6).
template <typename T> __global__ __launch_bounds__(256) void k_part(Args a) {
    using A = typename Acc<T>::type;
    __shared__ A lds[16];
    const int64_t n = blockIdx.x / a.splits;
    const int part = (int)(blockIdx.x % a.splits), from = part * a.width, to = from + a.width < a.V ? from + a.width : a.V;
    Soft<A> v = soft_row<T, 256, A>(reinterpret_cast<const T*>(a.x) + n * a.row, from, to, threadIdx.x, BaseOf<T>(a));
    soft_all<256, A>(v, BaseOf<T>(a), lds);
    if (threadIdx.x == 0) reinterpret_cast<Soft<A>*>(a.soft)[blockIdx.x] = v;
}

// Rows' losses, from the logits, or with JOIN from the rows' parts. 4,096 rows of 50,021 bf16 logits take 87 us (4.7 TB/s;
// loading the next round ahead of this one's arithmetic, or a maximum in fewer instructions, made no difference), 31,104 rows
// of 11 8 us (latency: a row's entries, their logits).
template <typename T, int TEAM, bool SHORT, bool JOIN> __global__ __launch_bounds__(256) void k_loss(Args a) {
    using A = typename Acc<T>::type;
    __shared__ A lds[16];
    __shared__ double rows[256 / TEAM][2], sums[4];
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const int64_t n = (int64_t)blockIdx.x * (256 / TEAM) + team;
    const bool on = n < a.N;
    const BaseOf<T> k(a);
    Soft<A> v = {lowest<A>(), 0};
    if (on) {
        const T* x = reinterpret_cast<const T*>(a.x) + n * a.row;
        if constexpr (JOIN) {
            for (int i = t; i < a.splits; i += TEAM) {
                const Soft<A> p = reinterpret_cast<const Soft<A>*>(a.soft)[n * a.splits + i];
                v.merge(p.m, p.s, k);
            }
        } else if constexpr (SHORT) {
            if (t < a.V) v.add((A)x[t], k);  // a column a thread
        } else {
            v = soft_row<T, TEAM, A>(x, 0, a.V, t, k);
        }
    }
    soft_all<TEAM, A>(v, k, lds);
    Stats<A> st = {v.m, v.s, 0, 0};
    const double sum = teach<T, TEAM, A>(a, n, st, t, on, lds, sums);
    if (t == 0) {
        const bool counted = on && st.ts != (A)0;
        const double loss = counted ? a.weight * sum : 0;
        if (on) {
            reinterpret_cast<Stats<A>*>(a.stats)[n] = st;
            if (a.reduction == EBR_REDUCE_NONE) reinterpret_cast<A*>(a.loss)[n] = (A)loss;
        }
        rows[team][0] = loss;
        rows[team][1] = counted;
    }
    if (a.reduction == EBR_REDUCE_NONE) return;
    __syncthreads();
    if (threadIdx.x == 0) {
        Partial<A> p = {0, 0};
        for (int i = 0; i < 256 / TEAM; ++i) {
            p.loss += rows[i][0];
            p.rows += rows[i][1];
        }
        if (gridDim.x == 1) finish<A>(a, p);
        else reinterpret_cast<Partial<A>*>(a.part)[blockIdx.x] = p;
    }
}

// The workgroups' sums together, in a fixed order; the mean's factor stays for the backward.
template <typename A> __global__ __launch_bounds__(1024) void k_total(Args a, int64_t parts) {
    __shared__ Partial<A> lds[16];
    Partial<A> v = {0, 0};
    const Partial<A>* p = reinterpret_cast<const Partial<A>*>(a.part);
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < parts; i += 1024) {
        const Partial<A> o = p[i];
        v.loss += o.loss;
        v.rows += o.rows;
    }
    v.loss = lanes_sum<64>(v.loss);
    v.rows = lanes_sum<64>(v.rows);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) {
            v.loss += lds[w].loss;
            v.rows += lds[w].rows;
        }
        finish<A>(a, v);
    }
}

// Rows of at most TEAM columns: a thread has a column and goes through the row's entries. 31,104 rows of 11 take 6 us.
template <typename T, int TEAM> __global__ __launch_bounds__(256) void k_grad_short(Args a) {
    using A = typename Acc<T>::type;
    const int t = threadIdx.x % TEAM;
    const int64_t n = (int64_t)blockIdx.x * (256 / TEAM) + threadIdx.x / TEAM;
    if (n >= a.N || t >= a.V) return;
    const BaseOf<T> k(a);
    const Stats<A> st = reinterpret_cast<const Stats<A>*>(a.stats)[n];
    A d = 0;
    if (st.ts != (A)0) {
        A p = 0;
        for (int i = 0; i < a.K; ++i)
            if (column(a, n * a.K + i) == t) p += k.power(teacher_at<A>(a, n * a.K + i) - st.tm);
        A c = reinterpret_cast<const A*>(a.grad)[n * a.grad_step] * (A)a.weight;
        if (a.scale) c *= *reinterpret_cast<const A*>(a.scale);
        d = c * (k.power((A)reinterpret_cast<const T*>(a.x)[n * a.row + t] - st.m) / st.s - p / st.ts);
    }
    reinterpret_cast<T*>(a.dx)[n * a.V + t] = (T)d;
}

// A row's columns, or a part of them, each from q alone; then the columns among them that the teacher names once more, each
// by the first of its entries, which adds the others of the same column in their order. The second write comes after a
// barrier, from the same workgroup.
//
// The stores go past the caches: otherwise what reads next waits for these lines to be written back. Of 4,096 rows of 50,021
// bf16 logits a loss and its gradient take 271 us through the caches and 251 past them; of 2,600 rows 168 and 139 us, with a
// sum of the gradient after it 253 and 224, and of 600 rows (60 MB, which the last-level cache would keep) 68 and 68. The
// gradient alone takes 148 us for the 4,096 rows (820 MB, 5.5 TB/s).
template <typename T, int TEAM> __global__ __launch_bounds__(256) void k_grad(Args a) {
    using A = typename Acc<T>::type;
    constexpr int VEC = 16 / (int)sizeof(T), AT_ONCE = 4;
    using V = Loose<T, VEC>;
    constexpr int TEAMS = 256 / TEAM;
    extern __shared__ __attribute__((aligned(16))) char shared[];
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    A* prob = reinterpret_cast<A*>(shared) + team * a.K;
    int* col = reinterpret_cast<int*>(reinterpret_cast<A*>(shared) + TEAMS * a.K) + team * a.K;
    uint32_t* seen = reinterpret_cast<uint32_t*>(shared + TEAMS * a.K * (int)(sizeof(A) + sizeof(int))) + team * (a.seen + 1);
    // the forward's last rows first: those that the last-level cache still has
    const uint32_t block = gridDim.x - 1 - blockIdx.x;
    const int64_t n = (int64_t)(block / a.splits) * (256 / TEAM) + team;
    const int from = (int)(block % a.splits) * a.width, to = from + a.width < a.V ? from + a.width : a.V;
    const bool on = n < a.N;
    const BaseOf<T> k(a);
    Stats<A> st = {};
    A c = 0, share = 0;
    bool counted = false;
    const T* x = reinterpret_cast<const T*>(a.x) + n * a.row;
    T* dx = reinterpret_cast<T*>(a.dx) + n * a.V;
    const auto q = [&](T v) { return k.power((A)v - st.m) * share; };  // c times the softmax
    // a bit for each column (or several, of a wide part) tells whether two entries may name the same: seen[a.seen] is set
    for (int i = t; i <= a.seen; i += TEAM) seen[i] = 0;
    __syncthreads();
    if (on) {
        st = reinterpret_cast<const Stats<A>*>(a.stats)[n];
        counted = st.ts != (A)0;
        c = reinterpret_cast<const A*>(a.grad)[n * a.grad_step] * (A)a.weight;
        if (a.scale) c *= *reinterpret_cast<const A*>(a.scale);
        share = c / st.s;
        for (int i = t; i < a.K; i += TEAM) {
            const int j = column(a, n * a.K + i);
            const bool mine = j >= from && j < to;
            col[i] = mine ? j : -1;
            prob[i] = mine ? k.power(teacher_at<A>(a, n * a.K + i) - st.tm) / st.ts : (A)0;
            if (!mine) continue;
            const uint32_t at = (uint32_t)(j - from) & (uint32_t)(a.seen * 32 - 1), bit = 1u << (at & 31);
            if (atomicOr(&seen[at >> 5], bit) & bit) seen[a.seen] = 1;
        }
        const int head = before_vectors(dx + from);
        if (t < head && from + t < to) dx[from + t] = counted ? (T)q(x[from + t]) : (T)0.f;
        int j = from + head + t * VEC;
        if (counted) {
            for (; j + (AT_ONCE - 1) * TEAM * VEC + VEC <= to; j += AT_ONCE * TEAM * VEC) {
                V p[AT_ONCE];
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) p[i] = *reinterpret_cast<const V*>(x + j + i * TEAM * VEC);
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) {
                    V o;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) o.e[e] = (T)q(p[i].e[e]);
                    store_past<T, VEC>(dx + j + i * TEAM * VEC, o);
                }
            }
            for (; j + VEC <= to; j += TEAM * VEC) {
                const V p = *reinterpret_cast<const V*>(x + j);
                V o;
#pragma unroll
                for (int e = 0; e < VEC; ++e) o.e[e] = (T)q(p.e[e]);
                store_past<T, VEC>(dx + j, o);
            }
            for (; j < to; ++j) dx[j] = (T)q(x[j]);
        } else {
            const V zero = {};
            for (; j + VEC <= to; j += TEAM * VEC) *reinterpret_cast<V*>(dx + j) = zero;
            for (; j < to; ++j) dx[j] = (T)0.f;
        }
    }
    __syncthreads();
    if (!counted) return;
    for (int i = t; i < a.K; i += TEAM) {
        const int j = col[i];
        if (j < 0) continue;
        A p = prob[i];
        bool first = true;
        if (seen[a.seen]) {
            p = 0;
            for (int o = 0; o < a.K; ++o)
                if (col[o] == j) {
                    first = first && o >= i;
                    p += prob[o];
                }
        }
        if (first) dx[j] = (T)(q(x[j]) - c * p);
    }
}

constexpr int SHORT_ROW = 32;  // columns of a row in which each has a thread

// k_grad's bits for the columns of a part: exact up to 2^17. Without them each entry goes through all the others: 20,000 rows
// of 4,001 bf16 logits with 256 entries take 312 us with their loss, 182 with them (fp32 361 and 303).
static int seen_of(int64_t width) {
    int w = 1;
    while (w < 4096 && (int64_t)w * 32 < width) w *= 2;
    return w;
}
static int64_t shared_of(int team, int K, int64_t width, int es) {
    return (int64_t)(256 / team) * (K * (int64_t)(es + 4) + 4 * (seen_of(width) + 1));
}

// Threads of a row: one a column for the shortest; then as many lanes as it has vectors, up to a wave (65,536 rows of 97
// bf16 take 104 us a wave each, 57 with 16 lanes), but not so few that the rows of a workgroup take more than 32 KiB of shared
// memory in the gradient; a workgroup for long rows.
static int team_of(int dtype, int64_t V, int K) {
    if (V > 2048) return 256;
    int t = 8;
    if (V <= SHORT_ROW) {
        while (t < V) t *= 2;
        return t;
    }
    const int es = dtype == EBR_DTYPE_F64 ? 8 : dtype == EBR_DTYPE_F32 ? 4 : 2, acc = es == 8 ? 8 : 4;
    while (t < 64 && (int64_t)t * (16 / es) < V) t *= 2;
    while (t < 64 && shared_of(t, K, V, acc) > 32768) t *= 2;
    return t < 64 || shared_of(t, K, V, acc) <= 32768 ? t : 256;
}

// Parts of a row: where rows of a workgroup each leave compute units without any, as many as give each of the 256 about
// four, with at least 4,096 columns (a round of loads) and at most 64 parts. An empty batch has no parts: nothing is launched
// for its rows.
static int splits_of(int64_t N, int64_t V) {
    if (V <= 2048 || N < 1 || N >= 512) return 1;
    int64_t s = 1024 / N;
    if (s > V / 4096) s = V / 4096;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}
static int width_of(int64_t V, int splits) { return (int)(((V + splits - 1) / splits + 7) / 8 * 8); }

static int64_t groups(int64_t N, int team) { return (N + 256 / team - 1) / (256 / team); }

static float low_of(double k) { return (float)(k - (double)(float)k); }

static int check(int dtype, int tdtype, int64_t N, int64_t V, int K, int64_t row, double T) {
    for (const int d : {dtype, tdtype})
        if (d != EBR_DTYPE_F32 && d != EBR_DTYPE_BF16 && d != EBR_DTYPE_F16 && d != EBR_DTYPE_F64) return EBR_ERR_DTYPE;
    // (T: so that its square, and what Base adds at 32 bits, are far from the largest float)
    if (N < 0 || N >= ((int64_t)1 << 31) || V < 1 || V >= ((int64_t)1 << 30) || K < 1 || K > K_MAX || row < V ||
        N * V >= ((int64_t)1 << 40) || row >= ((int64_t)1 << 40) || !(T >= 1e-15 && T <= 1e15) ||
        groups(N, team_of(dtype, V, K)) > MAX_BLOCKS)
        return EBR_ERR_SHAPE;
    return EBR_OK;
}

template <typename F> static int by_type(int dtype, F f) {
    switch (dtype) {
        case EBR_DTYPE_F32: return f(float());
        case EBR_DTYPE_BF16: return f(__bf16());
        case EBR_DTYPE_F16: return f(_Float16());
        default: return f(double());
    }
}

template <typename F> static void by_team(int team, int64_t V, F f) {
    const auto with = [&](auto t) {
        constexpr int TEAM = decltype(t)::value;
        if constexpr (TEAM <= SHORT_ROW)
            if (V <= SHORT_ROW) return f(t, std::true_type());
        f(t, std::false_type());
    };
    switch (team) {
        case 8: with(std::integral_constant<int, 8>()); break;
        case 16: with(std::integral_constant<int, 16>()); break;
        case 32: with(std::integral_constant<int, 32>()); break;
        case 64: with(std::integral_constant<int, 64>()); break;
        default: with(std::integral_constant<int, 256>()); break;
    }
}

}  // namespace ebr_distill

using namespace ebr_distill;

extern "C" {

int64_t ebr_block_distill_scratch(int dtype, int64_t N, int64_t V, int K) {
    if (check(dtype, dtype, N, V, K, V, 1.0)) return -1;
    const int splits = splits_of(N, V);
    const int64_t soft = splits > 1 ? N * splits * 2 * (dtype == EBR_DTYPE_F64 ? 8 : 4) : 0;
    return (soft + 15) / 16 * 16 + groups(N, splits > 1 ? 64 : team_of(dtype, V, K)) * (int64_t)sizeof(Partial<float>);
}

int ebr_block_distill(int dtype, int tdtype, int ids64, int64_t N, int64_t V, int K, int64_t row_stride, double temperature,
                      int reduction, const void* logits, const void* teacher, const void* ids, void* stats, void* loss,
                      void* scale, void* scratch, void* stream) {
    const int rc = check(dtype, tdtype, N, V, K, row_stride, temperature);
    if (rc) return rc;
    if (reduction != EBR_REDUCE_NONE && reduction != EBR_REDUCE_SUM && reduction != EBR_REDUCE_MEAN) return EBR_ERR_SHAPE;
    const bool one = reduction != EBR_REDUCE_NONE;
    if ((N > 0 && (!logits || !teacher || !ids || !stats)) || ((N > 0 || one) && !loss) || (one && !scale))
        return EBR_ERR_NULL;
    if (N > 0 && !scratch && (one || splits_of(N, V) > 1)) return EBR_ERR_SCRATCH;
    if (!aligned(stats, 16) || !aligned(scratch, 16)) return EBR_ERR_ALIGN;
    Args a = {logits, teacher, ids, N, row_stride, (int)V, K, tdtype, ids64 != 0, LOG2E / temperature,
              low_of(LOG2E / temperature), temperature * temperature * LN2, reduction, stats, loss, scale, scratch};
    hipStream_t s = (hipStream_t)stream;
    return by_type(dtype, [&](auto v) {
        using T = decltype(v);
        using A = typename Acc<T>::type;
        const int splits = splits_of(N, V), team = splits > 1 ? 64 : team_of(dtype, V, K);
        a.splits = splits;
        a.width = width_of(V, splits);
        if (splits > 1) {
            a.soft = scratch;
            const int64_t soft = N * splits * (int64_t)sizeof(Soft<A>);
            a.part = reinterpret_cast<char*>(scratch) + (soft + 15) / 16 * 16;
            hipLaunchKernelGGL((k_part<T>), dim3((unsigned)(N * splits)), dim3(256), 0, s, a);
            hipLaunchKernelGGL((k_loss<T, 64, false, true>), dim3((unsigned)groups(N, 64)), dim3(256), 0, s, a);
        } else if (N > 0) {
            by_team(team, V, [&](auto w, auto is_short) {
                hipLaunchKernelGGL((k_loss<T, decltype(w)::value, decltype(is_short)::value, false>),
                                   dim3((unsigned)groups(N, team)), dim3(256), 0, s, a);
            });
        }
        if (one && groups(N, team) != 1) hipLaunchKernelGGL((k_total<A>), dim3(1), dim3(1024), 0, s, a, groups(N, team));
        return launched();
    });
}

int ebr_block_distill_bwd(int dtype, int tdtype, int ids64, int64_t N, int64_t V, int K, int64_t row_stride,
                          double temperature, const void* logits, const void* teacher, const void* ids, const void* stats,
                          const void* scale, const void* grad, int64_t grad_stride, void* dx, void* stream) {
    const int rc = check(dtype, tdtype, N, V, K, row_stride, temperature);
    if (rc) return rc;
    if (grad_stride != 0 && grad_stride != 1) return EBR_ERR_SHAPE;
    if (N == 0) return EBR_OK;
    if (!logits || !teacher || !ids || !stats || !grad || !dx) return EBR_ERR_NULL;
    if (!aligned(stats, 16)) return EBR_ERR_ALIGN;
    Args a = {logits, teacher, ids, N, row_stride, (int)V, K, tdtype, ids64 != 0, LOG2E / temperature,
              low_of(LOG2E / temperature), temperature, EBR_REDUCE_NONE, const_cast<void*>(stats), nullptr,
              const_cast<void*>(scale), nullptr, grad, grad_stride, dx};
    return by_type(dtype, [&](auto v) {
        using T = decltype(v);
        using A = typename Acc<T>::type;
        const int team = team_of(dtype, V, K);
        a.splits = splits_of(N, V);
        a.width = width_of(V, a.splits);
        a.seen = seen_of(a.width);
        const size_t lds = (size_t)shared_of(team, K, a.width, sizeof(A));
        by_team(team, V, [&](auto w, auto is_short) {
            constexpr int TEAM = decltype(w)::value;
            const dim3 grid((unsigned)(groups(N, team) * a.splits));
            if constexpr (decltype(is_short)::value)
                hipLaunchKernelGGL((k_grad_short<T, TEAM>), grid, dim3(256), 0, (hipStream_t)stream, a);
            else
                hipLaunchKernelGGL((k_grad<T, TEAM>), grid, dim3(256), lds, (hipStream_t)stream, a);
        });
        return launched();
    });
}

}  // extern "C"
