// The gated projection y = silu(x Wg^T) * (x Wu^T) on gfx950, with its first and second derivatives (C ABI and formulas:
// include/ebr_block.h): products on the matrix cores with the activation, or its second derivative, in their epilogues.
//
// Every product is D[j][i] = sum over k of A(i, k) B(j, k), i being the direction in which D lies in memory. An operand lies
// with its rows' k side by side (K), or with its rows side by side for each k (M):
//   [g|u] = x W^T     A = W (K), rows of gate and up in turns of 32, so that a lane holds both at the same place; B = x (K).
//                     With B = rows of x and of c in turns of 32, a lane holds [cg|cu] = c W^T there as well
//   dx = [dg|du] W    A = W (M), B = [dg|du] (K)
//   dW = [dg|du]^T x  A = x (M), B = [dg|du] (M), the rows split among workgroups, partial sums added up in a fixed order
//
// The derivatives take g and u again: kept rounded they would double the gradients' errors, and kept in fp32 their product costs
// less than moving them for C below about a thousand (above it, 8192 x 2048 -> 5632, 403 us against some 145 for 369 MB written and
// read, but nothing has to be held from the forward to the backward).
//
// [dg|du] and [gg|gu] are rounded to the type, as the matrix instructions take them: in 16 bits the gradients are 2.3e-3 off in
// the mean square, where the rounding of the outputs alone makes 1.7e-3. Of up to 64 rows, whose products wait for the weight's bytes
// in any case, what the rounding leaves goes in as a second operand; of more, it would double dx's and dw's products.
//
// A workgroup's tile of TI x TJ steps through k in stages of 64 bytes an operand row, loaded straight into shared memory three
// stages ahead. The four buffers are separate arrays: the compiler then knows that the loads under way do not concern the
// reads, and does not wait for them. Rows' 16-byte chunks (64-byte chunks for operands of the
// second kind, which are read transposed) are exchanged by a function of the row, so that lanes meet no bank conflicts.
// Whatever lies outside the tensors is read as zero by the buffer loads' bounds.
//
// Tiles of 256 x 256 in 16 bits where there are enough of them: four waves of 128 x 128 (fewest bytes of shared memory a product),
// eight of 128 x 64 where the activation follows, whose arithmetic two waves a SIMD overlap (62208 x 256 -> 768: forward 88 us, 99
// with four; backward 118, 145; second 237, 275). Bound by the matrix cores at long k (8192 x 2048 -> 5632: forward 380 us, 995
// TFLOP/s, the library's product without the activation 396; backward's product 403; dx 320, 1,180; dw 357, 1,060), at k of some
// hundreds by prologue and epilogue. fp32 goes in tiles of 128, at the fp32 instructions' rate.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "../../include/ebr_block.h"
#include "glu_plan.hpp"
#include "rowwise.hpp"

namespace ebr_glu {

using namespace ebr_row;

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
#define EBR_LDS __attribute__((address_space(3)))

enum { K_ROWS = 0, M_ROWS = 1 };                                  // how an operand lies
enum { EP_OUT = 0, EP_PART = 1, EP_FWD = 2, EP_BWD = 3, EP_BWD2 = 4 };  // what becomes of D: y, [dg|du], or all of bwd2's
constexpr uint32_t OUTSIDE = 0x40000000;                          // an offset past a buffer's end

struct Args {
    const void *a[4], *b[4];  // pairs: the sum goes over the k of all of them, one after the other
    int64_t lda, ldb;         // elements between rows (of k, for M)
    int64_t ni, nj, nk;       // rows of A (gated: of the gate), of B, and k of one pair
    int pairs, splits;
    int64_t steps;            // stages of a split
    int ti, tj;               // tiles
    int tile0, count;         // those of this launch
    void *out, *dgu, *ggu;    // D, y or gdy; [dg|du]; [gg|gu]
    void *dgu2, *ggu2;        // what these lack of their values before rounding, or null
    const void *dy, *c;
    int64_t ldo;
};

template <typename T> struct Mma;
template <> struct Mma<__bf16> {
    static __device__ __forceinline__ f32x16 step(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mma<_Float16> {
    static __device__ __forceinline__ f32x16 step(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mma<float> {  // four values of k a lane, one a step
    static __device__ __forceinline__ f32x16 step(u32x4 a, u32x4 b, f32x16 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            c = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(float, (uint32_t)a[e]),
                                                     __builtin_bit_cast(float, (uint32_t)b[e]), c, 0, 0, 0);
        return c;
    }
};

// One operand's part of a workgroup: ROWS rows, of which WAVES waves load their share.
template <typename T, int LIES, int ROWS, int WAVES, bool PAIRED> struct Side {
    static constexpr int ES = (int)sizeof(T), EPC = 16 / ES, KS = STAGE / ES;  // elements of a chunk, k of a stage
    static constexpr int BYTES = ROWS * STAGE, LOADS = BYTES / 1024 / WAVES;
    static constexpr int ROWB = LIES == K_ROWS ? STAGE : ROWS * ES;  // bytes of a row in shared memory
    static constexpr int MASK = ROWB / 64 >= 4 ? 3 : ROWB / 64 - 1;
    static_assert(BYTES % (1024 * WAVES) == 0, "whole loads a wave");

    // The chunk (16 bytes) that lies at place p of a stage: its row (K) or k (M), and its first element there.
    static __device__ __forceinline__ void chunk(int p, int& row, int& at) {
        row = p * 16 / ROWB;
        const int c = p - row * (ROWB / 16);
        if constexpr (LIES == K_ROWS) at = (c ^ ((row >> 2) & 3)) * EPC;
        else at = ((((c >> 2) ^ (row & MASK)) << 2) | (c & 3)) * EPC;
    }
    // Row r of the tile that begins at row ``first``, in the operand, or -1 where there is none. PAIRED: rows of the two
    // operands of a pair in turns of 32, the same ones of each.
    static __device__ __forceinline__ int64_t source(int r, int64_t first, int64_t n) {
        const int64_t i = PAIRED ? first / 2 + (r >> 6) * 32 + (r & 31) : first + r;
        return i < n ? i : -1;
    }
    static __device__ __forceinline__ bool other(int r) { return PAIRED && ((r >> 5) & 1); }

    // This lane's byte offsets from the tile's place at the stage's k, past the end where a row is missing.
    uint32_t off[LOADS];
    int kat[LOADS];  // the k of its first element in a stage
    __device__ __forceinline__ void offsets(int64_t first, int64_t n, int64_t ld, int wave, int lane) {
#pragma unroll
        for (int q = 0; q < LOADS; ++q) {
            int row, at;
            chunk((wave * LOADS + q) * 64 + lane, row, at);
            if constexpr (LIES == K_ROWS) {
                const int64_t s = source(row, first, n);
                off[q] = s < 0 ? OUTSIDE : (uint32_t)(((s - (PAIRED ? first / 2 : first)) * ld + at) * ES);
                kat[q] = at;
            } else {
                off[q] = first + at < n ? (uint32_t)((row * ld + at) * ES) : OUTSIDE;
                kat[q] = row;
            }
        }
    }
    // How far the tile's place at k0 lies from the operand's.
    static __device__ __forceinline__ int64_t skip(int64_t first, int64_t ld, int64_t k0) {
        return LIES == K_ROWS ? (PAIRED ? first / 2 : first) * ld + k0 : first + k0 * ld;
    }
    // Loads the stage at p (and, of a pair's other operand, p2), of which ``left`` k exist, into ``to``.
    __device__ __forceinline__ void load(const T* p, const T* p2, int left, unsigned char* to, int wave) const {
#ifdef __HIP_DEVICE_COMPILE__  // (the host's pass has no buffers)
        constexpr int RAW = 0x00020000;  // dwords as they are
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)OUTSIDE, RAW);
        __amdgpu_buffer_rsrc_t r2 = r;
        if constexpr (PAIRED) r2 = __builtin_amdgcn_make_buffer_rsrc((void*)p2, 0, (int)OUTSIDE, RAW);
#pragma unroll
        for (int q = 0; q < LOADS; ++q) {
            const int at = wave * LOADS + q;  // (a load's 16 rows are of one operand)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(other(at * 16) ? r2 : r, (EBR_LDS void*)(to + at * 1024), 16,
                                                     kat[q] < left ? off[q] : OUTSIDE, 0, 0, 0);
        }
#endif
    }
    // The 32 rows from r0 (a multiple of 32) at step s of a stage: lane (row l % 32, half l / 32) gets EPC values of k.
    static __device__ __forceinline__ u32x4 read(const unsigned char* from, int r0, int s, int lane) {
        const int l32 = lane & 31, half = lane >> 5;
        if constexpr (LIES == K_ROWS) {
            const int row = r0 + l32;
            return *reinterpret_cast<const u32x4*>(from + row * ROWB + (((2 * s + half) ^ ((row >> 2) & 3)) << 4));
        } else if constexpr (ES == 2) {
            const int l16 = lane & 15, k = 16 * s + 8 * half + (l16 >> 2), col = (r0 + (lane & 16) + 4 * (l16 & 3)) * ES;
            const unsigned char* p = from + k * ROWB + ((((col >> 6) ^ (k & MASK)) << 6) | (col & 63));
            const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((EBR_LDS s16x4*)p));
            const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((EBR_LDS s16x4*)(p + 4 * ROWB)));
            return u32x4{lo[0], lo[1], hi[0], hi[1]};
        } else {
            u32x4 v;
            const int col = (r0 + l32) * ES;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int k = 8 * s + 4 * half + e;
                v[e] = *reinterpret_cast<const uint32_t*>(from + k * ROWB + ((((col >> 6) ^ (k & MASK)) << 6) | (col & 63)));
            }
            return v;
        }
    }
};

template <typename A> __device__ __forceinline__ A sigmoid(A g);
template <> __device__ __forceinline__ float sigmoid(float g) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896f * g));
}
template <> __device__ __forceinline__ double sigmoid(double g) { return 1.0 / (1.0 + exp(-g)); }

template <typename A> __device__ __forceinline__ A gated(A g, A u) { return g * sigmoid(g) * u; }
// Its gradients for g and u, and those of <c, (dg, du)> for g, u and dy.
template <typename A> __device__ __forceinline__ void first_of(A g, A u, A dy, A& dg, A& du) {
    const A s = sigmoid(g);
    dg = dy * u * (s * ((A)1 + g * ((A)1 - s)));
    du = dy * (g * s);
}
template <typename A>
__device__ __forceinline__ void second_of(A g, A u, A dy, A cg, A cu, A& gg, A& gu, A& gdy) {
    const A s = sigmoid(g), f1 = s * ((A)1 + g * ((A)1 - s)), f2 = s * ((A)1 - s) * ((A)2 + g * ((A)1 - (A)2 * s));
    gg = dy * (cg * u * f2 + cu * f1);
    gu = cg * dy * f1;
    gdy = cg * u * f1 + cu * (g * s);
}

// Four neighbours at p, of which ``n`` exist.
template <typename T> __device__ __forceinline__ void put4(T* p, const float (&v)[4], int64_t n, bool whole) {
    if (whole && n >= 4) {
        Pack<T, 4> x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x.e[e] = (T)v[e];
        stp<T, 4>(p, x);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) p[e] = (T)v[e];
    }
}
// The same whatever the alignment, in one access where there are four.
template <typename T> __device__ __forceinline__ void put4_anywhere(T* p, const float (&v)[4], int64_t n) {
    T x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (T)v[e];
    if (n >= 4) {
        __builtin_memcpy(p, x, sizeof(x));
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) p[e] = x[e];
    }
}
// What two fours lack of their values once rounded.
template <typename T>
__device__ __forceinline__ void put_rest(T* p, const float (&g)[4], const float (&u)[4], int64_t next, int64_t n, bool whole) {
    float rg[4], ru[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        rg[e] = g[e] - (float)(T)g[e];
        ru[e] = u[e] - (float)(T)u[e];
        if (!__builtin_isfinite(rg[e])) rg[e] = 0.f;  // (of a value past the type's range)
        if (!__builtin_isfinite(ru[e])) ru[e] = 0.f;
    }
    put4(p, rg, n, whole);
    put4(p + next, ru, n, whole);
}
template <typename T> __device__ __forceinline__ void get4(const T* p, float (&v)[4], int64_t n, bool whole) {
    if (whole && n >= 4) {
        const Pack<T, 4> x = ldp<T, 4>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)x.e[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = e < n ? (float)p[e] : 0.f;
    }
}

// All of a wave's reads of shared memory done, and all but its last N loads; and every wave there.
template <int N> __device__ __forceinline__ void stage_barrier() {
    static_assert(N < 64, "vmcnt");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Tile t: a block of GROUP tiles of j goes with all i before the next.
__device__ __forceinline__ void place_of(const Args& a, unsigned t, int& ti, int& tj) {
    constexpr int GROUP = 8;
    const unsigned block = t / (GROUP * a.ti), first = block * GROUP;
    const unsigned rows = a.tj - first < GROUP ? a.tj - first : GROUP, in = t - block * GROUP * a.ti;
    tj = (int)(first + in % rows);
    ti = (int)(in / rows);
}
// The tile of a workgroup: each of the 8 XCDs, which take workgroups in turns, gets neighbouring tiles.
__device__ __forceinline__ void tile_of(const Args& a, int& ti, int& tj, int& split, int& local) {
    const unsigned tiles = (unsigned)a.count, all = tiles * a.splits, b = blockIdx.x;
    const unsigned per = all / 8, more = all % 8, x = b % 8;
    const unsigned at = x * per + (x < more ? x : more) + b / 8;
    split = (int)(at / tiles);
    local = (int)(at % tiles);
    place_of(a, a.tile0 + local, ti, tj);
}

// A wave's way from its sums to rows of memory: planes of 32 rows of COLS values in shared memory, in chunks of 16 bytes exchanged
// by a function of the row. A lane holds four neighbours of one row; memory gets (and gives) whole chunks, a row's side by side.
template <typename O, int COLS> struct Plane {
    static constexpr int PER = 16 / (int)sizeof(O), ROWB = COLS * (int)sizeof(O), CHUNKS = ROWB / 16, BYTES = 32 * ROWB;
    static constexpr int SHIFT = ROWB == 256 ? 0 : ROWB == 128 ? 1 : 2, MOVES = BYTES / 1024;
    static_assert(ROWB == 64 || ROWB == 128 || ROWB == 256, "rows of whole banks");
    static __device__ __forceinline__ int place(int row, int chunk) {
        return row * ROWB + ((chunk ^ ((row >> SHIFT) & (CHUNKS - 1))) << 4);
    }
    // four values of ``row`` from column ``col`` (a multiple of 4) on
    static __device__ __forceinline__ unsigned char* four(unsigned char* at, int row, int col) {
        return at + place(row, col / PER) + col % PER * (int)sizeof(O);
    }
    static __device__ __forceinline__ void put(unsigned char* at, int row, int col, const float (&v)[4]) {
        Pack<O, 4> x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x.e[e] = (O)v[e];
        stp<O, 4>(reinterpret_cast<O*>(four(at, row, col)), x);
    }
    static __device__ __forceinline__ void get(unsigned char* at, int row, int col, float (&v)[4]) {
        const Pack<O, 4> x = ldp<O, 4>(reinterpret_cast<const O*>(four(at, row, col)));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)x.e[e];
    }
    // all of it to (from) rows of memory ``ld`` elements apart, of which ``rows`` and ``cols`` exist: a move takes STEP rows
    static constexpr int STEP = 64 / CHUNKS;
    static __device__ __forceinline__ uint32_t offset(int64_t ld, int lane) {
        return (uint32_t)(lane / CHUNKS * (int)ld + lane % CHUNKS * PER) * (uint32_t)sizeof(O);
    }
    static __device__ __forceinline__ bool there(int m, int rows, int cols, int lane) {
        return m * STEP + lane / CHUNKS < rows && lane % CHUNKS * PER < cols;
    }
    static __device__ __forceinline__ void store(const unsigned char* at, O* to, int64_t ld, int rows, int cols, int lane) {
        u32x4 v[MOVES];
#pragma unroll
        for (int m = 0; m < MOVES; ++m)
            v[m] = *reinterpret_cast<const u32x4*>(at + place(m * STEP + lane / CHUNKS, lane % CHUNKS));
        char* base = reinterpret_cast<char*>(to);
        const uint32_t off = offset(ld, lane);
#pragma unroll
        for (int m = 0; m < MOVES; ++m) {
            if (there(m, rows, cols, lane)) *reinterpret_cast<u32x4*>(base + off) = v[m];
            base += STEP * ld * (int64_t)sizeof(O);
        }
    }
    static __device__ __forceinline__ void load(unsigned char* at, const O* from, int64_t ld, int rows, int cols, int lane) {
        u32x4 v[MOVES];
        const char* base = reinterpret_cast<const char*>(from);
        const uint32_t off = offset(ld, lane);
#pragma unroll
        for (int m = 0; m < MOVES; ++m) {
            v[m] = there(m, rows, cols, lane) ? *reinterpret_cast<const u32x4*>(base + off) : u32x4{};
            base += STEP * ld * (int64_t)sizeof(O);
        }
#pragma unroll
        for (int m = 0; m < MOVES; ++m)
            *reinterpret_cast<u32x4*>(at + place(m * STEP + lane / CHUNKS, lane % CHUNKS)) = v[m];
    }
};

// How many of a plane's rows or columns there are: none where it lies outside.
__device__ __forceinline__ int left(int64_t n) { return n > 256 ? 256 : (int)n; }

// What becomes of a wave's sums, 32 rows at a time through ``at``, shared memory of its own.
template <typename T, int EP, int FI, int FJ>
__device__ __forceinline__ void finish(const Args& a, const f32x16 (&acc)[FI][FJ], int64_t ifrom, int64_t jfrom, float* part, int ldp,
                                       unsigned char* at, unsigned char* at4, int lane) {
    constexpr bool TWO = EP == EP_BWD2;
    const int l32 = lane & 31, il = 4 * (lane >> 5);
    if constexpr (EP < EP_FWD) {
        using O = std::conditional_t<EP == EP_PART, float, T>;
        constexpr int COLS = 128 / (int)sizeof(O), EACH = COLS / 32;  // a plane's tiles of 32
        using P = Plane<O, COLS>;
        O* out;  // at the wave's first place
        int64_t ldo = ldp;
        if constexpr (EP == EP_PART) out = part;
        else out = reinterpret_cast<O*>(a.out) + jfrom * a.ldo + ifrom, ldo = a.ldo;
#pragma unroll
        for (int j = 0; j < FJ; ++j)
#pragma unroll
            for (int i = 0; i < FI; i += EACH) {
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int e = 0; e < EACH; ++e)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const f32x16& s = acc[i + e][j];
                        const float v[4] = {s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]};
                        P::put(at + i / EACH * P::BYTES, l32, e * 32 + 8 * q + il, v);
                    }
                __builtin_amdgcn_wave_barrier();
                const int64_t row = jfrom + j * 32, col = ifrom + i * 32;
                P::store(at + i / EACH * P::BYTES, out + j * 32 * ldo + i * 32, ldo, left(a.nj - row), left(a.ni - col), lane);
            }
    } else {
        using P = Plane<T, FI * 16>;  // of gate or up, each half of the wave's rows of A
        enum { DY = 0, Y = 0, DG = 1, DU = 2, GG = 3 };  // and GU at ``at4``
        const int64_t col = ifrom / 2;
        const int cols = left(a.ni - col);
        T* const y = reinterpret_cast<T*>(a.out);
        T *const dgu = reinterpret_cast<T*>(a.dgu), *const ggu = reinterpret_cast<T*>(a.ggu);
#pragma unroll
        for (int j = 0; j < FJ; j += TWO ? 2 : 1) {
            const int64_t row = TWO ? jfrom / 2 + j * 16 : jfrom + j * 32;
            const int rows = left(a.nj - row);
            const int64_t one = row * a.ni + col, two = row * 2 * a.ni + col;
            __builtin_amdgcn_wave_barrier();
            if constexpr (EP != EP_FWD) P::load(at + DY * P::BYTES, reinterpret_cast<const T*>(a.dy) + one, a.ni, rows, cols, lane);
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < FI; i += 2)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int c = i * 16 + 8 * q + il;
                    float dy[4], o[4], og[4], ou[4], rg[4], ru[4];
                    if constexpr (EP != EP_FWD) P::get(at + DY * P::BYTES, l32, c, dy);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float g = acc[i][j][4 * q + e], u = acc[i + 1][j][4 * q + e];
                        if constexpr (EP == EP_FWD) o[e] = gated(g, u);
                        else first_of(g, u, dy[e], og[e], ou[e]);
                        if constexpr (TWO)
                            second_of(g, u, dy[e], acc[i][j + 1][4 * q + e], acc[i + 1][j + 1][4 * q + e], rg[e], ru[e], o[e]);
                    }
                    if constexpr (EP != EP_BWD) P::put(at + Y * P::BYTES, l32, c, o);
                    if constexpr (EP != EP_FWD) {
                        P::put(at + DG * P::BYTES, l32, c, og);
                        P::put(at + DU * P::BYTES, l32, c, ou);
                    }
                    if constexpr (TWO) {
                        P::put(at + GG * P::BYTES, l32, c, rg);
                        P::put(at4, l32, c, ru);
                    }
                    if constexpr (EP != EP_FWD) __builtin_amdgcn_sched_barrier(0);  // (several at once would not fit the registers)
                }
            __builtin_amdgcn_wave_barrier();
            if constexpr (EP != EP_BWD) P::store(at + Y * P::BYTES, y + one, a.ni, rows, cols, lane);
            if (EP == EP_BWD || (TWO && dgu)) {
                P::store(at + DG * P::BYTES, dgu + two, 2 * a.ni, rows, cols, lane);
                P::store(at + DU * P::BYTES, dgu + two + a.ni, 2 * a.ni, rows, cols, lane);
            }
            if (TWO && ggu) {
                P::store(at + GG * P::BYTES, ggu + two, 2 * a.ni, rows, cols, lane);
                P::store(at4, ggu + two + a.ni, 2 * a.ni, rows, cols, lane);
            }
        }
    }
}

// The same straight from the registers, for fp32 and for few rows (what [dg|du] lacks of its
// values before rounding is written here alone).
template <typename T, int EP, int FI, int FJ>
__device__ __forceinline__ void finish_few(const Args& a, const f32x16 (&acc)[FI][FJ], int64_t i0, int64_t j0, int wi, int wj,
                                           float* part, int ldp, int lane) {
    constexpr bool GATED = EP >= EP_FWD, TWO = EP == EP_BWD2;
    const int64_t jl = j0 + wj * FJ * 32 + (lane & 31);
    const int il = 4 * (lane >> 5);
    if constexpr (!GATED) {
#pragma unroll
        for (int j = 0; j < FJ; ++j) {
            const int64_t row = jl + j * 32;
            if (row >= a.nj) continue;
#pragma unroll
            for (int i = 0; i < FI; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int64_t col = i0 + (wi * FI + i) * 32 + 8 * q + il;
                    const float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                    if (col >= a.ni) continue;
                    if constexpr (EP == EP_OUT) {
                        put4(reinterpret_cast<T*>(a.out) + row * a.ldo + col, v, a.ni - col, true);
                    } else {
                        put4(part + (row - j0) * ldp + (col - i0), v, a.ni - col, true);
                    }
                }
        }
    } else {
#pragma unroll
        for (int j = 0; j < FJ; j += TWO ? 2 : 1) {
            const int64_t row = TWO ? j0 / 2 + (wj * FJ + j) * 16 + (lane & 31) : jl + j * 32;
            if (row >= a.nj) continue;
#pragma unroll
            for (int i = 0; i < FI; i += 2)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int64_t col = i0 / 2 + (wi * FI + i) * 16 + 8 * q + il;
                    if (col >= a.ni) continue;
                    const int64_t n = a.ni - col, at = row * a.ni + col, two = row * 2 * a.ni + col;
                    T* const dgu = reinterpret_cast<T*>(a.dgu) + two;
                    T* const ggu = reinterpret_cast<T*>(a.ggu) + two;
                    float dy[4], og[4], ou[4], o[4];
                    if constexpr (EP != EP_FWD) get4(reinterpret_cast<const T*>(a.dy) + at, dy, n, true);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float g = acc[i][j][4 * q + e], u = acc[i + 1][j][4 * q + e];
                        if constexpr (EP == EP_FWD) o[e] = gated(g, u);
                        else first_of(g, u, dy[e], og[e], ou[e]);
                    }
                    if constexpr (EP == EP_FWD) put4(reinterpret_cast<T*>(a.out) + at, o, n, true);
                    if (EP == EP_BWD || (TWO && a.dgu)) {
                        put4(dgu, og, n, true);
                        put4(dgu + a.ni, ou, n, true);
                        if (a.dgu2) put_rest(reinterpret_cast<T*>(a.dgu2) + two, og, ou, a.ni, n, true);
                    }
                    if constexpr (TWO) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            second_of(acc[i][j][4 * q + e], acc[i + 1][j][4 * q + e], dy[e], acc[i][j + 1][4 * q + e],
                                      acc[i + 1][j + 1][4 * q + e], og[e], ou[e], o[e]);
                        put4(reinterpret_cast<T*>(a.out) + at, o, n, true);
                        if (a.ggu) {
                            put4(ggu, og, n, true);
                            put4(ggu + a.ni, ou, n, true);
                            if (a.ggu2) put_rest(reinterpret_cast<T*>(a.ggu2) + two, og, ou, a.ni, n, true);
                        }
                    }
                }
        }
    }
}

template <typename T, int ALIES, int BLIES, int EP, int TI, int TJ, int WI, int WJ>
__global__ __launch_bounds__(64 * WI * WJ) void k_product(Args a) {
    constexpr int WAVES = WI * WJ, FI = TI / WI / 32, FJ = TJ / WJ / 32;
    constexpr bool GATED = EP >= EP_FWD, TWO = EP == EP_BWD2;
    constexpr bool STAGED = staged(sizeof(T), TI);  // four waves, an array each, or eight, half of one
    static_assert(!STAGED || WAVES == 4 || WAVES == 8, "an array a wave");
    static_assert(64 * WAVES == product_threads(sizeof(T), TI, TWO ? 2 : GATED), "the threads that sizes are checked for");
    static_assert((!GATED || FI % 2 == 0) && (!TWO || FJ % 2 == 0), "a wave's tile holds both of a pair");
    using SA = Side<T, ALIES, TI, WAVES, GATED>;
    using SB = Side<T, BLIES, TJ, WAVES, TWO>;
    constexpr int BUFFER = SA::BYTES + SB::BYTES;
    constexpr int FIFTH = TWO && WAVES == 8 ? BUFFER / 8 : 0;  // a wave's fifth plane, where half a buffer holds four
    __shared__ __attribute__((aligned(16))) unsigned char s0[BUFFER], s1[BUFFER], s2[BUFFER], s3[BUFFER], s4[FIFTH ? WAVES * FIFTH : 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave % WI, wj = wave / WI;
    int ti, tj, split, local;
    tile_of(a, ti, tj, split, local);
    const int64_t i0 = (int64_t)ti * TI, j0 = (int64_t)tj * TJ;
    f32x16 acc[FI][FJ];
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    const int64_t one = (a.nk + SA::KS - 1) / SA::KS, all = one * a.pairs;  // stages of a pair
    int64_t step = split * a.steps;
    const int64_t end = step + a.steps < all ? step + a.steps : all;
    u32x4 fa[2][FI], fb[2][FJ];
    const auto read = [&](const unsigned char* from, int s) {
#pragma unroll
        for (int i = 0; i < FI; ++i) fa[s][i] = SA::read(from, (wi * FI + i) * 32, s, lane);
#pragma unroll
        for (int j = 0; j < FJ; ++j) fb[s][j] = SB::read(from + SA::BYTES, (wj * FJ + j) * 32, s, lane);
    };
    // fp32: the sums of 64 k each, added up apart (one chain over all k is off by three times as much)
    constexpr bool IN_PARTS = sizeof(T) == 4;
    f32x16 sums[IN_PARTS ? FI : 1][IN_PARTS ? FJ : 1] = {};
    const auto take = [&]() {
        if constexpr (IN_PARTS) {
#pragma unroll
            for (int i = 0; i < FI; ++i)
#pragma unroll
                for (int j = 0; j < FJ; ++j) {
                    sums[i][j] += acc[i][j];
                    acc[i][j] = f32x16{};
                }
        }
    };
    const auto multiply = [&](int s) {
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int j = 0; j < FJ; ++j) acc[i][j] = Mma<T>::step(fa[s][i], fb[s][j], acc[i][j]);
        // the next fragments' reads (and the next stage's loads) between the first products, so that they are there after the
        // last ones
        constexpr int READS = FI * (ALIES == K_ROWS ? 1 : sizeof(T) == 2 ? 2 : 4) + FJ * (BLIES == K_ROWS ? 1 : sizeof(T) == 2 ? 2 : 4);
        constexpr int MM = FI * FJ * (sizeof(T) == 2 ? 1 : 4), EACH = (READS + MM / 2 - 1) / (MM / 2 > 0 ? MM / 2 : 1);
        constexpr int GO = (SA::LOADS + SB::LOADS + MM / 2 - 1) / (MM / 2 > 0 ? MM / 2 : 1);
#pragma unroll
        for (int g = 0; g < MM / 2; ++g) {
            __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);             // LDS reads
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                // a product
            if (s == 1) __builtin_amdgcn_sched_group_barrier(0x020, GO, 0);  // loads
        }
        __builtin_amdgcn_sched_barrier(0);  // (all fragments of a stage at once would not fit the registers)
    };
    SA sa;
    SB sb;
    sa.offsets(i0, a.ni, a.lda, wave, lane);
    sb.offsets(j0, a.nj, a.ldb, wave, lane);
    const T *pa, *pb, *pa2 = nullptr, *pb2 = nullptr;  // of the stage to be loaded next
    int rest;                                          // its k and those after it
    const int64_t sa_step = ALIES == K_ROWS ? SA::KS : SA::KS * a.lda, sb_step = BLIES == K_ROWS ? SB::KS : SB::KS * a.ldb;
    const auto advance = [&]() {
        rest -= SA::KS;
        pa += sa_step;
        pb += sb_step;
        if (GATED) pa2 += sa_step;
        if (TWO) pb2 += sb_step;
    };
    const auto load = [&](unsigned char* to) {
        const int left = rest < SA::KS ? rest : SA::KS;  // (none past the end: the loads read nothing and write zeros)
        sa.load(pa, pa2, left, to, wave);
        sb.load(pb, pb2, left, to + SA::BYTES, wave);
    };
    // A stage's last products run while the next one's first fragments are read, after the barrier that says that its loads
    // are there and that nobody reads this stage's buffer any more, which the loads of the fourth stage from here go to:
    // loads have three stages' time.
    constexpr int AHEAD = 2 * (SA::LOADS + SB::LOADS);  // of a wave, of the two stages after the next
    const auto stage = [&](unsigned char* here, const unsigned char* next) {
        read(here, 1);
        multiply(0);
        advance();
        stage_barrier<AHEAD>();
        load(here);
        read(next, 0);
        multiply(1);
    };
    for (int pair = 0; pair < (GATED ? 1 : a.pairs); ++pair) {
        // this split's stages of the pair: in fours, what lacks of them with zeros (which costs their products, but a branch
        // out of the loop's middle would cost a second copy of all sums)
        const int64_t from = step > pair * one ? step - pair * one : 0, to = end < (pair + 1) * one ? end - pair * one : one;
        if (from >= to) continue;
        const int64_t k0 = from * SA::KS, k1 = to * SA::KS < a.nk ? to * SA::KS : a.nk;
        const int64_t ia = SA::skip(i0, a.lda, k0), ib = SB::skip(j0, a.ldb, k0);
        pa = reinterpret_cast<const T*>(a.a[pair]) + ia;
        pb = reinterpret_cast<const T*>(a.b[pair]) + ib;
        if (GATED) pa2 = pa + a.ni * a.lda;
        if (TWO) pb2 = reinterpret_cast<const T*>(a.c) + ib;
        rest = (int)(k1 - k0);
        const int n = (int)(to - from);
        if (pair > 0) stage_barrier<0>();  // (the loads past the last pair's end are done with the buffers)
        load(s0);
        advance();
        load(s1);
        advance();
        load(s2);
        stage_barrier<AHEAD>();
        advance();
        load(s3);
        read(s0, 0);
        for (int s = 0; s < n; s += 4) {
            stage(s0, s1);
            stage(s1, s2);
            stage(s2, s3);
            stage(s3, s0);
            if constexpr (IN_PARTS) take();
        }
    }
    stage_barrier<0>();  // (the loads past the end, of zeros, are done with the buffers)

    if constexpr (IN_PARTS)
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int j = 0; j < FJ; ++j) acc[i][j] = sums[i][j];
    // the sums of a split: tile by tile
    float* const part = EP == EP_PART ? reinterpret_cast<float*>(a.out) + ((int64_t)split * a.count + local) * (TI * TJ) : nullptr;
    if constexpr (STAGED) {
        // (every wave is past its last read of the buffers: the last stage's barrier)
        constexpr int PER = WAVES / 4, MINE = BUFFER / PER;
        unsigned char* const own = (wave / PER == 0 ? s0 : wave / PER == 1 ? s1 : wave / PER == 2 ? s2 : s3) + wave % PER * MINE;
        constexpr int FOUR = 4 * 32 * FI * 16 * (int)sizeof(T);  // planes
        static_assert(!TWO || (FIFTH ? FOUR <= MINE && FOUR / 4 <= FIFTH : FOUR / 4 * 5 <= MINE), "a wave's planes");
        finish<T, EP, FI, FJ>(a, acc, i0 + wi * FI * 32, j0 + wj * FJ * 32, EP == EP_PART ? part + wj * FJ * 32 * TI + wi * FI * 32 : part,
                              TI, own, FIFTH ? s4 + wave * FIFTH : own + FOUR, lane);
    } else {
        finish_few<T, EP, FI, FJ>(a, acc, i0, j0, wi, wj, part, TI, lane);
    }
}

// Few rows of x: the weight, once, straight into registers, bound by its bytes. x, w and y may have any alignment. A workgroup's waves take 16 rows of gate and of
// up, and of their k 128 bytes in turns; the order of k within a product is the lanes' own (each brings 16 bytes of its row of
// either operand), so that a wave's loads take whole lines. The waves' sums are added up through shared memory.
//
// Against tiles of 64, weights from memory, us: bf16 C 2048 I 5632 14.5 : 18.7 for one row (3.2 TB/s), 19.4 : 18.8 for 17, 24.7 :
// 19.1 for 33; C 4096 I 11008 40 : 46 (4.5 TB/s), 53 : 53, 65 : 55; C 256 I 768 2.7 : 4.1, 3.2 : 4.1, 3.6 : 4.2; fp32 C 2048 I 5632
// 31 : 68, 45 : 68, 66 : 68. So for up to 32 rows.
template <typename T> struct Mma16;
template <> struct Mma16<__bf16> {
    static __device__ __forceinline__ f32x4 step(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mma16<_Float16> {
    static __device__ __forceinline__ f32x4 step(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mma16<float> {
    static __device__ __forceinline__ f32x4 step(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, (uint32_t)a[e]),
                                                     __builtin_bit_cast(float, (uint32_t)b[e]), c, 0, 0, 0);
        return c;
    }
};
template <typename T, int EP, int ROWS> __global__ __launch_bounds__(64 * FEW_WAVES) void k_few(Args a) {
    constexpr bool TWO = EP == EP_BWD2;
    constexpr int FJ = ROWS * (TWO ? 2 : 1);  // sixteens of x, then of c
    constexpr int EPC = 16 / (int)sizeof(T), TURN = 8 * EPC, AT_ONCE = FJ == 4 ? 2 : 4;  // k of a wave's turn; turns under way
    __shared__ f32x4 sums[FEW_WAVES][2][FJ][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, part = lane >> 4;
    // 16 bytes of a row from k on, or what it has of them; at the row's end the bytes before, taken out
    const auto chunk = [&](const T* p, int64_t k) {
        const int64_t at = k < a.nk - EPC ? k : a.nk - EPC, cut = (k - at) * 8 * (int)sizeof(T);
        u32x4 v;
        __builtin_memcpy(&v, p + at, 16);
        if (cut > 0)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int64_t n = cut - 32 * w;
                v[w] = n <= 0 ? v[w] : n < 32 ? v[w] & (~0u << n) : 0;
            }
        return v;
    };
    const int64_t i0 = (int64_t)blockIdx.x * 16, row = i0 + l16 < a.ni ? i0 + l16 : a.ni - 1;  // (the last one again past the end)
    const T* const gate = reinterpret_cast<const T*>(a.a[0]) + row * a.lda;
    const T* const up = gate + a.ni * a.lda;
    const T* const x = reinterpret_cast<const T*>(a.b[0]);
    f32x4 acc[2][FJ] = {};
    for (int64_t k0 = wave * TURN; k0 < a.nk; k0 += FEW_WAVES * TURN * AT_ONCE) {
        u32x4 g[AT_ONCE][2], u[AT_ONCE][2], b[AT_ONCE][2][FJ];
#pragma unroll
        for (int t = 0; t < AT_ONCE; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t k = k0 + t * FEW_WAVES * TURN + (part * 2 + h) * EPC;
                const bool in = k < a.nk;
                g[t][h] = in ? chunk(gate, k) : u32x4{};
                u[t][h] = in ? chunk(up, k) : u32x4{};
#pragma unroll
                for (int j = 0; j < FJ; ++j) {
                    const int64_t n = j % ROWS * 16 + l16;
                    const T* const from = j < ROWS ? x : reinterpret_cast<const T*>(a.c);
                    b[t][h][j] = in && n < a.nj ? chunk(from + n * a.ldb, k) : u32x4{};
                }
            }
#pragma unroll
        for (int t = 0; t < AT_ONCE; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < FJ; ++j) {
                    acc[0][j] = Mma16<T>::step(g[t][h], b[t][h][j], acc[0][j]);
                    acc[1][j] = Mma16<T>::step(u[t][h], b[t][h][j], acc[1][j]);
                }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < FJ; ++j) sums[wave][h][j][lane] = acc[h][j];
    __syncthreads();
    if (wave >= ROWS) return;
    const auto total = [&](int h, int j) {
        f32x4 v = {};
#pragma unroll
        for (int w = 0; w < FEW_WAVES; ++w) v += sums[w][h][j][lane];
        return v;
    };
    const f32x4 g = total(0, wave), u = total(1, wave);
    f32x4 cg = {}, cu = {};
    if constexpr (TWO) cg = total(0, wave + ROWS), cu = total(1, wave + ROWS);
    const int64_t n = wave * 16 + l16, i = i0 + 4 * part;
    if (n >= a.nj || i >= a.ni) return;
    const int64_t some = a.ni - i, at = n * a.ni + i, two = n * 2 * a.ni + i;
    const bool whole = a.ni % 4 == 0;
    T* const y = reinterpret_cast<T*>(a.out);
    float dy[4], o[4], og[4], ou[4], rg[4], ru[4];
    if constexpr (EP != EP_FWD) get4(reinterpret_cast<const T*>(a.dy) + at, dy, some, whole);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (EP == EP_FWD) o[e] = gated(g[e], u[e]);
        else first_of(g[e], u[e], dy[e], og[e], ou[e]);
        if constexpr (TWO) second_of(g[e], u[e], dy[e], cg[e], cu[e], rg[e], ru[e], o[e]);
    }
    if constexpr (EP == EP_FWD) put4_anywhere(y + at, o, some);
    if constexpr (EP == EP_BWD2) put4(y + at, o, some, whole);
    const auto both = [&](void* first, void* rest, const float (&vg)[4], const float (&vu)[4]) {
        if (!first) return;
        T* const p = reinterpret_cast<T*>(first) + two;
        put4(p, vg, some, whole);
        put4(p + a.ni, vu, some, whole);
        if (rest) put_rest(reinterpret_cast<T*>(rest) + two, vg, vu, a.ni, some, whole);
    };
    if constexpr (EP != EP_FWD) both(a.dgu, a.dgu2, og, ou);
    if constexpr (TWO) both(a.ggu, a.ggu2, rg, ru);
}

// fp64, for gradient checks: 64 x 64 of D (gated: of each half, and of both right operands) a workgroup, 4 x 4 a thread.
template <int ALIES, int BLIES, int EP> __global__ __launch_bounds__(256) void k_product64(Args a) {
    constexpr int NA = EP >= EP_FWD ? 2 : 1, NB = EP == EP_BWD2 ? 2 : 1;
    __shared__ double la[NA][16][65], lb[NB][16][65];
    const int ti = blockIdx.x % a.ti, tj = blockIdx.x / a.ti;
    const int64_t i0 = (int64_t)ti * 64, j0 = (int64_t)tj * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    double acc[NB][NA][4][4] = {};
    for (int pair = 0; pair < a.pairs; ++pair) {
        const double* pa = reinterpret_cast<const double*>(a.a[pair]);
        const double* pb[2] = {reinterpret_cast<const double*>(a.b[pair]), reinterpret_cast<const double*>(a.c)};
        for (int64_t k0 = 0; k0 < a.nk; k0 += 16) {
            __syncthreads();
            for (int p = threadIdx.x; p < 1024; p += 256) {
                const int r = p & 63, k = p >> 6;
                const bool in = k0 + k < a.nk;
                for (int h = 0; h < NA; ++h) {
                    const int64_t row = i0 + r + h * a.ni;
                    la[h][k][r] = in && i0 + r < a.ni ? pa[ALIES == K_ROWS ? row * a.lda + k0 + k : (k0 + k) * a.lda + row] : 0.0;
                }
                const int64_t row = j0 + r;
                for (int h = 0; h < NB; ++h)
                    lb[h][k][r] = in && row < a.nj ? pb[h][BLIES == K_ROWS ? row * a.ldb + k0 + k : (k0 + k) * a.ldb + row] : 0.0;
            }
            __syncthreads();
            for (int k = 0; k < 16; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        for (int f = 0; f < NB; ++f)
                            for (int h = 0; h < NA; ++h) acc[f][h][i][j] += la[h][k][tx + 16 * i] * lb[f][k][ty + 16 * j];
        }
    }
    double *const out = reinterpret_cast<double*>(a.out), *const dgu = reinterpret_cast<double*>(a.dgu);
    double* const ggu = reinterpret_cast<double*>(a.ggu);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t row = j0 + ty + 16 * j, col = i0 + tx + 16 * i;
            if (row >= a.nj || col >= a.ni) continue;
            const int64_t at = row * a.ni + col, two = row * 2 * a.ni + col;
            const double g = acc[0][0][i][j], u = acc[0][NA - 1][i][j];
            if constexpr (EP < EP_FWD) out[row * a.ldo + col] = g;
            if constexpr (EP == EP_FWD) out[at] = gated(g, u);
            if constexpr (EP > EP_FWD) {
                const double dy = reinterpret_cast<const double*>(a.dy)[at];
                double og, ou, o;
                if (a.dgu) first_of(g, u, dy, dgu[two], dgu[two + a.ni]);
                if constexpr (EP == EP_BWD2) {
                    second_of(g, u, dy, acc[NB - 1][0][i][j], acc[NB - 1][1][i][j], og, ou, o);
                    out[at] = o;
                    if (a.ggu) {
                        ggu[two] = og;
                        ggu[two + a.ni] = ou;
                    }
                }
            }
        }
}

// The splits' partial sums of the tiles from tile0 on added up, in their order.
template <typename T> __global__ __launch_bounds__(256) void k_join(Args a, int tile, const float* part, T* out) {
    const int per = tile * tile / 1024;  // workgroups of a tile
    int ti, tj;
    place_of(a, a.tile0 + blockIdx.x / per, ti, tj);
    const int at = (blockIdx.x % per * 256 + threadIdx.x) * 4;
    const int64_t row = (int64_t)tj * tile + at / tile, col = (int64_t)ti * tile + at % tile;
    if (row >= a.nj || col >= a.ni) return;
    float s[4] = {0, 0, 0, 0}, v[4];
    const float* p = part + (int64_t)(blockIdx.x / per) * tile * tile + at;
    for (int k = 0; k < a.splits; ++k, p += (int64_t)a.count * tile * tile) {
        get4(p, v, 4, true);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += v[e];
    }
    put4(out + row * a.ldo + col, s, a.ni - col, true);
}

// -- launches ----------------------------------------------------------------------------------------------------------

template <typename T, int ALIES, int BLIES, int EP> static void launch(hipStream_t s, const Cut& c, const Args& a) {
    const dim3 grid((unsigned)(a.count * a.splits));
    // (fp64 is not split; of few tiles alone dx is: of 64)
    constexpr bool SMALL = EP == EP_PART && ALIES == M_ROWS && BLIES == K_ROWS;
    if constexpr (std::is_same_v<T, double>) {
        if constexpr (EP != EP_PART) hipLaunchKernelGGL((k_product64<ALIES, BLIES, EP>), grid, dim3(256), 0, s, a);
    } else {
        if constexpr (sizeof(T) == 2 && !SMALL) {
            if (c.tile == 256) {
                constexpr int WJ = EP >= EP_FWD ? 4 : 2;
                hipLaunchKernelGGL((k_product<T, ALIES, BLIES, EP, 256, 256, 2, WJ>), grid, dim3(128 * WJ), 0, s, a);
                return;
            }
        }
        if constexpr (!SMALL) {
            if (c.tile == 128) {
                hipLaunchKernelGGL((k_product<T, ALIES, BLIES, EP, 128, 128, 2, 2>), grid, dim3(256), 0, s, a);
                return;
            }
        }
        if constexpr (EP == EP_BWD2) hipLaunchKernelGGL((k_product<T, ALIES, BLIES, EP, 64, 64, 1, 1>), grid, dim3(64), 0, s, a);
        else hipLaunchKernelGGL((k_product<T, ALIES, BLIES, EP, 64, 64, 1, 2>), grid, dim3(128), 0, s, a);
    }
}

// One product, whose operands, strides, sizes and outputs ``a`` holds.
template <int ALIES, int BLIES, int EP> static void product(int dtype, const Cut& c, Args& a, hipStream_t s) {
    constexpr bool PART = EP == EP_PART;  // its tiles that are split, else those that are not
    a.ti = (int)c.ti, a.tj = (int)c.tj, a.tile0 = PART ? (int)c.whole : 0, a.count = (int)(PART ? c.tiles() - c.whole : c.whole);
    a.splits = PART ? c.splits : 1;
    a.steps = PART ? c.steps : INT64_MAX / 4;
    const auto with = [&](auto v) {
        using T = decltype(v);
        launch<T, ALIES, BLIES, EP>(s, c, a);
    };
    switch (dtype) {
        case EBR_DTYPE_F32: with(float()); break;
        case EBR_DTYPE_BF16: with(__bf16()); break;
        case EBR_DTYPE_F16: with(_Float16()); break;
        default: with(double()); break;
    }
}

// [dg|du] or [gg|gu], rounded, and what they lack where the products take that as well (with_rest).
struct Grads {
    const void *g, *rest;
};

static void join(int dtype, const Cut& c, const Args& a, const float* part, void* out, hipStream_t s) {
    const dim3 grid((unsigned)(a.count * (c.tile * c.tile / 1024)));
    if (dtype == EBR_DTYPE_BF16) hipLaunchKernelGGL((k_join<__bf16>), grid, dim3(256), 0, s, a, c.tile, part, (__bf16*)out);
    else if (dtype == EBR_DTYPE_F16) hipLaunchKernelGGL((k_join<_Float16>), grid, dim3(256), 0, s, a, c.tile, part, (_Float16*)out);
    else hipLaunchKernelGGL((k_join<float>), grid, dim3(256), 0, s, a, c.tile, part, (float*)out);
}

// dx of dgu, and dw of (x, dgu) and, where there is one, a second pair.
static void input_grad(int dtype, int64_t N, int64_t C, int64_t I, const void* w, Grads dgu, void* dx, float* part, hipStream_t s) {
    Args a = {};
    a.a[0] = a.a[1] = w, a.b[0] = dgu.g, a.b[1] = dgu.rest, a.pairs = dgu.rest ? 2 : 1;
    a.lda = C, a.ldb = 2 * I, a.ni = C, a.nj = N, a.nk = 2 * I, a.out = dx, a.ldo = C;
    const Cut c = input_cut(dtype, N, C, I, a.pairs);
    if (c.splits == 1) {
        product<M_ROWS, K_ROWS, EP_OUT>(dtype, c, a, s);
        return;
    }
    a.out = part;
    product<M_ROWS, K_ROWS, EP_PART>(dtype, c, a, s);
    join(dtype, c, a, part, dx, s);
}

static void weight_grad(int dtype, int64_t N, int64_t C, int64_t I, const void* x, Grads dgu, const void* x2, Grads dgu2, void* dw,
                        float* part, hipStream_t s) {
    Args a = {};
    for (const auto& [of, grads] : {std::pair<const void*, Grads>(x, dgu), std::pair<const void*, Grads>(x2, dgu2)})
        for (const void* g : {grads.g, grads.rest})
            if (g) a.a[a.pairs] = of, a.b[a.pairs++] = g;
    const Cut c = weight_cut(dtype, N, C, I, a.pairs);
    a.lda = C, a.ldb = 2 * I, a.ni = C, a.nj = 2 * I, a.nk = N, a.out = dw, a.ldo = C;
    if (c.whole) product<M_ROWS, M_ROWS, EP_OUT>(dtype, c, a, s);
    if (c.splits == 1) return;
    a.out = part;
    product<M_ROWS, M_ROWS, EP_PART>(dtype, c, a, s);
    join(dtype, c, a, part, dw, s);
}

// The products of gate and up: of few rows, or of many.
template <int EP> static void gates(int dtype, Args& a, hipStream_t s) {
    if (!is_few(dtype, a.nj, a.nk)) {
        product<K_ROWS, K_ROWS, EP>(dtype, gates_cut(dtype, EP - EP_FWD, a.nj, a.nk, a.ni), a, s);
        return;
    }
    const auto with = [&](auto v) {
        using T = decltype(v);
        const dim3 grid((unsigned)((a.ni + 15) / 16)), threads(64 * FEW_WAVES);
        if (a.nj <= 16) hipLaunchKernelGGL((k_few<T, EP, 1>), grid, threads, 0, s, a);
        else hipLaunchKernelGGL((k_few<T, EP, 2>), grid, threads, 0, s, a);
    };
    if (dtype == EBR_DTYPE_F32) with(float());
    else if (dtype == EBR_DTYPE_BF16) with(__bf16());
    else with(_Float16());
}

static int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

// Widths that are no whole 16-byte chunks: the products run on copies with zeros up to the next chunk, which add nothing, and
// their outputs are copied back. (Reading such rows element by element took ten times as long: 8192 x 2048 -> 5631 bf16 with its
// gradients 15.8 ms, 1.7 so, 1.3 with 5632.)
struct Move {
    const void* from;
    void* to;
    int64_t rows, have_rows, ldf, ldt;
    int cols, have;  // written, and there to be read: zeros beyond
};
struct Moves {
    Move m[5];
    int first[6], count;
};
template <typename T> __global__ __launch_bounds__(256) void k_move(Moves a) {
    constexpr int VEC = 16 / (int)sizeof(T);
    int j = 0;
    while (j + 1 < a.count && (int)blockIdx.x >= a.first[j + 1]) ++j;
    const Move m = a.m[j];
    const int64_t skip = (int64_t)(a.first[j + 1] - a.first[j]) * 4;
    for (int64_t row = (int64_t)(blockIdx.x - a.first[j]) * 4 + threadIdx.x / 64; row < m.rows; row += skip) {
        const T* from = reinterpret_cast<const T*>(m.from) + row * m.ldf;
        T* to = reinterpret_cast<T*>(m.to) + row * m.ldt;
        for (int c = threadIdx.x % 64 * VEC; c < m.cols; c += 64 * VEC) {
            T v[VEC] = {};
            if (row < m.have_rows) {
                if (c + VEC <= m.have) __builtin_memcpy(v, from + c, 16);
                else
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        if (c + e < m.have) v[e] = from[c + e];
            }
            if (c + VEC <= m.cols) __builtin_memcpy(to + c, v, 16);
            else
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (c + e < m.cols) to[c + e] = v[e];
        }
    }
}

struct Padded {
    int dtype;
    int64_t N, C, I, Cp, Ip;
    char* at = nullptr;
    Moves in = {}, out = {};
    Padded(int dtype, int64_t N, int64_t C, int64_t I) : dtype(dtype), N(N), C(C), I(I) {
        Cp = padded(dtype, C), Ip = padded(dtype, I);
    }
    bool needed() const { return Cp != C || Ip != I; }
    int64_t bytes(int64_t rows, int64_t cols) const { return up16(rows * cols * size_of(dtype)); }
    // of x, w and y; of x, w, dy, dx and dw; of x, w, dy, c, gx, gdy and gw
    int64_t all(int order) const {
        if (!needed()) return 0;
        return (order == 0 ? 1 : order + 1) * bytes(N, Cp) + (order < 2 ? 1 : 2) * bytes(N, Ip) + (order == 0 ? 1 : 2) * bytes(2 * Ip, Cp);
    }
    void add(Moves& to, const Move& m) {
        to.m[to.count] = m;
        const int64_t want = (m.rows + 3) / 4;
        to.first[to.count + 1] = to.first[to.count] + (int)(want < 4096 ? want : 4096);
        ++to.count;
    }
    char* take(int64_t rows, int64_t cols) {
        char* p = at;
        at += bytes(rows, cols);
        return p;
    }
    const void* rows(const void* p, int64_t have, int64_t cols) {
        char* to = take(N, cols);
        add(in, {p, to, N, N, have, cols, (int)cols, (int)have});
        return to;
    }
    const void* weight(const void* w) {
        char* to = take(2 * Ip, Cp);
        for (int h = 0; h < 2; ++h)
            add(in, {(const char*)w + h * I * C * size_of(dtype), to + h * Ip * Cp * size_of(dtype), Ip, I, C, Cp, (int)Cp, (int)C});
        return to;
    }
    void* rows_out(void* p, int64_t have, int64_t cols) {
        if (!p) return nullptr;
        char* from = take(N, cols);
        add(out, {from, p, N, N, cols, have, (int)have, (int)have});
        return from;
    }
    void* weight_out(void* w) {
        if (!w) return nullptr;
        char* from = take(2 * Ip, Cp);
        for (int h = 0; h < 2; ++h)
            add(out, {from + h * Ip * Cp * size_of(dtype), (char*)w + h * I * C * size_of(dtype), I, I, Cp, C, (int)C, (int)C});
        return from;
    }
    void run(const Moves& m, hipStream_t s) const {
        const dim3 grid((unsigned)m.first[m.count]);
        if (m.count == 0) return;
        if (size_of(dtype) == 2) hipLaunchKernelGGL((k_move<uint16_t>), grid, dim3(256), 0, s, m);
        else hipLaunchKernelGGL((k_move<uint32_t>), grid, dim3(256), 0, s, m);
    }
};

static bool all_aligned(std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if (!aligned(p, 16)) return false;
    return true;
}

static void forward(int dtype, int64_t N, int64_t C, int64_t I, const void* x, const void* w, void* y, hipStream_t s) {
    Args a = {};
    a.a[0] = w, a.b[0] = x, a.lda = a.ldb = C, a.ni = I, a.nj = N, a.nk = C, a.pairs = 1, a.out = y;
    gates<EP_FWD>(dtype, a, s);
}
// Whether it takes rows of any width and alignment as they are.
static bool as_they_are(int dtype, int64_t N, int64_t C) { return dtype == EBR_DTYPE_F64 || is_few(dtype, N, C); }

static int64_t own_scratch(int dtype, int order, int64_t N, int64_t C, int64_t I) {
    if (order == 0) return 0;
    const int64_t each = with_rest(dtype, N) ? 2 : 1;
    // [dg|du], for order 2 [gg|gu] too, and a gradient's partial sums
    const int64_t part = std::max(weight_cut(dtype, N, C, I, (int)(order * each)).part_bytes(), input_cut(dtype, N, C, I, (int)each).part_bytes());
    return order * each * up16(N * 2 * I * size_of(dtype)) + part + 16;
}

static void backward(int dtype, int64_t N, int64_t C, int64_t I, const void* x, const void* w, const void* dy, void* dx, void* dw,
                     char* at, hipStream_t s) {
    Args a = {};
    a.a[0] = w, a.b[0] = x, a.lda = a.ldb = C, a.ni = I, a.nj = N, a.nk = C, a.pairs = 1, a.dy = dy;
    const int64_t rows = up16(N * 2 * I * size_of(dtype));
    a.dgu = at, at += rows;
    if (with_rest(dtype, N)) a.dgu2 = at, at += rows;
    gates<EP_BWD>(dtype, a, s);
    const Grads dgu = {a.dgu, a.dgu2};
    if (dx) input_grad(dtype, N, C, I, w, dgu, dx, reinterpret_cast<float*>(at), s);
    if (dw) weight_grad(dtype, N, C, I, x, dgu, nullptr, {}, dw, reinterpret_cast<float*>(at), s);
}

static void backward2(int dtype, int64_t N, int64_t C, int64_t I, const void* x, const void* w, const void* dy, const void* c,
                      void* gx, void* gdy, void* gw, char* at, hipStream_t s) {
    Args a = {};
    a.a[0] = w, a.b[0] = x, a.c = c, a.lda = a.ldb = C, a.ni = I, a.nj = N, a.nk = C, a.pairs = 1, a.out = gdy, a.dy = dy;
    const int64_t rows = up16(N * 2 * I * size_of(dtype));
    for (void** to : {gx || gw ? &a.ggu : nullptr, gw ? &a.dgu : nullptr}) {
        if (to) *to = at, at += rows;
        if (to && with_rest(dtype, N)) *(to == &a.ggu ? &a.ggu2 : &a.dgu2) = at, at += rows;
    }
    gates<EP_BWD2>(dtype, a, s);
    const Grads dgu = {a.dgu, a.dgu2}, ggu = {a.ggu, a.ggu2};
    if (gx) input_grad(dtype, N, C, I, w, ggu, gx, reinterpret_cast<float*>(at), s);
    if (gw) weight_grad(dtype, N, C, I, x, ggu, c, dgu, gw, reinterpret_cast<float*>(at), s);
}

}  // namespace ebr_glu

using namespace ebr_glu;

extern "C" {

int64_t ebr_block_swiglu_linear_scratch(int dtype, int order, int64_t N, int64_t C, int64_t I) {
    if (order < 0 || order > 2 || check(dtype, order, N, C, I)) return -1;
    if (order == 0 && as_they_are(dtype, N, C)) return 0;
    const Padded p(dtype, N, C, I);
    return own_scratch(dtype, order, N, p.Cp, p.Ip) + p.all(order);
}

int ebr_block_swiglu_linear(int dtype, int64_t N, int64_t C, int64_t I, const void* x, const void* w, void* y, void* scratch,
                            void* stream) {
    const int rc = check(dtype, 0, N, C, I);
    if (rc) return rc;
    if (!x || !w || !y) return EBR_ERR_NULL;
    hipStream_t s = (hipStream_t)stream;
    Padded p(dtype, N, C, I);
    if (as_they_are(dtype, N, C)) {
        forward(dtype, N, C, I, x, w, y, s);
    } else if (p.needed()) {
        if (!scratch) return EBR_ERR_SCRATCH;
        if (!aligned(scratch, 16)) return EBR_ERR_ALIGN;
        p.at = reinterpret_cast<char*>(scratch);
        x = p.rows(x, C, p.Cp), w = p.weight(w), y = p.rows_out(y, I, p.Ip);
        p.run(p.in, s);
        forward(dtype, N, p.Cp, p.Ip, x, w, y, s);
        p.run(p.out, s);
    } else {
        if (!all_aligned({x, w, y})) return EBR_ERR_ALIGN;
        forward(dtype, N, C, I, x, w, y, s);
    }
    return launched();
}

int ebr_block_swiglu_linear_bwd(int dtype, int64_t N, int64_t C, int64_t I, const void* x, const void* w, const void* dy,
                                void* dx, void* dw, void* scratch, void* stream) {
    const int rc = check(dtype, 1, N, C, I);
    if (rc) return rc;
    if (!x || !w || !dy) return EBR_ERR_NULL;
    if (!scratch) return EBR_ERR_SCRATCH;
    Padded p(dtype, N, C, I);
    if (!aligned(scratch, 16) || (!p.needed() && dtype != EBR_DTYPE_F64 && !all_aligned({x, w, dy, dx, dw}))) return EBR_ERR_ALIGN;
    if (!dx && !dw) return EBR_OK;
    hipStream_t s = (hipStream_t)stream;
    char* const own = reinterpret_cast<char*>(scratch) + p.all(1);
    if (p.needed()) {
        p.at = reinterpret_cast<char*>(scratch);
        x = p.rows(x, C, p.Cp), w = p.weight(w), dy = p.rows(dy, I, p.Ip);
        dx = p.rows_out(dx, C, p.Cp), dw = p.weight_out(dw);
    }
    p.run(p.in, s);
    backward(dtype, N, p.Cp, p.Ip, x, w, dy, dx, dw, own, s);
    p.run(p.out, s);
    return launched();
}

int ebr_block_swiglu_linear_bwd2(int dtype, int64_t N, int64_t C, int64_t I, const void* x, const void* w, const void* dy,
                                 const void* c, void* gx, void* gdy, void* gw, void* scratch, void* stream) {
    const int rc = check(dtype, 2, N, C, I);
    if (rc) return rc;
    if (!x || !w || !dy || !c || !gdy) return EBR_ERR_NULL;
    if (!scratch) return EBR_ERR_SCRATCH;
    Padded p(dtype, N, C, I);
    if (!aligned(scratch, 16) || (!p.needed() && dtype != EBR_DTYPE_F64 && !all_aligned({x, w, dy, c, gx, gdy, gw})))
        return EBR_ERR_ALIGN;
    hipStream_t s = (hipStream_t)stream;
    char* const own = reinterpret_cast<char*>(scratch) + p.all(2);
    if (p.needed()) {
        p.at = reinterpret_cast<char*>(scratch);
        x = p.rows(x, C, p.Cp), w = p.weight(w), dy = p.rows(dy, I, p.Ip), c = p.rows(c, C, p.Cp);
        gx = p.rows_out(gx, C, p.Cp), gdy = p.rows_out(gdy, I, p.Ip), gw = p.weight_out(gw);
    }
    p.run(p.in, s);
    backward2(dtype, N, p.Cp, p.Ip, x, w, dy, c, gx, gdy, gw, own, s);
    p.run(p.out, s);
    return launched();
}

}  // extern "C"
