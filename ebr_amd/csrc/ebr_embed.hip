// Embedding of tokens and its table's gradient on gfx950 (C ABI: include/ebr_block.h).
//
//   y[n, :]  = round(s w[id_n, :]), a row of zeros where id_n lies outside [0, V)
//   dw[v, :] = round(s sum over { n : id_n = v } of dy[n, :]), every row of the table written
//
// Both are bound by memory. The lookup reads the tokens' rows and writes y. The gradient has to read dy once and to write
// the whole table, most of it zeros for text; what costs is bringing a token's rows together. Atomic sums would do that in
// an order that changes from run to run, so the positions are sorted by token instead (a stable radix sort: equal tokens
// keep their order; few tokens, and small tables, need no sort), and a sum always adds the same rows in the same order, in 32
// bits.
#include <initializer_list>
#include <type_traits>

#include "rowwise.hpp"

namespace ebr_embed {

using namespace ebr_row;

struct Ids {
    const void* p;
    int wide;  // 64-bit tokens
    int V;
};

// A position's token, V for one outside the table.
__device__ __forceinline__ uint32_t token(const Ids& ids, int64_t n) {
    if (ids.wide) {
        const int64_t v = reinterpret_cast<const int64_t*>(ids.p)[n];
        return v >= 0 && v < ids.V ? (uint32_t)v : (uint32_t)ids.V;
    }
    const int v = reinterpret_cast<const int*>(ids.p)[n];
    return v >= 0 && v < ids.V ? (uint32_t)v : (uint32_t)ids.V;
}

// -- lookup ------------------------------------------------------------------------------------------------------------

// A row's threads, at most a wave of them, go over its columns VEC at a time (16 bytes of y), some rows side by side: a row's
// load waits for its token's, and the next rows' fill that time. 31,104 rows of 512 bf16 from an fp32 table of 11 take 9.5 us
// (3.3 TB/s of writes; the chain token, row, store is half of it), 32,768 rows of 2,048 from one of 100,003 67 us in a row of
// calls (4 TB/s). With 8 bytes of y a thread 10.2 and 71 us; with four rows of an fp32 table side by side 9.8 and 74, with two
// of a 16-bit one 11.4 and 51.8 where four take 10.3 and 52.5.
template <typename TW> constexpr int rows_of() { return sizeof(TW) == 2 ? 4 : 2; }
template <typename TW, typename TY, int VEC>
__global__ __launch_bounds__(256) void k_lookup(Ids ids, int64_t N, int C, int team, double scale, const TW* w, TY* y) {
    using A = typename Acc<TW>::type;
    constexpr int ROWS = rows_of<TW>();
    constexpr int PIECE = VEC * (int)sizeof(TW) > 16 ? 16 / (int)sizeof(TW) : VEC, PIECES = VEC / PIECE;
    using Raw = typename Words<PIECE * (int)sizeof(TW)>::type;
    const int t = threadIdx.x & (team - 1), per = 256 / team;
    for (int64_t n0 = (int64_t)blockIdx.x * per * ROWS + threadIdx.x / team; n0 < N; n0 += (int64_t)gridDim.x * per * ROWS) {
        uint32_t v[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) v[r] = n0 + r * per < N ? token(ids, n0 + r * per) : (uint32_t)ids.V;
        for (int c = t * VEC; c < C; c += team * VEC) {
            Raw x[ROWS][PIECES];  // (of row 0 where there is none)
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
#pragma unroll
                for (int i = 0; i < PIECES; ++i)
                    x[r][i] =
                        *reinterpret_cast<const Raw*>(w + (int64_t)(v[r] < (uint32_t)ids.V ? v[r] : 0) * C + c + i * PIECE);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                if (n0 + r * per >= N) break;
                Pack<TY, VEC> o;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    const Pack<TW, PIECE> p = unpacked<TW, PIECE>(x[r][i]);
#pragma unroll
                    for (int e = 0; e < PIECE; ++e)
                        o.e[i * PIECE + e] = v[r] < (uint32_t)ids.V ? (TY)((A)p.e[e] * (A)scale) : (TY)0.f;
                }
                stp<TY, VEC>(y + (n0 + r * per) * C + c, o);
            }
        }
    }
}

// -- positions sorted by token -----------------------------------------------------------------------------------------

// A workgroup ranks a tile of 1,024 positions a round, as many rounds as leave at most 128 workgroups (each reads all the
// others' counts); up to 4,096 positions are one workgroup's. 16,384 positions take 5.4 us a pass (and 3 the counts before it);
// in tiles of 4,096, which leave most of the card idle, 9.9. Latency bounds it: launches, and what one kernel wrote and the
// next reads on other XCDs. Nine bits a pass: one up to a vocabulary of 511, two up to 262,143.
constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64, SORT_ONE = 4096;
constexpr int SORT_BITS = 9, SORT_DIGITS = 1 << SORT_BITS;
constexpr int SORT_GROUPS = 128;

struct SortArgs {
    Ids ids;                     // read where kin is null
    const uint32_t *kin, *pin;   // tokens and positions
    uint32_t *kout, *pout;
    uint32_t* counts;            // [groups][SORT_DIGITS]
    int N, shift, bits, tiles;   // tiles: of each workgroup
};

// The lanes of this wave that hold the same digit.
__device__ __forceinline__ uint64_t alike(uint32_t digit, int bits, bool valid) {
    uint64_t m = __ballot(valid);
    for (int b = 0; b < bits; ++b) {
        const bool on = (digit >> b) & 1;
        const uint64_t s = __ballot(on);
        m &= on ? s : ~s;
    }
    return m;
}

__global__ __launch_bounds__(SORT_THREADS) void k_sort_count(SortArgs a) {
    __shared__ uint32_t count[SORT_DIGITS];
    for (int d = threadIdx.x; d < SORT_DIGITS; d += SORT_THREADS) count[d] = 0;
    __syncthreads();
    const int64_t from = (int64_t)blockIdx.x * a.tiles * SORT_THREADS;
    const int64_t to = from + (int64_t)a.tiles * SORT_THREADS < a.N ? from + (int64_t)a.tiles * SORT_THREADS : a.N;
    for (int64_t i = from + threadIdx.x; i < to; i += SORT_THREADS) {
        const uint32_t k = a.kin ? a.kin[i] : token(a.ids, i);
        atomicAdd(&count[(k >> a.shift) & ((1u << a.bits) - 1)], 1u);  // whole numbers: the order does not matter
    }
    __syncthreads();
    for (int d = threadIdx.x; d < SORT_DIGITS; d += SORT_THREADS) a.counts[(int64_t)blockIdx.x * SORT_DIGITS + d] = count[d];
}

// Exclusive prefix sums of v over SORT_DIGITS threads (the first ones of the workgroup), by wave and then over the waves.
__device__ __forceinline__ uint32_t digits_before(uint32_t v, uint32_t* waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t s = v;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const uint32_t o = __shfl_up(s, m, 64);
        if (lane >= m) s += o;
    }
    if (lane == 63) waves[wave] = s;
    __syncthreads();
    uint32_t base = 0;
    for (int w = 0; w < wave && w < SORT_DIGITS / 64; ++w) base += waves[w];
    return base + s - v;
}

// Ranks of a tile's keys among those with the same digit that come before them: count[wave][digit] ends as the number in
// the waves before, rank[k] as the number before in the wave. Positions run by wave, then by k, then by lane.
template <int KEYS>
__device__ __forceinline__ void rank_tile(const uint32_t (&key)[KEYS], const bool (&valid)[KEYS], int shift, int bits,
                                          uint32_t (*count)[SORT_DIGITS], uint32_t (&rank)[KEYS]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = lane; d < 1 << bits; d += 64) count[wave][d] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KEYS; ++k) {
        const uint32_t digit = (key[k] >> shift) & ((1u << bits) - 1);
        const uint64_t same = alike(digit, bits, valid[k]);
        const int first = same ? __ffsll((unsigned long long)same) - 1 : 0;
        uint32_t old = 0;
        if (valid[k] && lane == first) old = atomicAdd(&count[wave][digit], (uint32_t)__popcll(same));
        rank[k] = __shfl(old, first, 64) + (uint32_t)__popcll(same & ((1ull << lane) - 1));
    }
    __syncthreads();
}

__global__ __launch_bounds__(SORT_THREADS) void k_sort_place(SortArgs a) {
    __shared__ uint32_t count[SORT_WAVES][SORT_DIGITS];
    __shared__ uint32_t start[SORT_DIGITS], waves[SORT_WAVES];
    const int t = threadIdx.x, wave = t >> 6, digits = 1 << a.bits;
    const int64_t from = (int64_t)blockIdx.x * a.tiles * SORT_THREADS + t;
    const auto key_at = [&](int64_t i) { return i < a.N ? (a.kin ? a.kin[i] : token(a.ids, i)) : 0; };
    const auto pos_at = [&](int64_t i) { return i < a.N ? (a.kin ? a.pin[i] : (uint32_t)i) : 0; };
    uint32_t next_key = key_at(from), next_pos = pos_at(from);  // on their way while the counts come
    uint32_t before = 0, total = 0;
    if (t < digits) {
#pragma unroll 16
        for (int g = 0; g < (int)gridDim.x; ++g) {
            const uint32_t c = a.counts[(int64_t)g * SORT_DIGITS + t];
            total += c;
            if (g < (int)blockIdx.x) before += c;
        }
    }
    const uint32_t base = digits_before(total, waves);
    if (t < digits) start[t] = base + before;
    for (int tile = 0; tile < a.tiles; ++tile) {
        const int64_t i = from + (int64_t)tile * SORT_THREADS;
        const bool valid[1] = {i < a.N};
        const uint32_t key[1] = {next_key}, pos = next_pos;
        if (tile + 1 < a.tiles) {
            next_key = key_at(i + SORT_THREADS);
            next_pos = pos_at(i + SORT_THREADS);
        }
        uint32_t rank[1];
        rank_tile<1>(key, valid, a.shift, a.bits, count, rank);
        if (t < digits) {
            uint32_t sum = start[t];
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) {
                const uint32_t c = count[w][t];
                count[w][t] = sum;
                sum += c;
            }
            start[t] = sum;
        }
        __syncthreads();
        if (valid[0]) {
            const uint32_t to = count[wave][(key[0] >> a.shift) & (digits - 1)] + rank[0];
            a.kout[to] = key[0];
            a.pout[to] = pos;
        }
        __syncthreads();
    }
}

// Up to 4,096 positions: every pass in one workgroup, the keys going round through shared memory.
__global__ __launch_bounds__(SORT_THREADS) void k_sort_tile(SortArgs a, int passes) {
    __shared__ uint32_t count[SORT_WAVES][SORT_DIGITS];
    __shared__ uint32_t keys[SORT_ONE], waves[SORT_WAVES];
    __shared__ uint16_t places[SORT_ONE];
    constexpr int KEYS = SORT_ONE / SORT_THREADS;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, at = wave * (KEYS * 64) + lane;
    uint32_t key[KEYS], pos[KEYS], rank[KEYS];
    bool valid[KEYS];
#pragma unroll
    for (int k = 0; k < KEYS; ++k) {
        valid[k] = at + k * 64 < a.N;
        key[k] = valid[k] ? token(a.ids, at + k * 64) : 0;
        pos[k] = at + k * 64;
    }
    for (int p = 0; p < passes; ++p) {
        const int shift = p * a.bits;
        rank_tile<KEYS>(key, valid, shift, a.bits, count, rank);
        uint32_t sum = 0;
        if (t < 1 << a.bits)
            for (int w = 0; w < SORT_WAVES; ++w) {
                const uint32_t c = count[w][t];
                count[w][t] = sum;
                sum += c;
            }
        const uint32_t base = digits_before(sum, waves);
        if (t < 1 << a.bits)
            for (int w = 0; w < SORT_WAVES; ++w) count[w][t] += base;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < KEYS; ++k) {
            if (!valid[k]) continue;
            const uint32_t to = count[wave][(key[k] >> shift) & ((1u << a.bits) - 1)] + rank[k];
            keys[to] = key[k];
            places[to] = (uint16_t)pos[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < KEYS; ++k) {
            if (!valid[k]) continue;
            key[k] = keys[at + k * 64];
            pos[k] = places[at + k * 64];
        }
    }
#pragma unroll
    for (int k = 0; k < KEYS; ++k) {
        if (!valid[k]) continue;
        a.kout[at + k * 64] = key[k];
        a.pout[at + k * 64] = pos[k];
    }
}

// -- sums of equal tokens' rows ----------------------------------------------------------------------------------------

struct SumArgs {
    const uint32_t *key, *pos;  // sorted
    const void* dy;
    void* dw;
    void* part;  // [chunks][2][C]: a chunk's share of a run from the chunk before (0), and of one that goes on (1)
    int N, V, C, chunk, chunks, team, zero_rows;
    unsigned sum_blocks;
    double scale;
};

template <typename A, typename TW, int VEC>
__device__ __forceinline__ void put_row(TW* p, const A (&acc)[VEC], double scale) {
    TW o[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = (TW)(acc[e] * (A)scale);
    store_wide<TW, VEC>(p, o);
}

// The first of n sorted keys that is v or more, found by a wave: 64 probes a step, three steps for a quarter of a million.
__device__ __forceinline__ int first_from(const uint32_t* key, int n, uint32_t v) {
    const int lane = threadIdx.x & 63;
    int lo = 0, len = n;
    while (len > 0) {
        const int step = (len - 1) / 64 + 1;
        const int64_t at = (int64_t)lane * step;
        const int below = __popcll(__ballot(at < len && key[lo + (at < len ? at : 0)] < v));
        if (below == 0) break;
        const int64_t end = (int64_t)below * step < len ? (int64_t)below * step : len;
        lo += (below - 1) * step + 1;
        len = (int)(end - ((int64_t)(below - 1) * step + 1));
    }
    return lo;
}

constexpr int AHEAD = 8;  // rows whose loads are under way together (of 16 the sums take twice as long)

// The first workgroups sum: a team of lanes, as many as there are columns for and a wave at most, takes a chunk of the
// sorted positions and VEC columns a lane. A run of equal tokens inside the chunk is written to the table at once; a run
// over its border goes to part. The other workgroups write zeros to the rows of tokens that do not occur, found by
// search: these are most of the table for text, and their stores fill the time that the sums wait for their rows. They go
// past the caches, in whole lines: 16,384 tokens of 50,021 x 1,024 bf16 take 61 us with their gradient, through the caches 81
// (32 bytes a lane, which halves lines, cost the fp32 table of 100,003 x 2,048 150 us).
// Bound by memory: 21 us for those tokens (132 MB, 6.3 TB/s), 186 us for 32,768 tokens of that table (953 MB, 5.1 TB/s).
template <typename TW, typename TY, int VEC> __global__ __launch_bounds__(256) void k_sum(SumArgs a) {
    using A = typename Acc<TW>::type;
    using Raw = typename Words<VEC * (int)sizeof(TY)>::type;
    TW* dw = reinterpret_cast<TW*>(a.dw);
    if (blockIdx.x >= a.sum_blocks) {
        __shared__ uint8_t absent[256];
        __shared__ int ends[2];
        const int64_t r0 = (int64_t)(blockIdx.x - a.sum_blocks) * a.zero_rows;
        const int rows = (int)(a.V - r0 < a.zero_rows ? a.V - r0 : a.zero_rows), wave = threadIdx.x >> 6;
        if (wave < 2) {
            const int at = first_from(a.key, a.N, (uint32_t)(r0 + wave * rows));
            if ((threadIdx.x & 63) == 0) ends[wave] = at;
        }
        __syncthreads();
        if ((int)threadIdx.x < rows) {
            const uint32_t v = (uint32_t)(r0 + threadIdx.x);
            int lo = ends[0], hi = ends[1];
            while (lo < hi) {
                const int mid = lo + (hi - lo) / 2;
                if (a.key[mid] < v) lo = mid + 1;
                else hi = mid;
            }
            absent[threadIdx.x] = !(lo < ends[1] && a.key[lo] == v);
        }
        __syncthreads();
        constexpr int ZV = VEC < 16 / (int)sizeof(TW) ? VEC : 16 / (int)sizeof(TW);  // a wave's store covers whole lines
        const TW zero[ZV] = {};
        const int per = 256 / a.team, t = threadIdx.x & (a.team - 1);
        for (int r = threadIdx.x / a.team; r < rows; r += per) {
            if (!absent[r]) continue;
            for (int c = t * ZV; c < a.C; c += a.team * ZV) store_past<TW, ZV>(dw + (r0 + r) * a.C + c, zero);
        }
        return;
    }
    const int per = a.team * VEC, tiles = (a.C + per - 1) / per;
    const int64_t item = (int64_t)blockIdx.x * (256 / a.team) + threadIdx.x / a.team;
    if (item >= (int64_t)a.chunks * tiles) return;
    const int chunk = (int)(item / tiles), c = (int)(item % tiles) * per + (threadIdx.x & (a.team - 1)) * VEC;
    if (c >= a.C) return;
    const uint32_t V = (uint32_t)a.V;
    const int from = chunk * a.chunk, to = a.N - from > a.chunk ? from + a.chunk : a.N;  // (from + chunk may pass 32 bits)
    const TY* dy = reinterpret_cast<const TY*>(a.dy) + c;
    A* part = reinterpret_cast<A*>(a.part) + (int64_t)chunk * 2 * a.C + c;
    const uint32_t before = from > 0 ? a.key[from - 1] : V, after = to < a.N ? a.key[to] : V;
    uint32_t key[AHEAD], pos[AHEAD];
    const auto fetch = [&](int i) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int at = i + j < to ? i + j : to - 1;
            key[j] = a.key[at];
            pos[j] = a.pos[at];
        }
    };
    fetch(from);
    A acc[VEC];
    uint32_t cur = key[0];
    bool opened = cur == before;  // the run came from the chunk before
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0;
    const auto close = [&](bool goes_on) {
        if (cur >= V) return;  // positions without a token, which come last
        if (opened || goes_on) store_wide<A, VEC>(part + (opened ? 0 : a.C), acc);
        else put_row<A, TW, VEC>(dw + (int64_t)cur * a.C + c, acc, a.scale);
    };
    for (int i = from; i < to && key[0] < V; i += AHEAD) {  // (positions without a token come last)
        // no load depends on a condition (past the chunk's end it is the last row again), and rows stay as they lie in memory
        // until their turn: as elements behind conditions, each of 16 bits would have a register of its own
        Raw row[AHEAD];
        uint32_t k[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            k[j] = key[j];
            row[j] = *reinterpret_cast<const Raw*>(dy + (int64_t)pos[j] * a.C);
        }
        if (i + AHEAD < to) fetch(i + AHEAD);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (i + j >= to) break;
            if (k[j] != cur) {
                close(false);
                cur = k[j];
                opened = false;
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] = 0;
            }
            if (cur < V) {
                const Pack<TY, VEC> v = unpacked<TY, VEC>(row[j]);
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] += (A)v.e[e];
            }
        }
    }
    close(cur == after);
}

constexpr int JOIN_WAVES = 8;

// Runs over chunks' borders: the workgroup of the chunk in which a run begins adds its parts, its teams of lanes (as k_sum's)
// in turn, and the teams' sums in order. 4 to 10 us, most of it the launch. Few runs are that long; one wave for each takes
// 22 us where 11 tokens have 31,104 positions.
template <typename TW, int VEC> __global__ __launch_bounds__(64 * JOIN_WAVES) void k_join(SumArgs a) {
    using A = typename Acc<TW>::type;
    __shared__ A sums[JOIN_WAVES * 64 * VEC];
    const int lane = threadIdx.x & 63, teams = 64 * JOIN_WAVES / a.team, team = threadIdx.x / a.team;
    const int chunk = (int)blockIdx.x, at = (threadIdx.x & (a.team - 1)) * VEC, c = (int)blockIdx.y * a.team * VEC + at;
    const int from = chunk * a.chunk, next = from + a.chunk;
    const uint32_t k = a.key[next - 1];
    if (k >= (uint32_t)a.V || a.key[next] != k) return;                // nothing goes on (as for all that follow, of the
    if (a.key[from] == k && from > 0 && a.key[from - 1] == k) return;  // whole workgroup); it began before this chunk
    int end = chunk + 2;  // the first chunk that does not begin inside the run
    for (bool more = true; more;) {
        const int j = end + lane;
        const uint64_t out = __ballot(j >= a.chunks || a.key[(int64_t)j * a.chunk] != k);
        more = out == 0;
        end += more ? 64 : __ffsll((unsigned long long)out) - 1;
    }
    const A* part = reinterpret_cast<const A*>(a.part) + c;
    A acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0;
    if (c < a.C) {
        if (team == 0) load_wide<A, VEC>(part + ((int64_t)chunk * 2 + 1) * a.C, acc);
        int j = chunk + 1 + team;
        for (; j + 3 * teams < end; j += 4 * teams) {
            A x[4][VEC];
#pragma unroll
            for (int i = 0; i < 4; ++i) load_wide<A, VEC>(part + (int64_t)(j + i * teams) * 2 * a.C, x[i]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] += x[i][e];
        }
        for (; j < end; j += teams) {
            A x[VEC];
            load_wide<A, VEC>(part + (int64_t)j * 2 * a.C, x);
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += x[e];
        }
    }
    const int width = a.team * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) sums[team * width + at + e] = acc[e];
    const int used = end - chunk - 1 < teams ? end - chunk - 1 : teams;  // teams that had a part
    __syncthreads();
    if (team || c >= a.C) return;
    for (int w = 1; w < used; ++w)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += sums[w * width + at + e];
    put_row<A, TW, VEC>(reinterpret_cast<TW*>(a.dw) + (int64_t)k * a.C + c, acc, a.scale);
}

// -- few tokens --------------------------------------------------------------------------------------------------------

// A workgroup for each row of the table and 64 vectors of its columns: its four waves look through a quarter of the positions
// each, a position a lane, and add the rows of those that hold its token, AHEAD at a time; then the waves' sums go together in
// order. One launch in place of three, no scratch, nothing waited for: 81 tokens of 11 x 512 take 2.8 us in a row of calls,
// sorted 10.6, and of 16,000 x 2,048 29 and 33. 256 positions of one token, the slowest, 11 and 12; 32,768 rows of 64 columns,
// each a workgroup's, about the same.
constexpr int FEW = 256, FEW_ROWS = 32768;

template <typename TW, typename TY, int VEC>
__global__ __launch_bounds__(256) void k_few(Ids ids, int N, int C, double scale, const TY* dy, TW* dw) {
    using A = typename Acc<TW>::type;
    using Raw = typename Words<VEC * (int)sizeof(TY)>::type;
    __shared__ A sums[4][64 * VEC];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = lane * VEC;
    const int64_t c = (int64_t)blockIdx.y * 64 * VEC + at;
    const int per = (N + 3) / 4, n = wave * per + lane;
    const uint32_t v = blockIdx.x;
    uint64_t mine = __ballot(lane < per && n < N && token(ids, n) == v);
    const TY* from = dy + (int64_t)wave * per * C + (c < C ? c : 0);
    A acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0;
    while (mine) {
        Raw row[AHEAD];
        const int have = __popcll(mine);
        int p = 0;
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {  // past the last one it is that one again
            if (mine) p = __ffsll((unsigned long long)mine) - 1;
            mine &= mine - 1;
            row[j] = *reinterpret_cast<const Raw*>(from + (int64_t)p * C);
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (j >= have) break;
            const Pack<TY, VEC> x = unpacked<TY, VEC>(row[j]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += (A)x.e[e];
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) sums[wave][at + e] = acc[e];
    __syncthreads();
    if (wave || c >= C) return;
    for (int w = 1; w < 4; ++w)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += sums[w][at + e];
    put_row<A, TW, VEC>(dw + (int64_t)v * C + c, acc, scale);
}

// -- small tables ------------------------------------------------------------------------------------------------------

// A table of few rows has all its sums in shared memory, a set for each wave: rows of dy come in their order, TALLY of them
// under way, and go to their tokens' sums. A workgroup has a chunk of the positions, its waves a part of it each, and 64 vectors
// of the columns. Its sums together are its part of the gradient.
//
// 31,104 positions of 11 x 512 bf16 take 16 us with the join, where sorting and summing take 27 (32 MB, 6.7 us of them); the
// whole gradient of 65,536 x 2,048 (268 MB, 56 us) 62 us and 66 in a row of calls, where the last-level cache keeps part of dy,
// and 96 and 110 after other work. From 17 rows on, four waves' sums fill the memory: 32 rows take 20 us and 26 in the first
// case, 83 and 65 in the second, and more rows are slower than the sort in all. With the next rows' loads ahead of the sums,
// 11 rows take 59 us in place of 55 of the second case's kernel.
constexpr int TALLY = 16;
static bool small(int64_t N, int64_t V, int64_t C) { return N > 0 && (V <= 16 || (V <= 32 && N * C <= 1 << 25)); }

struct TallyArgs {
    Ids ids;
    const void* dy;
    void *part, *dw;  // part: [chunks][V][C]
    int N, C, per, chunks;  // per: positions of a wave
    double scale;
};

template <typename TW, typename TY, int VEC> __global__ __launch_bounds__(1024) void k_tally(TallyArgs a) {
    using A = typename Acc<TW>::type;
    using Raw = typename Words<VEC * (int)sizeof(TY)>::type;
    constexpr int WIDTH = 64 * VEC;
    extern __shared__ __attribute__((aligned(16))) char shared[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, V = a.ids.V, all = V * WIDTH;
    A* sums = reinterpret_cast<A*>(shared);
    A* mine = sums + wave * all + lane * VEC;
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < VEC; ++e) mine[v * WIDTH + e] = 0;
    const int c0 = (int)blockIdx.y * WIDTH, c = c0 + lane * VEC;
    const int64_t from = ((int64_t)blockIdx.x * waves + wave) * a.per, to = from + a.per < a.N ? from + a.per : a.N;
    const TY* dy = reinterpret_cast<const TY*>(a.dy) + (c < a.C ? c : 0);
    for (int64_t base = from; base < to; base += 64) {
        const uint32_t k = base + lane < to ? token(a.ids, base + lane) : (uint32_t)V;
        const int have = to - base < 64 ? (int)(to - base) : 64;
        for (int i = 0; i < have; i += TALLY) {
            Raw row[TALLY];
#pragma unroll
            for (int j = 0; j < TALLY; ++j)  // past the last position it is that one again
                row[j] = *reinterpret_cast<const Raw*>(dy + (base + (i + j < have ? i + j : have - 1)) * a.C);
#pragma unroll
            for (int j = 0; j < TALLY; ++j) {
                if (i + j >= have) break;
                const int v = __builtin_amdgcn_readlane((int)k, i + j);
                if (v >= V) continue;
                const Pack<TY, VEC> x = unpacked<TY, VEC>(row[j]);
#pragma unroll
                for (int e = 0; e < VEC; ++e) mine[v * WIDTH + e] += (A)x.e[e];
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < all; i += blockDim.x) {
        const int v = i / WIDTH, at = c0 + i % WIDTH;
        if (at >= a.C) continue;
        A s = sums[i];
        for (int w = 1; w < waves; ++w) s += sums[w * all + i];
        if (a.chunks > 1) reinterpret_cast<A*>(a.part)[((int64_t)blockIdx.x * V + v) * a.C + at] = s;
        else reinterpret_cast<TW*>(a.dw)[(int64_t)v * a.C + at] = (TW)(s * (A)a.scale);
    }
}

// The chunks' parts together: 64 sums a workgroup, its waves taking the chunks in turn, and then the waves' sums in order.
template <typename TW> __global__ __launch_bounds__(1024) void k_tally_join(TallyArgs a) {
    using A = typename Acc<TW>::type;
    __shared__ A sums[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t all = (int64_t)a.ids.V * a.C, i = (int64_t)blockIdx.x * 64 + lane;
    const A* part = reinterpret_cast<const A*>(a.part) + i;
    A s = 0;
    if (i < all)
#pragma unroll 8
        for (int k = wave; k < a.chunks; k += 16) s += part[k * all];
    sums[wave][lane] = s;
    __syncthreads();
    if (wave || i >= all) return;
    for (int w = 1; w < 16; ++w) s += sums[w][lane];
    reinterpret_cast<TW*>(a.dw)[i] = (TW)(s * (A)a.scale);
}

// -- launches ----------------------------------------------------------------------------------------------------------

static bool types_ok(int wt, int yt) {
    const bool known = wt == EBR_DTYPE_F32 || wt == EBR_DTYPE_BF16 || wt == EBR_DTYPE_F16 || wt == EBR_DTYPE_F64;
    return known && (wt == yt || (wt == EBR_DTYPE_F32 && (yt == EBR_DTYPE_BF16 || yt == EBR_DTYPE_F16)));
}

static int check(int wt, int yt, int64_t N, int64_t V, int64_t C) {
    if (!types_ok(wt, yt)) return EBR_ERR_DTYPE;
    if (N < 0 || N >= ((int64_t)1 << 31) - SORT_ONE || V < 1 || V >= ((int64_t)1 << 31) - 1 || C < 1 ||
        C >= (1 << 18) || N * C >= ((int64_t)1 << 40) || V * C >= ((int64_t)1 << 40))
        return EBR_ERR_SHAPE;
    return EBR_OK;
}

template <typename F> static int by_types(int wt, int yt, F f) {
    if (wt == EBR_DTYPE_F32 && yt == EBR_DTYPE_F32) return f(float(), float());
    if (wt == EBR_DTYPE_F32 && yt == EBR_DTYPE_BF16) return f(float(), __bf16());
    if (wt == EBR_DTYPE_F32) return f(float(), _Float16());
    if (wt == EBR_DTYPE_BF16) return f(__bf16(), __bf16());
    if (wt == EBR_DTYPE_F16) return f(_Float16(), _Float16());
    return f(double(), double());
}

// Sorted positions that a team adds up: 64, or fewer (down to one round of loads) as far as that takes to have 768 waves,
// three for each compute unit, of 512 columns each; more for very many positions, which bounds the parts that a run is in.
constexpr int CHUNK = 64, MIN_CHUNK = 8, MAX_CHUNKS = 8192;
constexpr int64_t MIN_COLUMNS = 768 * 512;

struct Plan {
    int passes, bits, groups, tiles, chunk, chunks;
    int64_t words, part;  // 32-bit words of keys and positions (both halves) and counts; elements of part
    Plan(int64_t N, int64_t V, int64_t C) {
        int width = 1;
        while ((V >> width) != 0) ++width;  // the tokens 0 .. V
        passes = (width + SORT_BITS - 1) / SORT_BITS;
        bits = (width + passes - 1) / passes;
        const int64_t all = (N + SORT_THREADS - 1) / SORT_THREADS;
        tiles = (int)((all + SORT_GROUPS - 1) / SORT_GROUPS);
        groups = tiles ? (int)((all + tiles - 1) / tiles) : 0;
        chunk = CHUNK;
        while (chunk > MIN_CHUNK && (N + chunk - 1) / chunk * C < MIN_COLUMNS) chunk /= 2;
        while ((N + chunk - 1) / chunk > MAX_CHUNKS) chunk *= 2;
        chunks = (int)((N + chunk - 1) / chunk);
        words = 4 * N + (int64_t)groups * SORT_DIGITS;
        words = (words + 3) / 4 * 4;
        part = (int64_t)chunks * 2 * C;
    }
};

static bool few(int64_t N, int64_t V) { return N > 0 && N <= FEW && V <= FEW_ROWS; }

// Of k_tally: waves whose sums fill 64 KiB, and chunks for two workgroups on each compute unit, of at least TALLY positions a
// wave.
struct Tally {
    int waves = 16, per, chunks;
    Tally(int64_t N, int64_t V, int64_t C) {
        while (waves > 1 && waves * V * 512 > 65536) waves /= 2;
        const int64_t tiles = (C + 127) / 128, each = (N * tiles + 512 * waves - 1) / (512 * waves);
        per = (int)((each + TALLY - 1) / TALLY * TALLY);
        chunks = (int)((N + (int64_t)waves * per - 1) / ((int64_t)waves * per));
    }
};

// Lanes of a row of C / vec vectors: the next power of two, at most a wave.
static int team_of(int C, int vec) {
    int t = 1;
    while (t < 64 && t * vec < C) t *= 2;
    return t;
}

// Columns that a thread takes at once: 16 bytes of TY, half of that, or one element, as C and the pointers allow.
template <typename TY, typename F> static void by_vector(int C, std::initializer_list<const void*> ps, F f) {
    constexpr int VEC = 16 / (int)sizeof(TY), HALF = VEC / 2;
    bool whole = true;
    for (const void* p : ps) whole = whole && aligned(p, 16);
    if (whole && C % VEC == 0) return f(std::integral_constant<int, VEC>());
    if (whole && C % HALF == 0) return f(std::integral_constant<int, HALF>());
    f(std::integral_constant<int, 1>());
}

template <typename TW, typename TY, int VEC> static void launch_sums(hipStream_t s, SumArgs a) {
    using A = typename Acc<TW>::type;
    a.team = team_of(a.C, VEC);
    const int64_t per = (int64_t)a.team * VEC, items = a.chunks * ((a.C + per - 1) / per), teams = 256 / a.team;
    a.sum_blocks = (unsigned)((items + teams - 1) / teams);
    // rows to a workgroup of zeros: about 32 KiB of them
    a.zero_rows = 4;
    while (a.zero_rows < 256 && (int64_t)a.zero_rows * a.C * (int64_t)sizeof(TW) < 32768) a.zero_rows *= 2;
    const int64_t zeros = ((int64_t)a.V + a.zero_rows - 1) / a.zero_rows;
    hipLaunchKernelGGL((k_sum<TW, TY, VEC>), dim3((unsigned)(a.sum_blocks + zeros)), dim3(256), 0, s, a);
    if (a.chunks > 1) {
        constexpr int JV = VEC < 16 / (int)sizeof(A) ? VEC : 16 / (int)sizeof(A);
        a.team = team_of(a.C, JV);
        const int64_t tiles = (a.C + a.team * JV - 1) / (a.team * JV);
        hipLaunchKernelGGL((k_join<TW, JV>), dim3(a.chunks - 1, (unsigned)tiles), dim3(64 * JOIN_WAVES), 0, s, a);
    }
}

}  // namespace ebr_embed

using namespace ebr_embed;

extern "C" {

int ebr_block_embed(int wdtype, int ydtype, int ids64, int64_t N, int64_t V, int C, double scale, const void* ids,
                    const void* w, void* y, void* stream) {
    const int rc = check(wdtype, ydtype, N, V, C);
    if (rc) return rc;
    if (!ids || !w || !y) return EBR_ERR_NULL;
    if (N == 0) return EBR_OK;
    const Ids i = {ids, ids64 != 0, (int)V};
    return by_types(wdtype, ydtype, [&](auto tw, auto ty) {
        using TW = decltype(tw);
        using TY = decltype(ty);
        const auto go = [&](auto vec) {
            constexpr int VN = decltype(vec)::value;
            const int team = team_of(C, VN);
            hipLaunchKernelGGL((k_lookup<TW, TY, VN>), dim3(blocks_for(N, rows_of<TW>() * (256 / team))), dim3(256), 0,
                               (hipStream_t)stream, i, N, C, team, scale, (const TW*)w, (TY*)y);
        };
        by_vector<TY>(C, {w, y}, go);
        return launched();
    });
}

int64_t ebr_block_embed_bwd_scratch(int wdtype, int64_t N, int64_t V, int C) {
    if (check(wdtype, wdtype, N, V, C)) return -1;
    if (small(N, V, C)) return Tally(N, V, C).chunks * V * C * (wdtype == EBR_DTYPE_F64 ? 8 : 4);
    const Plan p(N, V, C);
    return p.words * 4 + p.part * (wdtype == EBR_DTYPE_F64 ? 8 : 4);
}

int ebr_block_embed_bwd(int wdtype, int ydtype, int ids64, int64_t N, int64_t V, int C, double scale, const void* ids,
                        const void* dy, void* dw, void* scratch, void* stream) {
    const int rc = check(wdtype, ydtype, N, V, C);
    if (rc) return rc;
    if (!dw || (N > 0 && (!ids || !dy))) return EBR_ERR_NULL;
    if (N > 0 && !scratch) return EBR_ERR_SCRATCH;
    if (!aligned(scratch, 16)) return EBR_ERR_ALIGN;
    hipStream_t s = (hipStream_t)stream;
    if (few(N, V))
        return by_types(wdtype, ydtype, [&](auto tw, auto ty) {
            using TW = decltype(tw);
            using TY = decltype(ty);
            const auto go = [&](auto vec) {
                constexpr int VN = decltype(vec)::value;
                hipLaunchKernelGGL((k_few<TW, TY, VN>), dim3((unsigned)V, (C + 64 * VN - 1) / (64 * VN)), dim3(256), 0, s,
                                   Ids{ids, ids64 != 0, (int)V}, (int)N, C, scale, (const TY*)dy, (TW*)dw);
            };
            by_vector<TY>(C, {dy, dw}, go);
            return launched();
        });
    if (small(N, V, C))
        return by_types(wdtype, ydtype, [&](auto tw, auto ty) {
            using TW = decltype(tw);
            using TY = decltype(ty);
            constexpr int VEC = sizeof(TY) == 8 ? 1 : 2;
            const Tally p(N, V, C);
            const TallyArgs a = {{ids, ids64 != 0, (int)V}, dy, scratch, dw, (int)N, C, p.per, p.chunks, scale};
            const auto go = [&](auto vec) {
                constexpr int VN = decltype(vec)::value;
                using A = typename Acc<TW>::type;
                hipLaunchKernelGGL((k_tally<TW, TY, VN>), dim3(p.chunks, (C + 64 * VN - 1) / (64 * VN)), dim3(64 * p.waves),
                                   (size_t)p.waves * V * 64 * VN * sizeof(A), s, a);
            };
            if (C % VEC == 0 && aligned(dy, VEC * sizeof(TY))) go(std::integral_constant<int, VEC>());
            else go(std::integral_constant<int, 1>());
            if (p.chunks > 1)
                hipLaunchKernelGGL((k_tally_join<TW>), dim3((unsigned)((V * C + 63) / 64)), dim3(1024), 0, s, a);
            return launched();
        });
    const Plan p(N, V, C);
    uint32_t* w32 = reinterpret_cast<uint32_t*>(scratch);
    uint32_t *k0 = w32, *p0 = w32 + N, *k1 = w32 + 2 * N, *p1 = w32 + 3 * N, *counts = w32 + 4 * N;
    SortArgs so = {{ids, ids64 != 0, (int)V}, nullptr, nullptr, k0, p0, counts, (int)N, 0, p.bits, p.tiles};
    if (N > 0 && N <= SORT_ONE) {
        hipLaunchKernelGGL(k_sort_tile, dim3(1), dim3(SORT_THREADS), 0, s, so, p.passes);
    } else if (N > 0) {
        for (int i = 0; i < p.passes; ++i) {
            so.shift = i * p.bits;
            hipLaunchKernelGGL(k_sort_count, dim3(p.groups), dim3(SORT_THREADS), 0, s, so);
            hipLaunchKernelGGL(k_sort_place, dim3(p.groups), dim3(SORT_THREADS), 0, s, so);
            so.kin = so.kout;
            so.pin = so.pout;
            so.kout = so.kout == k0 ? k1 : k0;
            so.pout = so.pout == p0 ? p1 : p0;
        }
    }
    const bool swapped = N > SORT_ONE && p.passes % 2 == 0;
    return by_types(wdtype, ydtype, [&](auto tw, auto ty) {
        using TW = decltype(tw);
        using TY = decltype(ty);
        SumArgs a = {swapped ? k1 : k0, swapped ? p1 : p0, dy, dw, w32 + p.words, (int)N, (int)V, C, p.chunk, p.chunks,
                     0, 0, 0, scale};
        by_vector<TY>(C, {dy, dw}, [&](auto vec) { launch_sums<TW, TY, decltype(vec)::value>(s, a); });
        return launched();
    });
}

}  // extern "C"
