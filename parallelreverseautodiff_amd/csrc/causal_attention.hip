// Causal attention over packed sequences with grouped heads, in either element type, and its form for the newest tokens of a
// sequence against its cache.
//
//   S = scale Q K^T,  key j seen by query i of n (keys: m) iff j <= m - n + i,  P = softmax rows(S),  O = P V,  lse = log sum exp S
//   D = rowsum(dO (.) O),  P = exp(S - lse),  dV = P^T dO,  dS = P (.) (dO V^T - D),  dQ = scale dS K,  dK = scale dS^T Q
//
// One pass over the keys with the running maximum and sum of a row: scores never reach memory.  The rows of a tile are
// (token, head of the group) pairs - token r / group, head r % group - so the query heads that share a key/value head share its
// tiles, and their gradients of K and V add up in one workgroup in one order.
// Statistics and sums are held in the element type (32 or 64 bits); products run on the 16 x 16 x 4 matrix instructions, whose
// element order along the reduction is free as long as both operands agree: lane group g takes elements CH c + VEC g + t of
// chunk c, which makes its reads whole 16-byte vectors.
//
// Non-finite values.  A key row that holds one (in K or V) counts as zeros and its scores become NaN where they are seen: a
// query that sees it has a row of NaN, a query that does not is not touched by it - a product with a masked weight of zero
// would carry 0 * NaN into every row of the tile.
#include "common.h"

#include <algorithm>

namespace prad {

namespace {

typedef float f4v __attribute__((ext_vector_type(4)));
typedef double d4v __attribute__((ext_vector_type(4)));

template <typename T> struct Num;
template <> struct Num<float> {
    typedef f4v Acc;
    static __device__ __forceinline__ Acc mfma(float a, float b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ int row(int r, int g) { return 4 * g + r; }  // row of accumulator element r in lane group g
    // scores are kept in units of log2 e: the exponential is the hardware's power of two
    static __device__ __forceinline__ float unit() { return 1.4426950408889634f; }
    static __device__ __forceinline__ float exp_unit(float x) { return __builtin_amdgcn_exp2f(x); }
    static __device__ __forceinline__ float log_sum(float m, float l) { return (m + __log2f(l)) * 0.6931471805599453f; }
};
template <> struct Num<double> {
    typedef d4v Acc;
    static __device__ __forceinline__ Acc mfma(double a, double b, Acc c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ int row(int r, int g) { return 4 * r + g; }
    static __device__ __forceinline__ double unit() { return 1.0; }
    static __device__ __forceinline__ double exp_unit(double x) { return exp(x); }
    static __device__ __forceinline__ double log_sum(double m, double l) { return m + log(l); }
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

template <typename T> __device__ __forceinline__ bool is_finite(T x) { return fabs(x) < (T)INFINITY; }
template <typename T> __device__ __forceinline__ T nan_of() { return (T)NAN; }

// The rows and keys of one sequence.  Values that do not describe rows of the buffers are cut off to some that do.
struct Span {
    int64_t q0, nq, k0, nk;
};
__device__ __forceinline__ int64_t clamped(int64_t v, int64_t most) { return v < 0 ? 0 : v > most ? most : v; }

template <typename T>
__device__ __forceinline__ Span span_of(const CausalArgs<T>& p, int s) {
    Span r;
    r.q0 = clamped(p.q_off[s], p.q_rows);
    const int64_t q1 = clamped(p.q_off[s + 1], p.q_rows);
    r.nq = q1 > r.q0 ? q1 - r.q0 : 0;
    if (p.k_begin == nullptr) {
        r.k0 = r.q0;
        r.nk = r.nq;
    } else {
        r.k0 = clamped(p.k_begin[s], p.k_rows);
        const int64_t k1 = clamped(p.k_end[s], p.k_rows);
        r.nk = k1 > r.k0 ? k1 - r.k0 : 0;
    }
    return r;
}

// Makes a row that holds a non-finite value NaN throughout.
template <typename T, int CHUNKS>
__device__ __forceinline__ void poison_row(Pack<T, 16 / sizeof(T)> (&frag)[CHUNKS]) {
    constexpr int VEC = 16 / sizeof(T);
    int bad = 0;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int t = 0; t < VEC; ++t) bad |= is_finite(frag[c].v[t]) ? 0 : 1;
    bad |= __shfl_xor(bad, 16, 64);
    bad |= __shfl_xor(bad, 32, 64);
    if (bad) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
            for (int t = 0; t < VEC; ++t) frag[c].v[t] = nan_of<T>();
    }
}

// ---- units of work ----------------------------------------------------------------------------------------------------------
// A unit is 16 packed rows of one sequence and key/value head against its keys or a part of them, one workgroup each; in the
// gradients of K and V it is 16 keys against the rows.  Every workgroup finds the sequence of its unit for itself: lengths live
// on the device.  The wavefronts take every fourth tile of 16 keys (or rows) and add their sums up in LDS at the end, which gives
// short sequences four times the wavefronts.  (Against 64 rows a workgroup and tiles in LDS: 86 us for 301, the batch of doubles
// below; 401 for 743, two sequences of 1024, 8 heads of 64 doubles.  Eight wavefronts: 80 and 467.)
// Everything is transposed - S^T = K Q^T, O^T = V^T P^T - so that the weights come out of the first product in the lanes where
// the second wants them and a row's statistics sit in a lane; rows go from memory to the registers of the matrix instructions
// without LDS, along for a product over the head dimension and across for one over the rows.  The registers of an operand are
// filled again for the next tile as soon as its product has read them, so that loads are always in flight.
constexpr int WAVES = 4, MANY_WAVES = 8;
// Parts of the keys: the least keys in one, sequences that are not cut (300 keys in parts of 64 and joined: 15.2 us, whole: 13.2),
// units that run at once, two workgroups per compute unit.  Parts are as large as lets all units of a call run at once: the cache
// of 24 sequences below in 71 us, in parts of 256 keys in 86.
constexpr int LEAST_KEYS = 128, WHOLE_KEYS = 512, RUNNING = 512;

template <typename T>
struct Parts {
    uint32_t units;   // at most
    int most;         // of a sequence; 1: units are tiles
    T *stat, *data;   // of part i of (token, head) number n: {maximum, sum} and the weighted sum of values, at n * most + i
    int32_t* keys;    // how many keys make a part, for the join
};

// Parts of a sequence's keys: of `size` keys, or of more if there would be too many parts, whole tiles.
__device__ __forceinline__ int64_t part_keys(int64_t keys, int64_t size, int most_parts) {
    if (keys <= size * most_parts) return size;
    return ((keys + most_parts - 1) / most_parts + 15) / 16 * 16;
}
__device__ __forceinline__ uint32_t part_count(int64_t keys, uint32_t size, int most_parts) {
    if (keys <= WHOLE_KEYS || keys <= size || most_parts == 1) return 1;
    if (keys <= (int64_t)size * most_parts) return ((uint32_t)keys + size - 1) / size;
    const int64_t larger = part_keys(keys, size, most_parts);
    return (uint32_t)((keys + larger - 1) / larger);
}

// Sums over the lanes up to this one.
__device__ __forceinline__ uint32_t scan64(uint32_t x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // one lane up inside each 16, two, four, eight
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // the last lane of the 16 before; of the 32 before
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return x;
}

// The spans of sequences first + lane, and taking one of them from its lane (no value passes 31 bits).
template <typename T>
__device__ __forceinline__ Span lane_span(const CausalArgs<T>& p, int s) {
    Span sp = {0, 0, 0, 0};
    if (s < p.sequences) sp = span_of(p, s);
    return sp;
}
__device__ __forceinline__ Span span_from(const Span& sp, int lane) {
    return Span{__builtin_amdgcn_readlane((int)sp.q0, lane), __builtin_amdgcn_readlane((int)sp.nq, lane), __builtin_amdgcn_readlane((int)sp.k0, lane),
                __builtin_amdgcn_readlane((int)sp.nk, lane)};
}

// The last sequence s whose begin(s, its offset) is not above `value`, by a whole wavefront: its span and begin; false: none.
// A search that looks at 64 sequences at a time: one round of loads for up to 63 sequences, two for up to 4095.
template <typename T, typename Begin>
__device__ __forceinline__ bool find_span(const CausalArgs<T>& p, uint32_t value, int lane, Begin begin, Span* span, uint32_t* begun) {
    int64_t lo = 0, left = (int64_t)p.sequences + 1;  // it lies in [lo, lo + left); the end counts as a sequence without rows
    for (;;) {
        const int64_t step = (left + 63) / 64, s = lo + lane * step;
        const bool there = lane * step < left;
        const uint32_t mine = there ? begin((uint32_t)s, (uint32_t)clamped(p.q_off[s], p.q_rows)) : ~0u;
        const Span sp = lane_span(p, step == 1 && there ? (int)s : p.sequences);
        const uint64_t above = ~__ballot(there && mine <= value);
        const int at = above == 0 ? 63 : __builtin_ctzll(above) - 1;
        if (at < 0) return false;
        if (step == 1) {
            *span = span_from(sp, at);
            *begun = __builtin_amdgcn_readlane((int)mine, at);
            return true;
        }
        lo += at * step;
        left = left - at * step < step ? left - at * step : step;
    }
}

// Tile `tile` of the packed rows of `group` heads and its number in its sequence.  Tiles are numbered through all sequences
// without a table, sequence s from floor(offset group / 16) + s on, which leaves room for its ceil(n group / 16) tiles.
template <typename T>
__device__ __forceinline__ bool find_tile(const CausalArgs<T>& p, uint32_t group, uint32_t tile, int lane, Span* span, uint32_t* inside) {
    uint32_t first;
    if (!find_span(p, tile, lane, [group](uint32_t s, uint32_t offset) { return offset * group / 16 + s; }, span, &first)) return false;
    *inside = tile - first;
    return *inside < ((uint32_t)span->nq * group + 15) / 16;
}

// Unit `unit` where sequences have parts, by a whole wavefront: its sequence, how many parts that has, and the unit's number
// inside it; false: there are not so many.
template <typename T>
__device__ __forceinline__ bool find_unit(const CausalArgs<T>& p, int most_parts, uint32_t size, uint32_t unit, int lane, Span* span, uint32_t* parts, uint32_t* inside) {
    uint32_t before = 0;
    for (int s0 = 0; s0 < p.sequences; s0 += 64) {
        const Span sp = lane_span(p, s0 + lane);
        const uint32_t count = part_count(sp.nk, size, most_parts), units = ((uint32_t)sp.nq * (uint32_t)p.group + 15) / 16 * count;
        const uint32_t upto = before + scan64(units);
        const uint64_t behind = __ballot(upto > unit);
        if (behind != 0) {
            const int at = __builtin_ctzll(behind);
            *span = span_from(sp, at);
            *parts = __builtin_amdgcn_readlane(count, at);
            *inside = unit - __builtin_amdgcn_readlane(upto - units, at);
            return *inside < (uint32_t)__builtin_amdgcn_readlane(units, at);  // (offsets that overlap may wrap the sum)
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// Keys per part that make all units of a call few enough to run at once, each sequence having a part that is not whole.
template <typename T>
__device__ __forceinline__ uint32_t keys_per_part(const CausalArgs<T>& p, int lane) {
    float keys = 0, tiles = 0;
    for (int s0 = 0; s0 < p.sequences; s0 += 64) {
        const Span sp = lane_span(p, s0 + lane);
        const float here = (float)(((uint32_t)sp.nq * (uint32_t)p.group + 15) / 16);
        tiles += here;
        keys += here * (float)sp.nk;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        keys += __shfl_xor(keys, d, 64);
        tiles += __shfl_xor(tiles, d, 64);
    }
    const float room = fmaxf((float)(RUNNING / 2), RUNNING - tiles * p.kv_heads), share = keys * p.kv_heads / room;
    return __builtin_amdgcn_readfirstlane(((uint32_t)fminf(fmaxf(share, (float)LEAST_KEYS), 1e9f) + 63) / 64 * 64);
}

// N consecutive elements; columns past the row's end are read at its start, for which nothing uses the result.
template <typename T, int N, bool ALIGNED>
__device__ __forceinline__ Pack<T, N> load_some(const T* __restrict__ row, int d0, int head_dim) {
    Pack<T, N> v;
    if constexpr (ALIGNED) {
        v = *reinterpret_cast<const Pack<T, N>*>(row + (d0 < head_dim ? d0 : 0));
    } else {
#pragma unroll
        for (int t = 0; t < N; ++t) v.v[t] = row[d0 + t < head_dim ? d0 + t : 0];
    }
    return v;
}

// A row along the reduction of a product over the head dimension: elements CH c + VEC g + t.
template <typename T, int HDP, bool ALIGNED>
__device__ __forceinline__ void load_along(const T* __restrict__ row, int g, int head_dim, Pack<T, 16 / sizeof(T)> (&to)[HDP * sizeof(T) / 64]) {
    constexpr int VEC = 16 / sizeof(T);
#pragma unroll
    for (int c = 0; c < HDP / (4 * VEC); ++c) to[c] = load_some<T, VEC, ALIGNED>(row, 4 * VEC * c + VEC * g, head_dim);
}
template <typename T, int HDP>
__device__ __forceinline__ void zero_past(int g, int head_dim, Pack<T, 16 / sizeof(T)> (&frag)[HDP * sizeof(T) / 64]) {
    constexpr int VEC = 16 / sizeof(T);
#pragma unroll
    for (int c = 0; c < HDP / (4 * VEC); ++c)
#pragma unroll
        for (int t = 0; t < VEC; ++t) frag[c].v[t] = 4 * VEC * c + VEC * g + t < head_dim ? frag[c].v[t] : (T)0;
}
// A row across, a column per lane: columns 16 N y + N li + t.
template <typename T, int HDP> constexpr int columns_at_once() { return 16 / (int)sizeof(T) < HDP / 16 ? 16 / (int)sizeof(T) : HDP / 16; }
template <typename T, int HDP, bool ALIGNED>
__device__ __forceinline__ void load_across(const T* __restrict__ row, int li, int head_dim, Pack<T, columns_at_once<T, HDP>()> (&to)[HDP / 16 / columns_at_once<T, HDP>()]) {
    constexpr int N = columns_at_once<T, HDP>();
#pragma unroll
    for (int y = 0; y < HDP / 16 / N; ++y) to[y] = load_some<T, N, ALIGNED>(row, 16 * N * y + N * li, head_dim);
}
// Zeros for the non-finite values of a tile that is read across; returns a bit for each of its rows that has one.
template <typename T, int N, int COUNT>
__device__ __forceinline__ uint32_t zero_bad(Pack<T, N> (&v)[4][COUNT]) {
    T odd = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < COUNT; ++y)
#pragma unroll
            for (int t = 0; t < N; ++t) odd = fma(v[x][y].v[t], (T)0, odd);
    uint32_t rows = 0;
    if (__any(!(odd == 0))) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            bool fine = true;
#pragma unroll
            for (int y = 0; y < COUNT; ++y)
#pragma unroll
                for (int t = 0; t < N; ++t) {
                    fine = fine && is_finite(v[x][y].v[t]);
                    v[x][y].v[t] = is_finite(v[x][y].v[t]) ? v[x][y].v[t] : (T)0;
                }
            const uint64_t b = __ballot(!fine);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if ((b >> (16 * i)) & 0xFFFFu) rows |= 1u << Num<T>::row(x, i);
        }
    }
    return rows;
}
// The product of two tiles over the head dimension: rows of the accumulator are rows of a, columns rows of b.
template <typename T, int COUNT>
__device__ __forceinline__ typename Num<T>::Acc product(const Pack<T, 16 / sizeof(T)> (&a)[COUNT], const Pack<T, 16 / sizeof(T)> (&b)[COUNT]) {
    typename Num<T>::Acc acc = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < COUNT; ++c)
#pragma unroll
        for (int t = 0; t < 16 / (int)sizeof(T); ++t) acc = Num<T>::mfma(a[c].v[t], b[c].v[t], acc);
    return acc;
}
// out += rows that are read across, transposed, times the weights of those rows.
template <typename T, int N, int COUNT>
__device__ __forceinline__ void add_weighted(const Pack<T, N> (&v)[4][COUNT], typename Num<T>::Acc w, typename Num<T>::Acc (&out)[N * COUNT]) {
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < N * COUNT; ++y) out[y] = Num<T>::mfma(v[x][y / N].v[y % N], w[x], out[y]);
}
// A wavefront's sums to LDS: out[N y + t][x] is column 16 N y + N row(x, g) + t of row li.
template <typename T, int N, int TILES, int PITCH>
__device__ __forceinline__ void put_sums(const typename Num<T>::Acc (&out)[TILES], int li, int g, T* __restrict__ to) {
#pragma unroll
    for (int y = 0; y < TILES / N; ++y)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            Pack<T, N> e;
#pragma unroll
            for (int t = 0; t < N; ++t) e.v[t] = out[N * y + t][x];
            *reinterpret_cast<Pack<T, N>*>(&to[li * PITCH + 16 * N * y + N * Num<T>::row(x, g)]) = e;
        }
}

// x / group for x < group + 16
__device__ __forceinline__ uint32_t heads_over(uint32_t x, uint32_t group, uint32_t inverse) { return group < 16 ? x * inverse >> 16 : x >= group; }
__device__ __forceinline__ uint32_t inverse_of(uint32_t group) { return (65535 + group) / group; }  // of 2^16, rounded up

// ---- forward, and the newest tokens of a sequence against its cache ---------------------------------------------------------
// A cache is read once and bounds the call from some MB on: 24 sequences of 0 to 8192 keys, 16 heads on 4 of 128 floats, in
// 64 us, and 5 for joining the parts (332 MB, 4.5 TB/s of the 5.0 that a copy reaches).  Small calls are bound by their latency,
// about 1 us to find the sequence, 1.5 for the first rows, 1 per tile and 0.6 for the sums: 300 keys, 8 heads on 2 of 64
// floats, in 8.9 us.  Doubles, forward over sequences of 512, 256, 200 and 37, 6 heads on 3 of 32: 20 us.
template <typename T, int HDP, bool ALIGNED, bool CUT, int W>
__global__ void __launch_bounds__(64 * W, W == 4 && sizeof(T) == 4 && ALIGNED ? 2 : 1) attention_kernel(const CausalArgs<T> p, const Parts<T> cut) {
    constexpr int VEC = 16 / sizeof(T), CHUNKS = HDP / (4 * VEC), NY = HDP / 16, N = columns_at_once<T, HDP>(), PITCH = HDP + VEC;
    typedef typename Num<T>::Acc Acc;
    __shared__ __attribute__((aligned(16))) T sums[W][16 * PITCH];
    __shared__ T stat[W][2][16];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    // heads of a unit are neighbours, so that workgroups without a unit come last
    const uint32_t stride = gridDim.x / p.kv_heads;
    const int kv = (int)(blockIdx.x % p.kv_heads);
    const uint32_t keys_each = CUT ? keys_per_part(p, lane) : 0;
    if (CUT && blockIdx.x == 0 && threadIdx.x == 0) *cut.keys = (int32_t)keys_each;
    const T factor = p.scale * Num<T>::unit();
    // where the lane's rows of a whole tile lie (kept: 3 to 8 % faster; 128 doubles leave no registers for it)
    constexpr bool KEPT = sizeof(T) * HDP <= 512;
    const int64_t k_at = li * p.ldk, v_at[4] = {Num<T>::row(0, g) * p.ldv, Num<T>::row(1, g) * p.ldv, Num<T>::row(2, g) * p.ldv, Num<T>::row(3, g) * p.ldv};
    for (uint32_t unit = blockIdx.x / p.kv_heads; unit < cut.units; unit += stride) {
        Span sp;
        uint32_t parts = 1, inside;
        if constexpr (CUT) {
            if (!find_unit(p, cut.most, keys_each, unit, lane, &sp, &parts, &inside)) return;  // (nor are there any behind it)
        } else {
            if (!find_tile(p, p.group, unit, lane, &sp, &inside)) continue;
        }
        const uint32_t rows = (uint32_t)sp.nq * (uint32_t)p.group, tile = inside / parts, part = inside % parts, row0 = tile * 16;
        const int64_t lead = sp.nk - sp.nq;
        const uint32_t r = row0 + li < rows ? row0 + li : rows - 1;  // the lane's row; past the last it is the last one again
        const uint32_t first_token = row0 / p.group, ahead = (row0 % p.group + (r - row0)) / p.group;  // of the tile; of the row, from there
        const int64_t token = sp.q0 + first_token + ahead;
        const int head = kv * p.group + (int)(r - (first_token + ahead) * p.group);
        Pack<T, VEC> q[CHUNKS];
        load_along<T, HDP, ALIGNED>(p.Q + token * p.ldq + head * (int64_t)p.head_dim, g, p.head_dim, q);
        const int64_t first_last = lead + first_token, last = first_last + ahead;  // the last key that the tile's first row sees, that this one does
        const int64_t size = CUT ? part_keys(sp.nk, keys_each, cut.most) : 0, seen = clamped(first_last + (int)__builtin_amdgcn_readlane(ahead, 15) + 1, sp.nk);
        const int64_t from = part * size, to = parts == 1 || seen < from + size ? seen : from + size;
        const T* __restrict__ K = p.K + sp.k0 * p.ldk + kv * (int64_t)p.head_dim;
        const T* __restrict__ V = p.V + sp.k0 * p.ldv + kv * (int64_t)p.head_dim;
        T m = -(T)INFINITY, l = 0;  // l: this lane's share
        Acc o[NY];  // element x of o[N y + t]: column 16 N y + N row(x, g) + t of row li
#pragma unroll
        for (int y = 0; y < NY; ++y) o[y] = Acc{0, 0, 0, 0};
        Pack<T, VEC> k[CHUNKS];   // of key li
        Pack<T, N> v[4][NY / N];  // of keys row(x, g)
        // keys past the last are the last one again: their scores are masked
        auto load_k = [&](int64_t k0) {
            int64_t at = k_at;
            if (!KEPT || to - k0 < 16) at = (to - 1 - k0 < li ? to - 1 - k0 : li) * p.ldk;
            load_along<T, HDP, ALIGNED>(K + k0 * p.ldk + at, g, p.head_dim, k);
        };
        auto load_v = [&](int64_t k0) {
            int64_t at[4] = {v_at[0], v_at[1], v_at[2], v_at[3]};
            if (!KEPT || to - k0 < 16) {
#pragma unroll
                for (int x = 0; x < 4; ++x) at[x] = (to - 1 - k0 < Num<T>::row(x, g) ? to - 1 - k0 : Num<T>::row(x, g)) * p.ldv;
            }
            const T* __restrict__ first = V + k0 * p.ldv;
#pragma unroll
            for (int x = 0; x < 4; ++x) load_across<T, HDP, ALIGNED>(first + at[x], li, p.head_dim, v[x]);
        };
        int64_t k0 = from + 16 * wave;
        if (k0 < to) {
            load_k(k0);
            load_v(k0);
        }
        zero_past<T, HDP>(g, p.head_dim, q);
        poison_row<T, CHUNKS>(q);
        for (; k0 < to; k0 += 16 * W) {
            Acc sc = product<T>(k, q);
            // A key with a non-finite value is NaN for the rows that see it and zeros for the others.  In K it makes the scores
            // of its key non-finite whatever the rows hold, so that K is looked at only after such a score.
            uint32_t poisoned = 0;  // bit j: key k0 + j
            T odd = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) odd = fma(sc[x], (T)0, odd);
            if (__any(!(odd == 0))) {
                bool fine = true;
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                    for (int t = 0; t < VEC; ++t) fine = fine && is_finite(k[c].v[t]);
                const uint64_t b = __ballot(!fine);
                poisoned = (uint32_t)((b | (b >> 16) | (b >> 32) | (b >> 48)) & 0xFFFFu);
            }
            load_k(k0 + 16 * W);
            poisoned |= zero_bad<T>(v);
#pragma unroll
            for (int x = 0; x < 4; ++x) sc[x] *= factor;
            if (poisoned != 0 || k0 + 15 > first_last) {
                const int most = (int)clamped(last - k0 + 1, 16);  // keys of the tile that the row sees
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int j = Num<T>::row(x, g);
                    sc[x] = j >= most ? -(T)INFINITY : (poisoned >> j) & 1 ? nan_of<T>() : sc[x];
                }
            }
            T top = -(T)INFINITY;
#pragma unroll
            for (int x = 0; x < 4; ++x) top = fmax(top, sc[x]);
            // the maximum is raised for a tile only if one of its scores is above it
            if (__any(top > m)) {
                top = fmax(top, __shfl_xor(top, 16, 64));
                top = fmax(top, __shfl_xor(top, 32, 64));
                top = fmax(top, m);
                const T f = top == -(T)INFINITY ? (T)1 : Num<T>::exp_unit(m - top);
                m = top;
                l *= f;
#pragma unroll
                for (int y = 0; y < NY; ++y)
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[y][x] *= f;
            }
            const T ref = m == -(T)INFINITY ? (T)0 : m;  // nothing seen yet: every weight is exp(-inf) = 0
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                sc[x] = Num<T>::exp_unit(sc[x] - ref);
                l += sc[x];
            }
            add_weighted<T>(v, sc, o);
            load_v(k0 + 16 * W);
        }
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (g == 0) {
            stat[wave][0][li] = m;
            stat[wave][1][li] = l;
        }
        put_sums<T, N, NY, PITCH>(o, li, g, sums[wave]);
        __syncthreads();
        const int here = (int)(rows - row0 < 16 ? rows - row0 : 16);
        for (int at = threadIdx.x; at < here * (HDP / VEC); at += 64 * W) {
            const uint32_t row = at / (HDP / VEC), ahead_of = (row0 % p.group + row) / p.group;
            const int d = at % (HDP / VEC) * VEC;
            if (d >= p.head_dim) continue;
            const int64_t to_token = sp.q0 + first_token + ahead_of;
            const int to_head = kv * p.group + (int)(row0 + row - (first_token + ahead_of) * p.group);
            T top = stat[0][0][row], total = 0, sum[VEC];
#pragma unroll
            for (int w = 1; w < W; ++w) top = fmax(top, stat[w][0][row]);
            const T ref = top == -(T)INFINITY ? (T)0 : top;
#pragma unroll
            for (int t = 0; t < VEC; ++t) sum[t] = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const T f = Num<T>::exp_unit(stat[w][0][row] - ref);
                total = fma(stat[w][1][row], f, total);
                const Pack<T, VEC> e = *reinterpret_cast<const Pack<T, VEC>*>(&sums[w][row * PITCH + d]);
#pragma unroll
                for (int t = 0; t < VEC; ++t) sum[t] = fma(e.v[t], f, sum[t]);
            }
            T* __restrict__ dst;
            if (!CUT || parts == 1) {
                const bool any = first_last + ahead_of >= 0 && sp.nk > 0;
                const T by = any ? 1 / total : (T)0;
#pragma unroll
                for (int t = 0; t < VEC; ++t) sum[t] *= by;
                dst = p.O + to_token * p.ldo + to_head * (int64_t)p.head_dim;
                if (d == 0 && p.lse != nullptr) p.lse[to_head * p.q_rows + to_token] = any ? Num<T>::log_sum(top, total) : -(T)INFINITY;
            } else {
                const int64_t place = (to_token * p.heads + to_head) * cut.most + part;
                dst = cut.data + place * p.head_dim;
                if (d == 0) {
                    cut.stat[2 * place] = top;
                    cut.stat[2 * place + 1] = total;
                }
            }
#pragma unroll
            for (int t = 0; t < VEC; ++t)
                if (d + t < p.head_dim) dst[d + t] = sum[t];
        }
        __syncthreads();
    }
}

// Joins the parts of a row: a workgroup per (token, head), a wavefront every fourth part, whose loads are all in flight at once.
template <typename T>
__global__ void __launch_bounds__(64 * WAVES) cached_join_kernel(const CausalArgs<T> p, const Parts<T> cut) {
    __shared__ T sums[WAVES][128];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t at = blockIdx.x, token = at / p.heads;
    // rows in front of the first sequence and behind the last are left as they are
    Span sp;
    uint32_t first;
    if (!find_span(p, (uint32_t)token, lane, [](uint32_t, uint32_t offset) { return offset; }, &sp, &first)) return;
    if (token < sp.q0 || token >= sp.q0 + sp.nq) return;
    const int parts = (int)part_count(sp.nk, (uint32_t)*cut.keys, cut.most);
    if (parts == 1) return;
    const T m = lane < parts ? cut.stat[2 * (at * cut.most + lane)] : -(T)INFINITY;
    const T l = lane < parts ? cut.stat[2 * (at * cut.most + lane) + 1] : (T)0;
    constexpr int COUNT = 64 / WAVES;
    const T* __restrict__ mine = cut.data + at * cut.most * (int64_t)p.head_dim;
    T v[COUNT][2];
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
        const int i = wave + WAVES * j;
        v[j][0] = i < parts && lane < p.head_dim ? mine[(int64_t)i * p.head_dim + lane] : (T)0;
        v[j][1] = i < parts && lane + 64 < p.head_dim ? mine[(int64_t)i * p.head_dim + lane + 64] : (T)0;
    }
    T top = m;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmax(top, __shfl_xor(top, d, 64));
    T f = Num<T>::exp_unit(m - (top == -(T)INFINITY ? (T)0 : top)), total = l * f;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d, 64);
    f = sp.nk - sp.nq + (token - sp.q0) >= 0 ? f / total : (T)0;
    T sum[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
        const T w = __shfl(f, wave + WAVES * j, 64);
        sum[0] = fma(v[j][0], w, sum[0]);
        sum[1] = fma(v[j][1], w, sum[1]);
    }
    sums[wave][lane] = sum[0];
    sums[wave][lane + 64] = sum[1];
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= p.head_dim) return;
    T out = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) out += sums[w][d];
    p.O[token * p.ldo + at % p.heads * (int64_t)p.head_dim + d] = out;
}

// ---- backward -----------------------------------------------------------------------------------------------------------
// (Queries and keys are the same rows here: token i sees key j iff j <= i.  A row that sees a non-finite value has a NaN in lse,
// one of dO with a non-finite value a NaN in D: their weights are NaN, and the values themselves count as zeros.)

// The sums of the wavefronts of 16 rows, times `by`, to the rows' places.
template <typename T, int HDP, int W, typename RowOf>
__device__ __forceinline__ void write_sums(const T (&sums)[W][16 * (HDP + 16 / sizeof(T))], int here, int head_dim, T by, RowOf row_of) {
    constexpr int VEC = 16 / sizeof(T), PITCH = HDP + VEC;
    for (int at = threadIdx.x; at < here * (HDP / VEC); at += 64 * W) {
        const int row = at / (HDP / VEC), d = at % (HDP / VEC) * VEC;
        if (d >= head_dim) continue;
        T sum[VEC];
#pragma unroll
        for (int t = 0; t < VEC; ++t) sum[t] = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const Pack<T, VEC> e = *reinterpret_cast<const Pack<T, VEC>*>(&sums[w][row * PITCH + d]);
#pragma unroll
            for (int t = 0; t < VEC; ++t) sum[t] += e.v[t];
        }
        T* __restrict__ dst = row_of(row);
#pragma unroll
        for (int t = 0; t < VEC; ++t)
            if (d + t < head_dim) dst[d + t] = sum[t] * by;
    }
}

// Gradient of Q: 16 packed rows against the keys that they see.  Writes D = rowsum(dO (.) O) for the other kernel.  Bound by the
// latency of a tile (the batch of doubles above: 22 us, 2.3 us a tile).
template <typename T, int HDP, bool ALIGNED>
__global__ void __launch_bounds__(64 * WAVES) causal_bwd_q_kernel(const CausalArgs<T> p, uint32_t units) {
    constexpr int VEC = 16 / sizeof(T), CHUNKS = HDP / (4 * VEC), NY = HDP / 16, N = columns_at_once<T, HDP>(), PITCH = HDP + VEC;
    typedef typename Num<T>::Acc Acc;
    __shared__ __attribute__((aligned(16))) T sums[WAVES][16 * PITCH];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const uint32_t stride = gridDim.x / p.kv_heads;
    const int kv = (int)(blockIdx.x % p.kv_heads);
    const T factor = p.scale * Num<T>::unit();
    for (uint32_t unit = blockIdx.x / p.kv_heads; unit < units; unit += stride) {
        Span sp;
        uint32_t inside;
        if (!find_tile(p, p.group, unit, lane, &sp, &inside)) continue;
        const uint32_t rows = (uint32_t)sp.nq * (uint32_t)p.group, row0 = inside * 16;
        const uint32_t r = row0 + li < rows ? row0 + li : rows - 1;
        const uint32_t first_token = row0 / p.group, ahead = (row0 % p.group + (r - row0)) / p.group, last = first_token + ahead;
        const int64_t token = sp.q0 + last;
        const int head = kv * p.group + (int)(r - last * p.group);
        const int64_t at = head * p.q_rows + token, col = head * (int64_t)p.head_dim;
        Pack<T, VEC> q[CHUNKS], go[CHUNKS];
        load_along<T, HDP, ALIGNED>(p.Q + token * p.ldq + col, g, p.head_dim, q);
        load_along<T, HDP, ALIGNED>(p.dO + token * p.ldo + col, g, p.head_dim, go);
        T lse = p.lse[at] * Num<T>::unit(), dot = 0;
        {
            Pack<T, VEC> o[CHUNKS];
            load_along<T, HDP, ALIGNED>(p.O + token * p.ldo + col, g, p.head_dim, o);
            zero_past<T, HDP>(g, p.head_dim, o);
            zero_past<T, HDP>(g, p.head_dim, go);
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                for (int t = 0; t < VEC; ++t) dot = fma(go[c].v[t], o[c].v[t], dot);
            dot += __shfl_xor(dot, 16, 64);
            dot += __shfl_xor(dot, 32, 64);
            dot = is_finite(dot) ? dot : nan_of<T>();
            lse += dot - dot;  // NaN where D is
        }
        if (wave == 0 && g == 0 && row0 + li < rows) p.D[at] = dot;
        zero_past<T, HDP>(g, p.head_dim, q);
        const uint32_t seen = first_token + (uint32_t)__builtin_amdgcn_readlane(ahead, 15) + 1;  // (of nk = nq keys)
        const T* __restrict__ K = p.K + sp.k0 * p.ldk + kv * (int64_t)p.head_dim;
        const T* __restrict__ V = p.V + sp.k0 * p.ldv + kv * (int64_t)p.head_dim;
        Acc dq[NY];
#pragma unroll
        for (int y = 0; y < NY; ++y) dq[y] = Acc{0, 0, 0, 0};
        for (uint32_t k0 = 16 * wave; k0 < seen; k0 += 16 * WAVES) {
            const uint32_t most = seen - 1 - k0;
            const int64_t key = k0 + (li < most ? li : most);
            Pack<T, VEC> k[CHUNKS], v[CHUNKS];
            Pack<T, N> across[4][NY / N];
            load_along<T, HDP, ALIGNED>(K + key * p.ldk, g, p.head_dim, k);
            load_along<T, HDP, ALIGNED>(V + key * p.ldv, g, p.head_dim, v);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const uint32_t j = Num<T>::row(x, g);
                load_across<T, HDP, ALIGNED>(K + (int64_t)(k0 + (j < most ? j : most)) * p.ldk, li, p.head_dim, across[x]);
            }
            const Acc s = product<T>(k, q), dp = product<T>(v, go);
            Acc ds;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const T w = Num<T>::exp_unit(s[x] * factor - lse);
                ds[x] = k0 + Num<T>::row(x, g) <= last ? w * (dp[x] - dot) : (T)0;
            }
            zero_bad<T>(across);
            add_weighted<T>(across, ds, dq);
        }
        put_sums<T, N, NY, PITCH>(dq, li, g, sums[wave]);
        __syncthreads();
        write_sums<T, HDP, WAVES>(sums, (int)(rows - row0 < 16 ? rows - row0 : 16), p.head_dim, p.scale, [&](int row) {
            const uint32_t to = first_token + (row0 % p.group + row) / p.group;
            return p.dQ + (sp.q0 + to) * p.lddq + (kv * p.group + (int)(row0 + row - to * p.group)) * (int64_t)p.head_dim;
        });
        __syncthreads();
    }
}

// Gradients of K and V: 16 keys against the packed rows that see them, all heads of the group among them.  As above: 35 us, 8
// tiles of rows to a wavefront at most.  Reading a tile ahead in these two was measured: up to 16 % faster on sequences from
// 512 on, as much slower on many short ones, whose registers then let fewer wavefronts run; it was left out.
template <typename T, int HDP, bool ALIGNED, int W>
__global__ void __launch_bounds__(64 * W) causal_bwd_kv_kernel(const CausalArgs<T> p, uint32_t units) {
    constexpr int VEC = 16 / sizeof(T), CHUNKS = HDP / (4 * VEC), NY = HDP / 16, N = columns_at_once<T, HDP>(), PITCH = HDP + VEC;
    typedef typename Num<T>::Acc Acc;
    __shared__ __attribute__((aligned(16))) T sums[W][16 * PITCH];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const uint32_t stride = gridDim.x / p.kv_heads, group = p.group, inverse = inverse_of(group);
    const int kv = (int)(blockIdx.x % p.kv_heads);
    const T factor = p.scale * Num<T>::unit();
    for (uint32_t unit = blockIdx.x / p.kv_heads; unit < units; unit += stride) {
        Span sp;
        uint32_t inside;
        if (!find_tile(p, 1, unit, lane, &sp, &inside)) continue;
        const uint32_t keys = (uint32_t)sp.nk, rows = keys * group, key0 = inside * 16;
        const uint32_t key = key0 + li < keys ? key0 + li : keys - 1;
        Pack<T, VEC> k[CHUNKS], v[CHUNKS];
        load_along<T, HDP, ALIGNED>(p.K + (sp.k0 + key) * p.ldk + kv * (int64_t)p.head_dim, g, p.head_dim, k);
        load_along<T, HDP, ALIGNED>(p.V + (sp.k0 + key) * p.ldv + kv * (int64_t)p.head_dim, g, p.head_dim, v);
        zero_past<T, HDP>(g, p.head_dim, k);
        zero_past<T, HDP>(g, p.head_dim, v);
        Acc dk[NY], dv[NY];
#pragma unroll
        for (int y = 0; y < NY; ++y) dk[y] = dv[y] = Acc{0, 0, 0, 0};
        const T* __restrict__ Q = p.Q + sp.q0 * p.ldq + kv * (int64_t)group * p.head_dim;
        const T* __restrict__ G = p.dO + sp.q0 * p.ldo + kv * (int64_t)group * p.head_dim;
        const T* __restrict__ lses = p.lse + kv * (int64_t)group * p.q_rows + sp.q0;
        const T* __restrict__ dots = p.D + kv * (int64_t)group * p.q_rows + sp.q0;
        for (uint32_t r0 = key0 * group / 16 * 16 + 16 * wave; r0 < rows; r0 += 16 * W) {
            const uint32_t most = rows - 1 - r0, token0 = r0 / group, rest0 = r0 - token0 * group;
            Pack<T, VEC> q[CHUNKS], go[CHUNKS];
            Pack<T, N> q_across[4][NY / N], g_across[4][NY / N];
            {
                const uint32_t i = rest0 + (li < most ? li : most), ahead = heads_over(i, group, inverse);
                const int64_t token = token0 + ahead, col = (int64_t)(i - ahead * group) * p.head_dim;
                load_along<T, HDP, ALIGNED>(Q + token * p.ldq + col, g, p.head_dim, q);
                load_along<T, HDP, ALIGNED>(G + token * p.ldo + col, g, p.head_dim, go);
            }
            uint32_t sees[4];
            T lse[4], dot[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const uint32_t j = Num<T>::row(x, g), i = rest0 + (j < most ? j : most), ahead = heads_over(i, group, inverse);
                const int64_t token = token0 + ahead;
                const uint32_t head = i - ahead * group;
                load_across<T, HDP, ALIGNED>(Q + token * p.ldq + (int64_t)head * p.head_dim, li, p.head_dim, q_across[x]);
                load_across<T, HDP, ALIGNED>(G + token * p.ldo + (int64_t)head * p.head_dim, li, p.head_dim, g_across[x]);
                lse[x] = lses[head * p.q_rows + token];
                dot[x] = dots[head * p.q_rows + token];
                sees[x] = j <= most ? token0 + ahead + 1 : 0;  // how many keys the row sees
            }
            const Acc s = product<T>(q, k), dp = product<T>(go, v);  // rows are packed rows, columns keys
            Acc w, ds;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const T e = Num<T>::exp_unit(s[x] * factor - (lse[x] * Num<T>::unit() + (dot[x] - dot[x])));
                w[x] = key < sees[x] ? e : (T)0;
                ds[x] = key < sees[x] ? e * (dp[x] - dot[x]) : (T)0;
            }
            zero_bad<T>(g_across);
            add_weighted<T>(g_across, w, dv);
            zero_bad<T>(q_across);
            add_weighted<T>(q_across, ds, dk);
        }
        const int here = (int)(keys - key0 < 16 ? keys - key0 : 16);
        put_sums<T, N, NY, PITCH>(dv, li, g, sums[wave]);
        __syncthreads();
        write_sums<T, HDP, W>(sums, here, p.head_dim, (T)1, [&](int row) { return p.dV + (sp.k0 + key0 + row) * p.lddv + kv * (int64_t)p.head_dim; });
        __syncthreads();
        put_sums<T, N, NY, PITCH>(dk, li, g, sums[wave]);
        __syncthreads();
        write_sums<T, HDP, W>(sums, here, p.head_dim, p.scale, [&](int row) { return p.dK + (sp.k0 + key0 + row) * p.lddk + kv * (int64_t)p.head_dim; });
        __syncthreads();
    }
}

inline int64_t tile_slots(int64_t rows, int64_t group, int64_t sequences) { return rows * group / 16 + sequences; }

// Parts of a sequence's keys: one where a cache is short, no more than a lane each, and few enough that rows with many
// units do not need a large workspace.
template <typename T>
int most_parts(const CausalArgs<T>& a) {
    if (a.k_rows <= WHOLE_KEYS) return 1;
    const int64_t units = tile_slots(a.q_rows, a.group, a.sequences) * a.kv_heads;
    return (int)std::max<int64_t>(1, std::min<int64_t>({64, (a.k_rows + LEAST_KEYS - 1) / LEAST_KEYS, 8 * RUNNING / units}));
}

}  // namespace

// A launch of KERNEL<T, HDP, ALIGNED, ...> for the smallest padded head dimension that holds head_dim.
#define BY_HEAD_DIM(KERNEL, GROUPS, ARGS, ...)                                                                       \
    do {                                                                                                                \
        const dim3 grid((unsigned)(GROUPS)), block(64 * WAVES);                                                         \
        if (a.head_dim <= 32) hipLaunchKernelGGL((KERNEL<T, 32, __VA_ARGS__>), grid, block, 0, s, UNPACKED ARGS);       \
        else if (a.head_dim <= 64) hipLaunchKernelGGL((KERNEL<T, 64, __VA_ARGS__>), grid, block, 0, s, UNPACKED ARGS);  \
        else hipLaunchKernelGGL((KERNEL<T, 128, __VA_ARGS__>), grid, block, 0, s, UNPACKED ARGS);                       \
        if (hipError_t e = hipGetLastError()) return e;                                                                 \
    } while (0)
// With MANY_WAVES, for head dimensions of up to 256 bytes: more would not leave each wavefront the registers of a tile.
#define BY_HEAD_DIM_MANY(KERNEL, GROUPS, ARGS, ...)                                                                              \
    do {                                                                                                                         \
        const dim3 grid((unsigned)(GROUPS)), block(64 * MANY_WAVES);                                                             \
        if (a.head_dim <= 32) hipLaunchKernelGGL((KERNEL<T, 32, __VA_ARGS__, MANY_WAVES>), grid, block, 0, s, UNPACKED ARGS);    \
        else hipLaunchKernelGGL((KERNEL<T, 256 / sizeof(T), __VA_ARGS__, MANY_WAVES>), grid, block, 0, s, UNPACKED ARGS);        \
        if (hipError_t e = hipGetLastError()) return e;                                                                          \
    } while (0)
#define UNPACKED(...) __VA_ARGS__

// Workgroups for `tiles` units of every key/value head: one each, of very many some take several.
static int64_t workgroups(int64_t tiles, int64_t most, int64_t kv_heads) { return std::min(tiles, std::max<int64_t>(1, most / kv_heads)) * kv_heads; }
constexpr int64_t MOST_GROUPS = 1 << 20;

template <typename T, bool CUT>
static hipError_t launch_attention(const CausalArgs<T>& a, const Parts<T>& cut, int64_t most, hipStream_t s) {
    const int64_t groups = workgroups(cut.units, most, a.kv_heads);
    // No more units than compute units, of many keys: eight wavefronts each.  One token against 300 keys, 8 heads on 2 of 64, 9.7 us
    // for 10.2; 1024 tokens, 2 heads of 64, 19.1 for 21.3; level up to 256 keys, and for heads of 128; slower in double (four
    // sequences of doubles, forward, 23 for 21).
    if constexpr (!CUT && sizeof(T) == 4) {
        if (a.vec_q && a.vec_kv && a.head_dim <= 64 && groups <= RUNNING / 2 && a.k_rows > (int64_t)256 * a.sequences) {
            BY_HEAD_DIM_MANY(attention_kernel, groups, (a, cut), true, CUT);
            return hipSuccess;
        }
    }
    if (a.vec_q && a.vec_kv) BY_HEAD_DIM(attention_kernel, groups, (a, cut), true, CUT, WAVES);
    else BY_HEAD_DIM(attention_kernel, groups, (a, cut), false, CUT, WAVES);
    return hipSuccess;
}

template <typename T>
hipError_t launch_causal_fwd(const CausalArgs<T>& a, hipStream_t s) {
    return launch_attention<T, false>(a, {(uint32_t)tile_slots(a.q_rows, a.group, a.sequences), 1, nullptr, nullptr, nullptr}, MOST_GROUPS, s);
}

template <typename T>
size_t causal_bwd_workspace_bytes(const CausalArgs<T>& a) {
    return (size_t)a.heads * a.q_rows * sizeof(T);
}

template <typename T>
hipError_t launch_causal_bwd(CausalArgs<T> a, void* workspace, hipStream_t s) {
    a.D = static_cast<T*>(workspace);
    const int64_t tiles = tile_slots(a.q_rows, a.group, a.sequences), key_tiles = tile_slots(a.q_rows, 1, a.sequences);
    const int64_t groups = workgroups(tiles, MOST_GROUPS, a.kv_heads), key_groups = workgroups(key_tiles, MOST_GROUPS, a.kv_heads);
    const bool aligned = a.vec_q && a.vec_kv && a.vec_o;
    if (aligned) BY_HEAD_DIM(causal_bwd_q_kernel, groups, (a, (uint32_t)tiles), true);
    else BY_HEAD_DIM(causal_bwd_q_kernel, groups, (a, (uint32_t)tiles), false);
    // Few units of long walks: eight wavefronts each.  With the kernel above, the four sequences of doubles 56 us for 65; 1024
    // doubles, 8 heads of 32, 80 for 88; 700 floats, 8 heads on 2 of 32, 64 for 77; 800, 4 heads of 64, 50 for 53.  Beyond these
    // bounds: two sequences of 1024 doubles 150 for 137, ten of 100 39 for 28, eight of 64, 16 heads on 4 of 64 floats, 25 for
    // 23.  (The kernel above has nothing from it.)
    if (aligned && a.head_dim * sizeof(T) <= 256 && a.q_rows * a.kv_heads <= 16 * RUNNING && a.q_rows * a.group > (int64_t)256 * a.sequences)
        BY_HEAD_DIM_MANY(causal_bwd_kv_kernel, key_groups, (a, (uint32_t)key_tiles), true);
    else if (aligned) BY_HEAD_DIM(causal_bwd_kv_kernel, key_groups, (a, (uint32_t)key_tiles), true, WAVES);
    else BY_HEAD_DIM(causal_bwd_kv_kernel, key_groups, (a, (uint32_t)key_tiles), false, WAVES);
    return hipSuccess;
}

template <typename T>
size_t cached_workspace_bytes(const CausalArgs<T>& a) {
    const int parts = most_parts(a);
    return parts == 1 ? 0 : 16 + (size_t)a.q_rows * a.heads * parts * (a.head_dim + 2) * sizeof(T);
}

template <typename T>
hipError_t launch_cached_attention(const CausalArgs<T>& a, void* workspace, hipStream_t s) {
    Parts<T> cut;
    cut.most = most_parts(a);
    cut.keys = static_cast<int32_t*>(workspace);
    cut.data = static_cast<T*>(workspace) + 16 / sizeof(T);
    cut.stat = cut.data + a.q_rows * a.heads * (int64_t)cut.most * a.head_dim;
    const int64_t tiles = tile_slots(a.q_rows, a.group, a.sequences);
    cut.units = (uint32_t)(tiles * cut.most);
    if (cut.most == 1) return launch_attention<T, false>(a, cut, MOST_GROUPS, s);
    // where the units run at once there are no more than that of them
    if (hipError_t e = launch_attention<T, true>(a, cut, tiles * a.kv_heads <= RUNNING / 2 ? RUNNING : 4 * RUNNING, s)) return e;
    hipLaunchKernelGGL(cached_join_kernel<T>, dim3((unsigned)(a.q_rows * a.heads)), dim3(64 * WAVES), 0, s, a, cut);
    return hipGetLastError();
}

#define INSTANTIATE(T)                                                              \
    template hipError_t launch_causal_fwd<T>(const CausalArgs<T>&, hipStream_t);    \
    template size_t causal_bwd_workspace_bytes<T>(const CausalArgs<T>&);            \
    template hipError_t launch_causal_bwd<T>(CausalArgs<T>, void*, hipStream_t);    \
    template size_t cached_workspace_bytes<T>(const CausalArgs<T>&);                \
    template hipError_t launch_cached_attention<T>(const CausalArgs<T>&, void*, hipStream_t);
INSTANTIATE(float)
INSTANTIATE(double)
#undef INSTANTIATE

}  // namespace prad
