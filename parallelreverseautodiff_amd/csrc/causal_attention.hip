// Causal attention over packed sequences with grouped heads, in either element type, and its form for the newest tokens of a
// sequence against its cache.
//
//   S = scale Q K^T,  key j seen by query i of n (keys: m) iff j <= m - n + i,  P = softmax rows(S),  O = P V,  lse = log sum exp S
//   D = rowsum(dO (.) O),  P = exp(S - lse),  dV = P^T dO,  dS = P (.) (dO V^T - D),  dQ = scale dS K,  dK = scale dS^T Q
//
// One pass over the keys with the running maximum and sum of a row: scores never reach memory.  The rows of a tile are
// (token, head of the group) pairs - token r / group, head r % group - so the query heads that share a key/value head share its
// tiles, and their gradients of K and V add up in one workgroup's registers in one order.
// Statistics and sums are held in the element type (32 or 64 bits); products run on the 16 x 16 x 4 matrix instructions, whose
// element order along the reduction is free as long as both operands agree: lane group g takes elements CH c + VEC g + t of
// chunk c, which makes its reads whole 16-byte vectors.
//
// Non-finite values.  A key row that holds one (in K or V) is staged as zeros and its scores become NaN where they are seen: a
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

__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Reductions over the 16 lanes that share a lane group (a row of an accumulator).
template <typename T> __device__ __forceinline__ T max16(T v) {
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) v = fmax(v, __shfl_xor(v, m, 64));
    return v;
}
template <typename T> __device__ __forceinline__ T sum16(T v) {
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) v += __shfl_xor(v, m, 64);
    return v;
}

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

// Tiles of R packed rows are numbered through all sequences without a table: sequence s begins at number
// floor(offset G / R) + s, which leaves room for its ceil(n G / R) tiles.  Finds the sequence of a tile and the tile's number
// inside it; false: no such tile.
template <int R, typename T>
__device__ __forceinline__ bool find_tile(const CausalArgs<T>& p, int group, int64_t tile, int* sequence, int64_t* inside) {
    int lo = 0, hi = p.sequences;  // the last s whose first tile is not behind `tile` lies in [lo - 1, hi)
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (clamped(p.q_off[mid], p.q_rows) * group / R + mid <= tile) lo = mid + 1;
        else hi = mid;
    }
    if (lo == 0) return false;
    *sequence = lo - 1;
    *inside = tile - (clamped(p.q_off[lo - 1], p.q_rows) * group / R + (lo - 1));
    return true;
}

// Elements [d0, d0 + VEC) of a row of head_dim elements, zeros past it.
template <typename T>
__device__ __forceinline__ Pack<T, 16 / sizeof(T)> load_pack(const T* __restrict__ row, int d0, int head_dim, bool vec) {
    constexpr int VEC = 16 / sizeof(T);
    Pack<T, VEC> v;
#pragma unroll
    for (int t = 0; t < VEC; ++t) v.v[t] = (T)0;
    if (vec) {
        if (d0 < head_dim) v = *reinterpret_cast<const Pack<T, VEC>*>(row + d0);
    } else {
#pragma unroll
        for (int t = 0; t < VEC; ++t)
            if (d0 + t < head_dim) v.v[t] = row[d0 + t];
    }
    return v;
}

// A row as the A operand of the matrix instructions: frag[c][t] = element CH c + VEC g + t.
template <typename T, int HDP>
__device__ __forceinline__ void load_row(const T* __restrict__ row, int g, int head_dim, bool vec, Pack<T, 16 / sizeof(T)> (&frag)[HDP / (64 / sizeof(T))]) {
    constexpr int VEC = 16 / sizeof(T), CH = 4 * VEC;
#pragma unroll
    for (int c = 0; c < HDP / CH; ++c) {
        if (row != nullptr) {
            frag[c] = load_pack(row, CH * c + VEC * g, head_dim, vec);
        } else {
#pragma unroll
            for (int t = 0; t < VEC; ++t) frag[c].v[t] = (T)0;
        }
    }
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

// Stages two tiles of ROWS rows (of K and V, or of Q and dO) by 256 threads.  row_of(j, which) is the address of row j, nullptr
// for a row that is not there: zeros.  A row with a non-finite value in either tile is staged as zeros in that tile and marked
// with `tag`.
template <typename T, int HDP, int ROWS, int PITCH, typename RowOf>
__device__ __forceinline__ void stage_two(T* __restrict__ first, T* __restrict__ second, int* __restrict__ bad, int tag, int head_dim, bool vec, RowOf row_of) {
    constexpr int VEC = 16 / sizeof(T), PER_ROW = HDP / VEC, COUNT = ROWS * PER_ROW / 256;
    static_assert(ROWS * PER_ROW % 256 == 0, "whole rounds");
    Pack<T, VEC> v[2][COUNT];
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int u = 0; u < COUNT; ++u) {
            const int at = threadIdx.x + 256 * u, j = at / PER_ROW, d = (at % PER_ROW) * VEC;
            const T* __restrict__ row = row_of(j, which);
            if (row != nullptr) {
                v[which][u] = load_pack(row, d, head_dim, vec);
            } else {
#pragma unroll
                for (int t = 0; t < VEC; ++t) v[which][u].v[t] = (T)0;
            }
        }
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int u = 0; u < COUNT; ++u) {
            const int at = threadIdx.x + 256 * u, j = at / PER_ROW, d = (at % PER_ROW) * VEC;
            bool fine = true;
#pragma unroll
            for (int t = 0; t < VEC; ++t) fine = fine && is_finite(v[which][u].v[t]);
            if (!fine) {
                bad[j] = tag;
#pragma unroll
                for (int t = 0; t < VEC; ++t) v[which][u].v[t] = is_finite(v[which][u].v[t]) ? v[which][u].v[t] : (T)0;
            }
            *reinterpret_cast<Pack<T, VEC>*>((which == 0 ? first : second) + j * PITCH + d) = v[which][u];
        }
}

// C[16 x 16 y] = A . B^T over the head dimension: A fragments in registers, rows 16 y + li of a staged tile.
template <typename T, int HDP, int PITCH, int NY>
__device__ __forceinline__ void rows_product(const Pack<T, 16 / sizeof(T)> (&a)[HDP / (64 / sizeof(T))], const T* __restrict__ tile, int li, int g,
                                             typename Num<T>::Acc (&acc)[NY]) {
    constexpr int VEC = 16 / sizeof(T), CH = 4 * VEC;
#pragma unroll
    for (int y = 0; y < NY; ++y) acc[y] = typename Num<T>::Acc{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < HDP / CH; ++c) {
        Pack<T, VEC> b[NY];
#pragma unroll
        for (int y = 0; y < NY; ++y) b[y] = *reinterpret_cast<const Pack<T, VEC>*>(tile + (16 * y + li) * PITCH + CH * c + VEC * g);
#pragma unroll
        for (int t = 0; t < VEC; ++t)
#pragma unroll
            for (int y = 0; y < NY; ++y) acc[y] = Num<T>::mfma(a[c].v[t], b[y].v[t], acc[y]);
    }
}

// out[16 x HDP] += W . X: weights of 16 rows over COLS columns in the wavefront's tile w, staged rows of X.
template <typename T, int HDP, int COLS, int WPITCH, int PITCH>
__device__ __forceinline__ void weights_product(const T* __restrict__ w, const T* __restrict__ x, int li, int g, typename Num<T>::Acc (&out)[HDP / 16]) {
    constexpr int VEC = 16 / sizeof(T), CH = 4 * VEC;
#pragma unroll
    for (int c = 0; c < COLS / CH; ++c) {
        const Pack<T, VEC> a = *reinterpret_cast<const Pack<T, VEC>*>(w + li * WPITCH + CH * c + VEC * g);
#pragma unroll
        for (int t = 0; t < VEC; ++t)
#pragma unroll
            for (int y = 0; y < HDP / 16; ++y) out[y] = Num<T>::mfma(a.v[t], x[(CH * c + VEC * g + t) * PITCH + 16 * y + li], out[y]);
    }
}

// Columns of a tile and the pitches of the staged tiles: a 16-byte pad spreads the rows over the LDS banks.
template <typename T, int HDP> struct Tile {
    static constexpr int VEC = 16 / sizeof(T);
    static constexpr int COLS = sizeof(T) * HDP > 512 ? 16 : 32;
    static constexpr int PITCH = HDP + VEC, WPITCH = COLS + VEC, NY = COLS / 16;
};

// Running softmax statistics of the four rows a lane holds, over one tile of scores.  On return s holds the weights and the
// factors of the old sums.
template <typename T, int NY>
__device__ __forceinline__ void softmax_tile(typename Num<T>::Acc (&s)[NY], T (&m)[4], T (&l)[4], T (&factor)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        T top = s[0][r];
#pragma unroll
        for (int y = 1; y < NY; ++y) top = fmax(top, s[y][r]);
        top = fmax(m[r], max16(top));
        const T ref = top == -(T)INFINITY ? (T)0 : top;  // nothing seen yet: every weight below is exp(-inf) = 0
        factor[r] = Num<T>::exp_unit(m[r] - ref);
        T sum = 0;
#pragma unroll
        for (int y = 0; y < NY; ++y) {
            s[y][r] = Num<T>::exp_unit(s[y][r] - ref);
            sum += s[y][r];
        }
        l[r] = l[r] * factor[r] + sum16(sum);
        m[r] = top;
    }
}

// ---- forward ------------------------------------------------------------------------------------------------------------
// A workgroup takes 64 packed rows of a key/value head, a wavefront 16 of them; K and V pass through LDS in tiles of COLS keys.
template <typename T, int HDP>
__global__ void __launch_bounds__(256) causal_fwd_kernel(const CausalArgs<T> p) {
    typedef Tile<T, HDP> TL;
    typedef typename Num<T>::Acc Acc;
    constexpr int CHUNKS = HDP / (4 * TL::VEC);
    __shared__ __attribute__((aligned(16))) T ks[TL::COLS * TL::PITCH], vs[TL::COLS * TL::PITCH], ws[4][16 * TL::WPITCH];
    __shared__ int bad[TL::COLS];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int kv = blockIdx.y;
    int s;
    int64_t inside;
    if (!find_tile<64>(p, p.group, (int64_t)gridDim.x - 1 - blockIdx.x, &s, &inside)) return;  // (late tiles see the most keys: first)
    const Span sp = span_of(p, s);
    const int64_t rows = sp.nq * p.group, row0 = inside * 64;
    if (row0 >= rows) return;
    if (threadIdx.x < TL::COLS) bad[threadIdx.x] = -1;
    const int64_t lead = sp.nk - sp.nq;  // query i sees keys up to lead + i
    Pack<T, TL::VEC> q[CHUNKS];
    {
        const int64_t r = row0 + 16 * wave + li;
        const T* row = r < rows ? p.Q + (sp.q0 + r / p.group) * p.ldq + (kv * p.group + r % p.group) * (int64_t)p.head_dim : nullptr;
        load_row<T, HDP>(row, g, p.head_dim, p.vec_q, q);
        poison_row<T, CHUNKS>(q);
    }
    int64_t last[4];  // the last key that each of the lane's rows sees
#pragma unroll
    for (int r = 0; r < 4; ++r) last[r] = lead + (row0 + 16 * wave + Num<T>::row(r, g)) / p.group;
    T m[4], l[4];
    Acc o[HDP / 16];
#pragma unroll
    for (int r = 0; r < 4; ++r) { m[r] = -(T)INFINITY; l[r] = 0; }
#pragma unroll
    for (int y = 0; y < HDP / 16; ++y) o[y] = Acc{0, 0, 0, 0};
    const int64_t last_row = row0 + 63 < rows ? row0 + 63 : rows - 1;
    const int64_t seen = clamped(lead + last_row / p.group + 1, sp.nk);
    const T factor = p.scale * Num<T>::unit();
    const T* __restrict__ K = p.K + sp.k0 * p.ldk + kv * (int64_t)p.head_dim;
    const T* __restrict__ V = p.V + sp.k0 * p.ldv + kv * (int64_t)p.head_dim;
    for (int64_t k0 = 0; k0 < seen; k0 += TL::COLS) {
        const int tag = (int)(k0 / TL::COLS);
        __syncthreads();
        stage_two<T, HDP, TL::COLS, TL::PITCH>(ks, vs, bad, tag, p.head_dim, p.vec_kv, [&](int j, int which) -> const T* {
            if (k0 + j >= sp.nk) return nullptr;
            return which == 0 ? K + (k0 + j) * p.ldk : V + (k0 + j) * p.ldv;
        });
        __syncthreads();
        Acc acc[TL::NY];
        rows_product<T, HDP, TL::PITCH, TL::NY>(q, ks, li, g, acc);
#pragma unroll
        for (int y = 0; y < TL::NY; ++y) {
            const int64_t j = k0 + 16 * y + li;
            const bool poisoned = bad[16 * y + li] == tag;
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[y][r] = j > last[r] ? -(T)INFINITY : poisoned ? nan_of<T>() : acc[y][r] * factor;
        }
        T fac[4];
        softmax_tile<T, TL::NY>(acc, m, l, fac);
#pragma unroll
        for (int y = 0; y < HDP / 16; ++y)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[y][r] *= fac[r];
#pragma unroll
        for (int y = 0; y < TL::NY; ++y)
#pragma unroll
            for (int r = 0; r < 4; ++r) ws[wave][Num<T>::row(r, g) * TL::WPITCH + 16 * y + li] = acc[y][r];
        wave_sync();
        weights_product<T, HDP, TL::COLS, TL::WPITCH, TL::PITCH>(ws[wave], vs, li, g, o);
        wave_sync();
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int64_t row = row0 + 16 * wave + Num<T>::row(r, g);
        if (row >= rows) continue;
        const int64_t token = sp.q0 + row / p.group;
        const int head = kv * p.group + (int)(row % p.group);
        const bool any = last[r] >= 0;
        const T inv = any ? (T)1 / l[r] : (T)0;
        T* dst = p.O + token * p.ldo + head * (int64_t)p.head_dim;
#pragma unroll
        for (int y = 0; y < HDP / 16; ++y)
            if (16 * y + li < p.head_dim) dst[16 * y + li] = any ? o[y][r] * inv : (T)0;
        if (p.lse != nullptr && li == 0) p.lse[head * p.q_rows + token] = any ? Num<T>::log_sum(m[r], l[r]) : -(T)INFINITY;
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------------
// D = rowsum(dO (.) O) per token and head, 16 lanes to a row; NaN for a row of dO with a non-finite value.
template <typename T>
__global__ void __launch_bounds__(256) causal_dot_kernel(const CausalArgs<T> p) {
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4;
    const int lane = threadIdx.x & 15;
    if (at >= p.q_rows * p.heads) return;
    const int64_t token = at / p.heads;
    const int head = (int)(at % p.heads);
    const T* __restrict__ o = p.O + token * p.ldo + head * (int64_t)p.head_dim;
    const T* __restrict__ g = p.dO + token * p.ldo + head * (int64_t)p.head_dim;
    T sum = 0, check = 0;
    for (int d = lane; d < p.head_dim; d += 16) {
        sum += o[d] * g[d];
        check += is_finite(g[d]) ? (T)0 : nan_of<T>();
    }
    sum = sum16(sum + check);
    if (lane == 0) p.D[head * p.q_rows + token] = is_finite(sum) ? sum : nan_of<T>();
}

// Gradients of K and V: a workgroup owns 64 keys of a key/value head (a wavefront 16, its rows of K and V in registers) and
// walks the packed query rows that see them, all heads of the group among them, in tiles of COLS.
template <typename T, int HDP>
__global__ void __launch_bounds__(256) causal_bwd_kv_kernel(const CausalArgs<T> p) {
    typedef Tile<T, HDP> TL;
    typedef typename Num<T>::Acc Acc;
    constexpr int CHUNKS = HDP / (4 * TL::VEC);
    __shared__ __attribute__((aligned(16))) T qs[TL::COLS * TL::PITCH], gs[TL::COLS * TL::PITCH], ws[4][16 * TL::WPITCH];
    __shared__ T row_lse[TL::COLS], row_dot[TL::COLS];
    __shared__ int bad[TL::COLS];  // written by the staging; rows with a non-finite value already have a NaN in lse or D
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int kv = blockIdx.y;
    int s;
    int64_t inside;
    if (!find_tile<64>(p, 1, blockIdx.x, &s, &inside)) return;  // (tiles of keys are numbered like packed rows of one head)
    const Span sp = span_of(p, s);
    const int64_t key0 = inside * 64, rows = sp.nq * p.group;
    if (key0 >= sp.nk) return;
    const int64_t key = key0 + 16 * wave + li;
    Pack<T, TL::VEC> k[CHUNKS], v[CHUNKS];
    load_row<T, HDP>(key < sp.nk ? p.K + (sp.k0 + key) * p.ldk + kv * (int64_t)p.head_dim : nullptr, g, p.head_dim, p.vec_kv, k);
    load_row<T, HDP>(key < sp.nk ? p.V + (sp.k0 + key) * p.ldv + kv * (int64_t)p.head_dim : nullptr, g, p.head_dim, p.vec_kv, v);
    Acc dk[HDP / 16], dv[HDP / 16];
#pragma unroll
    for (int y = 0; y < HDP / 16; ++y) dk[y] = dv[y] = Acc{0, 0, 0, 0};
    const T factor = p.scale * Num<T>::unit();
    // (queries and keys are the same rows here: token i sees key j iff j <= i)
    for (int64_t r0 = key0 * p.group / TL::COLS * TL::COLS; r0 < rows; r0 += TL::COLS) {
        __syncthreads();
        if (threadIdx.x < TL::COLS) {
            const int64_t r = r0 + threadIdx.x;
            T lse = 0, dot = 0;
            if (r < rows) {
                const int64_t at = (kv * p.group + r % p.group) * p.q_rows + sp.q0 + r / p.group;
                dot = p.D[at];
                lse = p.lse[at] * Num<T>::unit() + (dot - dot);  // NaN where D is
            }
            row_lse[threadIdx.x] = lse;
            row_dot[threadIdx.x] = dot;
        }
        stage_two<T, HDP, TL::COLS, TL::PITCH>(qs, gs, bad, 0, p.head_dim, p.vec_q && p.vec_o, [&](int j, int which) -> const T* {
            const int64_t r = r0 + j;
            if (r >= rows) return nullptr;
            const int64_t token = sp.q0 + r / p.group, col = (kv * p.group + r % p.group) * (int64_t)p.head_dim;
            return which == 0 ? p.Q + token * p.ldq + col : p.dO + token * p.ldo + col;
        });
        __syncthreads();
        Acc st[TL::NY], dp[TL::NY];
        rows_product<T, HDP, TL::PITCH, TL::NY>(k, qs, li, g, st);   // S^T: rows are keys, columns query rows
        rows_product<T, HDP, TL::PITCH, TL::NY>(v, gs, li, g, dp);   // (dO V^T)^T
#pragma unroll
        for (int y = 0; y < TL::NY; ++y) {
            const int64_t r = r0 + 16 * y + li, token = r / p.group;
            const T lse = row_lse[16 * y + li], dot = row_dot[16 * y + li];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool seen = r < rows && key0 + 16 * wave + Num<T>::row(e, g) <= token;
                const T w = seen ? Num<T>::exp_unit(st[y][e] * factor - lse) : (T)0;
                st[y][e] = w;
                dp[y][e] = seen ? w * (dp[y][e] - dot) : (T)0;
            }
        }
#pragma unroll
        for (int y = 0; y < TL::NY; ++y)
#pragma unroll
            for (int e = 0; e < 4; ++e) ws[wave][Num<T>::row(e, g) * TL::WPITCH + 16 * y + li] = st[y][e];
        wave_sync();
        weights_product<T, HDP, TL::COLS, TL::WPITCH, TL::PITCH>(ws[wave], gs, li, g, dv);
        wave_sync();
#pragma unroll
        for (int y = 0; y < TL::NY; ++y)
#pragma unroll
            for (int e = 0; e < 4; ++e) ws[wave][Num<T>::row(e, g) * TL::WPITCH + 16 * y + li] = dp[y][e];
        wave_sync();
        weights_product<T, HDP, TL::COLS, TL::WPITCH, TL::PITCH>(ws[wave], qs, li, g, dk);
        wave_sync();
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int64_t j = key0 + 16 * wave + Num<T>::row(e, g);
        if (j >= sp.nk) continue;
        T* dst_k = p.dK + (sp.k0 + j) * p.lddk + kv * (int64_t)p.head_dim;
        T* dst_v = p.dV + (sp.k0 + j) * p.lddv + kv * (int64_t)p.head_dim;
#pragma unroll
        for (int y = 0; y < HDP / 16; ++y)
            if (16 * y + li < p.head_dim) {
                dst_k[16 * y + li] = dk[y][e] * p.scale;
                dst_v[16 * y + li] = dv[y][e];
            }
    }
}

// Gradient of Q: tiles as in the forward kernel, the rows of Q and dO in registers.
template <typename T, int HDP>
__global__ void __launch_bounds__(256) causal_bwd_q_kernel(const CausalArgs<T> p) {
    typedef Tile<T, HDP> TL;
    typedef typename Num<T>::Acc Acc;
    constexpr int CHUNKS = HDP / (4 * TL::VEC);
    __shared__ __attribute__((aligned(16))) T ks[TL::COLS * TL::PITCH], vs[TL::COLS * TL::PITCH], ws[4][16 * TL::WPITCH];
    __shared__ int bad[TL::COLS];  // written by the staging; rows that see such a key already have a NaN in lse
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int kv = blockIdx.y;
    int s;
    int64_t inside;
    if (!find_tile<64>(p, p.group, (int64_t)gridDim.x - 1 - blockIdx.x, &s, &inside)) return;
    const Span sp = span_of(p, s);
    const int64_t rows = sp.nq * p.group, row0 = inside * 64;
    if (row0 >= rows) return;
    Pack<T, TL::VEC> q[CHUNKS], go[CHUNKS];
    {
        const int64_t r = row0 + 16 * wave + li;
        const int64_t token = sp.q0 + r / p.group, col = (kv * p.group + r % p.group) * (int64_t)p.head_dim;
        load_row<T, HDP>(r < rows ? p.Q + token * p.ldq + col : nullptr, g, p.head_dim, p.vec_q, q);
        load_row<T, HDP>(r < rows ? p.dO + token * p.ldo + col : nullptr, g, p.head_dim, p.vec_o, go);
    }
    int64_t last[4];
    T lse[4], dot[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int64_t row = row0 + 16 * wave + Num<T>::row(r, g);
        last[r] = row < rows ? row / p.group : -1;
        lse[r] = dot[r] = 0;
        if (row < rows) {
            const int64_t at = (kv * p.group + row % p.group) * p.q_rows + sp.q0 + row / p.group;
            dot[r] = p.D[at];
            lse[r] = p.lse[at] * Num<T>::unit() + (dot[r] - dot[r]);
        }
    }
    Acc dq[HDP / 16];
#pragma unroll
    for (int y = 0; y < HDP / 16; ++y) dq[y] = Acc{0, 0, 0, 0};
    const int64_t last_row = row0 + 63 < rows ? row0 + 63 : rows - 1;
    const int64_t seen = last_row / p.group + 1;
    const T factor = p.scale * Num<T>::unit();
    const T* __restrict__ K = p.K + sp.k0 * p.ldk + kv * (int64_t)p.head_dim;
    const T* __restrict__ V = p.V + sp.k0 * p.ldv + kv * (int64_t)p.head_dim;
    for (int64_t k0 = 0; k0 < seen; k0 += TL::COLS) {
        __syncthreads();
        stage_two<T, HDP, TL::COLS, TL::PITCH>(ks, vs, bad, 0, p.head_dim, p.vec_kv, [&](int j, int which) -> const T* {
            if (k0 + j >= sp.nk) return nullptr;
            return which == 0 ? K + (k0 + j) * p.ldk : V + (k0 + j) * p.ldv;
        });
        __syncthreads();
        Acc st[TL::NY], dp[TL::NY];
        rows_product<T, HDP, TL::PITCH, TL::NY>(q, ks, li, g, st);
        rows_product<T, HDP, TL::PITCH, TL::NY>(go, vs, li, g, dp);
#pragma unroll
        for (int y = 0; y < TL::NY; ++y) {
            const int64_t j = k0 + 16 * y + li;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const T w = Num<T>::exp_unit(st[y][r] * factor - lse[r]);
                ws[wave][Num<T>::row(r, g) * TL::WPITCH + 16 * y + li] = j <= last[r] ? w * (dp[y][r] - dot[r]) : (T)0;
            }
        }
        wave_sync();
        weights_product<T, HDP, TL::COLS, TL::WPITCH, TL::PITCH>(ws[wave], ks, li, g, dq);
        wave_sync();
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int64_t row = row0 + 16 * wave + Num<T>::row(r, g);
        if (row >= rows) continue;
        T* dst = p.dQ + (sp.q0 + row / p.group) * p.lddq + (kv * p.group + row % p.group) * (int64_t)p.head_dim;
#pragma unroll
        for (int y = 0; y < HDP / 16; ++y)
            if (16 * y + li < p.head_dim) dst[16 * y + li] = dq[y][r] * p.scale;
    }
}

// ---- the newest tokens of a sequence against its cache --------------------------------------------------------------------
// Bound by reading the cache once.  Work is cut into units of one sequence: 16 packed rows against one part of its keys, one
// workgroup each, numbered through all sequences by a scan that every workgroup does for itself (lengths live on the device).
// A wavefront takes every fourth tile of 16 keys.  Everything is transposed - S^T = K Q^T, O^T = V^T P^T - so that the weights
// come out of the first product in the lanes where the second wants them, a row's statistics sit in a lane, and K and V go
// from memory to the registers of the matrix instructions without LDS.  Each operand's registers are filled again for the next
// tile as soon as its product has read them, so that loads are always in flight.
template <typename T>
struct CachedPlan {
    int most_parts;     // of a sequence
    T *stat, *data;     // of part i of packed row r: {maximum, sum} and the weighted sum of values, at r * most_parts + i
    int32_t* part_keys; // how many keys make a part, for the join
};
constexpr int CACHED_WAVES = 4, CACHED_LEAST = 128, CACHED_WHOLE = 512, CACHED_GROUPS = 512;

// Parts of a sequence's keys: of `size` keys, or of more if there would be too many parts, whole tiles.
__device__ __forceinline__ int64_t part_keys(int64_t keys, int64_t size, int most_parts) {
    if (keys <= size * most_parts) return size;
    return ((keys + most_parts - 1) / most_parts + 15) / 16 * 16;
}
__device__ __forceinline__ uint32_t part_count(int64_t keys, uint32_t size, int most_parts) {
    if (keys <= CACHED_WHOLE || keys <= size || most_parts == 1) return 1;
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

// The sequence of unit `unit` and the unit's number inside it, by a whole wavefront; false: there are not so many.  (Rows fit
// into 31 bits, so a sequence has less than 2^32 units.  Offsets that overlap may wrap the sum: the caller checks the number.)
template <typename T>
__device__ __forceinline__ bool find_unit(const CausalArgs<T>& p, int most_parts, uint32_t size, uint32_t unit, int lane, Span* span, uint32_t* parts, uint32_t* inside) {
    uint32_t before = 0;
    for (int s0 = 0; s0 < p.sequences; s0 += 64) {
        Span sp = {0, 0, 0, 0};
        uint32_t units = 0, count = 1;
        if (s0 + lane < p.sequences) {
            sp = span_of(p, s0 + lane);
            count = part_count(sp.nk, size, most_parts);
            units = ((uint32_t)sp.nq * (uint32_t)p.group + 15) / 16 * count;
        }
        const uint32_t upto = before + scan64(units);
        const uint64_t behind = __ballot(upto > unit);
        if (behind != 0) {
            const int at = __builtin_ctzll(behind);
            // (none of these passes 31 bits)
            span->q0 = __builtin_amdgcn_readlane((int)sp.q0, at);
            span->nq = __builtin_amdgcn_readlane((int)sp.nq, at);
            span->k0 = __builtin_amdgcn_readlane((int)sp.k0, at);
            span->nk = __builtin_amdgcn_readlane((int)sp.nk, at);
            *parts = __builtin_amdgcn_readlane(count, at);
            *inside = unit - __builtin_amdgcn_readlane(upto - units, at);
            return true;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// Keys per part that make all units of a call few enough to run at once, each sequence having a part that is not whole.
template <typename T>
__device__ __forceinline__ uint32_t keys_per_part(const CausalArgs<T>& p, int most_parts, int lane) {
    if (most_parts == 1) return 0;
    float keys = 0, tiles = 0;
    for (int s0 = 0; s0 < p.sequences; s0 += 64) {
        if (s0 + lane >= p.sequences) break;
        const Span sp = span_of(p, s0 + lane);
        const float here = (float)(((uint32_t)sp.nq * (uint32_t)p.group + 15) / 16);
        tiles += here;
        keys += here * (float)sp.nk;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        keys += __shfl_xor(keys, d, 64);
        tiles += __shfl_xor(tiles, d, 64);
    }
    const float room = fmaxf((float)(CACHED_GROUPS / 2), CACHED_GROUPS - tiles * p.kv_heads), share = keys * p.kv_heads / room;
    return __builtin_amdgcn_readfirstlane(((uint32_t)fminf(fmaxf(share, (float)CACHED_LEAST), 1e9f) + 63) / 64 * 64);
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

template <typename T, int HDP, bool ALIGNED>
__global__ void __launch_bounds__(64 * CACHED_WAVES, sizeof(T) == 4 && ALIGNED ? 2 : 1) cached_attention_kernel(const CausalArgs<T> p, const CachedPlan<T> plan) {
    constexpr int VEC = 16 / sizeof(T), CH = 4 * VEC, CHUNKS = HDP / CH, NY = HDP / 16, N = VEC < NY ? VEC : NY, W = CACHED_WAVES, PITCH = HDP + VEC;
    typedef typename Num<T>::Acc Acc;
    __shared__ __attribute__((aligned(16))) T sums[W][16 * PITCH];
    __shared__ T stat[W][2][16];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    // heads of a unit are neighbours, so that workgroups without a unit come last
    const uint32_t stride = gridDim.x / p.kv_heads;
    const int kv = (int)(blockIdx.x % p.kv_heads);
    const uint32_t keys_each = keys_per_part(p, plan.most_parts, lane);
    if (blockIdx.x == 0 && threadIdx.x == 0 && plan.most_parts > 1) *plan.part_keys = (int32_t)keys_each;
    for (uint32_t unit = blockIdx.x / p.kv_heads;; unit += stride) {
        Span sp;
        uint32_t parts, inside;
        if (!find_unit(p, plan.most_parts, keys_each, unit, lane, &sp, &parts, &inside)) return;
        const uint32_t rows = (uint32_t)sp.nq * (uint32_t)p.group, tile = inside / parts, part = inside % parts, row0 = tile * 16;
        if (tile >= (rows + 15) / 16) return;  // (a wrapped sum)
        const int64_t lead = sp.nk - sp.nq;
        const uint32_t r = row0 + li < rows ? row0 + li : rows - 1;  // the lane's row; past the last it is the last one again
        const uint32_t first_token = row0 / p.group, ahead = (row0 % p.group + (r - row0)) / p.group;  // of the tile; of the row, from there
        const int64_t token = sp.q0 + first_token + ahead;
        const int head = kv * p.group + (int)(r - (first_token + ahead) * p.group);
        Pack<T, VEC> q[CHUNKS];
        {
            const T* __restrict__ row = p.Q + token * p.ldq + head * (int64_t)p.head_dim;
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) q[c] = load_some<T, VEC, ALIGNED>(row, CH * c + VEC * g, p.head_dim);
        }
        const int64_t first_last = lead + first_token, last = first_last + ahead;  // the last key that the tile's first row sees, that this one does
        const int64_t size = part_keys(sp.nk, keys_each, plan.most_parts), seen = clamped(first_last + (int)__builtin_amdgcn_readlane(ahead, 15) + 1, sp.nk);
        const int64_t from = part * size, to = parts == 1 || seen < from + size ? seen : from + size;
        const T* __restrict__ K = p.K + sp.k0 * p.ldk + kv * (int64_t)p.head_dim;
        const T* __restrict__ V = p.V + sp.k0 * p.ldv + kv * (int64_t)p.head_dim;
        T m = -(T)INFINITY, l = 0;
        Acc o[NY];  // element r of o[N y + t]: column 16 N y + N row(r, g) + t of row li
#pragma unroll
        for (int y = 0; y < NY; ++y) o[y] = Acc{0, 0, 0, 0};
        const T factor = p.scale * Num<T>::unit();
        Pack<T, VEC> k[CHUNKS];   // key li, elements CH c + VEC g + t
        Pack<T, N> v[4][NY / N];  // keys row(x, g), columns 16 N y + N li + t
        // keys past the last are the last one again: their scores are masked
        auto load_k = [&](int64_t k0) {
            const int most = (int)(to - 1 - k0 < 15 ? to - 1 - k0 : 15);
            const T* __restrict__ row = K + k0 * p.ldk + (li < most ? li : most) * p.ldk;
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) k[c] = load_some<T, VEC, ALIGNED>(row, CH * c + VEC * g, p.head_dim);
        };
        auto load_v = [&](int64_t k0) {
            const int most = (int)(to - 1 - k0 < 15 ? to - 1 - k0 : 15);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int j = Num<T>::row(x, g);
                const T* __restrict__ row = V + k0 * p.ldv + (j < most ? j : most) * p.ldv;
#pragma unroll
                for (int y = 0; y < NY / N; ++y) v[x][y] = load_some<T, N, ALIGNED>(row, 16 * N * y + N * li, p.head_dim);
            }
        };
        int64_t k0 = from + 16 * wave;
        if (k0 < to) {
            load_k(k0);
            load_v(k0);
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
            for (int t = 0; t < VEC; ++t) q[c].v[t] = CH * c + VEC * g + t < p.head_dim ? q[c].v[t] : (T)0;
        poison_row<T, CHUNKS>(q);
        for (; k0 < to; k0 += 16 * W) {
            Acc sc = Acc{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                for (int t = 0; t < VEC; ++t) sc = Num<T>::mfma(k[c].v[t], q[c].v[t], sc);
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
            odd = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int y = 0; y < NY / N; ++y)
#pragma unroll
                    for (int t = 0; t < N; ++t) odd = fma(v[x][y].v[t], (T)0, odd);
            if (__any(!(odd == 0))) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    bool fine = true;
#pragma unroll
                    for (int y = 0; y < NY / N; ++y)
#pragma unroll
                        for (int t = 0; t < N; ++t) {
                            fine = fine && is_finite(v[x][y].v[t]);
                            v[x][y].v[t] = is_finite(v[x][y].v[t]) ? v[x][y].v[t] : (T)0;
                        }
                    const uint64_t b = __ballot(!fine);
#pragma unroll
                    for (int gg = 0; gg < 4; ++gg)
                        if ((b >> (16 * gg)) & 0xFFFFu) poisoned |= 1u << Num<T>::row(x, gg);
                }
            }
            T top = -(T)INFINITY;
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
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int y = 0; y < NY; ++y) o[y] = Num<T>::mfma(v[x][y / N].v[y % N], sc[x], o[y]);
            load_v(k0 + 16 * W);
        }
        // the wavefronts' sums, added in their order
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (g == 0) {
            stat[wave][0][li] = m;
            stat[wave][1][li] = l;
        }
        const int here = (int)(rows - row0 < 16 ? rows - row0 : 16);
        if (li < here) {
#pragma unroll
            for (int y = 0; y < NY / N; ++y)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    Pack<T, N> e;
#pragma unroll
                    for (int t = 0; t < N; ++t) e.v[t] = o[N * y + t][x];
                    *reinterpret_cast<Pack<T, N>*>(&sums[wave][li * PITCH + 16 * N * y + N * Num<T>::row(x, g)]) = e;
                }
        }
        __syncthreads();
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
            if (parts == 1) {
                const T by = first_last + ahead_of >= 0 && sp.nk > 0 ? 1 / total : (T)0;
#pragma unroll
                for (int t = 0; t < VEC; ++t) sum[t] *= by;
                dst = p.O + to_token * p.ldo + to_head * (int64_t)p.head_dim;
            } else {
                const int64_t place = (to_token * p.heads + to_head) * plan.most_parts + part;
                dst = plan.data + place * p.head_dim;
                if (d == 0) {
                    plan.stat[2 * place] = top;
                    plan.stat[2 * place + 1] = total;
                }
            }
#pragma unroll
            for (int t = 0; t < VEC; ++t)
                if (d + t < p.head_dim) dst[d + t] = sum[t];
        }
        if (unit > ~0u - stride) return;
        __syncthreads();
    }
}

// Joins the parts of a row: a wavefront per (token, head).
template <typename T>
__global__ void __launch_bounds__(256) cached_join_kernel(const CausalArgs<T> p, const CachedPlan<T> plan) {
    const int lane = threadIdx.x & 63;
    const int64_t at = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (at >= p.q_rows * p.heads) return;
    const int64_t token = at / p.heads;
    // the sequence of the token: rows in front of the first and behind the last are left as they are
    int begun = 0;  // offsets that are not behind the token
    for (int s0 = 0; s0 <= p.sequences; s0 += 64) {
        const int here = __popcll(__ballot(s0 + lane <= p.sequences && clamped(p.q_off[s0 + lane], p.q_rows) <= token));
        begun += here;
        if (here < 64) break;
    }
    begun = __builtin_amdgcn_readfirstlane(begun);
    if (begun == 0 || begun > p.sequences) return;
    const Span sp = span_of(p, begun - 1);
    if (token < sp.q0 || token >= sp.q0 + sp.nq) return;
    const int parts = (int)part_count(sp.nk, (uint32_t)*plan.part_keys, plan.most_parts);
    if (parts == 1) return;
    const T m = lane < parts ? plan.stat[2 * (at * plan.most_parts + lane)] : -(T)INFINITY;
    const T l = lane < parts ? plan.stat[2 * (at * plan.most_parts + lane) + 1] : (T)0;
    T top = m;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmax(top, __shfl_xor(top, d, 64));
    T f = Num<T>::exp_unit(m - (top == -(T)INFINITY ? (T)0 : top)), total = l * f;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d, 64);
    f = sp.nk - sp.nq + (token - sp.q0) >= 0 ? f / total : (T)0;
    const T* __restrict__ mine = plan.data + at * plan.most_parts * (int64_t)p.head_dim;
    T sum[2] = {0, 0};
    const int d0 = lane < p.head_dim ? lane : 0, d1 = lane + 64 < p.head_dim ? lane + 64 : 0;
#pragma unroll 8
    for (int i = 0; i < parts; ++i) {
        const T w = __shfl(f, i, 64);
        sum[0] += mine[(int64_t)i * p.head_dim + d0] * w;
        sum[1] += mine[(int64_t)i * p.head_dim + d1] * w;
    }
    T* __restrict__ dst = p.O + token * p.ldo + at % p.heads * (int64_t)p.head_dim;
    if (lane < p.head_dim) dst[lane] = sum[0];
    if (lane + 64 < p.head_dim) dst[lane + 64] = sum[1];
}

inline bool grid_fits(int64_t groups, int64_t lanes) { return groups * lanes < ((int64_t)1 << 32); }
inline int64_t tile_slots(int64_t rows, int64_t group, int64_t per_tile, int64_t sequences) { return rows * group / per_tile + sequences; }

}  // namespace

// A launch of KERNEL<T, HDP> for the smallest padded head dimension that holds head_dim.
#define BY_HEAD_DIM(KERNEL, GRID, ...)                                                                                  \
    do {                                                                                                                \
        if (a.head_dim <= 32) hipLaunchKernelGGL((KERNEL<T, 32>), GRID, dim3(256), 0, s, __VA_ARGS__);                  \
        else if (a.head_dim <= 64) hipLaunchKernelGGL((KERNEL<T, 64>), GRID, dim3(256), 0, s, __VA_ARGS__);             \
        else hipLaunchKernelGGL((KERNEL<T, 128>), GRID, dim3(256), 0, s, __VA_ARGS__);                                  \
        if (hipError_t e = hipGetLastError()) return e;                                                                 \
    } while (0)

#define BY_HEAD_DIM_CACHED(ALIGNED)                                                                                                       \
    do {                                                                                                                                  \
        const dim3 block(64 * CACHED_WAVES);                                                                                              \
        if (a.head_dim <= 32) hipLaunchKernelGGL((cached_attention_kernel<T, 32, ALIGNED>), grid, block, 0, s, a, plan);                  \
        else if (a.head_dim <= 64) hipLaunchKernelGGL((cached_attention_kernel<T, 64, ALIGNED>), grid, block, 0, s, a, plan);             \
        else hipLaunchKernelGGL((cached_attention_kernel<T, 128, ALIGNED>), grid, block, 0, s, a, plan);                                  \
    } while (0)

template <typename T>
hipError_t launch_causal_fwd(const CausalArgs<T>& a, hipStream_t s) {
    const int64_t slots = tile_slots(a.q_rows, a.group, 64, a.sequences);
    if (!grid_fits(slots, 256)) return hipErrorInvalidValue;
    BY_HEAD_DIM(causal_fwd_kernel, dim3((unsigned)slots, a.kv_heads), a);
    return hipSuccess;
}

template <typename T>
size_t causal_bwd_workspace_bytes(const CausalArgs<T>& a) {
    return (size_t)a.heads * a.q_rows * sizeof(T);
}

template <typename T>
hipError_t launch_causal_bwd(CausalArgs<T> a, void* workspace, hipStream_t s) {
    a.D = static_cast<T*>(workspace);
    const int64_t dots = (a.q_rows * a.heads + 15) / 16, key_slots = tile_slots(a.q_rows, 1, 64, a.sequences), slots = tile_slots(a.q_rows, a.group, 64, a.sequences);
    if (!grid_fits(dots, 256) || !grid_fits(slots, 256)) return hipErrorInvalidValue;
    hipLaunchKernelGGL(causal_dot_kernel<T>, dim3((unsigned)dots), dim3(256), 0, s, a);
    if (hipError_t e = hipGetLastError()) return e;
    BY_HEAD_DIM(causal_bwd_kv_kernel, dim3((unsigned)key_slots, a.kv_heads), a);
    BY_HEAD_DIM(causal_bwd_q_kernel, dim3((unsigned)slots, a.kv_heads), a);
    return hipSuccess;
}

// Parts of a sequence's keys at most: one where a cache is short, no more than a lane each, and few enough that rows with many
// units do not need a large workspace.
template <typename T>
static int most_cached_parts(const CausalArgs<T>& a) {
    if (a.k_rows <= CACHED_WHOLE) return 1;
    const int64_t units = tile_slots(a.q_rows, a.group, 16, a.sequences) * a.kv_heads;
    return (int)std::max<int64_t>(1, std::min<int64_t>({64, (a.k_rows + CACHED_LEAST - 1) / CACHED_LEAST, 8 * CACHED_GROUPS / units}));
}

template <typename T>
size_t cached_workspace_bytes(const CausalArgs<T>& a) {
    const int parts = most_cached_parts(a);
    return parts == 1 ? 0 : 16 + (size_t)a.q_rows * a.heads * parts * (a.head_dim + 2) * sizeof(T);
}

template <typename T>
hipError_t launch_cached_attention(const CausalArgs<T>& a, void* workspace, hipStream_t s) {
    CachedPlan<T> plan;
    plan.most_parts = most_cached_parts(a);
    plan.part_keys = static_cast<int32_t*>(workspace);
    plan.data = static_cast<T*>(workspace) + 16 / sizeof(T);
    plan.stat = plan.data + a.q_rows * a.heads * (int64_t)plan.most_parts * a.head_dim;
    // a workgroup per unit of a call whose units run at once; of larger calls some take several
    const int64_t tiles = tile_slots(a.q_rows, a.group, 16, a.sequences), rows = (a.q_rows * a.heads + 3) / 4;
    const int64_t groups = std::min(tiles * plan.most_parts, std::max<int64_t>(1, (tiles * a.kv_heads <= CACHED_GROUPS / 2 ? 1 : 4) * CACHED_GROUPS / a.kv_heads));
    if (!grid_fits(rows, 256) || a.q_rows > INT32_MAX / a.group - 16 || a.k_rows > INT32_MAX) return hipErrorInvalidValue;
    const dim3 grid((unsigned)(groups * a.kv_heads));
    if (a.vec_q && a.vec_kv) BY_HEAD_DIM_CACHED(true); else BY_HEAD_DIM_CACHED(false);
    if (hipError_t e = hipGetLastError()) return e;
    if (plan.most_parts > 1) {
        hipLaunchKernelGGL(cached_join_kernel<T>, dim3((unsigned)rows), dim3(256), 0, s, a, plan);
        if (hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
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
