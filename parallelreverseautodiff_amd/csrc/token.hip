// Between token ids and the layers: embedding lookup with its gradient, dropout, and the addition to an index vector.
// All of it is bound by memory (a large copy on this card moves 5.0 TB/s, both directions counted), or by the launches
// where the data is small.
#include "common.h"

#include <algorithm>
#include <initializer_list>

namespace prad {

namespace {

// N elements moved as one load or store.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

inline bool aligned16(std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
    return true;
}

// ---- lookup: out[i] = scale * table[ids[i]] ---------------------------------------------------------------------------
// A workgroup takes 1024 consecutive packs of the output, whatever the row length: four loads of ids, then four of the
// table are in flight per lane.  An id outside the table (padding) gives a row of zeros.  Bound by memory: 16384 rows of 1024
// floats in 23 us, 5.8 TB/s with the rows that are still in the caches.
constexpr int LOOKUP_UNROLL = 4;

template <typename T, int N>
__global__ void __launch_bounds__(256) embedding_fwd_kernel(const T* __restrict__ table, const int32_t* __restrict__ ids, T* __restrict__ out,
                                                            int64_t tokens, int64_t vocab, uint32_t packs, T scale) {
    typedef Pack<T, N> P;
    const int64_t base = (int64_t)blockIdx.x * (256 * LOOKUP_UNROLL);
    const int64_t row0 = base / packs;
    const uint32_t rem = (uint32_t)(base - row0 * packs);
    int64_t row[LOOKUP_UNROLL];
    uint32_t col[LOOKUP_UNROLL];
    int32_t id[LOOKUP_UNROLL];
#pragma unroll
    for (int u = 0; u < LOOKUP_UNROLL; ++u) {
        const uint64_t at = (uint64_t)rem + threadIdx.x + 256 * u;
        const uint32_t down = at <= 0xFFFFFFFFull ? (uint32_t)at / packs : (uint32_t)(at / packs);
        row[u] = row0 + down;
        col[u] = (uint32_t)(at - (uint64_t)down * packs);
        id[u] = row[u] < tokens ? ids[row[u]] : -1;
    }
    P v[LOOKUP_UNROLL];
#pragma unroll
    for (int u = 0; u < LOOKUP_UNROLL; ++u) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[u].v[e] = (T)0;
        if ((uint64_t)(int64_t)id[u] < (uint64_t)vocab) {
            v[u] = reinterpret_cast<const P*>(table)[(int64_t)id[u] * packs + col[u]];
#pragma unroll
            for (int e = 0; e < N; ++e) v[u].v[e] = v[u].v[e] * scale;
        }
    }
#pragma unroll
    for (int u = 0; u < LOOKUP_UNROLL; ++u)
        if (row[u] < tokens) reinterpret_cast<P*>(out)[row[u] * packs + col[u]] = v[u];
}

// ---- gradient: dtable[r] (+)= scale * sum over i with ids[i] == r of dout[i] -------------------------------------------
// The positions are brought into the order of their ids (equal ids in the order of their positions), so every sum has one
// order and one owner: no atomic touches a gradient and the result does not depend on how the launch was scheduled.
// Sums are held in double.

// Few tokens: one launch.  A wavefront owns a table row, finds its positions among the ids by ballots and adds them up.  Bound
// by its latency: 49 tokens, 1000 rows of 96 doubles in 2.9 us.  Against the three launches below, 512 tokens: 3.7 us for 17.2
// (1000 rows of 96 floats), 16 for 25 (32768 of 512); where all tokens are one, which a single wavefront then adds up, 35 for 14
// and 83 for 22.  With 1024 tokens that would be 71 and 161.
constexpr int EMB_DIRECT_TOKENS = 512;

template <typename T, int N>
__global__ void __launch_bounds__(256) embedding_bwd_direct_kernel(const T* __restrict__ dout, const int32_t* __restrict__ ids, T* __restrict__ dtable,
                                                                   int tokens, int64_t vocab, int64_t packs, double scale, int accumulate) {
    typedef Pack<T, N> P;
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (row >= vocab) return;
    uint64_t found[EMB_DIRECT_TOKENS / 64];
    uint64_t any = 0;
#pragma unroll
    for (int b = 0; b < EMB_DIRECT_TOKENS / 64; ++b) {
        const int i = 64 * b + lane;
        found[b] = __ballot(i < tokens && (int64_t)ids[i < tokens ? i : 0] == row);
        any |= found[b];
    }
    if (any == 0 && accumulate) return;
    for (int64_t c = lane; c < packs; c += 64) {
        double sum[N];
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = 0.0;
#pragma unroll
        for (int b = 0; b < EMB_DIRECT_TOKENS / 64; ++b) {
            uint64_t left = found[b];
            while (left != 0) {  // eight at a time, their loads in flight together
                const int n = __builtin_popcountll(left);
                P v[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (u >= n) break;
                    v[u] = reinterpret_cast<const P*>(dout)[(int64_t)(64 * b + __builtin_ctzll(left)) * packs + c];
                    left &= left - 1;
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (u >= n) break;
#pragma unroll
                    for (int e = 0; e < N; ++e) sum[e] += (double)v[u].v[e];
                }
            }
        }
        P* dst = reinterpret_cast<P*>(dtable) + row * packs + c;
        P r;
        if (accumulate) r = *dst;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const T g = (T)(sum[e] * scale);
            r.v[e] = accumulate ? r.v[e] + g : g;
        }
        *dst = r;
    }
}

// Many tokens, first launch: a workgroup owns `span` consecutive table rows and walks all ids twice - to count (its own
// ids, and how many lie below them: that is where its part of the order begins), then to place.  Each of its wavefronts
// walks a contiguous part of the positions, with write positions of its own per row, so equal ids keep the order of their
// positions without any exchange.  Rows without a token are cleared here.  The ids stay in the caches; what a walk costs is
// the comparison of every id by every workgroup, so there are no more of those than compute units (32768 ids, 32768 rows of
// 512 floats, lookup and gradient: 65.8 us with 256, 68.3 with 512, 66.7 with 128).
constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;
constexpr int SORT_MOST_SPAN = 960;  // 60 KB of counters

template <typename T, int N>
__global__ void __launch_bounds__(SORT_THREADS) embedding_sort_kernel(const int32_t* __restrict__ ids, int tokens, int64_t vocab, int span,
                                                                      int32_t* __restrict__ order, int32_t* __restrict__ order_ids,
                                                                      int32_t* __restrict__ valid, T* __restrict__ dtable, int64_t packs, int accumulate) {
    typedef Pack<T, N> P;
    extern __shared__ __attribute__((aligned(16))) int32_t cursor[];  // [wave][row of the span]
    __shared__ int32_t below_of[SORT_WAVES];
    __shared__ int32_t wave_total[SORT_WAVES];
    __shared__ uint64_t without_token[SORT_WAVES];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t first = (int64_t)blockIdx.x * span;
    const int rows = (int)(vocab - first < span ? vocab - first : span);
    for (int e = threadIdx.x; e < SORT_WAVES * span; e += SORT_THREADS) cursor[e] = 0;
    __syncthreads();
    // parts of whole wavefronts of positions
    const int64_t part = (((int64_t)tokens + SORT_WAVES - 1) / SORT_WAVES + 63) & ~(int64_t)63;
    const int64_t from = wave * part, to = from + part < tokens ? from + part : tokens;
    int32_t* __restrict__ mine = cursor + wave * span;
    const uint32_t first32 = (uint32_t)first, reach = (uint32_t)rows;  // (rows end below 2^31, where negative ids begin)
    int below = 0;
    for (int64_t i0 = from; i0 < to; i0 += 256) {
        int32_t id[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t i = i0 + 64 * u + lane;
            id[u] = i < to ? ids[i] : -1;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t r = (uint32_t)id[u] - first32;
            below += (uint32_t)id[u] < first32;
            if (r < reach) atomicAdd(&mine[r], 1);  // (a count: the order of the additions does not show)
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) below += __shfl_xor(below, off, 64);
    if (lane == 0) below_of[wave] = below;
    __syncthreads();
    // exclusive sums over (row, wave): first a row's wavefronts, then the rows
    int total = 0;  // of row threadIdx.x (span <= SORT_THREADS)
    const bool has_row = (int)threadIdx.x < rows;
    if (has_row)
        for (int w = 0; w < SORT_WAVES; ++w) {
            const int c = cursor[w * span + threadIdx.x];
            cursor[w * span + threadIdx.x] = total;
            total += c;
        }
    int before = total;  // inclusive sum over the lanes
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int v = __shfl_up(before, off, 64);
        if (lane >= off) before += v;
    }
    if (lane == 63) wave_total[wave] = before;
    __syncthreads();
    int base = 0;
    for (int w = 0; w < SORT_WAVES; ++w) {
        base += below_of[w];
        if (w < wave) base += wave_total[w];
    }
    const int begin = base + before - total;
    if (has_row)
        for (int w = 0; w < SORT_WAVES; ++w) cursor[w * span + threadIdx.x] += begin;
    if (first + rows == vocab && (int)threadIdx.x == rows - 1) *valid = begin + total;
    {
        const uint64_t empty = __ballot(has_row && total == 0);
        if (lane == 0) without_token[wave] = empty;
    }
    __syncthreads();
    // rows without a token: zeros, a wavefront to a row
    if (!accumulate) {
        for (int r = wave; r < rows; r += SORT_WAVES) {
            if (((without_token[r >> 6] >> (r & 63)) & 1) == 0) continue;
            P* dst = reinterpret_cast<P*>(dtable) + (first + r) * packs;
            P zero;
#pragma unroll
            for (int e = 0; e < N; ++e) zero.v[e] = (T)0;
            for (int64_t c = lane; c < packs; c += 64) dst[c] = zero;
        }
    }
    for (int64_t i0 = from; i0 < to; i0 += 256) {
        int32_t id[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t i = i0 + 64 * u + lane;
            id[u] = i < to ? ids[i] : -1;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            uint64_t left = __ballot((uint32_t)id[u] - first32 < reach);
            while (left != 0) {  // one round per id that occurs among the 64
                const int leader = __builtin_ctzll(left);
                const int32_t which = __builtin_amdgcn_readlane(id[u], leader);
                const uint64_t same = __ballot(id[u] == which);
                const int at = mine[which - first];
                if (id[u] == which) {
                    const int slot = at + __builtin_popcountll(same & ((1ull << lane) - 1));
                    order[slot] = (int32_t)(i0 + 64 * u + lane);
                    order_ids[slot] = which;
                }
                if (lane == leader) mine[which - first] = at + __builtin_popcountll(same);
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                left &= ~same;
            }
        }
    }
}

// Second launch: a wavefront adds up SUM_CHUNK consecutive entries of the order over 64 packs of columns.  A run of equal
// ids that lies inside the chunk is finished here; the parts of runs that cross its borders go to the workspace (the run
// that came in from the chunk before: `head`; the one that leaves it and began here: `tail`), for the third launch.
// Bound by memory: 32768 rows of 512 floats in 17 us, 67 MB read and, with 63 % of the rows of the table, 42 MB written.
constexpr int SUM_CHUNK = 32;

template <typename T, int N>
__global__ void __launch_bounds__(256) embedding_sum_kernel(const T* __restrict__ dout, const int32_t* __restrict__ order, const int32_t* __restrict__ order_ids,
                                                            const int32_t* __restrict__ valid, double* __restrict__ head, double* __restrict__ tail,
                                                            T* __restrict__ dtable, int64_t packs, double scale, int accumulate) {
    typedef Pack<T, N> P;
    typedef Pack<double, N> PD;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t chunk = (int64_t)blockIdx.x * 4 + wave;
    const int count = *valid;
    const int64_t e0 = chunk * SUM_CHUNK;
    if (e0 >= count) return;
    const int n = (int)(count - e0 < SUM_CHUNK ? count - e0 : SUM_CHUNK);
    const int64_t c = (int64_t)blockIdx.y * 64 + lane;
    const int64_t cc = c < packs ? c : packs - 1;
    // lane l < n holds entry l; lanes 62 and 63 the ids just before and just behind the chunk
    const int64_t mine = e0 + (lane < n ? lane : 0);
    const int32_t pos = order[mine];
    int32_t id = order_ids[mine];
    if (lane == 62) id = e0 > 0 ? order_ids[e0 - 1] : -1;
    if (lane == 63) id = e0 + n < count ? order_ids[e0 + n] : -1;
    const int32_t id_before = __builtin_amdgcn_readlane(id, 62), id_behind = __builtin_amdgcn_readlane(id, 63);
    double sum[N];
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] = 0.0;
    bool from_before = __builtin_amdgcn_readlane(id, 0) == id_before;
    for (int k0 = 0; k0 < n; k0 += 8) {
        P v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int64_t row = __builtin_amdgcn_readlane(pos, k0 + u < n ? k0 + u : n - 1);
            v[u] = reinterpret_cast<const P*>(dout)[row * packs + cc];
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (k0 + u >= n) break;
            const int32_t r = __builtin_amdgcn_readlane(id, k0 + u);
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] += (double)v[u].v[e];
            const bool last = k0 + u == n - 1;
            const int32_t next = last ? id_behind : __builtin_amdgcn_readlane(id, k0 + u + 1);
            if (!last && next == r) continue;
            if (c < packs) {
                if (from_before || next == r) {
                    PD part;
#pragma unroll
                    for (int e = 0; e < N; ++e) part.v[e] = sum[e];
                    reinterpret_cast<PD*>(from_before ? head : tail)[chunk * packs + c] = part;
                } else {
                    P* dst = reinterpret_cast<P*>(dtable) + (int64_t)r * packs + c;
                    P g;
                    if (accumulate) g = *dst;
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const T s = (T)(sum[e] * scale);
                        g.v[e] = accumulate ? g.v[e] + s : s;
                    }
                    *dst = g;
                }
            }
            from_before = false;
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] = 0.0;
        }
    }
}

// Third launch: the chunk in which a run that crosses borders began adds its tail and the heads of the chunks behind it.
// A frequent token's run spans many chunks: the four wavefronts take every fourth head.  (6 us behind the 17 above: a launch, and
// workgroups that find nothing to do.)
template <typename T, int N>
__global__ void __launch_bounds__(256) embedding_join_kernel(const int32_t* __restrict__ order_ids, const int32_t* __restrict__ valid,
                                                             const double* __restrict__ head, const double* __restrict__ tail, T* __restrict__ dtable,
                                                             int64_t packs, double scale, int accumulate) {
    typedef Pack<T, N> P;
    typedef Pack<double, N> PD;
    __shared__ PD parts[4][64];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t chunk = blockIdx.x;
    const int count = *valid;
    const int64_t end = (chunk + 1) * SUM_CHUNK;
    if (end >= count) return;  // nothing behind it
    const int32_t r = order_ids[end - 1];
    if (order_ids[end] != r) return;  // no run leaves the chunk
    if (chunk > 0 && order_ids[end - SUM_CHUNK] == r && order_ids[end - SUM_CHUNK - 1] == r) return;  // it came in from before
    const int64_t c = (int64_t)blockIdx.y * 64 + lane;
    const int64_t cc = c < packs ? c : packs - 1;
    const int64_t chunks = (count + SUM_CHUNK - 1) / SUM_CHUNK;
    double sum[N];
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] = 0.0;
    if (wave == 0) {
        const PD t = reinterpret_cast<const PD*>(tail)[chunk * packs + cc];
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = t.v[e];
    }
    for (int64_t j0 = chunk + 1; j0 < chunks; j0 += 64) {
        // how many of the next 64 chunks begin inside the run
        const uint64_t in_run = __ballot(j0 + lane < chunks && order_ids[(j0 + lane < chunks ? j0 + lane : chunk) * SUM_CHUNK] == r);
        const int m = ~in_run == 0 ? 64 : __builtin_ctzll(~in_run);
        for (int j = wave; j < m; j += 16) {
            PD h[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) h[u] = reinterpret_cast<const PD*>(head)[(j0 + (j + 4 * u < m ? j + 4 * u : j)) * packs + cc];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int e = 0; e < N; ++e) sum[e] += j + 4 * u < m ? h[u].v[e] : 0.0;
        }
        if (m < 64) break;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) parts[wave][lane].v[e] = sum[e];
    __syncthreads();
    if (wave == 0 && c < packs) {
        P* dst = reinterpret_cast<P*>(dtable) + (int64_t)r * packs + c;
        P g;
        if (accumulate) g = *dst;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const T s = (T)(((parts[0][lane].v[e] + parts[1][lane].v[e]) + (parts[2][lane].v[e] + parts[3][lane].v[e])) * scale);
            g.v[e] = accumulate ? g.v[e] + s : s;
        }
        *dst = g;
    }
}

// A launch holds fewer than 2^32 lanes.
inline bool grid_fits(int64_t groups, int64_t lanes) { return groups * lanes < ((int64_t)1 << 32); }

inline size_t round256(size_t b) { return (b + 255) & ~(size_t)255; }
// (a table of more rows than a launch has wavefronts takes the other launches, which have a workgroup for 960 rows)
inline bool one_launch(int64_t tokens, int64_t vocab) { return tokens <= EMB_DIRECT_TOKENS && grid_fits((vocab + 3) / 4, 256); }
inline int64_t sum_chunks(int64_t tokens) { return (tokens + SUM_CHUNK - 1) / SUM_CHUNK; }

template <typename T, int N>
hipError_t embedding_bwd_n(const T* dout, const int32_t* ids, T* dtable, int64_t tokens, int64_t vocab, int64_t width, double scale, int accumulate,
                           void* workspace, hipStream_t s) {
    const int64_t packs = width / N;
    if (one_launch(tokens, vocab)) {
        hipLaunchKernelGGL((embedding_bwd_direct_kernel<T, N>), dim3((unsigned)((vocab + 3) / 4)), dim3(256), 0, s, dout, ids, dtable, (int)tokens, vocab,
                           packs, scale, accumulate);
        return hipGetLastError();
    }
    char* at = static_cast<char*>(workspace);
    int32_t* valid = reinterpret_cast<int32_t*>(at);
    at += 256;
    int32_t* order = reinterpret_cast<int32_t*>(at);
    at += round256((size_t)tokens * 4);
    int32_t* order_ids = reinterpret_cast<int32_t*>(at);
    at += round256((size_t)tokens * 4);
    const int64_t chunks = sum_chunks(tokens);
    double* head = reinterpret_cast<double*>(at);
    double* tail = head + chunks * width;
    const unsigned slices = (unsigned)((packs + 63) / 64);
    if (slices > 65535 || !grid_fits(chunks, 256)) return hipErrorInvalidValue;
    const int span = (int)std::min<int64_t>(SORT_MOST_SPAN, (vocab + 255) / 256);
    hipLaunchKernelGGL((embedding_sort_kernel<T, N>), dim3((unsigned)((vocab + span - 1) / span)), dim3(SORT_THREADS), (size_t)SORT_WAVES * span * 4, s, ids,
                       (int)tokens, vocab, span, order, order_ids, valid, dtable, packs, accumulate);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL((embedding_sum_kernel<T, N>), dim3((unsigned)((chunks + 3) / 4), slices), dim3(256), 0, s, dout, order, order_ids, valid, head, tail,
                       dtable, packs, scale, accumulate);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL((embedding_join_kernel<T, N>), dim3((unsigned)chunks, slices), dim3(256), 0, s, order_ids, valid, head, tail, dtable, packs, scale,
                       accumulate);
    return hipGetLastError();
}

// ---- dropout ------------------------------------------------------------------------------------------------------------
// Philox4x32 with ten rounds (J. Salmon, M. Moraes, R. Dror, D. Shaw: Parallel random numbers: as easy as 1, 2, 3, SC 2011):
// four words from a counter and a key.  The counter is (element / 4 in two words, step, site), the key the seed; element e
// takes word e % 4.  So a mask is a function of its place alone and backward forms it again instead of reading it.
__device__ __forceinline__ void philox4x32(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1, uint32_t (&out)[4]) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    out[0] = c0; out[1] = c1; out[2] = c2; out[3] = c3;
}

// y = keep ? x * factor : 0, (+ residual).  One lane, one block of four elements, DROP_UNROLL blocks a workgroup apart.  An
// element that is dropped is selected away, not multiplied: what it held (an infinity, a NaN) does not show.  y may be x or
// the residual (a lane reads its elements before it writes them).  Bound by memory, the generator hides behind it: 8192 x 2048
// floats and a residual in 38 us, 5.3 TB/s; 49 x 96 doubles take 2.2 us, a launch.
constexpr int DROP_UNROLL = 2;

template <typename T, bool RES, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(const T* x, const T* res, T* y, int64_t n, uint32_t threshold,
                                                      T factor, uint32_t k0, uint32_t k1, uint32_t site, const int32_t* __restrict__ step) {
    typedef Pack<T, 16 / sizeof(T)> P;
    constexpr int PK = 16 / sizeof(T), PACKS = 4 / PK;
    const uint32_t at_step = step != nullptr ? (uint32_t)step[0] : 0u;
    const int64_t blocks = (n + 3) / 4;
    T v[DROP_UNROLL][4], rv[DROP_UNROLL][4];
#pragma unroll
    for (int u = 0; u < DROP_UNROLL; ++u) {
        const int64_t b = ((int64_t)blockIdx.x * DROP_UNROLL + u) * 256 + threadIdx.x;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[u][e] = rv[u][e] = (T)0;
        if (VEC && 4 * b + 3 < n) {
#pragma unroll
            for (int q = 0; q < PACKS; ++q) {
                const P p = reinterpret_cast<const P*>(x)[b * PACKS + q];
#pragma unroll
                for (int e = 0; e < PK; ++e) v[u][q * PK + e] = p.v[e];
                if (RES) {
                    const P w = reinterpret_cast<const P*>(res)[b * PACKS + q];
#pragma unroll
                    for (int e = 0; e < PK; ++e) rv[u][q * PK + e] = w.v[e];
                }
            }
        } else if (b < blocks) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * b + e < n) {
                    v[u][e] = x[4 * b + e];
                    if (RES) rv[u][e] = res[4 * b + e];
                }
        }
    }
#pragma unroll
    for (int u = 0; u < DROP_UNROLL; ++u) {
        const int64_t b = ((int64_t)blockIdx.x * DROP_UNROLL + u) * 256 + threadIdx.x;
        uint32_t word[4];
        philox4x32((uint32_t)b, (uint32_t)((uint64_t)b >> 32), at_step, site, k0, k1, word);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[u][e] = word[e] >= threshold ? v[u][e] * factor : (T)0;
            if (RES) v[u][e] = v[u][e] + rv[u][e];
        }
        if (VEC && 4 * b + 3 < n) {
#pragma unroll
            for (int q = 0; q < PACKS; ++q) {
                P p;
#pragma unroll
                for (int e = 0; e < PK; ++e) p.v[e] = v[u][q * PK + e];
                reinterpret_cast<P*>(y)[b * PACKS + q] = p;
            }
        } else if (b < blocks) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * b + e < n) y[4 * b + e] = v[u][e];
        }
    }
}

__global__ void __launch_bounds__(256) index_add_kernel(int32_t* __restrict__ v, int64_t n, int32_t delta) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) v[i] = (int32_t)((uint32_t)v[i] + (uint32_t)delta);
}

}  // namespace

template <typename T>
hipError_t launch_embedding_fwd(const T* table, const int32_t* ids, T* out, int64_t tokens, int64_t vocab, int64_t width, T scale, hipStream_t s) {
    constexpr int N = 16 / sizeof(T);
    const bool vec = width % N == 0 && aligned16({table, out});
    const int64_t packs = vec ? width / N : width;
    const int64_t per_block = 256 * LOOKUP_UNROLL;
    const int64_t groups = (tokens * packs + per_block - 1) / per_block;
    if (!grid_fits(groups, 256)) return hipErrorInvalidValue;
    const unsigned grid = (unsigned)groups;
    if (vec) hipLaunchKernelGGL((embedding_fwd_kernel<T, N>), dim3(grid), dim3(256), 0, s, table, ids, out, tokens, vocab, (uint32_t)packs, scale);
    else hipLaunchKernelGGL((embedding_fwd_kernel<T, 1>), dim3(grid), dim3(256), 0, s, table, ids, out, tokens, vocab, (uint32_t)packs, scale);
    return hipGetLastError();
}

size_t embedding_bwd_workspace_bytes(int64_t tokens, int64_t vocab, int64_t width) {
    if (one_launch(tokens, vocab)) return 0;
    return 256 + 2 * round256((size_t)tokens * 4) + 2 * (size_t)sum_chunks(tokens) * width * sizeof(double);
}

template <typename T>
hipError_t launch_embedding_bwd(const T* dout, const int32_t* ids, T* dtable, int64_t tokens, int64_t vocab, int64_t width, double scale, int accumulate,
                                void* workspace, hipStream_t s) {
    constexpr int N = 16 / sizeof(T);
    if (width % N == 0 && aligned16({dout, dtable})) return embedding_bwd_n<T, N>(dout, ids, dtable, tokens, vocab, width, scale, accumulate, workspace, s);
    return embedding_bwd_n<T, 1>(dout, ids, dtable, tokens, vocab, width, scale, accumulate, workspace, s);
}

template <typename T>
hipError_t launch_dropout(const T* x, const T* residual, T* y, int64_t n, double p, int64_t seed, int32_t site, const int32_t* step, hipStream_t s) {
    const uint32_t threshold = (uint32_t)(p * 4294967296.0);  // p < 1
    const T factor = (T)(1.0 / (1.0 - p));
    const uint32_t k0 = (uint32_t)(uint64_t)seed, k1 = (uint32_t)((uint64_t)seed >> 32);
    const int64_t blocks = (n + 3) / 4;
    const int64_t groups = (blocks + 256 * DROP_UNROLL - 1) / (256 * DROP_UNROLL);
    if (!grid_fits(groups, 256)) return hipErrorInvalidValue;
    const dim3 grid((unsigned)groups);
    const bool vec = aligned16({x, y}) && (residual == nullptr || aligned16({residual}));
    if (residual != nullptr) {
        if (vec) hipLaunchKernelGGL((dropout_kernel<T, true, true>), grid, dim3(256), 0, s, x, residual, y, n, threshold, factor, k0, k1, (uint32_t)site, step);
        else hipLaunchKernelGGL((dropout_kernel<T, true, false>), grid, dim3(256), 0, s, x, residual, y, n, threshold, factor, k0, k1, (uint32_t)site, step);
    } else {
        if (vec) hipLaunchKernelGGL((dropout_kernel<T, false, true>), grid, dim3(256), 0, s, x, residual, y, n, threshold, factor, k0, k1, (uint32_t)site, step);
        else hipLaunchKernelGGL((dropout_kernel<T, false, false>), grid, dim3(256), 0, s, x, residual, y, n, threshold, factor, k0, k1, (uint32_t)site, step);
    }
    return hipGetLastError();
}

hipError_t launch_index_add(int32_t* v, int64_t n, int32_t delta, hipStream_t s) {
    if (!grid_fits((n + 255) / 256, 256)) return hipErrorInvalidValue;
    hipLaunchKernelGGL(index_add_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, v, n, delta);
    return hipGetLastError();
}

#define INSTANTIATE(T)                                                                                                                          \
    template hipError_t launch_embedding_fwd<T>(const T*, const int32_t*, T*, int64_t, int64_t, int64_t, T, hipStream_t);                       \
    template hipError_t launch_embedding_bwd<T>(const T*, const int32_t*, T*, int64_t, int64_t, int64_t, double, int, void*, hipStream_t);      \
    template hipError_t launch_dropout<T>(const T*, const T*, T*, int64_t, double, int64_t, int32_t, const int32_t*, hipStream_t);
INSTANTIATE(float)
INSTANTIATE(double)
#undef INSTANTIATE

}  // namespace prad
