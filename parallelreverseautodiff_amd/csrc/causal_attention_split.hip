// Causal attention in float for long batches: the products run on the half-precision matrix instructions.
//
// A float x scaled by a power of two is held as two halves, x = hi + lo with hi the nearest half and lo the nearest half to the
// rest: 22 bits.  A product of two such numbers is three products of halves, hi hi + hi lo + lo hi, summed in float by the matrix
// instruction; what is left out, lo lo and the rest behind lo, is below 2^-21 of the product, the size of a float's own
// rounding.  The half instructions run at sixteen times the rate of the float ones, so three of them take a fifth of the time
// (library products on this card: 1060 TFLOP/s in half, 153 in float) - and they overlap with vector instructions, which the
// float ones do not.
//
// Scaling.  A half has 11 bits from 2^-14 on and ends at 2^-24, so an element keeps its 11 + 11 bits, off by 2^-23 of itself at most,
// down to 2^-2 or so; what is below that is off by 2^-25.  The rows of a tile (64 rows of one head) are scaled by one power of two that takes the largest
// magnitude in it to [2^11, 2^15), as long as no row's largest is more than 2^10 below that: every row is then right to 2^-23 of
// its own largest.  In an uneven tile each row has a power of its own; those go onto the scores, onto dP and onto the weights, row
// by row.  Where tiles are summed in one accumulator, the ratio of their powers is folded into the weights, in float.  The weights
// of a column (a query forward, a key or a query backward), with that ratio, are scaled by a power of two that belongs to the
// column and falls when one no longer fits into a half, the accumulators of the column with it: forward that is a running maximum
// beside the softmax's own, backward `fit`.  So it follows what really enters the sum: large values that a column does not see,
// or gives next to no weight, cost it no bits.
//
// Layout.  A first launch splits the operands and writes them in the order in which the 32 x 32 x 16 matrix instruction takes
// its fragments: lane l of a fragment holds 8 halves, row l % 32, elements 8 (l / 32) + e along the head dimension; a fragment is
// 1 KB, copied to LDS as it is and read back without bank conflicts.  Rows and columns past the end are zeros, so the
// main kernels check no bounds.  Which element of the reduction sits where is free as long as both operands agree: the weights
// come out of the first product with a column per lane and 4-row groups alternating between the lane halves, and the same
// fragments, read across by the transposing LDS loads, take the rows in that order, so weights go from one product into the next
// without leaving their lane and an operand is held once, whichever side it is needed from.
//
// A non-finite value is replaced by zero in the split operands and its row marked: where it is seen, scores (forward) or
// lse / D (backward) are NaN.
#include "common.h"

#include <algorithm>
#include <initializer_list>
#include <type_traits>

namespace prad {

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int NO_EXPONENT = -1000;   // of zeros
// How far (powers of two) the largest values of two rows of a tile lie apart before rows get powers of their own.
constexpr int MOST_SPREAD = 10;

// What the first launch notes about a tile of 64 rows.
struct Header {
    int e;                  // the power of its largest value: an even tile was scaled by 2^-e
    int uneven;             // rows were scaled by powers of their own
    uint32_t bad[2];        // rows that hold a non-finite value
};

__device__ __forceinline__ int64_t clamped(int64_t v, int64_t most) { return v < 0 ? 0 : v > most ? most : v; }
__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < INFINITY; }
// x < 2^power_of(x)
__device__ __forceinline__ int power_of(float x) {
    if (!(x > 0.f)) return NO_EXPONENT;
    int e;
    (void)frexpf(x, &e);
    return e;
}
// The power that takes the largest magnitude of some values to [2^11, 2^15).  A multiple of 4, so that tiles of about the same size
// have the same.
__device__ __forceinline__ int power_for(float top) { return top > 0.f ? (power_of(top) - 12) & ~3 : NO_EXPONENT; }
// 2^e, within the normal numbers
__device__ __forceinline__ float pow2(int e) { return __builtin_ldexpf(1.0f, e < -126 ? -126 : e > 127 ? 127 : e); }

// Tiles of 64 packed rows (token, head of the group) are numbered as in causal_attention.hip: sequence s begins at
// floor(offset G / R) + s.
// (Packed rows, with some tiles behind the last, are counted in 31 bits; tiles and sequences together in 32.)
__device__ __forceinline__ uint32_t first_tile(const CausalArgs<float>& p, int s, uint32_t group, uint32_t R) { return (uint32_t)clamped(p.q_off[s], p.q_rows) * group / R + s; }
__device__ __forceinline__ bool find_tile(const CausalArgs<float>& p, uint32_t group, uint32_t R, uint32_t tile, int* sequence, uint32_t* inside) {
    int lo = 0, hi = p.sequences;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (first_tile(p, mid, group, R) <= tile) lo = mid + 1;
        else hi = mid;
    }
    if (lo == 0) return false;
    *sequence = lo - 1;
    *inside = tile - first_tile(p, lo - 1, group, R);
    return true;
}
__device__ __forceinline__ void sequence_rows(const CausalArgs<float>& p, int s, uint32_t* q0, uint32_t* n) {
    *q0 = (uint32_t)clamped(p.q_off[s], p.q_rows);
    const uint32_t q1 = (uint32_t)clamped(p.q_off[s + 1], p.q_rows);
    *n = q1 > *q0 ? q1 - *q0 : 0;
}

// hi = nearest halves, lo = nearest halves to the rest.  `minus_one` is a register the compiler does not see through, which
// makes x - hi one mixed-precision instruction instead of a conversion and a subtraction.
__device__ __forceinline__ void split2(float a, float b, float minus_one, h2* hi, h2* lo) {
    const f2 v = {a, b};
    const h2 h = __builtin_convertvector(v, h2);
    const f2 r = {__builtin_fmaf((float)h.x, minus_one, a), __builtin_fmaf((float)h.y, minus_one, b)};
    *hi = h;
    *lo = __builtin_convertvector(r, h2);
}
__device__ __forceinline__ float opaque_minus_one() {
    float m = -1.0f;
    asm("" : "+s"(m));
    return m;
}
// Values are formed before this point: the compiler would otherwise move them past the next branch, towards their use and away
// from the matrix instructions they are meant to run beside.
__device__ __forceinline__ void keep_here(h8 (&hi)[2], h8 (&lo)[2]) { asm volatile("" : "+v"(hi[0]), "+v"(hi[1]), "+v"(lo[0]), "+v"(lo[1])); }
template <int N>
__device__ __forceinline__ void split_regs(const float (&x)[N], float minus_one, h8 (&hi)[N / 8], h8 (&lo)[N / 8]) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        h2 h, l;
        split2(x[i], x[i + 1], minus_one, &h, &l);
        hi[i / 8][i % 8] = h.x; hi[i / 8][i % 8 + 1] = h.y;
        lo[i / 8][i % 8] = l.x; lo[i / 8][i % 8 + 1] = l.y;
    }
}

// acc += (a_hi + a_lo) (b_hi + b_lo) without lo lo, the small parts first
__device__ __forceinline__ void mfma3(h8 a_hi, h8 a_lo, h8 b_hi, h8 b_lo, f16v& acc) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a_lo, b_hi, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a_hi, b_lo, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a_hi, b_hi, acc, 0, 0, 0);
}
// Row of accumulator element r in lane half h.
__device__ __forceinline__ int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// ---- first launch: split operands ------------------------------------------------------------------------------------------
// A block of 32 rows of a tile is 128 HDP bytes, [plane][HDP / 16][lane][8] with row l % 32 and columns 16 k + 8 (l / 32) + e in
// lane l of fragment k.  A tile is two blocks; tile and head (slot, kv) lie at (slot kv_heads + kv) 256 HDP bytes.
struct SplitSource {
    const float* src;
    int64_t ld;
    int group;         // heads per packed row group (1: keys)
    int vec;
    _Float16* split;
    Header* header;
    int* powers;       // of the 64 rows of a tile: scaled by 2^-power
    int dots;          // dO: D and lse of the rows as well
};
struct SplitArgs {
    CausalArgs<float> p;
    SplitSource t[4];
    int tensors;
    int4* order;       // schedules for the main kernels, see below
    int order_slots[2];
    int shift;
    float* row_notes;  // [slot][kv][2][64]: -lse log2 e (-inf for a row that is not there), then D
    int* e_dot;        // [slot][kv]: |D| < 2^e_dot
};

// The groups of 128 packed rows (which = 0) or 128 keys (1) of all sequences as (sequence, number inside it, first row of the
// sequence, its length), those with the most
// work first: the last workgroups to finish are then short ones.  Which of two with about equal work comes first is left to
// chance and shows in no result.  With an entry a workgroup knows all its addresses: its first copies wait for one load.  One workgroup, beside the ones that split.
constexpr int ORDER_BINS = 1024;
__device__ __forceinline__ void write_order(const CausalArgs<float>& p, int which, int slots, int shift, int4* __restrict__ order, int* bins) {
    __shared__ int wave_total[4];
    const int lane = threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const uint32_t group = which == 0 ? p.group : 1;
    for (int i = threadIdx.x; i < ORDER_BINS; i += 256) bins[i] = 0;
    __syncthreads();
    for (int pass = 0; pass < 2; ++pass) {
        for (int slot = threadIdx.x; slot < slots; slot += 256) {
            int s = -1;
            uint32_t inside = 0, q0 = 0, n = 0;
            int work = -1;  // in tiles of 64 keys or tokens
            if (find_tile(p, group, 128, slot, &s, &inside)) {
                sequence_rows(p, s, &q0, &n);
                if (inside < (n * group + 127) / 128) work = which == 0 ? (inside * 128 + 127) / group / 64 : (n - 1 - inside * 128) / 64;
            }
            const int bin = work < 0 ? ORDER_BINS - 1 : (work >> shift) > ORDER_BINS - 2 ? 0 : ORDER_BINS - 2 - (work >> shift);
            const int at = atomicAdd(&bins[bin], 1);
            if (pass == 1) order[at] = int4{work < 0 ? -1 : s, (int)inside, (int)q0, (int)n};
        }
        __syncthreads();
        if (pass == 1) break;
        // counts to first places
        int mine[ORDER_BINS / 256], total = 0;
#pragma unroll
        for (int i = 0; i < ORDER_BINS / 256; ++i) {
            mine[i] = total;
            total += bins[threadIdx.x * (ORDER_BINS / 256) + i];
        }
        int before = total;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int v = __shfl_up(before, off, 64);
            if (lane >= off) before += v;
        }
        if (lane == 63) wave_total[wave] = before;
        __syncthreads();
        int base = before - total;
        for (int w = 0; w < wave; ++w) base += wave_total[w];
#pragma unroll
        for (int i = 0; i < ORDER_BINS / 256; ++i) bins[threadIdx.x * (ORDER_BINS / 256) + i] = base + mine[i];
        __syncthreads();
    }
}

// Where lane l's 16 bytes lie among the 64 of fragment f.  Two bits of the row are turned over by the lane half and by the
// fragment's parity: a transposing load asks for 4 rows of 2 fragments and both halves at a time, which lie 1 KB and 512 bytes
// apart and would be in the same LDS banks.  (Fragments that are read along stay one KB in a row.)
__device__ __forceinline__ int place_in_fragment(int f, int l) { return l ^ (l >> 5) << 2 ^ (f & 1) << 3; }

// Over each LANES lanes, in all of them.
template <int LANES>
__device__ __forceinline__ float max_of(float x) {
    auto with = [&](int other) { x = fmaxf(x, __int_as_float(other)); };
    with(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xf, 0xf, true));
    with(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4E, 0xf, 0xf, true));
    with(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x141, 0xf, 0xf, true));
    if (LANES > 8) with(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x140, 0xf, 0xf, true));
    if (LANES > 16) x = fmaxf(x, __shfl_xor(x, 16, 64));
    return x;
}

template <int HDP>
__global__ void __launch_bounds__(256) causal_split_kernel(const SplitArgs a) {
    constexpr int PITCH = HDP + 4, PER_ROW = HDP / 4, COUNT = 64 * PER_ROW / 256;
    static_assert(64 * PITCH >= ORDER_BINS, "the tile's room also holds the bins of a schedule");
    __shared__ __attribute__((aligned(16))) float tile[64 * PITCH];
    __shared__ float row_top[64], row_dots[64];
    __shared__ int bad[64];
    const CausalArgs<float>& p = a.p;
    if ((int)blockIdx.z == a.tensors) {
        if (blockIdx.y == 0 && blockIdx.x < 2 && a.order_slots[blockIdx.x] > 0)
            write_order(p, blockIdx.x, a.order_slots[blockIdx.x], a.shift, a.order + (blockIdx.x == 0 ? 0 : a.order_slots[0]), reinterpret_cast<int*>(tile));
        return;
    }
    const SplitSource t = a.t[blockIdx.z];
    const int kv = blockIdx.y;
    int s;
    uint32_t inside, first, n;
    const uint32_t group = t.group;
    if (!find_tile(p, group, 64, blockIdx.x, &s, &inside)) return;
    sequence_rows(p, s, &first, &n);
    const uint32_t rows = n * group, row0 = inside * 64;
    if (inside >= (rows + 63) / 64) return;
    const int64_t q0 = first;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (threadIdx.x < 64) bad[threadIdx.x] = 0;
    __syncthreads();
    f4 v[COUNT];
#pragma unroll
    for (int u = 0; u < COUNT; ++u) {
        const int at = threadIdx.x + 256 * u, j = at / PER_ROW, d = (at % PER_ROW) * 4;
        const uint32_t r = row0 + j, token = r / group;
        v[u] = f4{0.f, 0.f, 0.f, 0.f};
        if (r < rows && d < p.head_dim) {
            const float* __restrict__ src = t.src + (q0 + token) * t.ld + (kv * group + (r - token * group)) * (int64_t)p.head_dim + d;
            if (t.vec) {
                v[u] = *reinterpret_cast<const f4*>(src);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < p.head_dim) v[u][e] = src[e];
            }
        }
    }
#pragma unroll
    for (int u = 0; u < COUNT; ++u) {
        const int j = (threadIdx.x + 256 * u) / PER_ROW;
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (!is_finite(v[u][e])) {
                v[u][e] = 0.f;
                bad[j] = 1;
            }
            top = fmaxf(top, fabsf(v[u][e]));
        }
        row_top[j] = max_of<PER_ROW>(top);  // (every lane of the row the same)
    }
    // D = rowsum(dO (.) O): the PER_ROW lanes that hold a row of dO
    if (t.dots) {
#pragma unroll
        for (int u = 0; u < COUNT; ++u) {
            const int at = threadIdx.x + 256 * u, j = at / PER_ROW, d = (at % PER_ROW) * 4;
            const uint32_t r = row0 + j, down = r / group;
            const int64_t token = q0 + down, head = kv * group + (r - down * group);
            float dot = 0.f;
            if (r < rows && d < p.head_dim) {
                const float* __restrict__ o = p.O + token * p.ldo + head * p.head_dim + d;
                f4 y = {0.f, 0.f, 0.f, 0.f};
                if (t.vec) {
                    y = *reinterpret_cast<const f4*>(o);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (d + e < p.head_dim) y[e] = o[e];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) dot = __builtin_fmaf(v[u][e], y[e], dot);
            }
#pragma unroll
            for (int m = 1; m < PER_ROW; m <<= 1) dot += __shfl_xor(dot, m, 64);
            row_dots[j] = dot;  // (every lane of the row the same)
        }
    }
    __syncthreads();
    // One power for the tile, or one for each row where some are far below the largest: each wavefront for itself, a row per lane.
    // (A row with a non-finite value does not count: whoever sees it gets NaN, and the others keep their bits.)
    const float top_here = row_top[lane], top = wave_max_t(top_here);
    const int e = power_for(top);
    const bool uneven = __ballot(row0 + lane < rows && bad[lane] == 0 && top > 0.f && power_of(top) - power_of(top_here) > MOST_SPREAD) != 0;
    const int64_t tile_at = (int64_t)blockIdx.x * p.kv_heads + kv;
    if (wave == 0) {
        const uint64_t marks = __ballot(bad[lane] != 0);
        if (lane == 0) t.header[tile_at] = Header{e, uneven, {(uint32_t)marks, (uint32_t)(marks >> 32)}};
        t.powers[tile_at * 64 + lane] = uneven ? power_for(top_here) : e;
        if (t.dots) {
            const uint32_t r = row0 + lane, down = r / group;
            const int64_t token = q0 + down, head = kv * group + (r - down * group);
            float dot = row_dots[lane], lse = -INFINITY, size = 0.f;
            if (r < rows) {
                if (!is_finite(dot) || bad[lane] != 0) dot = NAN;
                else size = fabsf(dot);
                lse = (dot - dot) - p.lse[head * p.q_rows + token] * LOG2E;  // NaN where D is
            }
            a.row_notes[tile_at * 128 + lane] = lse;
            a.row_notes[tile_at * 128 + 64 + lane] = dot;
            const int e_dot = power_of(wave_max_t(size));
            if (lane == 0) a.e_dot[tile_at] = e_dot;
        }
    }
#pragma unroll
    for (int u = 0; u < COUNT; ++u) {
        const int at = threadIdx.x + 256 * u, j = at / PER_ROW, d = (at % PER_ROW) * 4;
        const int by = uneven ? power_for(row_top[j]) : e;
        f4 w;
#pragma unroll
        for (int c = 0; c < 4; ++c) w[c] = top > 0.f ? __builtin_ldexpf(v[u][c], -by) : 0.f;
        *reinterpret_cast<f4*>(tile + j * PITCH + d) = w;
    }
    __syncthreads();
    const float minus_one = opaque_minus_one();
    const int64_t base = tile_at * (128 * HDP);  // halves
    constexpr int FRAGS = HDP / 16;  // per block and plane
#pragma unroll
    for (int u = 0; u < 2 * FRAGS * 64 / 256; ++u) {
        const int at = threadIdx.x + 256 * u, l = at & 63, f = (at >> 6) % FRAGS, block = (at >> 6) / FRAGS;
        const int64_t hi_at = base + (int64_t)(block * 2 * FRAGS + f) * 512 + place_in_fragment(f, l) * 8, lo_at = hi_at + FRAGS * 512;
        float x[8];
        h8 hi[1], lo[1];
        const float* __restrict__ row = tile + (32 * block + (l & 31)) * PITCH + 16 * f + 8 * (l >> 5);
#pragma unroll
        for (int c = 0; c < 8; ++c) x[c] = row[c];
        split_regs<8>(x, minus_one, hi, lo);
        *reinterpret_cast<h8*>(t.split + hi_at) = hi[0];
        *reinterpret_cast<h8*>(t.split + lo_at) = lo[0];
    }
}

// ---- staging ----------------------------------------------------------------------------------------------------------------
// Copies BYTES of split operands to LDS without passing through registers: 1 KB per instruction and wavefront.  As buffer loads:
// their flat form would count as an LDS access to the compiler, which then waits for all LDS reads wherever it waits for one.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* base, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00027000);
}
template <int BYTES, int WAVES>
__device__ __forceinline__ void stage(const _Float16* __restrict__ src, _Float16* dst, int wave, int lane) {
    static_assert(BYTES % (1024 * WAVES) == 0, "whole rounds");
    const __amdgpu_buffer_rsrc_t from = buffer_of(src, BYTES);
#pragma unroll
    for (int i = 0; i < BYTES / 1024 / WAVES; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)(dst + (i * WAVES + wave) * 512), 16, lane * 16,
                                                 (i * WAVES + wave) * 1024, 0, 0);
}
// The copies of every wavefront have arrived, and every wavefront is done with what they replace next.
__device__ __forceinline__ void staged() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}
__device__ __forceinline__ h8 frag(const _Float16* base, int f, int lane) { return *reinterpret_cast<const h8*>(base + f * 512 + place_in_fragment(f, lane) * 8); }

// Asks the scheduler for this order of instructions in a basic block: `n` LDS reads, `n` matrix instructions.  Without it the
// fragments are read right before they are used and every step waits for LDS.
__device__ __forceinline__ void then_reads(std::integral_constant<int, 2>) { __builtin_amdgcn_sched_group_barrier(0x100, 2, 0); }
__device__ __forceinline__ void then_reads(std::integral_constant<int, 4>) { __builtin_amdgcn_sched_group_barrier(0x100, 4, 0); }
__device__ __forceinline__ void then_products() { __builtin_amdgcn_sched_group_barrier(0x008, 3, 0); }

// A chain of STEPS products of fragments, the fragments of a step read while the step before it multiplies.  read(i, hi, lo),
// multiply(i, hi, lo).  BESIDE: vector instructions of the same basic block that do not depend on the chain go between its
// matrix instructions.
template <int STEPS, int READS, bool BESIDE = false, typename Read, typename Multiply>
__device__ __forceinline__ void product_chain(Read read, Multiply multiply) {
    h8 hi[2], lo[2];
    read(0, hi[0], lo[0]);
    then_reads(std::integral_constant<int, READS>());
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        if (i + 1 < STEPS) {
            read(i + 1, hi[(i + 1) & 1], lo[(i + 1) & 1]);
            then_reads(std::integral_constant<int, READS>());
        }
        multiply(i, hi[i & 1], lo[i & 1]);
        if constexpr (BESIDE) {
#pragma unroll
            for (int x = 0; x < 3; ++x) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
                __builtin_amdgcn_sched_group_barrier(0x400, 2, 0);
            }
        } else {
            then_products();
        }
    }
}
__device__ __forceinline__ void clear(f16v& acc) {
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0.f;
}
// first, second [32 rows x 32 columns] = A . B over the head dimension: two blocks, each against a column per lane.
template <int HDP>
__device__ __forceinline__ void rows_products(const _Float16* first_block, const h8 (&f_hi)[HDP / 16], const h8 (&f_lo)[HDP / 16], f16v& first,
                                              const _Float16* second_block, const h8 (&s_hi)[HDP / 16], const h8 (&s_lo)[HDP / 16], f16v& second, int lane) {
    constexpr int K = HDP / 16;
    clear(first);
    clear(second);
    product_chain<2 * K, 2>(
        [&](int i, h8& hi, h8& lo) {
            const _Float16* block = i < K ? first_block : second_block;
            hi = frag(block, i % K, lane);
            lo = frag(block, K + i % K, lane);
        },
        [&](int i, h8 hi, h8 lo) {
            if (i < K) mfma3(hi, lo, f_hi[i % K], f_lo[i % K], first);
            else mfma3(hi, lo, s_hi[i % K], s_lo[i % K], second);
        });
}
template <int HDP, bool BESIDE = false>
__device__ __forceinline__ void rows_product(const _Float16* block, const h8 (&b_hi)[HDP / 16], const h8 (&b_lo)[HDP / 16], f16v& acc, int lane) {
    constexpr int K = HDP / 16;
    clear(acc);
    product_chain<K, 2, BESIDE>(
        [&](int i, h8& hi, h8& lo) {
            hi = frag(block, i, lane);
            lo = frag(block, K + i, lane);
        },
        [&](int i, h8 hi, h8 lo) { mfma3(hi, lo, b_hi[i], b_lo[i], acc); });
}
// Fragment of a block read across, from LDS: lane l gets column 32 c + l % 32, rows acc_row(8 t + e, l / 32).  One transposing load
// gives each 16 lanes 4 rows of 16 columns: its lane i asks for columns 4 (i % 4) .. + 3 of row i / 4 and receives column i.
typedef short s4 __attribute__((ext_vector_type(4)));
struct Across {
    int at;  // of the lane, in halves; 8 rows on: the other value of that bit
    __device__ __forceinline__ explicit Across(int lane) {
        const int i = lane & 15;
        const int f = (lane >> 4) & 1, half = (i >> 1) & 1;
        at = f * 512 + place_in_fragment(f, 32 * half + 4 * (lane >> 5) + (i >> 2)) * 8 + (i & 1) * 4;
    }
    __device__ __forceinline__ h8 frag(const _Float16* plane, int c, int t) const {
        typedef __attribute__((address_space(3))) s4* lds;
        const _Float16* from = plane + c * 1024 + t * 128;
        const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(from + at)), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(from + (at ^ 64)));
        typedef short s8 __attribute__((ext_vector_type(8)));
        return __builtin_bit_cast(h8, s8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
    }
};
// out[HDP x 32 columns] += A^T . W: a block read across against the weights of its 32 rows.
template <int HDP, bool BESIDE = false>
__device__ __forceinline__ void columns_product(const _Float16* block, const h8 (&w_hi)[2], const h8 (&w_lo)[2], const Across& across, f16v (&out)[HDP / 32]) {
    product_chain<HDP / 16, 4, BESIDE>(
        [&](int i, h8& hi, h8& lo) {
            hi = across.frag(block, i / 2, i % 2);
            lo = across.frag(block + 32 * HDP, i / 2, i % 2);
        },
        [&](int i, h8 hi, h8 lo) { mfma3(hi, lo, w_hi[i % 2], w_lo[i % 2], out[i / 2]); });
}

__device__ __forceinline__ int wave_max_int(int v) {
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xf, 0xf, false));   // inside each 2 lanes, 4, 8, 16
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xf, 0xf, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xf, 0xf, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xf, 0xf, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xa, 0xf, false));  // with the 16 before, with the 32 before
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x143, 0xc, 0xf, false));
    return __builtin_amdgcn_readlane(v, 63);
}
// Over the two lanes that share a column (lane halves).
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---- forward ----------------------------------------------------------------------------------------------------------------
struct ForwardArgs {
    CausalArgs<float> p;
    const _Float16* k;
    const _Float16* v;
    const Header* hk;
    const Header* hv;
    const int* powers_k;
    const int* powers_v;
    const int4* order;
};

// A workgroup takes 128 packed rows of a key/value head, a wavefront 32 of them, a row per lane (of either half): S^T = K Q^T has
// a query's scores in its lane, its statistics are sums over registers.  K and V pass through LDS in tiles of 64 keys, the next
// one copied while this one is used.
template <int HDP, int KEYS>
struct ForwardTile {
    static constexpr int BLOCKS = KEYS / 32;
    _Float16 k[BLOCKS][64 * HDP];   // (a block of 32 rows: 2 planes of 32 HDP halves)
    _Float16 v[BLOCKS][64 * HDP];
};

// x[r] times 2^(power of its row + by): rows of a block of an uneven tile.
template <typename X>
__device__ __forceinline__ void take_powers(X& x, const int* __restrict__ powers, int by, int h) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int4 e = *reinterpret_cast<const int4*>(powers + 8 * q + 4 * h);
#pragma unroll
        for (int c = 0; c < 4; ++c) x[4 * q + c] = __builtin_ldexpf(x[4 * q + c], (&e.x)[c] + by);
    }
}
// The same for dP, with D and another power p2 of the row: (dP 2^(power + by) - D) 2^(p2 + by2).  D of the row, or of the lane.
__device__ __forceinline__ void take_powers(f16v& dp, const int* __restrict__ powers, int by, int h, const int* __restrict__ powers2, int by2, const float* dot,
                                            int dot_step = 1) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int4 e = *reinterpret_cast<const int4*>(powers + 8 * q + 4 * h), e2 = *reinterpret_cast<const int4*>(powers2 + 8 * q + 4 * h);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int out = (&e2.x)[c] + by2;
            dp[4 * q + c] = __builtin_ldexpf(dp[4 * q + c], (&e.x)[c] + by + out) - __builtin_ldexpf(dot[dot_step * (8 * q + 4 * h + c)], out);
        }
    }
}

// What the headers of a tile of keys say.  They are asked for with the copies of the tile and looked at (`uniform`) once those have
// arrived: touching them earlier would wait for the copies.
struct KeyNotes {
    Header k, v;
    int power;  // (of uniform()) K's, or one above all if the tile is uneven
    // the same value in every lane: to scalar registers
    __device__ __forceinline__ KeyNotes uniform() const {
        KeyNotes n;
        n.k.e = __builtin_amdgcn_readfirstlane(k.e);
        n.v.e = __builtin_amdgcn_readfirstlane(v.e);
        n.power = __builtin_amdgcn_readfirstlane((k.uneven | v.uneven) != 0 ? -NO_EXPONENT : k.e);
        n.k.bad[0] = __builtin_amdgcn_readfirstlane(k.bad[0] | v.bad[0]);
        n.k.bad[1] = __builtin_amdgcn_readfirstlane(k.bad[1] | v.bad[1]);
        return n;
    }
};

template <int HDP, int KEYS>
__device__ __forceinline__ void forward_stage(const ForwardArgs& a, ForwardTile<HDP, KEYS>& t, KeyNotes& notes, int64_t tile0, int kv, int k0, int wave,
                                              int lane) {
    const int64_t tile_at = (tile0 + k0 / 64) * a.p.kv_heads + kv;
    const int64_t at = tile_at * (128 * HDP) + (k0 / KEYS % (64 / KEYS)) * (2 * KEYS * HDP);
    notes.k = a.hk[tile_at];
    notes.v = a.hv[tile_at];
    stage<4 * KEYS * HDP, 4>(a.k + at, &t.k[0][0], wave, lane);
    stage<4 * KEYS * HDP, 4>(a.v + at, &t.v[0][0], wave, lane);
}

template <int HDP>
struct ForwardState {
    h8 q_hi[HDP / 16], q_lo[HDP / 16];
    f16v o[HDP / 32];
    float m, l;        // the maximum the sum refers to (in units of log2 e, whole): sum of 2^(score - m + 8), this lane half's share
    float x;           // the same for o: sum of 2^(score + e - x + 8) V 2^-e, e the power of V; behind the last tile x - m
    int e_row;         // exponent of the row of Q
    int last;          // the last key that the lane's row sees
};

// Masks and marks of a block of 32 scores per row, the first of them of key k0: only where some row does not see all the keys, or
// some key holds a non-finite value.
template <int HDP>
__device__ __forceinline__ void forward_mask(f16v& s, uint32_t marks, int k0, int wave_first, int h, const ForwardState<HDP>& st) {
    if (k0 + 31 > wave_first || marks != 0) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int j = acc_row(r, h);
            s[r] = k0 + j > st.last ? -INFINITY : ((marks >> j) & 1) != 0 ? NAN : s[r];
        }
    }
}
// Scores to weights, split.  A weight meets V scaled by 2^-e_tile: what enters the accumulators is 2^(score + e_tile), and the
// reference x of the weights follows the largest of those, so that a tile of large values whose weight is next to nothing takes no
// bits from the others.  The sum of the weights follows the largest score, m: it takes the weights of a block with the ratio of the
// two references, which are whole numbers.  Both are raised only when the largest has risen by more than 2^6 (weights reach
// 2^6 2^8), so that the accumulators are rarely rescaled (by the factor returned).  No key seen yet: -inf, and a top of -inf keeps
// the weights at 0.  (Scores of up to 2^MOST_SCORE: the references, and powers beside them, are whole numbers of 24 bits.)
constexpr float FAR = 60.f;
constexpr int MOST_SCORE = 23;
template <int HDP>
__device__ __forceinline__ float forward_weights(f16v& s, float c, float e_tile, float minus_one, ForwardState<HDP>& st, h8 (&hi)[2], h8 (&lo)[2], bool* far) {
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
    top = max_halves(top) * c;
    const bool raise = top > st.m + 6.f, raise_o = top + e_tile > st.x + 6.f;
    const float whole = ceilf(top), m = raise ? whole : st.m, x = raise_o ? whole + e_tile : st.x;
    const float f = __builtin_amdgcn_exp2f(raise ? st.m - m : 0.f), fo = __builtin_amdgcn_exp2f(raise_o ? st.x - x : 0.f);  // (-inf before: 0)
    st.m = m;
    st.x = x;
    // A tile so small that all of it is below 2^-40 of what the accumulators hold (or zeros): its weights are formed for the sum
    // alone, where the reference of the accumulators would take them below the smallest float.
    const float ref = fmaxf(fminf(x - (e_tile + 8.f), m + (FAR - 8.f)), -1e30f);  // (finite where both are not)
    *far = x - (e_tile + 8.f) > m + (FAR - 8.f);
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    float w[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        w[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -ref));
        sum[r & 3] += w[r];
    }
    st.l = __builtin_fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ref + 8.f - m), st.l * f);
    split_regs<16>(w, minus_one, hi, lo);
    keep_here(hi, lo);
    return fo;
}
// Before the weights of a block meet V: the accumulators follow the weights' reference.
template <int HDP>
__device__ __forceinline__ void forward_rescale(float f, bool far, ForwardState<HDP>& st, h8 (&hi)[2], h8 (&lo)[2]) {
    if (__ballot(f != 1.f) != 0) {
#pragma unroll
        for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) st.o[d][r] *= f;
    }
    if (__ballot(far) != 0) {
        const _Float16 keep = far ? 0.f : 1.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            hi[i] *= keep;
            lo[i] *= keep;
        }
    }
}

// `forward_weights` in uneven tiles (scores are in units of log2 e, `powers` those of the 32 values of the block) and for scores of
// any size: all that enters an exponential is a difference from m, and x is kept as one.
template <int HDP>
__device__ __forceinline__ float forward_uneven_weights(f16v& s, const int* __restrict__ powers, float minus_one, int h, ForwardState<HDP>& st, h8 (&hi)[2],
                                                        h8 (&lo)[2]) {
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
    top = max_halves(top);
    const bool raise = top - st.m > 6.f;
    const float m = raise ? ceilf(top) : st.m, down = raise ? st.m - m : 0.f, zero = m == -INFINITY ? 0.f : m;  // (m = -inf before: -inf)
    st.m = m;
    st.x += down;
    float sum = 0.f, top_o = -INFINITY;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int4 e = *reinterpret_cast<const int4*>(powers + 8 * q + 4 * h);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float z = s[4 * q + c] - zero;
            sum += __builtin_amdgcn_exp2f(z + 8.f);
            s[4 * q + c] = z + (float)(&e.x)[c];
            top_o = fmaxf(top_o, s[4 * q + c]);
        }
    }
    st.l = __builtin_fmaf(st.l, __builtin_amdgcn_exp2f(down), sum);
    top_o = max_halves(top_o);
    const bool raise_o = top_o - st.x > 6.f;
    const float x = raise_o ? ceilf(top_o) : st.x, f = __builtin_amdgcn_exp2f(raise_o ? st.x - x : 0.f);
    st.x = x;
    float w[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] = __builtin_amdgcn_exp2f(s[r] - (x - 8.f));
    split_regs<16>(w, minus_one, hi, lo);
    return f;
}

// A tile of KEYS keys against the wavefront's rows, block by block: the second block's scores are formed beside the first one's
// softmax, the first one's product with V beside the second one's softmax.  powers_k, powers_v: of the tile's keys.
template <int HDP, int KEYS, bool UNEVEN>
__device__ __forceinline__ void forward_tile(const ForwardTile<HDP, KEYS>& t, const KeyNotes& notes, const int* __restrict__ powers_k,
                                             const int* __restrict__ powers_v, int k0, int wave_first, float minus_one, int lane, ForwardState<HDP>& st) {
    const int h = lane >> 5, first_mark = k0 / 32 % 2;
    const Across across(lane);
    const float c = pow2(st.e_row + notes.k.e), e_v = (float)notes.v.e;
    f16v s[KEYS / 32];
    h8 hi[2], lo[2];
    bool far = false;
    auto weights = [&](f16v& s, int block, h8(&hi)[2], h8(&lo)[2]) __attribute__((always_inline)) {
        if constexpr (UNEVEN) return forward_uneven_weights<HDP>(s, powers_v + 32 * block, minus_one, h, st, hi, lo);
        else return forward_weights<HDP>(s, c, e_v, minus_one, st, hi, lo, &far);
    };
    rows_product<HDP>(&t.k[0][0], st.q_hi, st.q_lo, s[0], lane);
    if constexpr (UNEVEN) take_powers(s[0], powers_k, st.e_row, h);
    forward_mask<HDP>(s[0], notes.k.bad[KEYS == 64 ? 0 : first_mark], k0, wave_first, h, st);
    if constexpr (KEYS == 64) rows_product<HDP, true>(&t.k[1][0], st.q_hi, st.q_lo, s[1], lane);
    float f = weights(s[0], 0, hi, lo);
    forward_rescale<HDP>(f, far, st, hi, lo);
    if constexpr (KEYS == 64) {
        if constexpr (UNEVEN) take_powers(s[1], powers_k + 32, st.e_row, h);
        forward_mask<HDP>(s[1], notes.k.bad[1], k0 + 32, wave_first, h, st);
        columns_product<HDP, true>(&t.v[0][0], hi, lo, across, st.o);
        h8 hi2[2], lo2[2];
        f = weights(s[1], 1, hi2, lo2);
        forward_rescale<HDP>(f, far, st, hi2, lo2);
        columns_product<HDP>(&t.v[1][0], hi2, lo2, across, st.o);
    } else {
        columns_product<HDP>(&t.v[0][0], hi, lo, across, st.o);
    }
}

// Bound by the matrix instructions (busy 60 % of the time) and by what of the softmax does not hide behind them: 16 heads on 4 of
// keys, head dimension 64, 8192 tokens in 432 us, 318 TFLOP/s of the visible pairs, 954 with the three products each - 90 %
// of a large library product of halves.  Twelve sequences of up to 2048 in 75 us (busy 47 %: their lengths leave compute units idle at
// the end).  8 heads of 128, 4096 tokens, in 187 us: a workgroup to a compute unit, so that its latencies show (busy 45 %).  Where an
// uneven tile is met, the rest of a workgroup's walk takes its code: the 8192 tokens then 575 us for 444, with 4096 tokens and 8 heads
// of 128 300 us for 207, of 32 161 for 88 (calls with both launches).
template <int HDP, int KEYS>
__global__ void __launch_bounds__(256, HDP > 32 ? 2 : 3) causal_split_fwd_kernel(const ForwardArgs a) {
    __shared__ __attribute__((aligned(16))) ForwardTile<HDP, KEYS> even, odd;
    __shared__ int wave_power[4];
    const CausalArgs<float>& p = a.p;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
    // all heads of a group of rows next to each other: consecutive workgroups go to different chiplets, so a chiplet's cache
    // serves few heads
    const int kv = blockIdx.x % (unsigned)p.kv_heads;
    const int4 job = a.order[blockIdx.x / (unsigned)p.kv_heads];
    if (job.x < 0) return;
    const int q0 = job.z, rows = job.w * p.group, group_row0 = job.y * 128, row0 = group_row0 + 32 * wave, row = row0 + (lane & 31);
    // keys seen by the workgroup and by the wavefront; the first key that a row of the wavefront does not see is wave_first + 1
    const int seen = (min(group_row0 + 128, rows) - 1) / p.group + 1;
    const int wave_first = row0 < rows ? row0 / p.group : -1, wave_seen = row0 < rows ? (min(row0 + 32, rows) - 1) / p.group + 1 : 0;
    const int64_t tile0 = q0 / 64 + job.x;
    KeyNotes notes_even, notes_odd;
    forward_stage<HDP, KEYS>(a, even, notes_even, tile0, kv, 0, wave, lane);
    const float minus_one = opaque_minus_one();
    ForwardState<HDP> st;
    const int seen_by_row = row / p.group, head = kv * p.group + row - seen_by_row * p.group;
    const int64_t token = q0 + seen_by_row;
    bool row_bad = false;
    {
        // the row of Q, scaled by a power of two of its own; scale log2 e goes in as a factor in [1/2, 1) and another power
        const float* __restrict__ src = p.Q + token * p.ldq + head * (int64_t)p.head_dim;
        int e_factor = 0;
        const float factor = frexpf(p.scale * LOG2E, &e_factor);
        float x[HDP / 16][8], top = 0.f;
#pragma unroll
        for (int k = 0; k < HDP / 16; ++k)
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int d = 16 * k + 8 * h + 4 * v;
                f4 y = {0.f, 0.f, 0.f, 0.f};
                if (row < rows && d < p.head_dim) {
                    if (p.vec_q) {
                        y = *reinterpret_cast<const f4*>(src + d);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (d + e < p.head_dim) y[e] = src[d + e];
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    row_bad = row_bad || !is_finite(y[e]);
                    x[k][4 * v + e] = is_finite(y[e]) ? y[e] : 0.f;
                    top = fmaxf(top, fabsf(x[k][4 * v + e]));
                }
            }
        top = max_halves(top);
        row_bad = __shfl_xor((int)row_bad, 32, 64) != 0 || row_bad;
        int e = 0;
        if (top > 0.f) {
            (void)frexpf(top, &e);
            e -= 12;
        }
        st.e_row = e + e_factor;
        const int power = wave_max_int(top > 0.f ? st.e_row : NO_EXPONENT);
        if (lane == 0) wave_power[wave] = power;
#pragma unroll
        for (int k = 0; k < HDP / 16; ++k) {
            h8 hi[1], lo[1];
#pragma unroll
            for (int c = 0; c < 8; ++c) x[k][c] = __builtin_ldexpf(x[k][c], -e) * factor;
            split_regs<8>(x[k], minus_one, hi, lo);
            st.q_hi[k] = hi[0];
            st.q_lo[k] = lo[0];
        }
    }
    st.last = row < rows ? seen_by_row : job.w - 1;
    st.m = -INFINITY;
    st.l = 0.f;
    st.x = -INFINITY;
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) st.o[d][r] = 0.f;
    auto use = [&](auto uneven, const ForwardTile<HDP, KEYS>& t, const KeyNotes& notes, int k0) __attribute__((always_inline)) {
        const int64_t at = ((tile0 + k0 / 64) * p.kv_heads + kv) * 64 + k0 % 64;
        if (k0 < wave_seen) forward_tile<HDP, KEYS, uneven()>(t, notes, a.powers_k + at, a.powers_v + at, k0, wave_first, minus_one, lane, st);
    };
    // Scores are sums of up to 2^7 products of a row's values, below 2^12 times its power, and a key's, below 2^15.
    __syncthreads();
    const int most_power = MOST_SCORE - 34 - __builtin_amdgcn_readfirstlane(max(max(wave_power[0], wave_power[1]), max(wave_power[2], wave_power[3])));
    // From key k0 on, whose tile is being copied; returns where a tile is met that needs the uneven form, by the other one.  (The code
    // for those is apart, and used from there on: inside the common one its registers cost that up to 20 %.)
    auto walk = [&](auto uneven, int k0) __attribute__((always_inline)) {
        for (; k0 < seen; k0 += 2 * KEYS) {
            staged();
            KeyNotes notes = notes_even.uniform();
            if (!uneven() && notes.power > most_power) break;
            if (k0 + KEYS < seen) forward_stage<HDP, KEYS>(a, odd, notes_odd, tile0, kv, k0 + KEYS, wave, lane);
            use(uneven, even, notes, k0);
            if (k0 + KEYS >= seen) return seen;
            staged();
            notes = notes_odd.uniform();
            if (!uneven() && notes.power > most_power) return k0 + KEYS;
            if (k0 + 2 * KEYS < seen) forward_stage<HDP, KEYS>(a, even, notes_even, tile0, kv, k0 + 2 * KEYS, wave, lane);
            use(uneven, odd, notes, k0 + KEYS);
        }
        return k0;
    };
    const int at = walk(std::false_type(), 0);
    st.x = st.m == -INFINITY ? 0.f : st.x - st.m;
    if (__builtin_expect(at < seen, 0)) {
        // (all wavefronts are past what either buffer held before that tile)
        forward_stage<HDP, KEYS>(a, even, notes_even, tile0, kv, at, wave, lane);
        walk(std::true_type(), at);
    }
    if (row >= rows) return;
    const float l = sum_halves(st.l);
    const float inv = row_bad ? NAN : 1.f / l;
    float* __restrict__ dst = p.O + token * p.ldo + head * (int64_t)p.head_dim;
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int at = 32 * d + 8 * q + 4 * h;
            f4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = __builtin_ldexpf(st.o[d][4 * q + e] * inv, (int)st.x);
            if (at >= p.head_dim) continue;
            if (p.vec_o) {
                *reinterpret_cast<f4*>(dst + at) = y;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (at + e < p.head_dim) dst[at + e] = y[e];
            }
        }
    if (p.lse != nullptr && h == 0) {
        const float ref = st.m == -INFINITY ? 0.f : st.m - 8.f;
        p.lse[head * p.q_rows + token] = row_bad ? NAN : (ref + __log2f(l)) * LN2;
    }
}

// ---- backward ---------------------------------------------------------------------------------------------------------------
struct BackwardArgs {
    CausalArgs<float> p;
    const _Float16* q; const _Float16* g;   // g: dO
    const _Float16* k; const _Float16* v;
    const Header* hq; const Header* hg; const Header* hk; const Header* hv;
    const int* powers_q; const int* powers_g; const int* powers_k; const int* powers_v;
    const float* row_notes;
    const int* e_dot;
    const int4* row_order; const int4* key_order;
    int chunk_tiles, chunks;    // tiles of rows that a workgroup of the key kernel takes at most, and parts that makes of the longest
    float* part;                // [chunk][token][kv][dK | dV][hd4] where a group of keys has more than one part
    int hd4;                    // head_dim rounded up to whole vectors
};

// dP - D is below 2^(e - 1) in magnitude, e from the exponents of dO, V and D: a sum of up to 2^7 products of values below 2^15
__device__ __forceinline__ int e_difference(int e_g, int e_v, int e_dot) { return max(37 + e_g + e_v, e_dot + 1) + 1; }
// The largest of the values of the lanes up to lane n, or from lane n on; a lane asks with an n of its own (outside 0 .. 63: none of
// them, or all).
__device__ __forceinline__ int max_upto(int v, int n) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v = max(v, __shfl_up(v, off, 64));
    const int got = __shfl(v, n > 63 ? 63 : n < 0 ? 0 : n, 64);
    return n < 0 ? NO_EXPONENT : got;
}
__device__ __forceinline__ int max_from(int v, int n) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v = max(v, __shfl_down(v, off, 64));
    const int got = __shfl(v, n < 0 ? 0 : n > 63 ? 63 : n, 64);
    return n > 63 ? NO_EXPONENT : got;
}

// Makes weights fit into halves: where a column's largest has passed 2^15, the column and its accumulators come down to 2^11, so
// that it takes another factor of 16 before the next time.  x: the power of two that the column is scaled by.
// Weights start at 2^FIT_FROM times what is at most 1: a sum all of whose terms are below 2^-100 of the largest |dO||V| that it might have
// held - a weight of 2^-60 beside values 2^40 times the others' - loses bits, one with larger terms does not.
constexpr int FIT_FROM = 110;
template <int N>
__device__ __forceinline__ void fit(float (&w)[16], int& x, f16v (&acc)[N]) {
    float top = fabsf(w[0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, fabsf(w[r]));
    top = max_halves(top);
    const bool over = top >= 32768.f;
    if (__ballot(over) != 0) {
        int e = 0;
        (void)frexpf(top, &e);
        const int down = over ? e - 11 : 0;
        const float f = pow2(-down);
#pragma unroll
        for (int r = 0; r < 16; ++r) w[r] *= f;
#pragma unroll
        for (int d = 0; d < N; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] *= f;
        x -= down;
    }
}

template <int HDP>
__device__ __forceinline__ void load_fragments(const _Float16* __restrict__ block, int lane, h8 (&hi)[HDP / 16], h8 (&lo)[HDP / 16]) {
#pragma unroll
    for (int k = 0; k < HDP / 16; ++k) {
        hi[k] = frag(block, k, lane);
        lo[k] = frag(block, HDP / 16 + k, lane);
    }
}
// A column per lane of an accumulator to a row of `head_dim` floats.
template <int HDP>
__device__ __forceinline__ void store_column(float* __restrict__ dst, const f16v (&acc)[HDP / 32], float factor, int e, int h, int head_dim, bool vec) {
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int at = 32 * d + 8 * q + 4 * h;
            f4 y;
#pragma unroll
            for (int c = 0; c < 4; ++c) y[c] = __builtin_ldexpf(acc[d][4 * q + c], e) * factor;
            if (at >= head_dim) continue;
            if (vec) {
                *reinterpret_cast<f4*>(dst + at) = y;
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (at + c < head_dim) dst[at + c] = y[c];
            }
        }
}

// Gradients of K and V.  A workgroup owns 128 keys of a key/value head, a wavefront 32 of them, a key per lane, with their K and V
// in registers; blocks of 32 packed rows (all heads of the group) of Q and dO pass through LDS.  S = Q K^T and
// dP = dO V^T come out with a key per lane, so P and dS go straight into dV^T += dO^T P and dK^T += Q^T dS.
template <int HDP>
struct RowTile {
    _Float16 q[2][64 * HDP], g[2][64 * HDP];   // two blocks of 32 rows
    float lse[64], dot[64];
};
struct RowNotes {
    int e_q, e_g, uneven;
};

template <int HDP>
__device__ __forceinline__ void row_stage(const BackwardArgs& a, RowTile<HDP>& t, RowNotes& notes, int64_t tile_at, int wave, int lane) {
    const Header hq = a.hq[tile_at], hg = a.hg[tile_at];
    notes = RowNotes{hq.e, hg.e, hq.uneven | hg.uneven};
    stage<256 * HDP, 4>(a.q + tile_at * (128 * HDP), &t.q[0][0], wave, lane);
    stage<256 * HDP, 4>(a.g + tile_at * (128 * HDP), &t.g[0][0], wave, lane);
    if (wave < 2) {
        const __amdgpu_buffer_rsrc_t from = buffer_of(a.row_notes + tile_at * 128, 512);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)(t.lse + 64 * wave), 4, lane * 4, wave * 256, 0, 0);
    }
}

template <int HDP>
struct KeyState {
    h8 k_hi[HDP / 16], k_lo[HDP / 16], v_hi[HDP / 16], v_lo[HDP / 16];
    f16v dk[HDP / 32], dv[HDP / 32];
    int e_k, e_v;            // of the lane's key
    int x_v, x_k;            // the powers of two that the lane's key is scaled by in the weights of dV and dK
    int first_row;           // the first packed row that sees the lane's key
};

// powers_q, powers_g: of the block's rows.
template <int HDP, bool UNEVEN>
__device__ __forceinline__ void row_block(const RowTile<HDP>& t, int block, const RowNotes& notes, const int* __restrict__ powers_q,
                                          const int* __restrict__ powers_g, int row0, int wave_last, float factor, float minus_one, int lane, KeyState<HDP>& st) {
    const int h = lane >> 5;
    const Across across(lane);
    f16v s, dp;
    rows_products<HDP>(t.q[block], st.k_hi, st.k_lo, s, t.g[block], st.v_hi, st.v_lo, dp, lane);
    // The weights of dV are 2^x_v P with dO's power, those of dK 2^x_k P (dP - D) with Q's: what is made to fit into halves is what
    // really enters the sums.  (The power multiplies the exponential: as a part of its argument, a hundred or so, it would leave
    // that 17 bits behind the point.)  In an uneven tile the powers are those of the rows.
    if constexpr (UNEVEN) {
        take_powers(s, powers_q, st.e_k, h);
        take_powers(dp, powers_g, st.e_v, h, powers_q, st.x_k, t.dot + 32 * block);
    }
    const float c = __builtin_ldexpf(factor, UNEVEN ? 0 : notes.e_q + st.e_k);
    const int e_one = UNEVEN ? 2 * NO_EXPONENT : notes.e_q + st.x_k;  // (D is in dP already: what is left of it is 0, or NaN)
    const float a1 = __builtin_ldexpf(1.f, UNEVEN ? 0 : notes.e_g + st.e_v + e_one), f = pow2(UNEVEN ? 0 : notes.e_g + st.x_v);
    float w[16], ds[16];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const f4 lse = *reinterpret_cast<const f4*>(t.lse + 32 * block + 8 * q + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * q + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * q + e], c, lse[e]));
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const f4 dot = *reinterpret_cast<const f4*>(t.dot + 32 * block + 8 * q + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) ds[4 * q + e] = w[4 * q + e] * __builtin_fmaf(dp[4 * q + e], a1, -__builtin_ldexpf(dot[e], e_one));
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] *= f;
    if constexpr (UNEVEN) take_powers(w, powers_g, st.x_v, h);
    if (row0 < wave_last) {  // some key is not seen by some row (whose weight, D or dP may be anything)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const bool seen = row0 + acc_row(r, h) >= st.first_row;
            w[r] = seen ? w[r] : 0.f;
            ds[r] = seen ? ds[r] : 0.f;
        }
    }
    fit(w, st.x_v, st.dv);
    h8 hi[2], lo[2];
    split_regs<16>(w, minus_one, hi, lo);
    columns_product<HDP>(t.g[block], hi, lo, across, st.dv);
    fit(ds, st.x_k, st.dk);
    split_regs<16>(ds, minus_one, hi, lo);
    columns_product<HDP>(t.q[block], hi, lo, across, st.dk);
}

// Bound by vector instructions beside the products (two exponent-sized passes, two splits and two looks for the largest weight per
// score) and, one third, by the last workgroups: 16 heads on 4 of keys, head dimension 64, sequences of 2048, 1901, 1536, 1000,
// 800, 511, 300 and 64 tokens in 177 us, 4 of the 7 products of a training step (matrix instructions busy 56 % of the time).  With
// uneven tiles all through 5 to 40 % slower.
template <int HDP>
__global__ void __launch_bounds__(256, HDP > 64 ? 1 : 2) causal_split_bwd_kv_kernel(const BackwardArgs a) {
    __shared__ __attribute__((aligned(16))) RowTile<HDP> even, odd;
    const CausalArgs<float>& p = a.p;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
    // later parts exist for long groups only and are as large as a part gets: first.  (The parts of a group must not be neighbours:
    // with consecutive workgroups on different chiplets, every second chiplet would only get parts that do not exist.)
    const unsigned per_chunk = gridDim.x / (unsigned)a.chunks;
    const int kv = blockIdx.x % (unsigned)p.kv_heads, chunk = a.chunks - 1 - (int)(blockIdx.x / per_chunk);
    const int4 job = a.key_order[blockIdx.x % per_chunk / (unsigned)p.kv_heads];
    if (job.x < 0) return;
    const int q0 = job.z, n = job.w, rows = n * p.group, group_key0 = job.y * 128, key0 = group_key0 + 32 * wave;
    const bool active = key0 < n;
    const int64_t row_tile0 = (int64_t)q0 * p.group / 64 + job.x;
    // tiles of rows: the last part is a whole one, the first what remains
    const int all_first = group_key0 * p.group / 64, all_tiles = (rows + 63) / 64, parts = (all_tiles - all_first + a.chunk_tiles - 1) / a.chunk_tiles;
    if (chunk >= parts) return;
    const int first = max(all_first, all_tiles - (parts - chunk) * a.chunk_tiles), tiles = all_tiles - (parts - 1 - chunk) * a.chunk_tiles;
    RowNotes notes_even, notes_odd;
    auto tile_at = [&](int i) { return (row_tile0 + i) * p.kv_heads + kv; };
    row_stage<HDP>(a, even, notes_even, tile_at(first), wave, lane);
    const float minus_one = opaque_minus_one();
    KeyState<HDP> st;
    {
        const int from = active ? key0 : group_key0;
        const int64_t key_tile = ((int64_t)q0 / 64 + job.x + from / 64) * p.kv_heads + kv;
        const int64_t at = key_tile * (128 * HDP) + from / 32 % 2 * (64 * HDP);
        load_fragments<HDP>(a.k + at, lane, st.k_hi, st.k_lo);
        load_fragments<HDP>(a.v + at, lane, st.v_hi, st.v_lo);
        st.e_k = a.powers_k[key_tile * 64 + from % 64 + (lane & 31)];
        st.e_v = a.powers_v[key_tile * 64 + from % 64 + (lane & 31)];
        // tiles of rows that see all of the wavefront's keys, then those of which some rows do not see some key
        const int first_row = (key0 + (lane & 31)) * p.group, whole = max(first, ((key0 + 31) * p.group + 63) / 64);
        int tq = NO_EXPONENT, tg = NO_EXPONENT, td = NO_EXPONENT;
        for (int tile = whole + lane; tile < tiles; tile += 64) {
            tq = max(tq, a.hq[tile_at(tile)].e);
            tg = max(tg, a.hg[tile_at(tile)].e);
            td = max(td, a.e_dot[tile_at(tile)]);
        }
        tq = wave_max_int(tq);
        tg = wave_max_int(tg);
        td = wave_max_int(td);
        for (int tile = max(first, key0 * p.group / 64); tile < min(whole, tiles); ++tile) {
            const int64_t at = tile_at(tile);
            const int from_row = first_row - 64 * tile;
            tq = max(tq, max_from(a.powers_q[at * 64 + lane], from_row));
            tg = max(tg, max_from(a.powers_g[at * 64 + lane], from_row));
            td = max(td, max_from(power_of(fabsf(a.row_notes[at * 128 + 64 + lane])), from_row));
        }
        // P is at most 1, |P (dP - D)| 2^(1 - e_difference) too
        st.x_v = FIT_FROM - tg;
        st.x_k = FIT_FROM + 1 - e_difference(tg, st.e_v, td) - tq;
    }
    st.first_row = (key0 + (lane & 31)) * p.group;
    const int wave_first = key0 * p.group, wave_last = (key0 + 31) * p.group;
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) st.dk[d][r] = st.dv[d][r] = 0.f;
    const float factor = p.scale * LOG2E;
    auto uniform = [](const RowNotes& x) {
        return RowNotes{__builtin_amdgcn_readfirstlane(x.e_q), __builtin_amdgcn_readfirstlane(x.e_g), __builtin_amdgcn_readfirstlane(x.uneven)};
    };
    auto use = [&](auto uneven, const RowTile<HDP>& t, const RowNotes& notes, int i) __attribute__((always_inline)) {
#pragma unroll
        for (int block = 0; block < 2; ++block)
            if (active && 64 * i + 32 * block + 31 >= wave_first)
                row_block<HDP, uneven()>(t, block, notes, a.powers_q + tile_at(i) * 64 + 32 * block, a.powers_g + tile_at(i) * 64 + 32 * block,
                                         64 * i + 32 * block, wave_last, factor, minus_one, lane, st);
    };
    auto walk = [&](auto uneven, int i) __attribute__((always_inline)) {  // (as in the forward kernel)
        for (; i < tiles; i += 2) {
            staged();
            RowNotes notes = uniform(notes_even);
            if (!uneven() && notes.uneven != 0) break;
            if (i + 1 < tiles) row_stage<HDP>(a, odd, notes_odd, tile_at(i + 1), wave, lane);
            use(uneven, even, notes, i);
            if (i + 1 >= tiles) return tiles;
            staged();
            notes = uniform(notes_odd);
            if (!uneven() && notes.uneven != 0) return i + 1;
            if (i + 2 < tiles) row_stage<HDP>(a, even, notes_even, tile_at(i + 2), wave, lane);
            use(uneven, odd, notes, i + 1);
        }
        return i;
    };
    const int at = walk(std::false_type(), first);
    if (__builtin_expect(at < tiles, 0)) {
        row_stage<HDP>(a, even, notes_even, tile_at(at), wave, lane);
        walk(std::true_type(), at);
    }
    const int64_t key = key0 + (lane & 31);
    if (key >= n) return;
    float* dst_k = p.dK + (q0 + key) * p.lddk + kv * (int64_t)p.head_dim;
    float* dst_v = p.dV + (q0 + key) * p.lddv + kv * (int64_t)p.head_dim;
    int width = p.head_dim;
    bool vec = p.vec_dkv;
    if (parts > 1) {
        dst_k = a.part + ((chunk * p.q_rows + q0 + key) * p.kv_heads + kv) * (2 * a.hd4);
        dst_v = dst_k + a.hd4;
        width = a.hd4;  // (columns past the head dimension are zeros)
        vec = true;
    }
    store_column<HDP>(dst_k, st.dk, p.scale, -st.x_k, h, width, vec);
    store_column<HDP>(dst_v, st.dv, 1.f, -st.x_v, h, width, vec);
}

// Adds the parts of the groups of keys that have several, in their order (16 us behind the 177 above, by memory).
__global__ void __launch_bounds__(256) causal_split_join_kernel(const BackwardArgs a) {
    const CausalArgs<float>& p = a.p;
    const int kv = blockIdx.x % (unsigned)p.kv_heads;
    const int4 job = a.key_order[blockIdx.x / (unsigned)p.kv_heads];
    if (job.x < 0) return;
    const int64_t q0 = job.z;
    const int n = job.w, key0 = job.y * 128, total = (n * p.group + 63) / 64 - key0 * p.group / 64;
    const int parts = (total + a.chunk_tiles - 1) / a.chunk_tiles;
    if (parts <= 1) return;
    const int per_row = a.hd4 / 2;  // vectors of both gradients
    for (int i = (int)(blockIdx.y * 256 + threadIdx.x); i < 128 * per_row; i += 256 * gridDim.y) {
        const int64_t key = key0 + i / per_row;
        const int c = i % per_row * 4;
        if (key >= n) break;
        f4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int x = 0; x < parts; ++x) sum += *reinterpret_cast<const f4*>(a.part + ((x * p.q_rows + q0 + key) * p.kv_heads + kv) * (2 * a.hd4) + c);
        const bool is_v = c >= a.hd4;
        const int d = is_v ? c - a.hd4 : c;
        float* dst = (is_v ? p.dV + (q0 + key) * p.lddv : p.dK + (q0 + key) * p.lddk) + kv * (int64_t)p.head_dim + d;
        if (p.vec_dkv) {
            *reinterpret_cast<f4*>(dst) = sum;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < p.head_dim) dst[e] = sum[e];
        }
    }
}

// Gradient of Q: 128 packed rows to a workgroup, a row per lane, Q and dO in registers; blocks of 32 keys of K and V pass
// through LDS.  S^T = K Q^T and dP^T = V dO^T, then dQ^T += K^T dS^T.
template <int HDP>
struct KeyTile {
    _Float16 k[2][64 * HDP], v[2][64 * HDP];   // two blocks of 32 keys
};
struct BlockNotes {
    int e_k, e_v, uneven;
};

template <int HDP>
__device__ __forceinline__ void key_stage(const BackwardArgs& a, KeyTile<HDP>& t, BlockNotes& notes, int64_t tile_at, int wave, int lane) {
    const Header hk = a.hk[tile_at], hv = a.hv[tile_at];
    notes = BlockNotes{hk.e, hv.e, hk.uneven | hv.uneven};
    stage<256 * HDP, 4>(a.k + tile_at * (128 * HDP), &t.k[0][0], wave, lane);
    stage<256 * HDP, 4>(a.v + tile_at * (128 * HDP), &t.v[0][0], wave, lane);
}

template <int HDP>
struct RowState {
    h8 q_hi[HDP / 16], q_lo[HDP / 16], g_hi[HDP / 16], g_lo[HDP / 16];
    f16v dq[HDP / 32];
    float lse, dot;
    int e_q, e_g;   // of the lane's row
    int x_q;        // the power of two that the lane's row is scaled by in the weights
    int last;       // the last key that the lane's row sees
};

// powers_k, powers_v: of the block's keys.
template <int HDP, bool UNEVEN>
__device__ __forceinline__ void key_block(const KeyTile<HDP>& t, int block, const BlockNotes& notes, const int* __restrict__ powers_k,
                                          const int* __restrict__ powers_v, int k0, int wave_first, float factor, float minus_one, int lane, RowState<HDP>& st) {
    const int h = lane >> 5;
    const Across across(lane);
    f16v s, dp;
    rows_products<HDP>(t.k[block], st.q_hi, st.q_lo, s, t.v[block], st.g_hi, st.g_lo, dp, lane);
    if constexpr (UNEVEN) {  // (as above)
        take_powers(s, powers_k, st.e_q, h);
        take_powers(dp, powers_v, st.e_g, h, powers_k, st.x_q, &st.dot, 0);
    }
    const float c = __builtin_ldexpf(factor, UNEVEN ? 0 : st.e_q + notes.e_k);
    const int e_one = UNEVEN ? 2 * NO_EXPONENT : notes.e_k + st.x_q;
    const float a1 = __builtin_ldexpf(1.f, UNEVEN ? 0 : st.e_g + notes.e_v + e_one), b = -__builtin_ldexpf(st.dot, e_one);
    float ds[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, st.lse)) * __builtin_fmaf(dp[r], a1, b);
    if (k0 + 31 > wave_first) {  // some key is not seen by some row (whose weight or dP may be anything)
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] = k0 + acc_row(r, h) <= st.last ? ds[r] : 0.f;
    }
    fit(ds, st.x_q, st.dq);
    h8 hi[2], lo[2];
    split_regs<16>(ds, minus_one, hi, lo);
    columns_product<HDP>(t.k[block], hi, lo, across, st.dq);
}

// Bound as the forward kernel: the batch above in 115 us, 3 products of the 7.
template <int HDP>
__global__ void __launch_bounds__(256, 2) causal_split_bwd_q_kernel(const BackwardArgs a) {
    __shared__ __attribute__((aligned(16))) KeyTile<HDP> even, odd;
    const CausalArgs<float>& p = a.p;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
    const int kv = blockIdx.x % (unsigned)p.kv_heads;
    const int4 job = a.row_order[blockIdx.x / (unsigned)p.kv_heads];
    if (job.x < 0) return;
    const int q0 = job.z, rows = job.w * p.group, group_row0 = job.y * 128, row0 = group_row0 + 32 * wave, row = row0 + (lane & 31);
    const bool active = row0 < rows;
    const int seen = (min(group_row0 + 128, rows) - 1) / p.group + 1, tiles = (seen + 63) / 64;
    const int wave_first = row0 / p.group, wave_seen = active ? (min(row0 + 32, rows) - 1) / p.group + 1 : 0;
    const int64_t key_tile0 = q0 / 64 + job.x;
    BlockNotes notes_even, notes_odd;
    auto tile_at = [&](int i) { return (key_tile0 + i) * p.kv_heads + kv; };
    key_stage<HDP>(a, even, notes_even, tile_at(0), wave, lane);
    const float minus_one = opaque_minus_one();
    RowState<HDP> st;
    {
        const int from = active ? row0 : group_row0;
        const int64_t row_tile = ((int64_t)q0 * p.group / 64 + job.x + from / 64) * p.kv_heads + kv, at = row_tile * (128 * HDP) + from / 32 % 2 * (64 * HDP);
        load_fragments<HDP>(a.q + at, lane, st.q_hi, st.q_lo);
        load_fragments<HDP>(a.g + at, lane, st.g_hi, st.g_lo);
        st.lse = a.row_notes[row_tile * 128 + from % 64 + (lane & 31)];
        st.dot = a.row_notes[row_tile * 128 + 64 + from % 64 + (lane & 31)];
        st.e_q = a.powers_q[row_tile * 64 + from % 64 + (lane & 31)];
        st.e_g = a.powers_g[row_tile * 64 + from % 64 + (lane & 31)];
        // tiles of keys that all of the wavefront's rows see, then those of which some rows do not see some key
        const int last = row < rows ? row / p.group : job.w - 1, whole = min((wave_first + 1) / 64, tiles);
        int tk = NO_EXPONENT, tv = NO_EXPONENT;
        for (int tile = lane; tile < whole; tile += 64) {
            tk = max(tk, a.hk[tile_at(tile)].e);
            tv = max(tv, a.hv[tile_at(tile)].e);
        }
        tk = wave_max_int(tk);
        tv = wave_max_int(tv);
        for (int tile = whole; 64 * tile < wave_seen; ++tile) {
            tk = max(tk, max_upto(a.powers_k[tile_at(tile) * 64 + lane], last - 64 * tile));
            tv = max(tv, max_upto(a.powers_v[tile_at(tile) * 64 + lane], last - 64 * tile));
        }
        st.x_q = FIT_FROM + 1 - e_difference(st.e_g, tv, power_of(fabsf(st.dot))) - tk;
    }
    const int seen_by_row = row / p.group;
    st.last = row < rows ? seen_by_row : job.w - 1;
#pragma unroll
    for (int d = 0; d < HDP / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) st.dq[d][r] = 0.f;
    const float factor = p.scale * LOG2E;
    auto uniform = [](const BlockNotes& x) {
        return BlockNotes{__builtin_amdgcn_readfirstlane(x.e_k), __builtin_amdgcn_readfirstlane(x.e_v), __builtin_amdgcn_readfirstlane(x.uneven)};
    };
    auto use = [&](auto uneven, const KeyTile<HDP>& t, const BlockNotes& notes, int i) __attribute__((always_inline)) {
#pragma unroll
        for (int block = 0; block < 2; ++block)
            if (64 * i + 32 * block < wave_seen)
                key_block<HDP, uneven()>(t, block, notes, a.powers_k + tile_at(i) * 64 + 32 * block, a.powers_v + tile_at(i) * 64 + 32 * block,
                                         64 * i + 32 * block, wave_first, factor, minus_one, lane, st);
    };
    auto walk = [&](auto uneven, int i) __attribute__((always_inline)) {  // (as in the forward kernel)
        for (; i < tiles; i += 2) {
            staged();
            BlockNotes notes = uniform(notes_even);
            if (!uneven() && notes.uneven != 0) break;
            if (i + 1 < tiles) key_stage<HDP>(a, odd, notes_odd, tile_at(i + 1), wave, lane);
            use(uneven, even, notes, i);
            if (i + 1 >= tiles) return tiles;
            staged();
            notes = uniform(notes_odd);
            if (!uneven() && notes.uneven != 0) return i + 1;
            if (i + 2 < tiles) key_stage<HDP>(a, even, notes_even, tile_at(i + 2), wave, lane);
            use(uneven, odd, notes, i + 1);
        }
        return i;
    };
    const int at = walk(std::false_type(), 0);
    if (__builtin_expect(at < tiles, 0)) {
        key_stage<HDP>(a, even, notes_even, tile_at(at), wave, lane);
        walk(std::true_type(), at);
    }
    if (row >= rows) return;
    store_column<HDP>(p.dQ + ((int64_t)q0 + seen_by_row) * p.lddq + (kv * p.group + row - seen_by_row * p.group) * (int64_t)p.head_dim, st.dq, p.scale,
                      -st.x_q, h, p.head_dim, p.vec_dq);
}

// ---- workspace --------------------------------------------------------------------------------------------------------------
inline size_t round256(size_t b) { return (b + 255) & ~(size_t)255; }
inline int64_t tile_slots(int64_t rows, int64_t group, int64_t per_tile, int64_t sequences) { return rows * group / per_tile + sequences; }
inline int padded(int head_dim) { return head_dim <= 32 ? 32 : head_dim <= 64 ? 64 : 128; }

// Hands out parts of the workspace; with a null base it only counts.
struct Carver {
    char* base;
    size_t used = 0;
    template <typename U>
    U* take(size_t bytes) {
        U* at = base == nullptr ? nullptr : reinterpret_cast<U*>(base + used);
        used += round256(bytes);
        return at;
    }
};

// Work is at most q_rows / 64 tiles: this many bits less of it tell ORDER_BINS - 1 kinds apart.
inline int order_shift(int64_t q_rows) {
    int shift = 0;
    while ((q_rows / 64) >> shift >= ORDER_BINS - 1) ++shift;
    return shift;
}

struct ForwardPlan {
    SplitArgs split;
    ForwardArgs main;
    size_t bytes;
};
ForwardPlan forward_plan(const CausalArgs<float>& p, void* workspace) {
    const int hdp = padded(p.head_dim);
    const int64_t key_tiles = tile_slots(p.q_rows, 1, 64, p.sequences) * p.kv_heads;
    Carver c{static_cast<char*>(workspace)};
    ForwardPlan f{};
    _Float16* k = c.take<_Float16>((size_t)key_tiles * 256 * hdp);
    _Float16* v = c.take<_Float16>((size_t)key_tiles * 256 * hdp);
    Header* hk = c.take<Header>((size_t)key_tiles * sizeof(Header));
    Header* hv = c.take<Header>((size_t)key_tiles * sizeof(Header));
    int* powers_k = c.take<int>((size_t)key_tiles * 64 * sizeof(int));
    int* powers_v = c.take<int>((size_t)key_tiles * 64 * sizeof(int));
    const int64_t row_groups = tile_slots(p.q_rows, p.group, 128, p.sequences);
    f.split.order = c.take<int4>((size_t)row_groups * sizeof(int4));
    f.split.order_slots[0] = (int)row_groups;
    f.split.tensors = 2;
    f.split.shift = order_shift(p.q_rows);
    f.split.p = p;
    f.split.t[0] = {p.K, p.ldk, 1, p.vec_kv, k, hk, powers_k, 0};
    f.split.t[1] = {p.V, p.ldv, 1, p.vec_kv, v, hv, powers_v, 0};
    f.main = {p, k, v, hk, hv, powers_k, powers_v, f.split.order};
    f.bytes = c.used;
    return f;
}

constexpr int MOST_PARTS = 32, CHUNK_FROM = 16;
struct BackwardPlan {
    SplitArgs split;
    BackwardArgs main;
    size_t bytes;
};
BackwardPlan backward_plan(const CausalArgs<float>& p, void* workspace) {
    const int hdp = padded(p.head_dim);
    const int64_t key_tiles = tile_slots(p.q_rows, 1, 64, p.sequences) * p.kv_heads, row_tiles = tile_slots(p.q_rows, p.group, 64, p.sequences) * p.kv_heads;
    Carver c{static_cast<char*>(workspace)};
    BackwardPlan b{};
    _Float16* split[4];
    Header* headers[4];
    int* powers[4];
    for (int i = 0; i < 4; ++i) {  // Q, dO, K, V
        const int64_t tiles = i < 2 ? row_tiles : key_tiles;
        split[i] = c.take<_Float16>((size_t)tiles * 256 * hdp);
        headers[i] = c.take<Header>((size_t)tiles * sizeof(Header));
        powers[i] = c.take<int>((size_t)tiles * 64 * sizeof(int));
    }
    float* notes = c.take<float>((size_t)row_tiles * 128 * 4);
    int* e_dot = c.take<int>((size_t)row_tiles * sizeof(int));
    b.split.p = p;
    b.split.t[0] = {p.Q, p.ldq, p.group, p.vec_q, split[0], headers[0], powers[0], 0};
    b.split.t[1] = {p.dO, p.ldo, p.group, p.vec_o, split[1], headers[1], powers[1], 1};
    b.split.t[2] = {p.K, p.ldk, 1, p.vec_kv, split[2], headers[2], powers[2], 0};
    b.split.t[3] = {p.V, p.ldv, 1, p.vec_kv, split[3], headers[3], powers[3], 0};
    const int64_t row_groups = tile_slots(p.q_rows, p.group, 128, p.sequences), key_groups = tile_slots(p.q_rows, 1, 128, p.sequences);
    b.split.order = c.take<int4>((size_t)(row_groups + key_groups) * sizeof(int4));
    b.split.order_slots[0] = (int)row_groups;
    b.split.order_slots[1] = (int)key_groups;
    b.split.tensors = 4;
    b.split.shift = order_shift(p.q_rows);
    // Parts of the rows that see a group of keys.  If the sequences were equally long, 512 workgroups (two to a compute unit) would
    // have `share` tiles of rows each; half of it keeps the longest group from being what the others wait for.  At most
    // MOST_PARTS parts and 256 MB of them.
    const int hd4 = (p.head_dim + 3) & ~3;
    const int64_t part_bytes = p.q_rows * p.kv_heads * 2 * hd4 * 4, most_tiles = (p.q_rows * p.group + 63) / 64;
    const int64_t most_parts = std::max<int64_t>(1, std::min<int64_t>(MOST_PARTS, ((int64_t)256 << 20) / part_bytes));
    const int64_t share = (int64_t)((double)p.q_rows * p.q_rows / p.sequences * p.group * p.kv_heads / (2.0 * 128 * 64 * 512));
    const int64_t chunk = std::max<int64_t>({CHUNK_FROM, share / 2, (most_tiles + most_parts - 1) / most_parts});
    const int chunks = (int)((most_tiles + chunk - 1) / chunk);
    float* part = chunks > 1 ? c.take<float>((size_t)(part_bytes * chunks)) : nullptr;
    b.split.row_notes = notes;
    b.split.e_dot = e_dot;
    b.main = {p, split[0], split[1], split[2], split[3], headers[0], headers[1], headers[2], headers[3], powers[0], powers[1], powers[2], powers[3], notes, e_dot,
              b.split.order, b.split.order + row_groups, (int)chunk, chunks, part, hd4};
    b.bytes = c.used;
    return b;
}

}  // namespace

// Whether a batch is large enough for these kernels; smaller ones are faster with units of 16 rows.  Three products on halves
// cost less than one on floats and tiles of 128 rows read less, but their workgroups take more rows each: they want
// rows * heads >= 2^14 to fill the card, and they have a kernel more to launch and longer prologues, which pay from
// rows * heads * (mean length) = 2^22 on - in the gradients of shared keys, where there are fewer tiles of keys, from twice
// that.  Measured, these against the units of 16, head dimension 64, 8 heads on 8 of keys, forward / backward in us:
//   1024 rows of length 64: 15 / 26 against 9 / 19;  2048 of 64: 18 / 34 against 14 / 31;  2048 of 256: 22 / 46 against 23 / 59;
//   4096 of 1024: 47 / 108 against 82 / 243;  8 heads on 2 of keys, 2048 of 256: 19 / 86 against 23 / 65, of 1024: 38 / 121
//   against 47 / 193.
// And sequences have to fill the tiles of 128 packed rows and 64 keys, of which each takes whole ones: from 40 packed rows a sequence
// on, in the gradients from 32 keys too.  (The mean stands for the lengths, which the host does not know.)  As above, by mean length,
// 32768 rows, forward / backward in us:
//   8 heads on 8: 16: 383 / 791 against 233 / 673;  32: 208 / 444 against 159 / 429;  48: 155 / 357 against 188 / 554;
//   16 heads on 4: 8: 454 / 942 against 331 / 625;  16: 243 / 618 against 282 / 604;  24: 190 / 539 against 280 / 522;
//   32: 156 / 457 against 279 / 507.
static bool split_pays(const CausalArgs<float>& p, int64_t least, int64_t least_keys) {
    const int64_t rows = p.q_rows * p.heads;
    return rows >= ((int64_t)1 << 14) && (double)rows * p.q_rows / p.sequences >= (double)least && p.q_rows >= least_keys * p.sequences &&
           p.q_rows * p.group >= (int64_t)40 * p.sequences;
}
// The other kernels take what these cannot: launches of 2^32 lanes, and a workspace that is out of proportion - head dimensions are
// padded to 32, so that it can be many times the operands - where it is large.
static bool split_fits(const CausalArgs<float>& p, std::initializer_list<int64_t> groups, size_t bytes) {
    for (int64_t g : groups)
        if (g * 256 >= ((int64_t)1 << 32)) return false;
    return bytes <= std::max((size_t)1 << 32, (size_t)(8 * sizeof(float) * 2) * p.q_rows * (p.heads + p.kv_heads) * p.head_dim);
}
bool causal_split_fwd_pays(const CausalArgs<float>& p) {
    return split_pays(p, 1 << 22, 0) && split_fits(p, {tile_slots(p.q_rows, 1, 64, p.sequences), tile_slots(p.q_rows, p.group, 128, p.sequences) * p.kv_heads}, causal_split_fwd_workspace_bytes(p));
}
bool causal_split_bwd_pays(const CausalArgs<float>& p) {
    if (!split_pays(p, p.group == 1 ? 1 << 22 : 1 << 23, 32)) return false;
    const BackwardPlan b = backward_plan(p, nullptr);
    return split_fits(p, {tile_slots(p.q_rows, p.group, 64, p.sequences), tile_slots(p.q_rows, p.group, 128, p.sequences) * p.kv_heads,
                          tile_slots(p.q_rows, 1, 128, p.sequences) * p.kv_heads * b.main.chunks}, b.bytes);
}

size_t causal_split_fwd_workspace_bytes(const CausalArgs<float>& p) { return forward_plan(p, nullptr).bytes; }

hipError_t launch_causal_split_fwd(const CausalArgs<float>& p, void* workspace, hipStream_t s) {
    const ForwardPlan f = forward_plan(p, workspace);
    const int64_t key_slots = tile_slots(p.q_rows, 1, 64, p.sequences), slots = tile_slots(p.q_rows, p.group, 128, p.sequences);
    const dim3 split((unsigned)key_slots, p.kv_heads, 3), grid((unsigned)(slots * p.kv_heads)), block(256);
    switch (padded(p.head_dim)) {
        case 32:
            hipLaunchKernelGGL(causal_split_kernel<32>, split, block, 0, s, f.split);
            hipLaunchKernelGGL((causal_split_fwd_kernel<32, 64>), grid, block, 0, s, f.main);
            break;
        case 64:
            hipLaunchKernelGGL(causal_split_kernel<64>, split, block, 0, s, f.split);
            hipLaunchKernelGGL((causal_split_fwd_kernel<64, 64>), grid, block, 0, s, f.main);
            break;
        default:
            hipLaunchKernelGGL(causal_split_kernel<128>, split, block, 0, s, f.split);
            hipLaunchKernelGGL((causal_split_fwd_kernel<128, 32>), grid, block, 0, s, f.main);
            break;
    }
    return hipGetLastError();
}

size_t causal_split_bwd_workspace_bytes(const CausalArgs<float>& p) { return backward_plan(p, nullptr).bytes; }

template <int HDP>
static void enqueue_backward(const BackwardPlan& b, dim3 split, unsigned key_groups, dim3 row_grid, hipStream_t s) {
    hipLaunchKernelGGL(causal_split_kernel<HDP>, split, dim3(256), 0, s, b.split);
    hipLaunchKernelGGL(causal_split_bwd_kv_kernel<HDP>, dim3(key_groups * b.main.chunks), dim3(256), 0, s, b.main);
    if (b.main.chunks > 1) hipLaunchKernelGGL(causal_split_join_kernel, dim3(key_groups, HDP / 32), dim3(256), 0, s, b.main);
    hipLaunchKernelGGL(causal_split_bwd_q_kernel<HDP>, row_grid, dim3(256), 0, s, b.main);
}

hipError_t launch_causal_split_bwd(const CausalArgs<float>& p, void* workspace, hipStream_t s) {
    const BackwardPlan b = backward_plan(p, workspace);
    const int64_t row_tiles = tile_slots(p.q_rows, p.group, 64, p.sequences), key_groups = tile_slots(p.q_rows, 1, 128, p.sequences),
                  row_groups = tile_slots(p.q_rows, p.group, 128, p.sequences);
    // (at least two wide: the workgroups 0 and 1 of the last plane make the schedules, however few tiles there are)
    const dim3 split((unsigned)std::max<int64_t>(row_tiles, 2), p.kv_heads, 5), row_grid((unsigned)(row_groups * p.kv_heads));
    switch (padded(p.head_dim)) {
        case 32: enqueue_backward<32>(b, split, (unsigned)(key_groups * p.kv_heads), row_grid, s); break;
        case 64: enqueue_backward<64>(b, split, (unsigned)(key_groups * p.kv_heads), row_grid, s); break;
        default: enqueue_backward<128>(b, split, (unsigned)(key_groups * p.kv_heads), row_grid, s); break;
    }
    return hipGetLastError();
}

}  // namespace prad
