// Pieces shared by the attention kernels: matrix products of 32 x 32 x 16, tiles in shared memory that are read by rows and
// transposed, the place of a block among packed sequences.
//
// Operand layouts of the product (64 lanes, lane = 32 h + m): A holds row m, B column m, both with the eight elements
// k = 8 h .. 8 h + 7 of the summed axis; the result holds column m, its i-th value the row (i & 3) + 8 (i >> 2) + 4 h.  The
// summed axis may go in any order that is the same in A and B: the eight results of a lane i = 8 s .. 8 s + 7 are therefore a
// B operand as they stand, if A takes its elements from rows 16 s + 4 h + (0..3) and 16 s + 8 + 4 h + (0..3), which is what two
// transposing reads of four rows each give.
#pragma once
#include "seq_common.h"

#include <cmath>
#include <initializer_list>

namespace seqamd {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
using Frag = T __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x16 product(Frag<bf16> a, Frag<bf16> b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 product(Frag<f16> a, Frag<f16> b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ f32x16 zeros16()
{
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.0f;
    return z;
}

// row of the result's i-th value
__device__ __forceinline__ int row_in(int i, int half) { return (i & 3) + 8 * (i >> 2) + 4 * half; }

// The larger value; NaN where there is one, so that the compiler need not quieten its operands first, an instruction for each
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float larger(float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); }

// the other half's value
__device__ __forceinline__ float swapped(float x)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// A tile in shared memory: rows of DP 16-bit elements, in chunks of eight, whose places in the row are exchanged by the
// row's number: the 8 rows of a read by rows and the 8 rows of a transposing read (each 64 bytes wide) then lie in
// different banks (64 banks of 4 bytes).
template <int DP>
struct Tile {
    static constexpr int kChunks = DP / 8, kRowBytes = DP * 2;
    static __device__ __forceinline__ int swizzle(int row)
    {
        static_assert(DP == 64 || DP == 128, "");
        return DP == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    }
    static __device__ __forceinline__ int at(int row, int chunk) { return row * kRowBytes + ((chunk ^ swizzle(row)) << 4); }
};

// An operand by rows: lane (h, m) takes eight elements of row m.  at[k]: byte in the tile for summed elements 16 k .. 16 k + 15
template <int DP>
struct RowRead {
    int at[DP / 16];
    __device__ __forceinline__ RowRead(int lane)
    {
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) at[k] = Tile<DP>::at(lane & 31, 2 * k + (lane >> 5));
    }
    // row0: a multiple of 32
    template <typename T>
    __device__ __forceinline__ Frag<T> get(const char* tile, int row0, int k) const
    {
        return *reinterpret_cast<const Frag<T>*>(tile + row0 * Tile<DP>::kRowBytes + at[k]);
    }
};

// A transposed operand: lane (h, m) takes column 32 b + m of the rows 16 s + 4 h + (0..3) and 16 s + 8 + 4 h + (0..3).
// A transposing read takes 8 bytes from each of 16 lanes, four lanes to a row, and gives lane i column i of the four rows.
template <int DP>
struct ColumnRead {
    int at[DP / 32][2];
    __device__ __forceinline__ ColumnRead(int lane)
    {
        const int h = lane >> 5, group = (lane >> 4) & 1, i = lane & 15;
#pragma unroll
        for (int b = 0; b < DP / 32; ++b)
#pragma unroll
            for (int t = 0; t < 2; ++t) at[b][t] = Tile<DP>::at(8 * t + 4 * h + (i >> 2), 4 * b + 2 * group + ((i & 3) >> 1)) + (i & 1) * 8;
    }
    // row0: a multiple of 16
    template <typename T>
    __device__ __forceinline__ Frag<T> get(const char* tile, int row0, int b) const
    {
        typedef __attribute__((address_space(3))) i16x4* Shared;
        struct {
            i16x4 x[2];
        } r;
#pragma unroll
        for (int t = 0; t < 2; ++t) r.x[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Shared)(tile + row0 * Tile<DP>::kRowBytes + at[b][t]));
        return __builtin_bit_cast(Frag<T>, r);
    }
};

// The operand is there from here on: a load that is still under way when a loop begins would be waited for in each turn of
// it, with all loads of that turn that are meant to go on meanwhile.
template <typename T>
__device__ __forceinline__ void arrive(Frag<T>& f)
{
    u32x4 w = __builtin_bit_cast(u32x4, f);
    asm volatile("" : "+v"(w));
    f = __builtin_bit_cast(Frag<T>, w);
}

// 16 bytes at a byte offset from an address that is the same for the whole wave
__device__ __forceinline__ u32x4 load_at(const char* base, unsigned offset)
{
    u32x4 x;
    __builtin_memcpy(&x, base + offset, 16);
    return x;
}

// eight results as an operand, rounded to nearest: the one rounding between the two products
template <typename T>
__device__ __forceinline__ Frag<T> rounded(const f32x16& x, int first)
{
    Frag<T> f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = T(x[first + i]);
    return f;
}

// eight elements of a row as an operand, zeros behind its end
template <typename T>
__device__ __forceinline__ Frag<T> load_row(const T* row, int d, int dim)
{
    u32x4 x = {0, 0, 0, 0};
    if (d < dim) __builtin_memcpy(&x, row + d, 16);
    return __builtin_bit_cast(Frag<T>, x);
}

// a lane's column of results, multiplied, as a row of `dim` values
template <typename T, int DP>
__device__ __forceinline__ void store_row(T* to, const f32x16* x, float times, int dim, int half)
{
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int ch = 32 * d + row_in(i, half);
            if (ch < dim) {
                float y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = x[d][i + j] * times;
                Pack<T, 4> pack;
                pack.set(y);
                store_pack<T, 4>(to + ch, pack);
            }
        }
}

// Values that are not finite, at keys that some queries of a tile do not see: a weight of zero times them would not be zero.  Tiles
// with hidden keys are put into shared memory with zeros in their place; which keys had them is noted, and what they are is
// added to the stored rows of the queries that see them.
template <typename T>
__device__ __forceinline__ unsigned not_finite(unsigned two)
{
    constexpr unsigned kLow = __is_same(T, bf16) ? 0x7f80u : 0x7c00u, kBoth = kLow << 16 | kLow;
    const unsigned e = two & kBoth;
    return ((e & 0xffffu) == kLow ? 0xffffu : 0u) | ((e >> 16) == kLow ? 0xffff0000u : 0u);
}

// zeros in their place; returns whether there were any
template <typename T>
__device__ __forceinline__ bool take_them_out(u32x4& x)
{
    unsigned any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned m = not_finite<T>(x[i]);
        x[i] &= ~m;
        any |= m;
    }
    return any != 0;
}

// Adds the values that are not finite of the row `v` to the channels of a stored row that a lane has stored (in memory and out of
// line: a rare case takes no registers from the common one)
template <typename T, typename O>
__device__ __attribute__((noinline)) void add_them(const T* v, O* to, int dim, int half)
{
#pragma unroll 1
    for (int ch = 4 * half; ch < dim; ch += (ch & 3) == 3 ? 5 : 1) {
        const float x = static_cast<float>(v[ch]);
        if (!__builtin_isfinite(x)) to[ch] = O(static_cast<float>(to[ch]) + x);
    }
}

// Packed sequences.  Offsets are read on the device and kept inside the tensors whatever they hold.
struct Packed {
    const int *q_offsets, *k_offsets, *k_lengths;
    int64_t q_rows, k_rows;
    int n;
    const int* map;      // more than kMapped sequences: the number of tiles, then (sequence, tile) of each, see map_kernel
};

constexpr int kMapped = 64;

// How a sequence is cut into tiles: by its keys, or by its queries times `mult`
struct Tiling {
    bool keys;
    int size, mult;
};

struct Span {
    int64_t q0, k0;      // first rows
    int nq, nk;
    int tile, seq;       // tile among the sequence's; seq < 0: none
};

__device__ __forceinline__ void span_of(const Packed& p, int seq, Span& s)
{
    s.seq = seq;
    s.q0 = kept(p.q_offsets[seq], 0, p.q_rows);
    s.nq = int(kept(p.q_offsets[seq + 1], s.q0, p.q_rows) - s.q0);
    s.k0 = kept(p.k_offsets[seq], 0, p.k_rows);
    const int64_t room = kept(p.k_offsets[seq + 1], s.k0, p.k_rows) - s.k0;
    s.nk = int(p.k_lengths ? kept(p.k_lengths[seq], 0, room) : room);
}

__device__ __forceinline__ int wave_sum(int x)
{
#pragma unroll
    for (int m = 1; m < 64; m *= 2) x += __shfl_xor(x, m);
    return x;
}

__device__ __forceinline__ int wave_max(int x)
{
#pragma unroll
    for (int m = 1; m < 64; m *= 2) x = max(x, __shfl_xor(x, m));
    return x;
}

// inclusive sum over the lanes
__device__ __forceinline__ long long wave_scan(long long x)
{
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const long long left = __shfl_up(x, m);
        if (int(threadIdx.x & 63) >= m) x += left;
    }
    return x;
}

// a lane's span, for all
__device__ __forceinline__ Span taken(const Span& own, int lane, int seq, int tile)
{
    Span s;
    s.q0 = __shfl(int(own.q0), lane);
    s.k0 = __shfl(int(own.k0), lane);
    s.nq = __shfl(own.nq, lane);
    s.nk = __shfl(own.nk, lane);
    s.seq = seq;
    s.tile = tile;
    return s;
}

// In which order tiles are handed out, from the dearest to the cheapest where up to 64 sequences allow it: by their distance
// from the sequence's first tile (a causal tile of queries sees the keys before it), or from its last (a tile of keys is
// seen by the queries behind it).
enum class Dear { kLast, kFirst };

__device__ __forceinline__ int tiles_of(const Tiling& t, const Span& s)
{
    return t.keys ? (s.nk + t.size - 1) / t.size : int((int64_t(s.nq) * t.mult + t.size - 1) / t.size);
}

__device__ __forceinline__ Span any_tile(const Packed& p, const Tiling& how, int wanted, Dear dear)
{
    Span s;
    s.seq = -1;
    auto count = [&](const Span& one) { return tiles_of(how, one); };
    const int lane = threadIdx.x & 63;
    if (p.n == 1) {
        span_of(p, 0, s);
        const int tiles = count(s);
        s.tile = dear == Dear::kLast ? tiles - 1 - wanted : wanted;
        if (wanted >= tiles) s.seq = -1;
        return s;
    }
    if (p.n <= kMapped) {
        // a sequence to a lane.  Level by level (a level: the tiles at the same distance), the levels below r hold
        // sum of min(tiles, r); r by bisection, bit by bit
        Span own{};
        if (lane < p.n) span_of(p, lane, own);
        const int tiles = lane < p.n ? count(own) : 0;
        const int target = wave_sum(tiles) - 1 - wanted;
        if (target < 0) return s;
        const int most = wave_max(tiles);
        int level = 0, below = 0;
        for (int bit = 31 - __clz(most); bit >= 0; --bit) {
            const int r = level + (1 << bit), c = wave_sum(min(tiles, r));
            if (c <= target) level = r, below = c;
        }
        const unsigned long long there = __ballot(tiles > level), mine = 1ull << lane;
        const int holder = __ffsll(__ballot((there & mine) && __popcll(there & (mine - 1)) == target - below)) - 1;
        return taken(own, holder, holder, dear == Dear::kLast ? level : __shfl(tiles, holder) - 1 - level);
    }
    const int target = p.map[0] - 1 - wanted;
    if (target < 0) return s;
    const int seq = p.map[2 + 2 * target], tile = p.map[3 + 2 * target];
    span_of(p, seq, s);
    s.tile = tile;
    if (dear == Dear::kFirst) s.tile = count(s) - 1 - tile;
    return s;
}

// The `wanted`-th tile over all sequences; each wave finds it by itself, and holds it in scalar registers.
__device__ __forceinline__ Span find_tile(const Packed& p, const Tiling& how, int wanted, Dear dear)
{
    const Span v = any_tile(p, how, wanted, dear);
    Span s;
    s.q0 = __builtin_amdgcn_readfirstlane(int(v.q0));
    s.k0 = __builtin_amdgcn_readfirstlane(int(v.k0));
    s.nq = __builtin_amdgcn_readfirstlane(v.nq);
    s.nk = __builtin_amdgcn_readfirstlane(v.nk);
    s.tile = __builtin_amdgcn_readfirstlane(v.tile);
    s.seq = __builtin_amdgcn_readfirstlane(v.seq);
    return s;
}

// The tiles of many sequences, listed once for all blocks of the kernels behind it: a block to a tiling.
struct MapArgs {
    Packed packed;
    Tiling how[2];
    int* map[2];
    int room[2];             // tiles that a map holds: offsets that do not ascend could name more
};

constexpr int kMapThreads = 1024;

static __global__ void __launch_bounds__(kMapThreads) map_kernel(MapArgs p)
{
    __shared__ long long s_sums[kMapThreads / 64];          // offsets that do not ascend can name more tiles than 32 bits count
    const int tid = threadIdx.x, lane = tid & 63;
    const Tiling how = blockIdx.x ? p.how[1] : p.how[0];
    int* const map = blockIdx.x ? p.map[1] : p.map[0];
    const int room = blockIdx.x ? p.room[1] : p.room[0];
    long long done = 0;
    for (int64_t base = 0; base < p.packed.n; base += kMapThreads) {
        Span one{};
        const int seq = int(base + tid);
        if (base + tid < p.packed.n) span_of(p.packed, seq, one);
        const int own = base + tid < p.packed.n ? tiles_of(how, one) : 0;
        const long long upto = wave_scan(own);
        __syncthreads();
        if (lane == 63) s_sums[tid >> 6] = upto;
        __syncthreads();
        long long before = done + upto - own;
        for (int w = 0; w < kMapThreads / 64; ++w) {
            if (w < (tid >> 6)) before += s_sums[w];
            done += s_sums[w];
        }
        for (int i = 0; i < own && before + i < room; ++i) {
            map[2 + 2 * (before + i)] = seq;
            map[3 + 2 * (before + i)] = i;
        }
    }
    if (tid == 0) map[0] = done < room ? int(done) : room;
}

// offsets of a tile's rows are 32-bit
inline void check_strides(std::initializer_list<int64_t> tokens)
{
    for (const int64_t t : tokens) require(t >= 0 && t < (int64_t(1) << 23), "tokens are at most 2^23 elements apart");
}

// most tiles of `size` rows that n sequences with `rows` rows in all have
inline int64_t most_tiles(int64_t rows, int64_t n, int64_t size) { return rows / size + (rows < n ? rows : n); }

inline size_t map_bytes(int64_t tiles, int64_t n) { return n > kMapped ? (size_t(tiles + 1) * 2 * sizeof(int) + 255) / 256 * 256 : 0; }

}  // namespace seqamd
