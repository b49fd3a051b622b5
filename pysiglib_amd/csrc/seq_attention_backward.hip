// Gradients of the attention over packed sequences.
//
// Mathematics.  With the forward's log-sums, P = 2^(scale' S - lse') is formed again tile by tile.  delta = rowsum(dO . O),
// dS = P . (dO V^T - delta), dQ = scale dS K, dK = scale dS^T Q, dV = P^T dO.
//
// Two kernels, one with its queries fixed (dQ and delta), one with its keys fixed (dK and dV, over all query heads that share
// them): seven products instead of the five that one kernel would form, but every sum belongs to one block, so nothing is
// added through memory in an order that changes from call to call.
//
// Keys fixed: a wave cannot hold sums, keys and values of 64 keys of 128 channels at once with two waves to a SIMD, so waves
// work in pairs.  The first forms P of a tile of queries and adds to dV, the second, one tile behind, takes P from shared
// memory, forms dS and adds to dK.  Operands are rounded to the inputs' type (P, dS), sums are 32-bit.  In shared memory P is the
// upper three bytes of its 32-bit float: its whole range, so that keys with little weight beside another have dK as exact as
// others, and 2^-15 of its size, an eighth of float16's rounding at the least, which dS gets next.
#include "seq_attention.h"

namespace seqamd {
namespace {

struct GradArgs {
    const void *q, *k, *v, *out, *grad;       // out and grad: [q_rows][heads][dim]
    const float* lse;
    void *dq, *dk, *dv;                       // contiguous
    float* delta;                             // [q_rows][heads]
    Packed packed, k_packed;                  // the second with the map of tiles of keys
    int64_t q_token, q_head, k_token, k_head, v_token, v_head, g_token, g_head;
    int heads, kv_heads, dim, causal;
    float scale, scale2;                      // scale2 = scale * log2(e)
    unsigned first_block;                     // of a launch
};

constexpr float kLog2e = 1.44269504088896341f;
constexpr int kExact = 512;               // keys up to which delta is summed from its definition, 128 channels, causal

// Weights between two waves: the upper halves of eight floats in four words, the bytes below these of four floats in one
__device__ __forceinline__ u32x4 upper_halves(const f32x16& x, int first)
{
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(__float_as_uint(x[first + 2 * i + 1]), __float_as_uint(x[first + 2 * i]), 0x07060302u);
    return w;
}

__device__ __forceinline__ u32x4 third_bytes(const f32x16& x)
{
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = __builtin_amdgcn_perm(__float_as_uint(x[4 * i + 1]), __float_as_uint(x[4 * i]), 0x0c0c0501u) |
               __builtin_amdgcn_perm(__float_as_uint(x[4 * i + 3]), __float_as_uint(x[4 * i + 2]), 0x05010c0cu);
    return w;
}

// the i-th of the eight
__device__ __forceinline__ float weight_of(u32x4 upper, unsigned third, int i)
{
    return __uint_as_float(__builtin_amdgcn_perm(upper[i / 2], third, (i & 1 ? 0x07060000u : 0x05040000u) | unsigned(i & 3) << 8 | 0x0cu));
}

// the power of two that brings a size near 1
__device__ __forceinline__ float towards_one(float size)
{
    return size > 0.0f && size < INFINITY ? ldexpf(1.0f, min(-ilogbf(size), 126)) : 1.0f;
}

// float16 holds dS, as large as gradients times values, only near 1, and P only down to 2^-24.  Those of a lane's column go into their
// product multiplied by a power of two, of the lane's own, that brought the largest so far near 1; one that is 2^10 times as large
// moves it, and what is summed up with it.  Smaller ones lose bits only where they are small beside the largest of the same sum.
struct Lift {
    float times = 1.0f, most = 0.0f;          // most: of what it is good for
};

template <int BLOCKS>
__device__ __forceinline__ void fit(Lift& lift, const f32x16& x, f32x16* sums)
{
    auto size = [&](int i) { return __builtin_fabsf(x[i]); };
    float most = larger(size(0), size(1), size(2));
#pragma unroll
    for (int i = 3; i < 15; i += 2) most = larger(most, size(i), size(i + 1));
    most = larger(most, size(15));
    most = larger(most, swapped(most));
    if (__any(most > lift.most)) {
        const bool moves = most > lift.most;
        const float times = moves ? towards_one(most) : lift.times, change = times / lift.times;
        if (moves) lift.most = most < INFINITY ? 1024.0f / times : INFINITY;
        lift.times = times;
#pragma unroll
        for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) sums[d][i] *= change;
    }
}

// Operands that are not finite, of keys that a query does not see or queries that do not see a key: neither a weight of zero nor dS,
// set to zero there, makes zero with them in the second product.  They are taken out of the tiles that hide some from others, and put
// back at the end into the sums that they belong to.  P knows of them all the same: by the log-sum of a query that is or sees such a
// one, which is not finite then, unless the key's score was -infinity: P is set to zero there.  Where they are multiplied with dS, which
// they make zero or not finite, it is not a number that they leave.
template <typename T>
__device__ __attribute__((noinline)) void spoil(const T* row, T* to, int dim, int half)
{
#pragma unroll 1
    for (int ch = 4 * half; ch < dim; ch += (ch & 3) == 3 ? 5 : 1)
        if (!__builtin_isfinite(static_cast<float>(row[ch]))) to[ch] = T(__builtin_nanf(""));
}

// ---- queries fixed: 32 to a wave, tiles of kKeys keys.  Bound: the matrix units, busy 40 % of the cycles, between them the
// exponentials that wait for the products (4 sequences of 1600 to 2047, 32 heads on 8 of 128, bfloat16: 248 to 268 us) ----
template <typename T, int DP, int WAVES, int kKeys>
__global__ void __launch_bounds__(WAVES * 64, 2) dq_kernel(GradArgs p)
{
    constexpr int kThreads = WAVES * 64, kRows = 32 * WAVES, kSlices = DP / 16, kBlocks = DP / 32;
    constexpr int kTileBytes = kKeys * Tile<DP>::kRowBytes, kLoads = kKeys * Tile<DP>::kChunks / kThreads;
    static_assert(kLoads * kThreads == kKeys * Tile<DP>::kChunks, "");
    static_assert(kKeys == 32, "");
    __shared__ __attribute__((aligned(16))) char s_tiles[2][2][kTileBytes];
    constexpr int kHiding = kRows / kKeys + 2;          // tiles that hide keys from some queries of the block, at most
    __shared__ unsigned s_bad[kHiding], s_any;          // their keys that are not finite, and whether there are any
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (tid < kHiding) s_bad[tid] = 0;
    if (tid == 0) s_any = 0;
    const unsigned block = p.first_block + blockIdx.x;
    const int turn = block % p.heads, head = (turn % p.kv_heads) * (p.heads / p.kv_heads) + turn / p.kv_heads, kv = turn % p.kv_heads;
    const Span at = find_tile(p.packed, Tiling{false, kRows, 1}, block / p.heads, Dear::kLast);
    if (at.seq < 0) return;
    const int q_first = at.tile * kRows, shift = at.nk - at.nq;
    const int q_past = q_first + kRows < at.nq ? q_first + kRows : at.nq;
    int keys = at.nk;
    if (p.causal && q_past + shift < keys) keys = q_past + shift < 0 ? 0 : q_past + shift;
    const int tiles = (keys + kKeys - 1) / kKeys;

    const RowRead<DP> rows(lane);
    const ColumnRead<DP> columns(lane);
    const int query = q_first + wave * 32 + (lane & 31), row = query < at.nq ? query : at.nq - 1;
    Frag<T> q[kSlices], g[kSlices];
    float delta = 0.0f;
    {
        const T* from = static_cast<const T*>(p.q) + (at.q0 + row) * p.q_token + head * p.q_head;
        const T* grad = static_cast<const T*>(p.grad) + (at.q0 + row) * p.g_token + head * p.g_head;
        const T* out = static_cast<const T*>(p.out) + ((at.q0 + row) * p.heads + head) * p.dim;
#pragma unroll
        for (int k = 0; k < kSlices; ++k) {
            const int d = 16 * k + 8 * half;
            q[k] = load_row<T>(from, d, p.dim);
            g[k] = load_row<T>(grad, d, p.dim);
            const Frag<T> y = load_row<T>(out, d, p.dim);
#pragma unroll
            for (int i = 0; i < 8; ++i) delta = fmaf(static_cast<float>(g[k][i]), static_cast<float>(y[i]), delta);
        }
        delta += swapped(delta);
    }
    const int64_t place = (at.q0 + row) * p.heads + head;
    Lift lift;
    const float lse = p.lse[place] == -INFINITY ? INFINITY : p.lse[place] * kLog2e;
    const int last = p.causal && query + shift < at.nk - 1 ? query + shift : at.nk - 1;
    // The output's rounding makes delta wrong by u |dO| |O|, which matters where few keys share the weight: dS, differences from
    // delta, is as small there as that.  64 channels: e, the sum of dS, is what delta is short of, and dQ is short of e P K, which
    // is summed beside it (when it was chosen, 24 sequences of up to 2000, 16 heads on 4, the whole gradient: 418 us, without it 390;
    // sequences of 17 to 129: 66 us, 74 when they went over their keys twice; now 440 and 69).  128 channels: no registers for these sums; queries go over up to
    // `exact` keys twice.  Every query has them all where none are hidden, and the error's share falls with the channels: there
    // they do so to longer lengths (8 sequences of 1000, 16 heads on 8, nothing hidden: 381 us, once 321; dQ's error against 64
    // bits, in those of a result that is rounded once: 1.43 and 1.55).
    constexpr bool kMend = DP == 64;
    const int exact = kExact * (p.causal ? 1 : 4) * (p.dim > 96 ? 1 : 2);
    f32x16 dq[kBlocks], pk[kMend ? kBlocks : 1];
    float short_of = 0.0f;
#pragma unroll
    for (int d = 0; d < kBlocks; ++d) {
        dq[d] = zeros16();
        if (kMend) pk[d] = zeros16();
    }

    u32x4 next[2][kLoads];
    unsigned k_at[kLoads], v_at[kLoads];
    auto offsets = [&](int left) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int e = i * kThreads + tid, r = min(e / Tile<DP>::kChunks, left - 1), ch = min(e % Tile<DP>::kChunks * 8, p.dim - 8);
            k_at[i] = unsigned((r * int(p.k_token) + ch) * int(sizeof(T)));
            v_at[i] = unsigned((r * int(p.v_token) + ch) * int(sizeof(T)));
        }
    };
    const char* const k_base = reinterpret_cast<const char*>(static_cast<const T*>(p.k) + at.k0 * p.k_token + kv * p.k_head);
    const char* const v_base = reinterpret_cast<const char*>(static_cast<const T*>(p.v) + at.k0 * p.v_token + kv * p.v_head);
    auto fetch = [&](int tile) __attribute__((always_inline)) {
        if (tile == 0 || (tile + 1) * kKeys > at.nk) offsets(min(at.nk - tile * kKeys, kKeys));
        const char *kp = k_base + tile * int64_t(kKeys * sizeof(T)) * p.k_token, *vp = v_base + tile * int64_t(kKeys * sizeof(T)) * p.v_token;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            next[0][i] = load_at(kp, k_at[i]);
            next[1][i] = load_at(vp, v_at[i]);
        }
    };
    const int hiding = min(at.nk, p.causal ? max(q_first + shift + 1, 0) : at.nk) / kKeys;       // the first tile that hides a key from a query
    // keys' channels past the head's are zero: zeros of the query make no zero with what is not finite
    static_assert(kThreads % Tile<DP>::kChunks == 0, "");
    const bool there = tid % Tile<DP>::kChunks * 8 < p.dim;
    auto put = [&](int buffer, int tile) __attribute__((always_inline)) {
        auto place = [&](int i) { return Tile<DP>::at((i * kThreads + tid) / Tile<DP>::kChunks, (i * kThreads + tid) % Tile<DP>::kChunks); };
#pragma unroll
        for (int i = 0; i < kLoads; ++i) *reinterpret_cast<u32x4*>(s_tiles[buffer][1] + place(i)) = next[1][i];
        if (tile >= hiding) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                u32x4 x = there ? next[0][i] : u32x4{0, 0, 0, 0};
                if (take_them_out<T>(x)) {
                    atomicOr(&s_bad[tile - hiding], 1u << (i * kThreads + tid) / Tile<DP>::kChunks);
                    s_any = 1;
                }
                *reinterpret_cast<u32x4*>(s_tiles[buffer][0] + place(i)) = x;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) *reinterpret_cast<u32x4*>(s_tiles[buffer][0] + place(i)) = there ? next[0][i] : u32x4{0, 0, 0, 0};
        }
    };
    // S^T and dP^T of 32 keys
    auto pair_products = [&](const char* kt, const char* vt, int row0, f32x16& s, f32x16& dp) __attribute__((always_inline)) {
        s = zeros16(), dp = zeros16();
#pragma unroll
        for (int k = 0; k < kSlices; ++k) {
            s = product(rows.template get<T>(kt, row0, k), q[k], s);
            dp = product(rows.template get<T>(vt, row0, k), g[k], dp);
        }
    };
    if (tiles) {
        fetch(0);
        if (hiding == 0) __syncthreads();       // s_bad is clear
        put(0, 0);
    }
#pragma unroll
    for (int k = 0; k < kSlices; ++k) {
        arrive<T>(q[k]);
        arrive<T>(g[k]);
    }
    auto hides = [&](int key0) { return key0 + 32 > at.nk || (p.causal && key0 + 31 > q_first + wave * 32 + shift); };
    // P of 32 keys from their S; hidden ones have none, and no dP
    auto weigh = [&](f32x16& s, f32x16& dp, int tile) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], p.scale2, -lse));
        if (hides(tile * kKeys)) {
            const unsigned bad = s_bad[tile - hiding] >> 4 * half;
            const int past = last - tile * kKeys - 4 * half;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (row_in(i, 0) > past) s[i] = dp[i] = 0.0f;
                if ((bad >> row_in(i, 0) & 1) != 0 && s[i] == s[i]) s[i] = 0.0f;
            }
        }
    };
    int buffer = 0;
    if (!kMend && keys <= exact && tiles) {       // first to sum P dP, which is delta
        float sum = 0.0f;
        for (int tile = 0; tile < tiles; ++tile, buffer ^= 1) {
            __syncthreads();
            const int after = tile + 1 < tiles ? tile + 1 : 0;
            fetch(after);
            f32x16 s, dp;
            pair_products(s_tiles[buffer][0], s_tiles[buffer][1], 0, s, dp);
            weigh(s, dp, tile);
#pragma unroll
            for (int i = 0; i < 16; ++i) sum = fmaf(s[i], dp[i], sum);
            put(buffer ^ 1, after);
        }
        delta = sum + swapped(sum);
    }
    for (int tile = 0; tile < tiles; ++tile, buffer ^= 1) {
        __syncthreads();
        if (tile + 1 < tiles) fetch(tile + 1);
        const char *kt = s_tiles[buffer][0], *vt = s_tiles[buffer][1];
        const int key0 = tile * kKeys;
        if (!p.causal || key0 <= q_first + wave * 32 + 31 + shift) {        // otherwise none of the wave's queries sees these
            f32x16 s, dp;
            pair_products(kt, vt, 0, s, dp);
            weigh(s, dp, tile);
            Frag<T> w[2];
            if (kMend) w[0] = rounded<T>(s, 0), w[1] = rounded<T>(s, 8);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] *= dp[i] - delta;
                if (kMend) short_of += s[i];
            }
            if constexpr (__is_same(T, f16)) {
                fit<kBlocks>(lift, s, dq);
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] *= lift.times;
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Frag<T> ds = rounded<T>(s, 8 * u);
#pragma unroll
                for (int d = 0; d < kBlocks; ++d) {
                    const Frag<T> f = columns.template get<T>(kt, 16 * u, d);
                    dq[d] = product(f, ds, dq[d]);
                    if (kMend) pk[d] = product(f, w[u], pk[d]);
                }
            }
        }
        if (tile + 1 < tiles) put(buffer ^ 1, tile + 1);
    }
    if (kMend) {
        short_of += swapped(short_of);
        delta += short_of;
        short_of *= lift.times;
#pragma unroll
        for (int d = 0; d < kBlocks; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) dq[d][i] = fmaf(-short_of, pk[d][i], dq[d][i]);
    }
    if (query >= at.nq) return;
    if (half == 0) p.delta[place] = delta;
    T* const to = static_cast<T*>(p.dq) + place * p.dim;
    store_row<T, DP>(to, dq, p.scale / lift.times, p.dim, half);
    if (__builtin_expect(s_any != 0, 0))
        for (int k = hiding * kKeys; k <= last; ++k) spoil(static_cast<const T*>(p.k) + (at.k0 + k) * p.k_token + kv * p.k_head, to, p.dim, half);
}

// ---- keys fixed: 32 to a pair of waves, PAIRS pairs to a block; queries in steps of kQueries.  Bound: as above, 41 % (the same
// sequences: 319 to 348 us) ----
template <typename T, int DP, int PAIRS, int kQueries>
__global__ void __launch_bounds__(PAIRS * 128, 2) dkv_kernel(GradArgs p)
{
    constexpr int kThreads = PAIRS * 128, kRows = 32 * PAIRS, kSlices = DP / 16, kBlocks = DP / 32, kParts = kQueries / 32;
    constexpr int kTileBytes = kQueries * Tile<DP>::kRowBytes, kLoads = kQueries * Tile<DP>::kChunks / kThreads;
    static_assert(kLoads * kThreads == kQueries * Tile<DP>::kChunks, "");
    __shared__ __attribute__((aligned(16))) char s_tiles[3][2][kTileBytes];
    __shared__ __attribute__((aligned(16))) float s_lse[3][kQueries], s_delta[3][kQueries];
    __shared__ __attribute__((aligned(16))) u32x4 s_weights[2][PAIRS][kParts][3][64];
    __shared__ unsigned s_any;          // whether operands that are not finite were taken out
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6), pair = wave % PAIRS;
    const bool second = wave >= PAIRS;
    if (tid == 0) s_any = 0;
    const unsigned block = p.first_block + blockIdx.x;
    const int kv = block % p.kv_heads, group = p.heads / p.kv_heads;
    const Span at = find_tile(p.k_packed, Tiling{true, kRows, 1}, block / p.kv_heads, Dear::kFirst);
    if (at.seq < 0) return;
    const int k_first = at.tile * kRows, shift = at.nk - at.nq;
    // the first query that sees any of the block's keys
    int q_begin = p.causal ? k_first - shift : 0;
    q_begin = q_begin < 0 ? 0 : (q_begin > at.nq ? at.nq : q_begin);
    const int tiles = (at.nq - q_begin + kQueries - 1) / kQueries, steps = tiles * group;

    const RowRead<DP> rows(lane);
    const ColumnRead<DP> columns(lane);
    const int key0 = k_first + pair * 32, key = key0 + (lane & 31);
    Frag<T> fixed[kSlices];             // keys, in the second wave values
    f32x16 sums[kBlocks];               // dV, in the second wave dK
    {
        const int64_t r = at.k0 + min(key, at.nk - 1);
        const T* from = second ? static_cast<const T*>(p.v) + r * p.v_token + kv * p.v_head : static_cast<const T*>(p.k) + r * p.k_token + kv * p.k_head;
#pragma unroll
        for (int k = 0; k < kSlices; ++k) fixed[k] = load_row<T>(from, 16 * k + 8 * half, p.dim);
#pragma unroll
        for (int d = 0; d < kBlocks; ++d) sums[d] = zeros16();
    }
    Lift lift;

    u32x4 next[2][kLoads];
    float next_lse, next_delta;
    bool next_in, next_hides;
    // queries up to `seen` and of the tiles that begin before it: some of them do not see some of the block's keys
    const int seen = p.causal ? k_first + kRows - 1 - shift : 0;
    auto fetch = [&](int head, int tile) __attribute__((always_inline)) {
        const int q0 = q_begin + tile * kQueries, left = at.nq - q0 - 1;
        const char* qp = reinterpret_cast<const char*>(static_cast<const T*>(p.q) + (at.q0 + q0) * p.q_token + head * p.q_head);
        const char* gp = reinterpret_cast<const char*>(static_cast<const T*>(p.grad) + (at.q0 + q0) * p.g_token + head * p.g_head);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int e = i * kThreads + tid, r = min(e / Tile<DP>::kChunks, left), ch = min(e % Tile<DP>::kChunks * 8, p.dim - 8);
            next[0][i] = load_at(qp, unsigned((r * int(p.q_token) + ch) * int(sizeof(T))));
            next[1][i] = load_at(gp, unsigned((r * int(p.g_token) + ch) * int(sizeof(T))));
        }
        const int64_t first = (at.q0 + q0) * p.heads + head;
        const int mine = tid % kQueries, place = min(mine, left) * p.heads;
        next_lse = p.lse[first + place];
        next_delta = p.delta[first + place];
        next_in = mine <= left;
        next_hides = q0 < seen;
    };
    auto put = [&](int buffer) __attribute__((always_inline)) {
        auto place = [&](int i) { return Tile<DP>::at((i * kThreads + tid) / Tile<DP>::kChunks, (i * kThreads + tid) % Tile<DP>::kChunks); };
        if (next_hides) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                u32x4 x = next[0][i], y = next[1][i];
                // a query that is not finite has a log-sum that is not either, and P from that
                const bool one = take_them_out<T>(x), two = take_them_out<T>(y);
                if (one || two) s_any = 1;
                *reinterpret_cast<u32x4*>(s_tiles[buffer][0] + place(i)) = x;
                *reinterpret_cast<u32x4*>(s_tiles[buffer][1] + place(i)) = y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                *reinterpret_cast<u32x4*>(s_tiles[buffer][0] + place(i)) = next[0][i];
                *reinterpret_cast<u32x4*>(s_tiles[buffer][1] + place(i)) = next[1][i];
            }
        }
        if (tid < kQueries) {           // queries past the end, and those that see nothing, have no weights
            const bool none = !next_in || next_lse == -INFINITY;
            s_lse[buffer][tid] = none ? INFINITY : next_lse * kLog2e;
            s_delta[buffer][tid] = none ? 0.0f : next_delta;
        }
    };
    // a tile's rows times the fixed operand, its parts of 32 rows side by side: products of one part wait for each other
    auto by_rows = [&](const char* tile, f32x16* x) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < kParts; ++c) x[c] = zeros16();
#pragma unroll
        for (int k = 0; k < kSlices; ++k)
#pragma unroll
            for (int c = 0; c < kParts; ++c) x[c] = product(rows.template get<T>(tile, 32 * c, k), fixed[k], x[c]);
    };
    // adds the columns of 32 rows times the two operands
    auto by_columns = [&](const char* tile, int row0, const Frag<T>* w) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int d = 0; d < kBlocks; ++d) sums[d] = product(columns.template get<T>(tile, row0 + 16 * u, d), w[u], sums[d]);
    };
    // nothing of the 32 queries from q0 on that do not see the key
    auto hide = [&](f32x16& x, int q0) __attribute__((always_inline)) {
        if (p.causal && q0 + shift < key0 + 31)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (key > q0 + row_in(i, half) + shift) x[i] = 0.0f;
    };
    if (steps) {
        fetch(kv * group, 0);
        __syncthreads();                // s_any is clear
        put(0);
    }
#pragma unroll
    for (int k = 0; k < kSlices; ++k) arrive<T>(fixed[k]);
    int now = 0, before = 2;            // buffers of this step and of the one before it
    int head = kv * group, tile = 0;    // of this step
    for (int step = 0; step <= steps && steps; ++step) {
        __syncthreads();
        const int after = now == 2 ? 0 : now + 1;
        const int q0 = q_begin + tile * kQueries;
        if (++tile == tiles) tile = 0, ++head;
        if (step + 1 < steps) fetch(head, tile);
        if (!second && step < steps) {
            f32x16 parts[kParts];
            by_rows(s_tiles[now][0], parts);
#pragma unroll
            for (int c = 0; c < kParts; ++c) {
                f32x16& s = parts[c];
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], p.scale2, -s_lse[now][32 * c + row_in(i, half)]));
                hide(s, q0 + 32 * c);
#pragma unroll
                for (int u = 0; u < 2; ++u) s_weights[step & 1][pair][c][u][lane] = upper_halves(s, 8 * u);
                s_weights[step & 1][pair][c][2][lane] = third_bytes(s);
                if constexpr (__is_same(T, f16)) {
                    fit<kBlocks>(lift, s, sums);
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] *= lift.times;
                }
                const Frag<T> w[2] = {rounded<T>(s, 0), rounded<T>(s, 8)};
                by_columns(s_tiles[now][1], 32 * c, w);
            }
        }
        if (second && step > 0) {
            f32x16 parts[kParts];
            by_rows(s_tiles[before][1], parts);
#pragma unroll
            for (int c = 0; c < kParts; ++c) {
                f32x16& x = parts[c];
                const u32x4 third = s_weights[(step - 1) & 1][pair][c][2][lane];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const u32x4 upper = s_weights[(step - 1) & 1][pair][c][u][lane];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float d = x[8 * u + i] - s_delta[before][32 * c + row_in(8 * u + i, half)];
                        x[8 * u + i] = weighed(weight_of(upper, third[2 * u + i / 4], i), d);
                    }
                }
                if constexpr (__is_same(T, f16)) {
                    fit<kBlocks>(lift, x, sums);
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] *= lift.times;
                }
                const Frag<T> ds[2] = {rounded<T>(x, 0), rounded<T>(x, 8)};
                by_columns(s_tiles[before][0], 32 * c, ds);
            }
        }
        if (step + 1 < steps) put(after);
        before = now;
        now = after;
    }
    if (key >= at.nk) return;
    T* const to = static_cast<T*>(second ? p.dk : p.dv) + ((at.k0 + key) * p.kv_heads + kv) * p.dim;
    store_row<T, DP>(to, sums, (second ? p.scale : 1.0f) / lift.times, p.dim, half);
    if (__builtin_expect(steps != 0 && s_any != 0, 0))
        for (int h = kv * group; h < (kv + 1) * group; ++h)
            for (int i = max(key - shift, 0); i < min(seen + kQueries, at.nq); ++i) {
                if (second) spoil(static_cast<const T*>(p.q) + (at.q0 + i) * p.q_token + h * p.q_head, to, p.dim, half);
                else add_them(static_cast<const T*>(p.grad) + (at.q0 + i) * p.g_token + h * p.g_head, to, p.dim, half);
            }
}

// Blocks by the average length of the sequences, from times of whole calls (16 heads on 4 of 64 channels, 16000 tokens, and 32 on
// 8 of 128, 8000 tokens).
// Queries fixed, waves of a block: 64 channels, sequences of 64: 2 waves 90 us, 4 waves 99; of 400: 169 and 174; of 2000: 360 and 356;
// one of 8192: 852 and 842.  128 channels, of 16: 2 waves 178 us, 8 waves 232; of 400: 4 waves 250; of 2000: 4 waves 466 us, 8 waves 480; one of 8192: 8 waves 1934 us.
// Keys fixed: 64 channels, 2 pairs, sequences of 16: steps of 32 queries 94 us, of 64 132; of 400: 150 and 139; of 8192: 895
// and 804.  128 channels, of 64: 2 pairs and 32 queries 172 us, 4 pairs and 64 queries 191; of 1000: 493 and 498; 4 of 1600 to
// 2047: 546 and 508; two of 4096: 1057 and 955.
struct Blocks {
    int waves, pairs, queries;
};

Blocks blocks_of(int64_t q_rows, int64_t k_rows, int64_t n, int64_t dim)
{
    const int64_t queries = q_rows / n, keys = k_rows / n;
    if (dim <= 64) return Blocks{queries <= 1400 ? 2 : 4, 2, keys <= 200 ? 32 : 64};
    return Blocks{queries <= 200 ? 2 : (queries <= 2048 ? 4 : 8), keys <= 700 ? 2 : 4, keys <= 700 ? 32 : 64};
}

struct Space {
    size_t q_map, k_map, all;
};

Space space_of(int64_t q_rows, int64_t k_rows, int64_t n, int64_t heads, int64_t dim)
{
    const Blocks b = blocks_of(q_rows, k_rows, n, dim);
    Space s;
    s.q_map = map_bytes(most_tiles(q_rows, n, 32 * b.waves), n);
    s.k_map = map_bytes(most_tiles(k_rows, n, 32 * b.pairs), n);
    s.all = s.q_map + s.k_map + size_t(q_rows) * heads * sizeof(float);
    return s;
}

template <typename T, int DP>
void backward(GradArgs& p, void* workspace, hipStream_t stream)
{
    const Blocks b = blocks_of(p.packed.q_rows, p.packed.k_rows, p.packed.n, p.dim);
    const Space space = space_of(p.packed.q_rows, p.packed.k_rows, p.packed.n, p.heads, p.dim);
    char* const at = static_cast<char*>(workspace);
    p.delta = reinterpret_cast<float*>(at + space.q_map + space.k_map);
    const int64_t q_blocks = most_tiles(p.packed.q_rows, p.packed.n, 32 * b.waves) * p.heads;
    const int64_t k_blocks = most_tiles(p.packed.k_rows, p.packed.n, 32 * b.pairs) * p.kv_heads;
    require(q_blocks < (int64_t(1) << 31) && k_blocks < (int64_t(1) << 31), "too many queries and heads");
    p.k_packed = p.packed;
    if (space.q_map) {
        MapArgs m{};
        m.packed = p.packed;
        m.how[0] = Tiling{false, 32 * b.waves, 1};
        m.how[1] = Tiling{true, 32 * b.pairs, 1};
        m.map[0] = reinterpret_cast<int*>(at);
        m.map[1] = reinterpret_cast<int*>(at + space.q_map);
        m.room[0] = int(most_tiles(p.packed.q_rows, p.packed.n, 32 * b.waves));
        m.room[1] = int(most_tiles(p.packed.k_rows, p.packed.n, 32 * b.pairs));
        p.packed.map = m.map[0];
        p.k_packed.map = m.map[1];
        hipLaunchKernelGGL(map_kernel, dim3(2), dim3(kMapThreads), 0, stream, m);
        SIG_HIP(hipGetLastError());
    }
    switch (b.waves) {
    case 2: launch_all(dq_kernel<T, DP, 2, 32>, q_blocks, 128, stream, p); break;
    case 4: launch_all(dq_kernel<T, DP, 4, 32>, q_blocks, 256, stream, p); break;
    default: launch_all(dq_kernel<T, 128, 8, 32>, q_blocks, 512, stream, p); break;
    }
    if (b.queries == 32) launch_all(dkv_kernel<T, DP, 2, 32>, k_blocks, 256, stream, p);
    else launch_all(dkv_kernel<T, DP, DP == 64 ? 2 : 4, 64>, k_blocks, DP == 64 ? 256 : 512, stream, p);
}

}  // namespace
}  // namespace seqamd

using namespace seqamd;

extern "C" {

__attribute__((visibility("default"))) uint64_t cusig_amd_attention_backprop_workspace(uint64_t q_rows, uint64_t k_rows, uint64_t sequences, uint64_t heads, uint64_t dim) noexcept
{
    // never nothing: the workspace is a pointer in every call
    const uint64_t bytes = sequences ? space_of(int64_t(q_rows), int64_t(k_rows), int64_t(sequences), int64_t(heads), int64_t(dim)).all : 0;
    return bytes ? bytes : 256;
}

__attribute__((visibility("default"))) int cusig_amd_attention_backprop(
    int dtype, const void* grad_out, const void* q, const void* k, const void* v, const void* out, const float* lse, const int* q_offsets,
    const int* k_offsets, void* dq, void* dk, void* dv, uint64_t q_rows, uint64_t k_rows, uint64_t sequences, uint64_t heads, uint64_t kv_heads, uint64_t dim,
    int64_t q_token, int64_t q_head, int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head, int64_t grad_token, int64_t grad_head, float scale,
    bool causal, void* workspace, uint64_t workspace_bytes, void* stream) noexcept
{
    return sigamd::guarded([&] {
        require(q_rows < (uint64_t(1) << 31) && k_rows < (uint64_t(1) << 31) && sequences < (uint64_t(1) << 31), "too many rows or sequences");
        require(dim >= 8 && dim <= 128 && dim % 8 == 0, "a head has 8 to 128 channels, a multiple of 8");
        require(kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads < (1u << 20), "heads are a multiple of the key heads");
        require(scale > 0.0f && std::isfinite(scale), "the scale is positive and finite");
        check_workspace(workspace, workspace_bytes, cusig_amd_attention_backprop_workspace(q_rows, k_rows, sequences, heads, dim));
        check_strides({q_token, k_token, v_token, grad_token});
        if (sequences == 0) return;
        require(q_offsets && k_offsets && (q_rows == 0 || (grad_out && q && out && lse && dq)) && (k_rows == 0 || (k && v && dk && dv)), "a tensor is missing");
        GradArgs p{};
        p.q = q, p.k = k, p.v = v, p.out = out, p.grad = grad_out, p.lse = lse, p.dq = dq, p.dk = dk, p.dv = dv;
        p.packed = Packed{q_offsets, k_offsets, nullptr, int64_t(q_rows), int64_t(k_rows), int(sequences), nullptr};
        p.q_token = q_token, p.q_head = q_head, p.k_token = k_token, p.k_head = k_head, p.v_token = v_token, p.v_head = v_head;
        p.g_token = grad_token, p.g_head = grad_head;
        p.heads = int(heads), p.kv_heads = int(kv_heads), p.dim = int(dim), p.causal = causal;
        p.scale = scale, p.scale2 = scale * kLog2e;
        const hipStream_t s = static_cast<hipStream_t>(stream);
        switch (dtype) {
        case kBF16: dim <= 64 ? backward<bf16, 64>(p, workspace, s) : backward<bf16, 128>(p, workspace, s); break;
        case kF16: dim <= 64 ? backward<f16, 64>(p, workspace, s) : backward<f16, 128>(p, workspace, s); break;
        default: throw std::invalid_argument("attention takes bfloat16 or float16");
        }
    });
}

}  // extern "C"
