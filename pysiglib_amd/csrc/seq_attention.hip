// Attention over packed sequences: O = softmax(scale Q K^T) V with a query's visible keys, forward.
//
// Mathematics.  One pass over the keys with the running maximum m and sum l of each query: a tile's scores S change them to
// m' = max(m, max S), l' = 2^(m - m') l + sum 2^(S - m'), O' = 2^(m - m') O + 2^(S - m') V, and at the end O / l.  Queries see the
// keys up to their own place, counted from the sequences' ends; a query that sees none gets 0 and a log-sum of -infinity.
// Everything but the operands of the products is 32-bit; the weights 2^(S - m) are rounded to the inputs' type for the second
// product, which is the only rounding before the last.
//
// The products are formed transposed, S^T = K Q^T and O^T = V^T P^T: a lane then holds scores of a single query, its maximum
// and sum need one exchange between lanes, and the weights are the second product's operand where they stand.
//
// Bound: 128 channels, the matrix units: one sequence of 8192, 32 heads on 8, bfloat16, 525 to 605 us by the card (0.91 to 1.05 PFLOP/s;
// a large library product reaches 1.19), and the order of reads around the products no longer changes that.  64 channels, the
// softmax: 15 vector instructions to a matrix one, 24 sequences of up to 2000, 16 heads on 4, float16, 141 us (0.53 PFLOP/s).  Heads of
// other widths take the time of the next of these two (4 sequences of 2000, 16 heads on 4, bfloat16: 32 channels 61 us, 64 58, 80 89, 96 91,
// 128 95).
// Single queries, HBM: 48 against caches of up to 12000 keys of 8 heads of 128, 242 us (5.1 TB/s).
#include "seq_attention.h"

namespace seqamd {
namespace {

struct AttentionArgs {
    const void *q, *k, *v;
    void* out;               // [q_rows][heads][dim]
    float* lse;              // [q_rows][heads]
    Packed packed;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;
    float* parts;            // of the splits
    int heads, kv_heads, dim, causal, splits;
    float scale;             // times log2(e)
    unsigned first_block;    // of a launch
};

// The maximum is taken over where it grew by more than kSlack, in powers of two.  Weights in float16 stand 2^kRaise above what they are: up
// to 2^15, so that those of keys with little weight beside another's keep their bits down to 2^-25 of the largest, not to 2^-14.
template <typename T>
constexpr float kSlack = __is_same(T, f16) ? 4.0f : 8.0f;
template <typename T>
constexpr float kRaise = __is_same(T, f16) ? 11.0f : 0.0f;

// WAVES waves of 32 queries each, tiles of kKeys keys: what a block reads serves all its waves, the next tile on its way meanwhile.
template <typename T, int DP, int WAVES, int kKeys>
__global__ void __launch_bounds__(WAVES * 64, DP == 64 ? 4 : 2) attention_kernel(AttentionArgs p)
{
    constexpr int kThreads = WAVES * 64, kRows = 32 * WAVES, kSlices = DP / 16, kBlocks = DP / 32;
    constexpr int kTileBytes = kKeys * Tile<DP>::kRowBytes, kLoads = kKeys * Tile<DP>::kChunks / kThreads;
    static_assert(kLoads * kThreads == kKeys * Tile<DP>::kChunks, "");
    __shared__ __attribute__((aligned(16))) char s_tiles[2][2][kTileBytes];
    constexpr int kHiding = kRows / kKeys + 2;       // tiles that hide keys from some queries of the block, at most
    __shared__ unsigned s_bad[kHiding][kKeys / 32], s_any;       // their keys whose values are not finite, and whether there are any
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (tid < kHiding)
        for (unsigned& bad : s_bad[tid]) bad = 0;
    if (tid == 0) s_any = 0;
    // the heads that share keys and values follow each other at a distance of kv_heads: on the same die where that is a multiple of 8
    const unsigned block = p.first_block + blockIdx.x;
    const int turn = block % p.heads, head = (turn % p.kv_heads) * (p.heads / p.kv_heads) + turn / p.kv_heads, kv = turn % p.kv_heads;
    // the last tiles see the most keys: they begin first
    const Span at = find_tile(p.packed, Tiling{false, kRows, 1}, block / p.heads, Dear::kLast);
    if (at.seq < 0) return;
    const int q_first = at.tile * kRows, shift = at.nk - at.nq;
    // keys that any query of the block sees
    const int q_past = q_first + kRows < at.nq ? q_first + kRows : at.nq;
    int keys = at.nk;
    if (p.causal && q_past + shift < keys) keys = q_past + shift < 0 ? 0 : q_past + shift;
    const int tiles = (keys + kKeys - 1) / kKeys;

    const RowRead<DP> rows(lane);
    const ColumnRead<DP> columns(lane);
    const int query = q_first + wave * 32 + (lane & 31);
    Frag<T> q[kSlices];
    f32x16 o[kBlocks];
    float top = -INFINITY, sum = 0.0f;
    {
        const T* from = static_cast<const T*>(p.q) + (at.q0 + min(query, at.nq - 1)) * p.q_token + head * p.q_head;
#pragma unroll
        for (int k = 0; k < kSlices; ++k) q[k] = load_row<T>(from, 16 * k + 8 * half, p.dim);
    }
#pragma unroll
    for (int d = 0; d < kBlocks; ++d) o[d] = zeros16();

    // A tile's rows at fixed offsets from its first: only the last tile, whose rows may end early, forms them anew
    u32x4 next[2][kLoads];
    unsigned k_at[kLoads], v_at[kLoads];
    auto offsets = [&](unsigned* to, int64_t token, int left) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int e = i * kThreads + tid, row = min(e / Tile<DP>::kChunks, left - 1), ch = min(e % Tile<DP>::kChunks * 8, p.dim - 8);
            to[i] = unsigned((row * int(token) + ch) * int(sizeof(T)));        // rows past the end have no weight, channels meet zeros or are not stored
        }
    };
    const char* const k_base = reinterpret_cast<const char*>(static_cast<const T*>(p.k) + at.k0 * p.k_token + kv * p.k_head);
    const char* const v_base = reinterpret_cast<const char*>(static_cast<const T*>(p.v) + at.k0 * p.v_token + kv * p.v_head);
    offsets(k_at, p.k_token, min(at.nk, kKeys));
    offsets(v_at, p.v_token, min(at.nk, kKeys));
    auto fetch = [&](int tile) __attribute__((always_inline)) {
        if ((tile + 1) * kKeys > at.nk) {
            offsets(k_at, p.k_token, at.nk - tile * kKeys);
            offsets(v_at, p.v_token, at.nk - tile * kKeys);
        }
        const char *kp = k_base + tile * int64_t(kKeys * sizeof(T)) * p.k_token, *vp = v_base + tile * int64_t(kKeys * sizeof(T)) * p.v_token;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            next[0][i] = load_at(kp, k_at[i]);
            next[1][i] = load_at(vp, v_at[i]);
        }
    };
    // A key is hidden past the sequence's end, or behind a query's place.  Tiles from `hiding` on hide some from some of the block's
    // queries, from `hiding_wave` on from some of the wave's; from `unseen` on the wave's queries see none of them.
    const int hiding = min(at.nk, p.causal ? max(q_first + shift + 1, 0) : at.nk) / kKeys;
    const int hiding_wave = min(at.nk, p.causal ? max(q_first + wave * 32 + shift + 1, 0) : at.nk) / kKeys;
    const int unseen = p.causal ? min(max(q_first + wave * 32 + 31 + shift + kKeys, 0) / kKeys, tiles) : tiles;
    // keys' channels past the head's are zero: zeros of the query make no zero with what is not finite
    static_assert(kThreads % Tile<DP>::kChunks == 0, "");
    const bool there = tid % Tile<DP>::kChunks * 8 < p.dim;
    auto put = [&](int tile) __attribute__((always_inline)) {
        auto place = [&](int i) { return Tile<DP>::at((i * kThreads + tid) / Tile<DP>::kChunks, (i * kThreads + tid) % Tile<DP>::kChunks); };
#pragma unroll
        for (int i = 0; i < kLoads; ++i) *reinterpret_cast<u32x4*>(s_tiles[tile & 1][0] + place(i)) = there ? next[0][i] : u32x4{0, 0, 0, 0};
        if (tile >= hiding) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int row = (i * kThreads + tid) / Tile<DP>::kChunks;
                u32x4 x = next[1][i];
                if (take_them_out<T>(x)) {
                    atomicOr(&s_bad[tile - hiding][row / 32], 1u << row % 32);
                    s_any = 1;
                }
                *reinterpret_cast<u32x4*>(s_tiles[tile & 1][1] + place(i)) = x;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) *reinterpret_cast<u32x4*>(s_tiles[tile & 1][1] + place(i)) = next[1][i];
        }
    };
    const int last = p.causal && query + shift < at.nk - 1 ? query + shift : at.nk - 1;
    f32x16 s[kKeys / 32];
    Frag<T> w[kKeys / 16];
    auto scores = [&](int tile) __attribute__((always_inline)) {
        const char* kt = s_tiles[tile & 1][0];
#pragma unroll
        for (int c = 0; c < kKeys / 32; ++c) s[c] = zeros16();
#pragma unroll
        for (int k = 0; k < kSlices; ++k)
#pragma unroll
            for (int c = 0; c < kKeys / 32; ++c) s[c] = product(rows.template get<T>(kt, 32 * c, k), q[k], s[c]);
    };
    auto weights = [&](int tile) __attribute__((always_inline)) {
        const int key0 = tile * kKeys;
        if (tile >= hiding_wave) {
#pragma unroll
            for (int c = 0; c < kKeys / 32; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (key0 + 32 * c + row_in(i, half) > last) s[c][i] = -INFINITY;
        }
        float part[4];           // chains of their own: each waits for itself alone
#pragma unroll
        for (int j = 0; j < 4; ++j) part[j] = larger(s[0][j], s[0][j + 4], s[0][j + 8]);
#pragma unroll
        for (int j = 0; j < 4; ++j) part[j] = kKeys == 64 ? larger(part[j], s[0][j + 12], s[kKeys / 32 - 1][j]) : larger(part[j], s[0][j + 12]);
        if constexpr (kKeys == 64)
#pragma unroll
            for (int j = 0; j < 4; ++j) part[j] = larger(larger(part[j], s[1][j + 4], s[1][j + 8]), s[1][j + 12]);
        float most = larger(larger(part[0], part[1], part[2]), part[3]);
        most = larger(most, swapped(most)) * p.scale;
        const bool grows = most > top + kSlack<T> || (top == -INFINITY && most > top);
        if (__any(grows)) {             // each query by itself: its roundings are no matter of the others'
            const float now = grows ? most : top, shrink = top == now ? 1.0f : exp2f(top - now);
            top = now;
            sum *= shrink;
#pragma unroll
            for (int d = 0; d < kBlocks; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= shrink;
        }
        const float base = top == -INFINITY ? 0.0f : top - kRaise<T>;
#pragma unroll
        for (int j = 0; j < 4; ++j) part[j] = 0.0f;
#pragma unroll
        for (int c = 0; c < kKeys / 32; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[c][i] = __builtin_amdgcn_exp2f(fmaf(s[c][i], p.scale, -base));
                part[i & 3] += s[c][i];
            }
        sum += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
        for (int c = 0; c < kKeys / 16; ++c) w[c] = rounded<T>(s[c / 2], 8 * (c & 1));
    };
    auto values = [&](int tile) __attribute__((always_inline)) {
        const char* vt = s_tiles[tile & 1][1];
#pragma unroll
        for (int c = 0; c < kKeys / 16; ++c)
#pragma unroll
            for (int d = 0; d < kBlocks; ++d) o[d] = product(columns.template get<T>(vt, 16 * c, d), w[c], o[d]);
    };
    if (tiles) {
        fetch(0);
        if (hiding == 0) __syncthreads();       // s_bad is clear
        put(0);
    }
#pragma unroll
    for (int k = 0; k < kSlices; ++k) arrive<T>(q[k]);
    for (int tile = 0; tile < tiles; ++tile) {
        __syncthreads();
        if (tile + 1 < tiles) fetch(tile + 1);
        if (tile < unseen) {
            scores(tile);
            weights(tile);
            values(tile);
        }
        if (tile + 1 < tiles) put(tile + 1);
    }
    top -= kRaise<T>;
    const float total = sum + swapped(sum);
    if (query >= at.nq) return;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int64_t row = (at.q0 + query) * p.heads + head;
    if (half == 0) p.lse[row] = total == 0.0f ? -INFINITY : 0.69314718055994531f * (top + log2f(total));
    T* const to = static_cast<T*>(p.out) + row * p.dim;
    store_row<T, DP>(to, o, inv, p.dim, half);
    if (__builtin_expect(s_any != 0, 0))
        for (int tile = hiding; tile < tiles; ++tile)
            for (int part = 0; part < kKeys / 32; ++part)
                for (unsigned bad = s_bad[tile - hiding][part]; bad; bad &= bad - 1) {
                    const int key = tile * kKeys + 32 * part + __ffs(bad) - 1;
                    if (key <= last) add_them<T, T>(static_cast<const T*>(p.v) + (at.k0 + key) * p.v_token + kv * p.v_head, to, p.dim, half);
                }
}

// ---- few queries to many keys: rows of a tile are the pairs (query, head) that share a key head ----
// The four waves of a block take tiles of 32 keys in turn, each with its own maxima and sums, joined at the end; a sequence's
// keys are cut into p.splits ranges that blocks take beside each other, joined by join_kernel.
template <typename T, int DP>
__global__ void __launch_bounds__(256, 2) few_kernel(AttentionArgs p)
{
    constexpr int kSlices = DP / 16, kBlocks = DP / 32, kWaves = 4, kTile = 32;
    constexpr int kTileBytes = kTile * Tile<DP>::kRowBytes, kLoads = kTile * Tile<DP>::kChunks / 64;
    __shared__ __attribute__((aligned(16))) char s_tiles[kWaves][2][kTileBytes];
    __shared__ float s_top[kWaves][32], s_sum[kWaves][32];
    __shared__ unsigned s_bad[4], s_any;     // of the tiles that hide keys from some of the pairs: keys whose values are not finite
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned block = p.first_block + blockIdx.x;
    const int group = p.heads / p.kv_heads, kv = block % p.kv_heads, split = block / p.kv_heads % p.splits;
    const Span at = find_tile(p.packed, Tiling{false, 32, group}, block / p.kv_heads / p.splits, Dear::kLast);
    if (at.seq < 0) return;
    const int pairs = at.nq * group, shift = at.nk - at.nq, pair = at.tile * 32 + (lane & 31);
    const int own = pair < pairs ? pair : pairs - 1, query = own / group, head = kv * group + own % group;
    // keys that any query of the tile sees, of those this split's
    const int last_query = (at.tile * 32 + 31 < pairs ? at.tile * 32 + 31 : pairs - 1) / group;
    int keys = p.causal && last_query + 1 + shift < at.nk ? last_query + 1 + shift : at.nk;
    keys = keys < 0 ? 0 : keys;
    const int each = ((keys + p.splits - 1) / p.splits + kTile - 1) / kTile * kTile;
    const int begin = int64_t(split) * each < keys ? split * each : keys, past = begin + each < keys ? begin + each : keys;
    const int tiles = (past - begin + kTile - 1) / kTile;

    Frag<T> q[kSlices];
    {
        const T* from = static_cast<const T*>(p.q) + (at.q0 + query) * p.q_token + head * p.q_head;
#pragma unroll
        for (int k = 0; k < kSlices; ++k) q[k] = load_row<T>(from, 16 * k + 8 * half, p.dim);
    }
    const RowRead<DP> rows(lane);
    const ColumnRead<DP> columns(lane);
    f32x16 o[kBlocks];
#pragma unroll
    for (int d = 0; d < kBlocks; ++d) o[d] = zeros16();
    float top = -INFINITY, sum = 0.0f;
    const int last = p.causal && query + shift < past - 1 ? query + shift : past - 1;

    char *kt = s_tiles[wave][0], *vt = s_tiles[wave][1];
    const bool there = lane % Tile<DP>::kChunks * 8 < p.dim;          // keys' channels past the head's are zero, as above
    u32x4 next[2][kLoads];
    auto fetch = [&](int tile) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int e = i * 64 + lane, row = e / Tile<DP>::kChunks, chunk = e % Tile<DP>::kChunks;
            const int at_key = begin + tile * kTile + row, key = at_key < past ? at_key : past - 1;
            const int ch = chunk * 8 < p.dim ? chunk * 8 : p.dim - 8;
            __builtin_memcpy(&next[0][i], static_cast<const T*>(p.k) + (at.k0 + key) * p.k_token + kv * p.k_head + ch, 16);
            __builtin_memcpy(&next[1][i], static_cast<const T*>(p.v) + (at.k0 + key) * p.v_token + kv * p.v_head + ch, 16);
        }
    };
    const int first_query = at.tile * 32 / group;
    auto hides = [&](int tile) { return (tile + 1) * kTile > past - begin || (p.causal && begin + (tile + 1) * kTile - 1 > first_query + shift); };
    const int hiding = min(p.causal ? max(first_query + shift + 1 - begin, 0) / kTile : tiles, tiles - 1);      // the first of them, or one before it
    if (wave < tiles) fetch(wave);
    if (tid < 4) s_bad[tid] = 0;
    if (tid == 4) s_any = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSlices; ++k) arrive<T>(q[k]);
    for (int tile = wave; tile < tiles; tile += kWaves) {
        const bool hidden = hides(tile);
        if (hidden)
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                if (take_them_out<T>(next[1][i])) {
                    atomicOr(&s_bad[tile - hiding], 1u << (i * 64 + lane) / Tile<DP>::kChunks);
                    s_any = 1;
                }
        // the wave's own tiles: shared memory serves a wave in order, no barrier is needed
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int e = i * 64 + lane, to = Tile<DP>::at(e / Tile<DP>::kChunks, e % Tile<DP>::kChunks);
            *reinterpret_cast<u32x4*>(kt + to) = there ? next[0][i] : u32x4{0, 0, 0, 0};
            *reinterpret_cast<u32x4*>(vt + to) = next[1][i];
        }
        __builtin_amdgcn_wave_barrier();
        if (tile + kWaves < tiles) fetch(tile + kWaves);
        const int key0 = begin + tile * kTile;
        f32x16 s = zeros16();
#pragma unroll
        for (int k = 0; k < kSlices; ++k) s = product(rows.template get<T>(kt, 0, k), q[k], s);
        if (hidden)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (key0 + row_in(i, half) > last) s[i] = -INFINITY;
        float most = larger(s[0], s[1], s[2]);
#pragma unroll
        for (int i = 3; i < 15; i += 2) most = larger(most, s[i], s[i + 1]);
        most = larger(most, s[15]);
        most = larger(most, swapped(most)) * p.scale;
        const bool grows = most > top + kSlack<T> || (top == -INFINITY && most > top);
        if (__any(grows)) {             // each query by itself: its roundings are no matter of the others'
            const float now = grows ? most : top, shrink = top == now ? 1.0f : exp2f(top - now);
            top = now;
            sum *= shrink;
#pragma unroll
            for (int d = 0; d < kBlocks; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= shrink;
        }
        const float base = top == -INFINITY ? 0.0f : top - kRaise<T>;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], p.scale, -base));
            sum += s[i];
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const Frag<T> w = rounded<T>(s, 8 * u);
#pragma unroll
            for (int d = 0; d < kBlocks; ++d) o[d] = product(columns.template get<T>(vt, 16 * u, d), w, o[d]);
        }
        __builtin_amdgcn_wave_barrier();
    }
    // the waves' parts together: maxima and sums of all, then the weighted values, two waves into two, one into one
    sum += swapped(sum);
    top -= kRaise<T>;
    if (half == 0) {
        s_top[wave][lane] = top;
        s_sum[wave][lane] = sum;
    }
    __syncthreads();
    float most = -INFINITY, total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) most = fmaxf(most, s_top[w][lane & 31]);
    const float base = most == -INFINITY ? 0.0f : most;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += s_sum[w][lane & 31] * exp2f(s_top[w][lane & 31] - base);
    const float mine = exp2f(top - base);
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= mine;
    float* const shared = reinterpret_cast<float*>(&s_tiles[0][0][0]);       // two parts of 64 lanes' sums, 64 KB at most
    constexpr int kPart = kBlocks * 16 * 64;
    static_assert(2 * kPart * sizeof(float) <= sizeof s_tiles, "");
#pragma unroll
    for (int step = 2; step > 0; step /= 2) {
        __syncthreads();
        if (wave >= step && wave < 2 * step)
#pragma unroll
            for (int d = 0; d < kBlocks; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) shared[(wave - step) * kPart + (d * 16 + i) * 64 + lane] = o[d][i];
        __syncthreads();
        if (wave < step)
#pragma unroll
            for (int d = 0; d < kBlocks; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] += shared[wave * kPart + (d * 16 + i) * 64 + lane];
    }
    if (wave || pair >= pairs) return;
    auto correct = [&](auto* to) {
        if (__builtin_expect(s_any != 0, 0))
            for (int tile = hiding; tile < tiles; ++tile)
                for (unsigned bad = s_bad[max(tile - hiding, 0)]; bad; bad &= bad - 1) {
                    const int key = begin + tile * kTile + __ffs(bad) - 1;
                    if (key <= last) add_them(static_cast<const T*>(p.v) + (at.k0 + key) * p.v_token + kv * p.v_head, to, p.dim, half);
                }
    };
    const int64_t row = (at.q0 + query) * p.heads + head;
    if (p.splits > 1) {
        // [splits][q_rows * heads] of (maximum, sum), then [splits][q_rows * heads][dim]
        const int64_t all = p.packed.q_rows * p.heads, place = split * all + row;
        float* const to = p.parts + 2 * p.splits * all + place * p.dim;
        if (half == 0) {
            p.parts[2 * place] = most;
            p.parts[2 * place + 1] = total;
        }
#pragma unroll
        for (int d = 0; d < kBlocks; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int ch = 32 * d + row_in(i, half);
                if (ch < p.dim) {
                    typedef float f32x4 __attribute__((ext_vector_type(4)));
                    *reinterpret_cast<f32x4*>(to + ch) = f32x4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
                }
            }
        correct(to);
        return;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    if (half == 0) p.lse[row] = total == 0.0f ? -INFINITY : 0.69314718055994531f * (most + log2f(total));
    T* const to = static_cast<T*>(p.out) + row * p.dim;
    store_row<T, DP>(to, o, inv, p.dim, half);
    correct(to);
}

// the splits of one (query, head) to a wave, a lane to one or two channels pairwise
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(AttentionArgs p)
{
    const int64_t all = p.packed.q_rows * p.heads, row = (int64_t(p.first_block) + blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    // rows before the first sequence and behind the last have no parts
    const int64_t first_row = kept(p.packed.q_offsets[0], 0, p.packed.q_rows), past_row = kept(p.packed.q_offsets[p.packed.n], first_row, p.packed.q_rows);
    if (row < first_row * p.heads || row >= past_row * p.heads) return;
    float most = -INFINITY;
    for (int s = lane; s < p.splits; s += 64) most = fmaxf(most, p.parts[2 * (s * all + row)]);
#pragma unroll
    for (int m = 1; m < 64; m *= 2) most = fmaxf(most, __shfl_xor(most, m));
    const float base = most == -INFINITY ? 0.0f : most;
    const int ch = min(2 * lane, p.dim - 2);
    const float* from = p.parts + 2 * p.splits * all + row * p.dim + ch;
    float total = 0.0f, x[2] = {0.0f, 0.0f};
    for (int first = 0; first < p.splits; first += 64) {
        // a split's maximum and sum to a lane; then the splits' values, whose loads wait for nothing
        float w = 0.0f;
        if (first + lane < p.splits) {
            const int64_t place = (first + lane) * all + row;
            w = exp2f(p.parts[2 * place] - base);
            total += w * p.parts[2 * place + 1];
        }
        const int count = min(64, p.splits - first);
        for (int s = 0; s < count; s += 8)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float ws = __shfl(w, s + j);
                const Pack<float, 2> v = load_pack<float, 2>(from + min(first + s + j, p.splits - 1) * all * p.dim);
                const bool there = s + j < count;               // the last split's values in the place of those past it may be infinite
                x[0] = there ? fmaf(ws, v.get(0), x[0]) : x[0];
                x[1] = there ? fmaf(ws, v.get(1), x[1]) : x[1];
            }
    }
#pragma unroll
    for (int m = 1; m < 64; m *= 2) total += __shfl_xor(total, m);
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    if (lane == 0) p.lse[row] = total == 0.0f ? -INFINITY : 0.69314718055994531f * (most + log2f(total));
    if (2 * lane < p.dim) {
        x[0] *= inv;
        x[1] *= inv;
        Pack<T, 2> pack;
        pack.set(x);
        store_pack<T, 2>(static_cast<T*>(p.out) + row * p.dim + 2 * lane, pack);
    }
}

// How a call is cut, by averages: the lengths are not known here.  (A prompt of 4096 beside 63 single tokens against 2000 keys, 32 heads
// on 8 of 128, bfloat16: 384 us; the prompt in a call of its own 152, the tokens 121.)  few: pairs of (query, head) in tiles of 32 instead of a head's queries in tiles of 32 to a wave.
struct Cut {
    bool few;
    int waves, splits;
    int64_t tiles;           // over all sequences, at most
    size_t map, parts;       // bytes of workspace
};

Cut cut_of(int64_t q_rows, int64_t k_rows, int64_t n, int64_t heads, int64_t kv_heads, int64_t dim)
{
    Cut c;
    const int64_t group = heads / kv_heads;
    const int64_t queries = q_rows / n, keys = k_rows / n;         // of a sequence, on average
    // One tile for the pairs of all heads that share keys: against keys enough to cut in ranges, or for a handful of queries
    // (4000 sequences of 4, 16 heads on 4: 109 us, by heads 268; 1000 of 16: 66 us, by heads 41)
    c.few = (queries * group < 64 && keys >= 256) || (queries * group < 32 && group > 1);
    // Small blocks for short sequences (16 heads on 4 of 64 channels, 16000 tokens in sequences of 64: 2 waves 34 us, 8 waves
    // 69; of 400: 55 and 64; of 1000: 88 and 82.  32 heads on 8 of 128, 8000 tokens in sequences of 100: 2 waves 64 us, 4 waves
    // 73; of 1000: 138, 128, 8 waves 152; one of 8192: 8 waves 597, 4 waves 621)
    c.waves = dim <= 64 ? (queries <= 512 ? 2 : 8) : (queries <= 200 ? 2 : (queries <= 2048 ? 4 : 8));
    c.splits = 1;
    if (c.few) {
        c.tiles = most_tiles(q_rows * group, q_rows < n ? q_rows : n, 32);
        // ranges of 256 keys and more, until there are about 16 blocks for each of the 256 compute units
        const int64_t by_blocks = 4096 / (c.tiles * kv_heads ? c.tiles * kv_heads : 1), by_keys = k_rows / n / 256;
        const int64_t splits = by_blocks < by_keys ? by_blocks : by_keys;
        c.splits = int(splits < 1 ? 1 : (splits > 256 ? 256 : splits));
    } else {
        c.tiles = most_tiles(q_rows, n, 32 * c.waves);
    }
    c.map = map_bytes(c.tiles, n);
    c.parts = c.splits > 1 ? size_t(c.splits) * q_rows * heads * (dim + 2) * sizeof(float) : 0;
    return c;
}

template <typename T, int DP>
void forward(const AttentionArgs& p, const Cut& cut, hipStream_t stream)
{
    if (cut.few) {
        const int64_t blocks = cut.tiles * p.kv_heads * p.splits, rows = p.packed.q_rows * p.heads;
        launch_all(few_kernel<T, DP>, blocks, 256, stream, p);
        if (p.splits > 1) launch_all(join_kernel<T>, (rows + 3) / 4, 256, stream, p);
        return;
    }
    const int64_t blocks = cut.tiles * p.heads;
    switch (cut.waves) {
    case 2: return launch_all(attention_kernel<T, DP, 2, 32>, blocks, 128, stream, p);
    case 4: return launch_all(attention_kernel<T, 128, 4, 64>, blocks, 256, stream, p);
    default: return launch_all(attention_kernel<T, DP, 8, 64>, blocks, 512, stream, p);
    }
}

}  // namespace
}  // namespace seqamd

using namespace seqamd;

extern "C" {

__attribute__((visibility("default"))) uint64_t cusig_amd_attention_workspace(uint64_t q_rows, uint64_t k_rows, uint64_t sequences, uint64_t heads,
                                                                            uint64_t kv_heads, uint64_t dim) noexcept
{
    if (!sequences || !kv_heads || !heads || heads % kv_heads) return 0;
    const Cut c = cut_of(int64_t(q_rows), int64_t(k_rows), int64_t(sequences), int64_t(heads), int64_t(kv_heads), int64_t(dim));
    return c.map + c.parts;
}

__attribute__((visibility("default"))) int cusig_amd_attention(
    int dtype, const void* q, const void* k, const void* v, const int* q_offsets, const int* k_offsets, const int* k_lengths, void* out, float* lse,
    uint64_t q_rows, uint64_t k_rows, uint64_t sequences, uint64_t heads, uint64_t kv_heads, uint64_t dim, int64_t q_token, int64_t q_head, int64_t k_token,
    int64_t k_head, int64_t v_token, int64_t v_head, float scale, bool causal, void* workspace, uint64_t workspace_bytes, void* stream) noexcept
{
    return sigamd::guarded([&] {
        require(q_rows < (uint64_t(1) << 31) && k_rows < (uint64_t(1) << 31) && sequences < (uint64_t(1) << 31), "too many rows or sequences");
        require(dim >= 8 && dim <= 128 && dim % 8 == 0, "a head has 8 to 128 channels, a multiple of 8");
        require(kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads < (1u << 20), "heads are a multiple of the key heads");
        require(scale > 0.0f && std::isfinite(scale), "the scale is positive and finite");
        check_strides({q_token, k_token, v_token});
        if (q_rows == 0 || sequences == 0) return;
        require(q && q_offsets && k_offsets && out && lse && (k_rows == 0 || (k && v)), "a tensor is missing");
        AttentionArgs p{};
        p.q = q, p.k = k, p.v = v, p.out = out, p.lse = lse;
        p.packed = Packed{q_offsets, k_offsets, k_lengths, int64_t(q_rows), int64_t(k_rows), int(sequences), nullptr};
        p.q_token = q_token, p.q_head = q_head, p.k_token = k_token, p.k_head = k_head, p.v_token = v_token, p.v_head = v_head;
        p.heads = int(heads), p.kv_heads = int(kv_heads), p.dim = int(dim), p.causal = causal;
        p.scale = scale * 1.44269504088896341f;
        const Cut cut = cut_of(p.packed.q_rows, p.packed.k_rows, p.packed.n, p.heads, p.kv_heads, p.dim);
        check_workspace(workspace, workspace_bytes, cut.map + cut.parts);
        p.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + cut.map);
        p.splits = cut.splits;
        require(cut.tiles * (cut.few ? p.kv_heads * int64_t(p.splits) : p.heads) < (int64_t(1) << 31), "too many queries and heads");
        const hipStream_t s = static_cast<hipStream_t>(stream);
        if (cut.map) {
            p.packed.map = static_cast<const int*>(workspace);
            MapArgs m{};
            m.packed = p.packed;
            m.how[0] = cut.few ? Tiling{false, 32, p.heads / p.kv_heads} : Tiling{false, 32 * cut.waves, 1};
            m.map[0] = static_cast<int*>(workspace);
            m.room[0] = int(cut.tiles);
            hipLaunchKernelGGL(map_kernel, dim3(1), dim3(kMapThreads), 0, s, m);
            SIG_HIP(hipGetLastError());
        }
        switch (dtype) {
        case kBF16: dim <= 64 ? forward<bf16, 64>(p, cut, s) : forward<bf16, 128>(p, cut, s); break;
        case kF16: dim <= 64 ? forward<f16, 64>(p, cut, s) : forward<f16, 128>(p, cut, s); break;
        default: throw std::invalid_argument("attention takes bfloat16 or float16");
        }
    });
}

}  // extern "C"
