// Shared by the selective scan's two directions (seq_selective.hip, seq_selective_backward.hip): how the channels and states lie on a wave,
// how sequences are cut into segments, what a tile of rows holds.
//
// h_t = exp(dt_t a) h_{t-1} + dt_t x_t b_t for each channel and state, y_t = sum over the states of c_t h_t, plus d x_t, times
// z_t sigmoid(z_t); dt = softplus(delta + bias), or delta + bias.  Every channel has its own a, x, delta; b and c are those of its group.
//
// Layout.  Four lanes (a quad) hold four channels: their registers the channels, the lanes neighbouring states, so that a step's
// dt x_i b_n of 16 pairs is one matrix instruction (16 blocks of 4 x 4, one product each) that adds them to the decayed states.  A lane holds
// four such quadruples: four groups of four states of four channels (16 states), two groups of eight channels (8), one of 16 (4);
// 32 and 64 states are those of 2 and 4 quads.  Q = states / 4 counts lanes to a channel, 16 pairs being a lane's: a wave has 256 / Q channels,
// b and c are read once for four channels, dt once for four states, and the sums over states (y) and over channels (the
// gradients of b and c) each cross few lanes.
// Room for more states than there are holds the first ones again.  Copies of a state go through the same steps, and each has an equal part of its c
// and of its final gradient: 1, 1/2 or 1/4 of it, which rounds no normal number.  Sums over the room are then sums over the states, and nothing infinite
// meets a zero that the formula does not have.  Gradients that are not sums over states are those of one copy times the number of copies.
#pragma once
#include "seq_common.h"

#include <initializer_list>
#include <type_traits>

namespace seqamd {
namespace selective {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

typedef float Four __attribute__((ext_vector_type(4)));

template <int Q>
struct Shape {
    static constexpr int kRows = Q == 1 ? 4 : (Q == 2 ? 8 : 16);        // of a tile
    static constexpr int kChannels = 256 / Q;                           // of a wave
    static constexpr int kEach = kRows * kChannels / 128;               // pairs of neighbouring channels of a tile's rows to a lane
    static constexpr int kOwn = kChannels > 128 ? 2 : 1;                // different channels among them: so many pairs
    static constexpr int kStates = 4 * Q;
    static constexpr int kPacks = kRows * 2 * Q;                        // of four values of b or c in a tile
    static constexpr int kPacksEach = (kPacks + 63) / 64;
    static constexpr int kGroups = Q < 4 ? Q : 4;                       // of four states of a lane
    static constexpr int kSets = 4 / kGroups;                           // of four channels of a lane
    static constexpr int kQuads = Q < 4 ? 1 : Q / 4;                    // with the same channels
    static constexpr int kSaved = kRows < 8 ? kRows : 8;                // backward: rows between two states that are stored

    // pair i of a lane: its row in the tile, and its first channel in the wave
    static constexpr int kRowsAtOnce = kChannels < 128 ? 128 / kChannels : 1;
    static constexpr int row(int i) { return i * 128 / kChannels; }      // of the wave's first lanes
    static __device__ __forceinline__ int row(int i, int lane) { return row(i) + (kRowsAtOnce > 1 ? lane / (kChannels / 2) : 0); }

    // where state n lies among the wave's in shared memory: a lane's groups beside each other
    static __host__ __device__ constexpr int place(int n) { return n / 16 * 16 + n % 4 * kGroups + n % 16 / 4; }
};

// which state place n holds, where there are places for up to twice as many as there are (for four times one)
__device__ __forceinline__ int state_at(int n, int states) { return n < states ? n : min(n - states, states - 1); }

// how many of `room` places hold state n: a power of two
__device__ __forceinline__ float copies_of(int n, int states, int room) { return n + states >= room ? 1.0f : (n + 2 * states >= room ? 2.0f : 4.0f); }

struct Args {
    const void *x, *delta, *b, *c, *z, *grad;   // z may be null; grad: of y, backward
    const float *a, *d, *bias;                  // a [channels][states]; d and bias may be null
    const float* begin;                         // initial states [n][channels][states] or null
    const float* grad_end;                      // gradients of the final states or null, backward
    float* end;                                 // final states; backward: gradients of the initial ones
    void *out, *ddelta, *dz;                    // y; backward: the gradients of x, delta and z
    const int* offsets;                         // [n + 1] rows where sequences begin, or null: n sequences of `length` rows
    // states as the lanes hold them: [columns][4][64 lanes][4], columns: a wave's channels
    Four* carry;                                // [slots] the segments' own last states, then the states before them
    Four* back;                                 // the same for the gradients of states, the other way
    float* span;                                // [slots][channels] sum of dt over a segment
    Four* tile_state;                           // backward: [tiles] states before a tile's rows, of a segment's own
    float* tile_span;                           // [tiles][channels] sum of dt from the segment's first row on
    float* shared_parts;                        // backward: [blocks of a group][rows][groups][2][4 Q] sums of the gradients of b and c
    float* own_parts;                           // [pieces][channels][states + 2] those of a, d and bias
    int64_t rows, length, n, segment, slots, per_sequence;
    int64_t x_step, delta_step, z_step, grad_step, b_step, b_group, c_step, c_group;
    int channels, states, groups, per_group, tiles;     // tiles: of a group's channels
    int group_blocks, pieces;                           // backward: blocks to a group, pieces of the slots
    bool softplus;
    unsigned first_block;
};

// log(1 + e^v) = max(v, 0) + log(1 + w), w = e^-|v|: the logarithm of u = 1 + w as it was rounded, and what the rounding left out, over u, which is 1
// wherever that counts.  The hardware's logarithm is off by two roundings on all of [1, 2], the whole by |v| (the exponential's) and four.
__device__ __forceinline__ float softplus_of(float v)
{
    const float w = __builtin_amdgcn_exp2f(-fabsf(v) * kLog2e), u = 1.0f + w;
    return fmaxf(v, 0.0f) + fmaf(__builtin_amdgcn_logf(u), kLn2, w - (u - 1.0f));
}

__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-v * kLog2e)); }

// the lane whose number differs as CTRL says; all of them are there
template <int CTRL>
__device__ __forceinline__ float moved(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// the sum over the lanes of a channel, in all of them
template <int Q>
__device__ __forceinline__ float over_states(float v)
{
    v += moved<0xB1>(v);                            // neighbours
    v += moved<0x4E>(v);                            // pairs
    if constexpr (Q >= 8) v += moved<0x141>(v);     // mirrored halves of a row of 16: the other four
    if constexpr (Q >= 16) v += moved<0x140>(v);    // the other eight
    return v;
}

// state + x_i b_n for 16 pairs of a quad: x the channels' in its four lanes, b the states'
__device__ __forceinline__ Four add_products(float x, float b, Four state) { return __builtin_amdgcn_mfma_f32_4x4x1f32(x, b, state, 0, 0, 0); }

// Orders the shared memory of ONE wave.  The hardware serves its accesses in the order of their issue, so lanes see what others wrote before, and
// no wait is needed; only the compiler, to which a lane's accesses are its own, has to be kept from moving them across this point.
__device__ __forceinline__ void wave_sync()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}

// The rows of a segment: `first` up to `past` of the sequence `seq`, number `k` of its segments
struct Segment {
    int64_t seq, first, past, begin, end;       // begin, end: of the sequence
    bool there, first_one, last_one;
};

// The rows of sequence i, kept inside the tensors whatever the offsets hold
__device__ __forceinline__ void rows_of(const Args& p, int64_t i, int64_t& first, int64_t& past)
{
    if (p.offsets) {
        first = kept(p.offsets[i], 0, p.rows);
        past = kept(p.offsets[i + 1], first, p.rows);
    } else {
        first = i * p.length;
        past = first + p.length;
    }
}

// Slots.  Packed, sequence i has those from first / segment + i on: one more than whole segments lie between its first row and the next
// sequence's, which is room for all it has.
__device__ __forceinline__ int64_t slot_of(const Args& p, int64_t i, int64_t first) { return p.offsets ? first / p.segment + i : i * p.per_sequence; }

__device__ __forceinline__ Segment segment_of(const Args& p, int64_t slot)
{
    Segment s;
    int64_t k;
    if (p.offsets) {
        int64_t lo = 0, hi = p.n - 1;           // the last sequence that begins at or before the slot
        while (lo < hi) {
            const int64_t mid = (lo + hi + 1) / 2;
            if (slot_of(p, mid, kept(p.offsets[mid], 0, p.rows)) <= slot) lo = mid;
            else hi = mid - 1;
        }
        s.seq = lo;
        rows_of(p, lo, s.begin, s.end);
        k = slot - slot_of(p, lo, s.begin);
    } else {
        s.seq = slot / p.per_sequence;
        rows_of(p, s.seq, s.begin, s.end);
        k = slot - s.seq * p.per_sequence;
    }
    s.first = s.begin + k * p.segment;
    s.past = s.first + p.segment < s.end ? s.first + p.segment : s.end;
    s.first_one = k == 0;
    s.there = k >= 0 && (s.first < s.end || k == 0);
    s.last_one = s.past == s.end;
    return s;
}

// the tiles of a segment are numbered like slots: those of the rows before it, and one more for every slot
__device__ __forceinline__ int64_t tile_of(int64_t slot, const Segment& s, int rows) { return s.first / rows + slot; }

// What the wave's lanes have of the channels and states
template <typename T, int Q>
struct Column {
    using S = Shape<Q>;
    static constexpr int kG = S::kGroups, kSets = S::kSets;
    int lane, j, part, at;          // j: in the quad, part: which 16 states, at: the lane's first channel in the wave
    int first, count;               // the wave's channels: the first, and how many there are
    int group, column;
    int pair[S::kOwn];              // the first channels of the lane's pairs.  Where the last one would be behind the channels it is the last two
                                    // again: what two lanes form, they form alike
    Four a[4];                      // a log2(e), zero where there is no channel; of set u / kG, group u % kG
    float bias[S::kOwn][2], d[S::kOwn][2];

    __device__ __forceinline__ int channel(int u) const { return at + 4 * (u / kG); }
    __device__ __forceinline__ int state(int u) const { return part * 16 + 4 * (u % kG) + j; }
    // the lane's number, unknown to the compiler: what is formed from it is formed where it is used and takes no registers through a loop
    __device__ __forceinline__ int lane_again() const
    {
        int l = lane;
        asm volatile("" : "+v"(l));
        return l;
    }
    __device__ __forceinline__ int state_of(int l, int u, int states) const { return state_at(l / 4 % S::kQuads * 16 + 4 * (u % kG) + l % 4, states); }

    __device__ __forceinline__ void init(const Args& p, int group_, int tile)
    {
        lane = threadIdx.x & 63;
        j = lane % 4;
        part = lane / 4 % S::kQuads;
        at = lane / 4 / S::kQuads * 4 * kSets;
        group = group_;
        column = group * p.tiles + tile;
        first = group * p.per_group + tile * S::kChannels;
        count = min(p.per_group - tile * S::kChannels, S::kChannels);
        load_state(p, p.a, a);
#pragma unroll
        for (int u = 0; u < 4; ++u) a[u] *= kLog2e;
#pragma unroll
        for (int i = 0; i < S::kOwn; ++i) {
            const int ch = 2 * ((lane + 64 * i) % (S::kChannels / 2));
            pair[i] = max(min(ch, count - 2), 0);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const bool there = pair[i] + k < count;
                bias[i][k] = p.bias && there ? p.bias[first + pair[i] + k] : 0.0f;
                d[i][k] = p.d && there ? p.d[first + pair[i] + k] : 0.0f;
            }
        }
    }
    __device__ __forceinline__ int channel_of(int i) const { return pair[i % S::kOwn]; }
    // whether the lane is the one that counts this channel of its pair i
    __device__ __forceinline__ bool counts(int i, int k) const
    {
        const int ch = 2 * ((lane + 64 * (i % S::kOwn)) % (S::kChannels / 2));
        return channel_of(i) + k >= ch && channel_of(i) + k < count;
    }

    // the lane's values of [channels][states] from `from` on; zero where there are none
    __device__ __forceinline__ void load_state(const Args& p, const float* from, Four (&h)[4]) const
    {
        const int l = lane_again();
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                h[u][i] = from && channel(u) + i < count ? from[int64_t(first + channel(u) + i) * p.states + state_of(l, u, p.states)] : 0.0f;
    }
    // each copy's part of its state's, or (ALL) what all copies of a state have, of one's
    template <bool ALL>
    __device__ __forceinline__ void over_copies(const Args& p, Four (&h)[4]) const
    {
        if (p.states == S::kStates) return;
        const int l = lane_again();
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float n = copies_of(state_of(l, u, p.states), p.states, S::kStates);
            h[u] *= ALL ? n : 1.0f / n;
        }
    }
    __device__ __forceinline__ void store_state(const Args& p, float* to, const Four (&h)[4]) const
    {
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (channel(u) + i < count && state(u) < p.states) to[int64_t(first + channel(u) + i) * p.states + state(u)] = h[u][i];
    }
    // the same as the lanes hold it
    __device__ __forceinline__ int64_t place(const Args& p, int64_t row) const { return (row * p.groups * p.tiles + column) * 256 + lane; }
    __device__ __forceinline__ void load_own(const Args& p, const Four* from, int64_t row, Four (&h)[4]) const
    {
        const Four* const q = from + place(p, row);
#pragma unroll
        for (int u = 0; u < 4; ++u) h[u] = q[64 * u];
    }
    __device__ __forceinline__ void store_own(const Args& p, Four* to, int64_t row, const Four (&h)[4]) const
    {
        Four* const q = to + place(p, row);
#pragma unroll
        for (int u = 0; u < 4; ++u) q[64 * u] = h[u];
    }
    // one number for each of the lane's channels, [channels] from `from` on
    __device__ __forceinline__ void load_line(const float* from, Four (&v)[kSets]) const
    {
#pragma unroll
        for (int s = 0; s < kSets; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[s][i] = at + 4 * s + i < count ? from[first + at + 4 * s + i] : 0.0f;
    }
    __device__ __forceinline__ void store_line(float* to, const Four (&v)[kSets]) const
    {
        if (j == 0 && part == 0)
#pragma unroll
            for (int s = 0; s < kSets; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at + 4 * s + i < count) to[first + at + 4 * s + i] = v[s][i];
    }

    // the lane's pairs of `rows` rows from t0 on; rows behind them are the last one again.  The rows' address is the same for all lanes, each at a
    // distance of its own.
    __device__ __forceinline__ void load(const void* from, int64_t step, int64_t t0, int rows, Pack<T, 2> (&to)[S::kEach]) const
    {
        const T* const base = static_cast<const T*>(from) + t0 * step + first;
        if (rows == S::kRows && count >= 2) {
            const unsigned more = S::kRowsAtOnce > 1 ? unsigned(lane / (S::kChannels / 2) * int(step)) : 0u;
#pragma unroll
            for (int i = 0; i < S::kEach; ++i) to[i] = load_pack<T, 2>(base + S::row(i) * step + (more + channel_of(i)));
        } else {
#pragma unroll
            for (int i = 0; i < S::kEach; ++i) to[i] = load_some<T, 2>(base + unsigned(min(S::row(i, lane), rows - 1) * int(step) + channel_of(i)), count);
        }
    }
    __device__ __forceinline__ void store(void* to, int64_t channels, int64_t t0, int rows, const float (&v)[S::kEach][2]) const
    {
        T* const base = static_cast<T*>(to) + t0 * channels + first;
        Pack<T, 2> o;
        if (rows == S::kRows && count >= 2) {
            const unsigned more = S::kRowsAtOnce > 1 ? unsigned(lane / (S::kChannels / 2) * int(channels)) : 0u;
#pragma unroll
            for (int i = 0; i < S::kEach; ++i) {
                o.set(v[i]);
                store_pack<T, 2>(base + S::row(i) * channels + (more + channel_of(i)), o);
            }
        } else {
#pragma unroll
            for (int i = 0; i < S::kEach; ++i) {
                o.set(v[i]);
                if (S::row(i, lane) < rows) store_some<T, 2>(base + unsigned(S::row(i, lane) * int(channels) + channel_of(i)), o, count);
            }
        }
    }
    // a pair's two numbers in a row of shared memory
    __device__ __forceinline__ void put(float* row, int i, float a, float b) const
    {
        row[channel_of(i)] = a;
        row[channel_of(i) + 1] = b;
    }
    // the packs of b and c
    __device__ __forceinline__ void load_shared(const Args& p, int64_t t0, int rows, Pack<T, 4> (&to)[S::kPacksEach]) const
    {
        const T *const b = static_cast<const T*>(p.b) + t0 * p.b_step + group * p.b_group, *const c = static_cast<const T*>(p.c) + t0 * p.c_step + group * p.c_group;
#pragma unroll
        for (int i = 0; i < S::kPacksEach; ++i) {
            const int e = i * 64 + lane, r = min(e / (2 * Q), rows - 1), n = e % Q * 4;
            to[i] = Pack<T, 4>{};
            if (e < S::kPacks) {
                const T* const row = e / Q % 2 ? c + r * p.c_step : b + r * p.b_step;
                if (n + 4 <= p.states) {
                    to[i] = load_pack<T, 4>(row + n);
                } else {
                    const int from = lane_again() % Q * 4;          // 64 is a multiple of Q
#pragma unroll
                    for (int k = 0; k < 4; ++k) to[i].put(k, row[state_at(from + k, p.states)]);
                }
            }
        }
    }
    __device__ __forceinline__ void put_shared(const Args& p, const Pack<T, 4> (&from)[S::kPacksEach], float (*to)[2][S::kStates]) const
    {
#pragma unroll
        for (int i = 0; i < S::kPacksEach; ++i) {
            const int e = i * 64 + lane;
            if (e < S::kPacks) {
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = from[i].get(k);
                if (p.states != S::kStates) {           // each copy's part of c
                    const int l = lane_again();
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] *= (i * 64 + l) / Q % 2 ? 1.0f / copies_of(state_at(l % Q * 4 + k, p.states), p.states, S::kStates) : 1.0f;
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) to[e / (2 * Q)][e / Q % 2][S::place(e % Q * 4 + k)] = v[k];
            }
        }
    }
    // the lane's values of b or c of one row
    __device__ __forceinline__ void read_shared(const float* row, float (&to)[kG]) const
    {
        const float* const q = row + part * 16 + j * kG;
        if constexpr (kG == 4) {
            const Four v = *reinterpret_cast<const Four*>(q);
#pragma unroll
            for (int g = 0; g < 4; ++g) to[g] = v[g];
        } else {
#pragma unroll
            for (int g = 0; g < kG; ++g) to[g] = q[g];
        }
    }
    // dt of the pairs
    __device__ __forceinline__ void steps(const Args& p, const Pack<T, 2> (&delta)[S::kEach], float (&dt)[S::kEach][2]) const
    {
#pragma unroll
        for (int i = 0; i < S::kEach; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) dt[i][k] = delta[i].get(k) + bias[i % S::kOwn][k];
        if (p.softplus)
#pragma unroll
            for (int i = 0; i < S::kEach; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) dt[i][k] = softplus_of(dt[i][k]);
    }
    // v times the gates
    __device__ __forceinline__ void gate(const Pack<T, 2> (&z)[S::kEach], float (&v)[S::kEach][2]) const
    {
#pragma unroll
        for (int i = 0; i < S::kEach; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) v[i][k] *= z[i].get(k) * sigmoid(z[i].get(k));
    }
};

// the decays of a quadruple
__device__ __forceinline__ Four decays(Four dt, Four a)
{
    Four e;
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(dt[i] * a[i]);
    return e;
}

// how the rows are cut
struct Plan {
    int q, tiles;
    int waves;              // to a block, backward
    int64_t segment, slots, per_sequence;
    bool several;           // a sequence may have more than one segment
};

inline int lanes_of(int states)
{
    int q = 1;
    while (4 * q < states) q *= 2;
    return q;
}

inline int tile_rows(int q) { return q == 1 ? 4 : (q == 2 ? 8 : 16); }

Plan plan_of(bool packed, int64_t rows, int64_t n, int64_t length, int channels, int states, int groups, bool back);
void check_sizes(uint64_t rows, uint64_t n, uint64_t channels, uint64_t states, uint64_t groups);
void check_strides(std::initializer_list<int64_t> strides);
void join_segments(const Args& p, bool back, hipStream_t stream);

constexpr int kMostStates = 64;
constexpr int64_t kMostStride = 1 << 24;      // of x, delta, z and y's gradient: distances in a tile are 32-bit

// calls body with the lanes to a channel as a type
template <typename F>
void with_lanes(int q, F&& body)
{
    switch (q) {
    case 1: return body(std::integral_constant<int, 1>{});
    case 2: return body(std::integral_constant<int, 2>{});
    case 4: return body(std::integral_constant<int, 4>{});
    case 8: return body(std::integral_constant<int, 8>{});
    default: return body(std::integral_constant<int, 16>{});
    }
}

}  // namespace selective
}  // namespace seqamd
