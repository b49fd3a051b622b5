// Shared by the selective scan's two directions (seq_selective.hip, seq_selective_backward.hip): how the channels and states lie on a wave,
// how sequences are cut into segments, what a tile of rows holds.
//
// h_t = exp(dt_t a) h_{t-1} + dt_t x_t b_t for each channel and state, y_t = sum over the states of c_t h_t, plus d x_t, times
// z_t sigmoid(z_t); dt = softplus(delta + bias), or delta + bias.  Every channel has its own a, x, delta; b and c are those of its group.
//
// Layout.  Q lanes share a channel, four states each (4 Q are at least the states); a lane has four channels.  So a wave holds 256 / Q
// channels with all their states in 16 registers a lane, b and c are read once for four channels, dt and dt x once for four
// states, and the sums over states (y) and over channels (the gradients of b and c) each cross few lanes.
#pragma once
#include "seq_common.h"

#include <type_traits>

namespace seqamd {
namespace selective {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

template <int Q>
struct Shape {
    static constexpr int kRows = Q == 1 ? 4 : (Q == 2 ? 8 : 16);        // of a tile
    static constexpr int kChannels = 256 / Q;                           // of a wave
    static constexpr int kEach = kRows * kChannels / 64;                // elements of a tile to a lane
    static constexpr int kOwn = kChannels >= 64 ? kChannels / 64 : 1;   // different channels among them
    static constexpr int kStates = 4 * Q;
    static constexpr int kPacks = kRows * 2 * Q;                        // of four values of b or c in a tile
    static constexpr int kPacksEach = (kPacks + 63) / 64;

    // element i of a lane: its row in the tile and its channel in the wave
    static __device__ __forceinline__ int row(int i, int lane) { return i * 64 / kChannels + (kChannels < 64 ? lane / kChannels : 0); }
    static __device__ __forceinline__ int channel(int i, int lane) { return kChannels < 64 ? lane % kChannels : i * 64 % kChannels + lane; }
    static constexpr int own(int i) { return kChannels < 64 ? 0 : i * 64 % kChannels / 64; }
};

struct Args {
    const void *x, *delta, *b, *c, *z, *grad;   // z may be null; grad: of y, backward
    const float *a, *d, *bias;                  // a [channels][states]; d and bias may be null
    const float* begin;                         // initial states [n][channels][states] or null
    const float* grad_end;                      // gradients of the final states or null, backward
    float* end;                                 // final states; backward: gradients of the initial ones
    void *out, *ddelta, *dz;                    // y; backward: the gradients of x, delta and z
    const int* offsets;                         // [n + 1] rows where sequences begin, or null: n sequences of `length` rows
    float* carry;                               // [slots][channels][states] the segments' own last states, then the ones before them
    float* back;                                // the same for the gradients of states, the other way
    float* span;                                // [slots][channels] sum of dt over a segment
    float* tile_state;                          // backward: [tiles][channels][states] states at the tiles' first rows, from zero ones at the segment's
    float* tile_span;                           // [tiles][channels] sum of dt from the segment's first row on
    float* shared_parts;                        // backward: [blocks of a group][rows][groups][2][4 Q] sums of the gradients of b and c
    float* own_parts;                           // [pieces][channels][states + 2] those of a, d and bias
    int64_t rows, length, n, segment, slots, per_sequence;
    int64_t x_step, delta_step, z_step, grad_step, b_step, b_group, c_step, c_group;
    int channels, states, groups, per_group, tiles;     // tiles: of a group's channels
    int waves, group_blocks, pieces;                    // backward: waves to a block (they divide the tiles), blocks to a group, pieces of the slots
    bool softplus, several;                             // several: a sequence may have more than one segment
    unsigned first_block;
};

// log(1 + e^v) = max(v, 0) + log1p(w), w = e^-|v|; log1p(w) = 2 atanh(s) with s = w / (2 + w) <= 1/3, and atanh(s) / s as a polynomial
// in s^2, fitted on that range (off by 4e-9; the whole by four roundings)
__device__ __forceinline__ float softplus_of(float v)
{
    const float w = __builtin_amdgcn_exp2f(-fabsf(v) * kLog2e), s = w * __builtin_amdgcn_rcpf(2.0f + w), u = s * s;
    const float f = fmaf(fmaf(fmaf(fmaf(0.14089162647724152f, u, 0.13980302214622498f), u, 0.20012454688549042f), u, 0.3333315849304199f), u, 1.0f);
    return fmaxf(v, 0.0f) + 2.0f * s * f;
}

__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-v * kLog2e)); }

// the lane whose number differs as CTRL says; all of them are there
template <int CTRL>
__device__ __forceinline__ float moved(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// the sum over the Q lanes of a channel, in all of them
template <int Q>
__device__ __forceinline__ float over_states(float v)
{
    if constexpr (Q >= 2) v += moved<0xB1>(v);      // neighbours
    if constexpr (Q >= 4) v += moved<0x4E>(v);      // pairs
    if constexpr (Q >= 8) v += moved<0x141>(v);     // mirrored halves of a row of 16: the other four
    if constexpr (Q >= 16) v += moved<0x140>(v);    // the other eight
    return v;
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

// What the wave's lanes have of the channels
template <typename T, int Q>
struct Column {
    using S = Shape<Q>;
    int lane, q, at;                // at: the lane's first channel in the wave
    int first, count;               // the wave's channels: the first, and how many there are
    int group;
    float a[4][4];                  // a log2(e), zero where there is no channel or state
    float bias[S::kOwn], d[S::kOwn];

    __device__ __forceinline__ void init(const Args& p, int group_, int tile)
    {
        lane = threadIdx.x & 63;
        q = lane % Q;
        at = lane / Q * 4;
        group = group_;
        first = group * p.per_group + tile * S::kChannels;
        count = p.per_group - tile * S::kChannels;
        count = count < S::kChannels ? count : S::kChannels;
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
            const bool there = at + ch < count;
            Pack<float, 4> v{};
            if (there && 4 * q < p.states) v = load_some<float, 4>(p.a + int64_t(first + at + ch) * p.states + 4 * q, p.states - 4 * q);
#pragma unroll
            for (int k = 0; k < 4; ++k) a[ch][k] = v.get(k) * kLog2e;
        }
#pragma unroll
        for (int i = 0; i < S::kOwn; ++i) {
            const int ch = S::channel(i, lane);
            bias[i] = p.bias && ch < count ? p.bias[first + ch] : 0.0f;
            d[i] = p.d && ch < count ? p.d[first + ch] : 0.0f;
        }
    }

    // a state of the lane's channels and states, [channels][states] from `from` on
    __device__ __forceinline__ void load_state(const Args& p, const float* from, float (&h)[4][4]) const
    {
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
            Pack<float, 4> v{};
            if (from && at + ch < count && 4 * q < p.states) v = load_some<float, 4>(from + int64_t(first + at + ch) * p.states + 4 * q, p.states - 4 * q);
#pragma unroll
            for (int k = 0; k < 4; ++k) h[ch][k] = v.get(k);
        }
    }
    __device__ __forceinline__ void store_state(const Args& p, float* to, const float (&h)[4][4]) const
    {
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
            if (at + ch >= count || 4 * q >= p.states) continue;
            Pack<float, 4> v;
            v.set(h[ch]);
            store_some<float, 4>(to + int64_t(first + at + ch) * p.states + 4 * q, v, p.states - 4 * q);
        }
    }

    // the lane's elements of a tile of rows from t0 on; rows from `past` on are the last one again, as are channels behind the last
    __device__ __forceinline__ void load(const void* from, int64_t step, int64_t t0, int64_t past, T (&to)[S::kEach]) const
    {
#pragma unroll
        for (int i = 0; i < S::kEach; ++i) {
            const int64_t t = t0 + S::row(i, lane), row = t < past ? t : past - 1;
            const int ch = S::channel(i, lane);
            to[i] = static_cast<const T*>(from)[row * step + first + (ch < count ? ch : 0)];
        }
    }
    // the packs of b and c
    __device__ __forceinline__ void load_shared(const Args& p, int64_t t0, int64_t past, Pack<T, 4> (&to)[S::kPacksEach]) const
    {
#pragma unroll
        for (int i = 0; i < S::kPacksEach; ++i) {
            const int e = i * 64 + lane, r = e / (2 * Q), n = e % Q * 4;
            const bool c = e / Q % 2;
            const int64_t t = t0 + r, row = t < past ? t : past - 1;
            to[i] = Pack<T, 4>{};
            if (e < S::kPacks && n < p.states)
                to[i] = load_some<T, 4>(c ? static_cast<const T*>(p.c) + row * p.c_step + group * p.c_group + n : static_cast<const T*>(p.b) + row * p.b_step + group * p.b_group + n, p.states - n);
        }
    }
    __device__ __forceinline__ void put_shared(const Pack<T, 4> (&from)[S::kPacksEach], float (*to)[2][S::kStates]) const
    {
#pragma unroll
        for (int i = 0; i < S::kPacksEach; ++i) {
            const int e = i * 64 + lane;
            if (e < S::kPacks) *reinterpret_cast<float4*>(&to[e / (2 * Q)][e / Q % 2][e % Q * 4]) = float4{from[i].get(0), from[i].get(1), from[i].get(2), from[i].get(3)};
        }
    }
};

__device__ __forceinline__ void read4(const float* from, float (&to)[4])
{
    const float4 v = *reinterpret_cast<const float4*>(from);
    to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
}

// how the rows are cut, for `most` waves in all
struct Plan {
    int q, tiles;
    int64_t segment, slots, per_sequence;
    bool several;
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
void join_segments(const Args& p, bool back, hipStream_t stream);

constexpr int kMostStates = 64;

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
