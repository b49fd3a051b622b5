// The selective scan forward, and one step of it against a kept state.
//
// Bound: vector instructions.  A state's step is a product, an exponential, a product and two multiply-adds; the reads and writes of HBM take
// about a third of their time.  The exponentials and the state never leave registers; rows come in tiles, whose dt, dt x, b and c a
// wave puts into shared memory of its own, so no wave waits for another.
// Sequences too few to fill the chip are cut into segments: each forms its own last state from a zero one at its beginning, these are
// joined one after the other with the decay of whole segments, exp(a sum dt), and then every segment runs with the state before it.
// Measured, one sequence of 8192 steps, 4096 channels of 16 states, bfloat16 (5.4e8 steps of states): the segments' own states 111 us, their joining 13, the outputs
// 148, each kernel by itself under a profiler; the call takes 254.  Vector instructions issue in 83 % of the two passes' cycles; the reads and writes alone would take
// 53 us.  One token of 64 such streams 11 us.
#include "seq_selective.h"

#include <algorithm>
#include <type_traits>

namespace seqamd {
namespace selective {
namespace {

// Waves to a SIMD that registers are kept for: three, but two where float32's rows, twice as wide, and few states to a channel, so that a wave has many channels, would
// spill.  Three leave room for all but a few in five kernels: the outputs' of 16-bit types keep 10 registers in memory with 16 states and 7 with up to four, of float32 2 with
// 32, outside their loops over rows.  (Forward, two and three: one sequence of 8192, 4096 channels of 16, bfloat16, 266 and 257 us; 16 of 1000, 1024 channels of 4, bfloat16, 87 and 86; in float32 50003
// steps of 256 of 8 113 and 122, 16 of 1000, 1024 of 16, 158 and 173, 512 of 32 144 and 137; a segment's own states of 1024 of 4 with two 105, with three 108.)
template <typename T>
constexpr int waves_of(int q, bool out) { return sizeof(T) == 4 && q < (out ? 8 : 2) ? 2 : 3; }

// OUT: the outputs and the sequences' last states; otherwise the segments' own last states and the sums of dt
template <typename T, int Q, bool OUT>
__global__ void __launch_bounds__(kThreads, waves_of<T>(Q, OUT)) scan_kernel(Args p)
{
    using S = Shape<Q>;
    constexpr int R = S::kRows, E = S::kEach, G = S::kGroups, kSets = S::kSets;
    __shared__ __attribute__((aligned(16))) float s_in[kWaves][R][2][S::kChannels];
    __shared__ __attribute__((aligned(16))) float s_bc[kWaves][R][2][S::kStates];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), columns = p.groups * p.tiles;
    const int64_t id = (int64_t(p.first_block) + blockIdx.x) * kWaves + wave, slot = id / columns;
    if (slot >= p.slots) return;
    const Segment s = segment_of(p, slot);
    if (!s.there || (!OUT && s.last_one)) return;
    Column<T, Q> col;
    col.init(p, int(id % columns) / p.tiles, int(id % columns) % p.tiles);
    const int64_t size = int64_t(p.channels) * p.states;
    Four h[4], span[kSets];
    if (s.first_one) {
        col.load_state(p, p.begin ? p.begin + s.seq * size : nullptr, h);
    } else if constexpr (OUT) {
        col.load_own(p, p.carry, slot, h);
    } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) h[u] = Four{};
    }
#pragma unroll
    for (int i = 0; i < kSets; ++i) span[i] = Four{};
    auto& in = s_in[wave];
    auto& bc = s_bc[wave];
    Pack<T, 2> x[E], delta[E], z[E];
    Pack<T, 4> shared[S::kPacksEach];
    auto fetch = [&](int64_t t0) __attribute__((always_inline)) {
        const int rows = s.past - t0 < R ? int(s.past - t0) : R;
        col.load(p.x, p.x_step, t0, rows, x);
        col.load(p.delta, p.delta_step, t0, rows, delta);
        if (OUT && p.z) col.load(p.z, p.z_step, t0, rows, z);
        col.load_shared(p, t0, rows, shared);
    };
    if (s.first < s.past) fetch(s.first);
    for (int64_t t0 = s.first; t0 < s.past; t0 += R) {
        const int rows = s.past - t0 < R ? int(s.past - t0) : R;
        Pack<T, 2> x_now[E], z_now[E];
        {
            float dt[E][2];
            col.steps(p, delta, dt);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                auto& row = in[S::row(i, col.lane)];
                col.put(row[0], i, dt[i][0], dt[i][1]);
                col.put(row[1], i, dt[i][0] * x[i].get(0), dt[i][1] * x[i].get(1));
                x_now[i] = x[i], z_now[i] = z[i];
            }
        }
        col.put_shared(p, shared, bc);
        wave_sync();
        if (t0 + R < s.past) fetch(t0 + R);
        auto step = [&](int t) __attribute__((always_inline)) {
            float b[G], c[G];
            col.read_shared(bc[t][0], b);
            if constexpr (OUT) col.read_shared(bc[t][1], c);
#pragma unroll
            for (int i = 0; i < kSets; ++i) {
                const Four dt = *reinterpret_cast<const Four*>(&in[t][0][col.at + 4 * i]);
                const float du = in[t][1][col.at + 4 * i + col.j];
                Four y{};
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    Four& state = h[i * G + g];
                    state = add_products(du, b[g], state * decays(dt, col.a[i * G + g]));
                    if constexpr (OUT)
#pragma unroll
                        for (int k = 0; k < 4; ++k) y[k] = fmaf(c[g], state[k], y[k]);
                }
                if constexpr (OUT) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) y[k] = over_states<Q>(y[k]);
                    *reinterpret_cast<Four*>(&in[t][0][col.at + 4 * i]) = y;
                } else {
                    span[i] += dt;
                }
            }
        };
        if (rows == R) {
#pragma unroll 4
            for (int t = 0; t < R; ++t) step(t);
        } else {
#pragma unroll 1
            for (int t = 0; t < rows; ++t) step(t);
        }
        wave_sync();
        if constexpr (OUT) {
            float y[E][2];
#pragma unroll
            for (int i = 0; i < E; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) y[i][k] = fmaf(col.d[i % S::kOwn][k], x_now[i].get(k), in[S::row(i, col.lane)][0][col.channel_of(i) + k]);
            if (p.z) col.gate(z_now, y);
            col.store(p.out, p.channels, t0, rows, y);
            wave_sync();
        }
    }
    if constexpr (OUT) {
        if (s.last_one) col.store_state(p, p.end + s.seq * size, h);
    } else {
        col.store_own(p, p.carry, slot, h);
        col.store_line(p.span + slot * p.channels, span);
    }
}

// Sequences with several segments: the segments' own last states become the states before them, and (BACK) their own gradients the gradients behind
// them.  P threads to a state take neighbouring segments, whose maps meet in shared memory; eight segments' numbers are on their way at once.
template <bool BACK, int Q, int P>
__global__ void __launch_bounds__(kThreads) join_kernel(Args p, int blocks)
{
    using S = Shape<Q>;
    constexpr int kLanes = kThreads / P, kAtOnce = 8;
    __shared__ float s_a[P][kLanes], s_b[P][kLanes];
    const int64_t block = int64_t(p.first_block) + blockIdx.x, seq = block / blocks;
    if (seq >= p.n) return;
    int64_t first, past;
    rows_of(p, seq, first, past);
    const int64_t count = (past - first + p.segment - 1) / p.segment, slot = slot_of(p, seq, first);
    if (count < 2 || slot + count > p.slots) return;
    const int lane = threadIdx.x % kLanes, piece = threadIdx.x / kLanes;
    const int64_t each = (count + P - 1) / P, size = int64_t(p.groups) * p.tiles * 1024;
    for (int64_t base = (block % blocks) * kLanes; base < size; base += int64_t(blocks) * kLanes) {
        // e as the lanes hold it: column, quadruple, lane, channel of it
        const int64_t e = base + lane;
        const int column = int(e / 1024), u = int(e / 256) % 4, l = int(e / 4) % 64, i = int(e % 4);
        const int ch = (column % p.tiles) * S::kChannels + l / 4 / S::kQuads * 4 * S::kSets + 4 * (u / S::kGroups) + i;
        const int state = l / 4 % S::kQuads * 16 + 4 * (u % S::kGroups) + l % 4;
        const bool there = ch < p.per_group;
        const int channel = column / p.tiles * p.per_group + ch;
        const float a = there ? p.a[int64_t(channel) * p.states + state_at(state, p.states)] * kLog2e : 0.0f;
        // BACKWARD: from the last segment to the first.  A segment's map takes the state before it to the one behind it; the last one's is not
        // known, and not asked for.
        auto join = [&](Four* at, auto backward) __attribute__((always_inline)) {
            constexpr bool kBackward = decltype(backward)::value;
            float* const own = reinterpret_cast<float*>(at) + e;
            const int64_t low = min(piece * each, count), high = min(low + each, count);        // in the order of the walk
            auto segment = [&](int64_t k) { return slot + (kBackward ? count - 1 - k : k); };
            auto walk = [&](auto&& take) __attribute__((always_inline)) {
                for (int64_t k0 = low; k0 < high; k0 += kAtOnce) {
                    float v[kAtOnce], d[kAtOnce];
#pragma unroll
                    for (int n = 0; n < kAtOnce; ++n) {
                        const bool known = k0 + n < high && k0 + n < count - 1;
                        v[n] = known ? own[segment(k0 + n) * size] : 0.0f;
                        d[n] = known && there ? p.span[segment(k0 + n) * p.channels + channel] : 0.0f;
                    }
#pragma unroll
                    for (int n = 0; n < kAtOnce; ++n)
                        if (k0 + n < high) take(k0 + n, __builtin_amdgcn_exp2f(a * d[n]), v[n]);
                }
            };
            float h = 0.0f;
            if constexpr (P > 1) {
                float ma = 1.0f, mb = 0.0f;
                walk([&](int64_t, float d, float v) {
                    mb = fmaf(mb, d, v);
                    ma *= d;
                });
                __syncthreads();
                s_a[piece][lane] = ma, s_b[piece][lane] = mb;
                __syncthreads();
                for (int n = 0; n < piece; ++n) h = fmaf(h, s_a[n][lane], s_b[n][lane]);
            }
            walk([&](int64_t k, float d, float v) {
                own[segment(k) * size] = h;
                h = fmaf(h, d, v);
            });
        };
        join(p.carry, std::false_type{});
        if constexpr (BACK) join(p.back, std::true_type{});
    }
}

// One token of each row: Q lanes to a channel, four neighbouring states to a lane.  Bound: vector instructions, in 72 % of the cycles, 213 to a wave, of which the formula
// needs some 60 and the addresses the most: a division of 64 bits for the row, one for the group, products of rows and distances.  (34 MB of states of the 64 streams above,
// read and written, at 3.0 TB/s; four rows to a thread, whose a is then read once, took 11.6 us in place of 12.3, and the call with its host side the same.)
template <typename T, int Q>
__global__ void __launch_bounds__(kThreads) step_kernel(Args p)
{
    const int64_t e = (int64_t(p.first_block) + blockIdx.x) * (kThreads / Q) + threadIdx.x / Q, row = e / p.channels;
    if (row >= p.rows) return;              // all the lanes of a channel together
    const int ch = int(e - row * p.channels), q = threadIdx.x % Q, group = ch / p.per_group;
    const int count = 4 * q < p.states ? p.states - 4 * q : 0;
    float* const at = p.end + e * p.states + 4 * q;
    Pack<float, 4> h{}, a{};
    Pack<T, 4> b{}, c{};
    if (count) {
        h = load_some<float, 4>(at, count);
        a = load_some<float, 4>(p.a + int64_t(ch) * p.states + 4 * q, count);
        b = load_some<T, 4>(static_cast<const T*>(p.b) + row * p.b_step + group * p.b_group + 4 * q, count);
        c = load_some<T, 4>(static_cast<const T*>(p.c) + row * p.c_step + group * p.c_group + 4 * q, count);
    }
    const float x = float(static_cast<const T*>(p.x)[row * p.x_step + ch]), raw = float(static_cast<const T*>(p.delta)[row * p.delta_step + ch]) + (p.bias ? p.bias[ch] : 0.0f);
    const float dt = p.softplus ? softplus_of(raw) : raw, du = dt * x;
    float now[4], y = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) now[k] = fmaf(h.get(k), __builtin_amdgcn_exp2f(dt * (a.get(k) * kLog2e)), du * b.get(k));
    if (count < 4)          // where there is no state an infinite du has made NaN
#pragma unroll
        for (int k = 0; k < 4; ++k) now[k] = k < count ? now[k] : 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) y = fmaf(c.get(k), now[k], y);
#pragma unroll
    for (int m = 1; m < Q; m *= 2) y += __shfl_xor(y, m);
    if (p.d) y = fmaf(p.d[ch], x, y);
    if (p.z) {
        const float z = float(static_cast<const T*>(p.z)[row * p.z_step + ch]);
        y *= z * sigmoid(z);
    }
    if (count) {
        h.set(now);
        store_some<float, 4>(at, h, count);
    }
    if (q == 0) static_cast<T*>(p.out)[e] = T(y);
}

}  // namespace

void check_sizes(uint64_t rows, uint64_t n, uint64_t channels, uint64_t states, uint64_t groups)
{
    require(states >= 1 && states <= kMostStates, "a channel has 1 to 64 states");
    require(rows < (uint64_t(1) << 31) && n < (uint64_t(1) << 31) && channels < (uint64_t(1) << 24) && groups < (uint64_t(1) << 24), "too many rows, channels or sequences");
    require(groups >= 1 && channels % groups == 0, "the channels are a multiple of the groups");
}

void check_strides(std::initializer_list<int64_t> strides)
{
    for (const int64_t stride : strides) require(stride >= 0 && stride <= kMostStride, "rows are too far apart");
}

// Segments: as long as makes 4096 waves over all rows forward, 2048 backward, where two waves fill a SIMD, and with up to eight states, whose
// segments would be short; at least a tile: few rows end sooner in many short segments (3000 steps of 100 channels of 16, bfloat16, forward 27 us, with
// four tiles to a segment 57; with gradients 95 and 200).  (16 sequences of 1024, 2048 channels of 16, bfloat16: 258 us, with 2048 waves 270;
// 3 of 3000, 1000 channels of 64, float16: 265 and 287; but one of 50000, 256 channels of 8, bfloat16: 115 and 102, of 4: 119 and 94.)
// Backward no more than that: the waves are all there at once, and one more would run behind them.  A packed sequence ends half a segment
// early on average.  (24 sequences of up to 900, 770 channels in two groups, float16, forward and gradients: 385 us, with 2352 waves and an idle one in eight 473.)
// Backward four waves to a block add up their sums over channels where all four have all their channels, which is 1 % sooner than each alone (4 sequences of
// 2048, 2048 channels of 16, bfloat16, forward and gradients: 589 and 594 us); with idle ones it is slower (64 of 1024, 192 channels: 548 and 492; 64 channels: 439 and 215).
Plan plan_of(bool packed, int64_t rows, int64_t n, int64_t length, int channels, int states, int groups, bool back)
{
    Plan p;
    p.q = lanes_of(states);
    const int wide = 256 / p.q, tile = tile_rows(p.q);
    p.tiles = (channels / groups + wide - 1) / wide;
    p.waves = channels / groups % (kWaves * wide) ? 1 : kWaves;
    const int64_t columns = int64_t(groups) * p.tiles;
    int64_t most = back || p.q <= 2 ? 2048 : 4096, segment;
    if (packed) {
        most = std::max(most - n * columns / 2, most / 2);
        segment = (rows * columns + most - 1) / most;
    } else {
        const int64_t each = std::max<int64_t>(most / std::max<int64_t>(n * columns, 1), 1);
        segment = (length + each - 1) / each;
    }
    segment = (std::max<int64_t>(segment, 1) + tile - 1) / tile * tile;
    const int64_t longest = packed ? rows : length;
    p.several = longest > segment;
    p.segment = p.several ? segment : std::max<int64_t>((longest + tile - 1) / tile * tile, tile);
    p.per_sequence = packed ? 0 : std::max<int64_t>((length + p.segment - 1) / p.segment, 1);
    p.slots = n == 0 ? 0 : (packed ? rows / p.segment + n : n * p.per_sequence);
    return p;
}

// Many segments to a sequence are joined by several threads to a state: one of 50003, 256 channels of 8, float32, forward with 16 threads to a state 108 us, with one
// 197; 8 of 2048, 256 channels of 16, bfloat16, 128 segments each, 66 and 68; 64 segments of 16 such sequences 96 and 87: there are then threads enough, and
// the maps go by shared memory for nothing.
void join_segments(const Args& p, bool back, hipStream_t stream)
{
    const int64_t states = int64_t(p.groups) * p.tiles * 1024, count = p.offsets ? p.rows / p.segment / p.n : p.per_sequence;        // on average
    with_lanes(lanes_of(p.states), [&](auto q) {
        constexpr int Q = decltype(q)::value;
        auto launch = [&](auto kernel, int pieces) {
            // no more blocks than some for every compute unit: most sequences may have one segment
            const int64_t most = states * pieces / kThreads, blocks = std::max<int64_t>(std::min(most, 8192 / std::max<int64_t>(p.n, 1)), 1);
            in_launches(blocks * p.n, kThreads, [&](unsigned first, dim3 grid) {
                Args a = p;
                a.first_block = first;
                hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, a, int(blocks));
            });
        };
        if (count > 64) launch(back ? join_kernel<true, Q, 16> : join_kernel<false, Q, 16>, 16);
        else launch(back ? join_kernel<true, Q, 1> : join_kernel<false, Q, 1>, 1);
    });
}

}  // namespace selective
}  // namespace seqamd

using namespace seqamd;
using namespace seqamd::selective;

namespace {

uint64_t up(uint64_t bytes) { return (bytes + 255) / 256 * 256; }

uint64_t carry_bytes(const Plan& p, uint64_t groups) { return up(uint64_t(p.slots) * groups * p.tiles * 4096); }

uint64_t forward_workspace(const Plan& p, uint64_t channels, uint64_t groups) { return p.several ? carry_bytes(p, groups) + up(uint64_t(p.slots) * channels * 4) : 0; }

}  // namespace

extern "C" {

__attribute__((visibility("default"))) uint64_t cusig_amd_selective_scan_workspace(bool packed, uint64_t sequences, uint64_t length, uint64_t rows, uint64_t channels,
                                                                                    uint64_t states, uint64_t groups) noexcept
{
    uint64_t bytes = 0;
    sigamd::guarded([&] {
        check_sizes(rows, sequences, channels, states, groups);
        bytes = forward_workspace(plan_of(packed, int64_t(rows), int64_t(sequences), int64_t(length), int(channels), int(states), int(groups), false), channels, groups);
    });
    return bytes;
}

__attribute__((visibility("default"))) int cusig_amd_selective_scan(
    int dtype, const void* x, const void* delta, const float* a, const void* b, const void* c, const float* d, const void* z, const float* delta_bias,
    const float* initial_state, void* y, float* final_state, const int* offsets, uint64_t sequences, uint64_t length, uint64_t rows, uint64_t channels,
    uint64_t states, uint64_t groups, int64_t x_stride, int64_t delta_stride, int64_t z_stride, int64_t b_stride, int64_t b_group, int64_t c_stride,
    int64_t c_group, bool softplus, void* workspace, uint64_t workspace_bytes, void* stream) noexcept
{
    return sigamd::guarded([&] {
        check_sizes(rows, sequences, channels, states, groups);
        if (!offsets) check_rows(sequences, length, rows);
        check_strides({x_stride, delta_stride, z_stride});
        if (sequences * channels == 0) return;
        require(a && final_state && (rows == 0 || (x && delta && b && c && y)), "a tensor is missing");
        const Plan plan = plan_of(offsets, int64_t(rows), int64_t(sequences), int64_t(length), int(channels), int(states), int(groups), false);
        check_workspace(workspace, workspace_bytes, forward_workspace(plan, channels, groups));
        Args p{};
        p.x = x, p.delta = delta, p.a = a, p.b = b, p.c = c, p.d = d, p.z = z, p.bias = delta_bias, p.begin = initial_state, p.out = y, p.end = final_state;
        p.offsets = offsets, p.n = int64_t(sequences), p.length = int64_t(length), p.rows = int64_t(rows);
        p.channels = int(channels), p.states = int(states), p.groups = int(groups), p.per_group = int(channels / groups), p.tiles = plan.tiles;
        p.x_step = x_stride, p.delta_step = delta_stride, p.z_step = z_stride, p.b_step = b_stride, p.b_group = b_group, p.c_step = c_stride, p.c_group = c_group;
        p.softplus = softplus;
        p.segment = plan.segment, p.slots = plan.slots, p.per_sequence = plan.per_sequence;
        p.carry = static_cast<Four*>(workspace);
        p.span = reinterpret_cast<float*>(static_cast<char*>(workspace) + (plan.several ? carry_bytes(plan, groups) : 0));
        const int64_t waves = p.slots * p.groups * p.tiles, blocks = (waves + kWaves - 1) / kWaves;
        const auto s = static_cast<hipStream_t>(stream);
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            with_lanes(plan.q, [&](auto q) {
                constexpr int Q = decltype(q)::value;
                if (plan.several) {
                    launch_all(scan_kernel<T, Q, false>, blocks, kThreads, s, p);
                    join_segments(p, false, s);
                }
                launch_all(scan_kernel<T, Q, true>, blocks, kThreads, s, p);
            });
        });
    });
}

__attribute__((visibility("default"))) int cusig_amd_selective_scan_step(
    int dtype, const void* x, const void* delta, const float* a, const void* b, const void* c, const float* d, const void* z, const float* delta_bias, float* state,
    void* y, uint64_t rows, uint64_t channels, uint64_t states, uint64_t groups, int64_t x_stride, int64_t delta_stride, int64_t z_stride, int64_t b_stride,
    int64_t b_group, int64_t c_stride, int64_t c_group, bool softplus, void* stream) noexcept
{
    return sigamd::guarded([&] {
        check_sizes(rows, rows, channels, states, groups);
        if (rows * channels == 0) return;
        require(x && delta && a && b && c && state && y, "a tensor is missing");
        Args p{};
        p.x = x, p.delta = delta, p.a = a, p.b = b, p.c = c, p.d = d, p.z = z, p.bias = delta_bias, p.out = y, p.end = state;
        p.rows = int64_t(rows), p.channels = int(channels), p.states = int(states), p.per_group = int(channels / groups);
        p.x_step = x_stride, p.delta_step = delta_stride, p.z_step = z_stride, p.b_step = b_stride, p.b_group = b_group, p.c_step = c_stride, p.c_group = c_group;
        p.softplus = softplus;
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            with_lanes(lanes_of(p.states), [&](auto q) {
                constexpr int Q = decltype(q)::value;
                launch_all(step_kernel<T, Q>, (p.rows * p.channels * Q + kThreads - 1) / kThreads, kThreads, static_cast<hipStream_t>(stream), p);
            });
        });
    });
}

}  // extern "C"
