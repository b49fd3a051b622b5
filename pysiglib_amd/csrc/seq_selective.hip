// The selective scan forward, and one step of it against a kept state.
//
// Bound: vector instructions.  A state's step is a product, an exponential, a product and two multiply-adds; the reads and writes of HBM take
// about a third of their time.  The exponentials and the state never leave registers; rows come in tiles, whose dt, dt x, b and c a
// wave puts into shared memory of its own, so no wave waits for another.
// Sequences too few to fill the chip are cut into segments: each forms its own last state from a zero one at its beginning, these are
// joined one after the other with the decay of whole segments, exp(a sum dt), and then every segment runs with the state before it.
#include "seq_selective.h"

#include <algorithm>
#include <type_traits>

namespace seqamd {
namespace selective {
namespace {

// OUT: the outputs and the sequences' last states; otherwise the segments' own last states and the sums of dt
template <typename T, int Q, bool OUT>
__global__ void __launch_bounds__(kThreads, 2) scan_kernel(Args p)
{
    using S = Shape<Q>;
    constexpr int R = S::kRows, E = S::kEach;
    __shared__ __attribute__((aligned(16))) float s_in[kWaves][R][2][S::kChannels];
    __shared__ __attribute__((aligned(16))) float s_bc[kWaves][R][2][S::kStates];
    const int wave = threadIdx.x / 64, columns = p.groups * p.tiles;
    const int64_t id = (int64_t(p.first_block) + blockIdx.x) * kWaves + wave, slot = id / columns;
    if (slot >= p.slots) return;
    const Segment s = segment_of(p, slot);
    if (!s.there || (!OUT && s.last_one)) return;
    Column<T, Q> col;
    col.init(p, int(id % columns) / p.tiles, int(id % columns) % p.tiles);
    const int64_t size = int64_t(p.channels) * p.states;
    float h[4][4], span[4];
    col.load_state(p, !OUT ? nullptr : (s.first_one ? (p.begin ? p.begin + s.seq * size : nullptr) : p.carry + slot * size), h);
#pragma unroll
    for (int ch = 0; ch < 4; ++ch) span[ch] = 0.0f;
    auto& in = s_in[wave];
    auto& bc = s_bc[wave];
    T x[E], delta[E], z[E];
    Pack<T, 4> shared[S::kPacksEach];
    auto fetch = [&](int64_t t0) __attribute__((always_inline)) {
        col.load(p.x, p.x_step, t0, s.past, x);
        col.load(p.delta, p.delta_step, t0, s.past, delta);
        if (OUT && p.z) col.load(p.z, p.z_step, t0, s.past, z);
        col.load_shared(p, t0, s.past, shared);
    };
    if (s.first < s.past) fetch(s.first);
    for (int64_t t0 = s.first; t0 < s.past; t0 += R) {
        T x_now[E], z_now[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float raw = float(delta[i]) + col.bias[S::own(i)], dt = p.softplus ? softplus_of(raw) : raw;
            in[S::row(i, col.lane)][0][S::channel(i, col.lane)] = dt;
            in[S::row(i, col.lane)][1][S::channel(i, col.lane)] = dt * float(x[i]);
            x_now[i] = x[i], z_now[i] = z[i];
        }
        col.put_shared(shared, bc);
        if (t0 + R < s.past) fetch(t0 + R);
        auto step = [&](int t) __attribute__((always_inline)) {
            float dt[4], du[4], b[4], c[4], y[4];
            read4(&in[t][0][col.at], dt);
            read4(&in[t][1][col.at], du);
            read4(&bc[t][0][4 * col.q], b);
            if constexpr (OUT) read4(&bc[t][1][4 * col.q], c);
#pragma unroll
            for (int ch = 0; ch < 4; ++ch) {
                y[ch] = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    h[ch][k] = fmaf(h[ch][k], __builtin_amdgcn_exp2f(dt[ch] * col.a[ch][k]), du[ch] * b[k]);
                    if constexpr (OUT) y[ch] = fmaf(c[k], h[ch][k], y[ch]);
                }
                if constexpr (OUT) y[ch] = over_states<Q>(y[ch]);
                else span[ch] += dt[ch];
            }
            if constexpr (OUT) *reinterpret_cast<float4*>(&in[t][0][col.at]) = float4{y[0], y[1], y[2], y[3]};
        };
        const int count = s.past - t0 < R ? int(s.past - t0) : R;
        if (count == R) {
#pragma unroll 4
            for (int t = 0; t < R; ++t) step(t);
        } else {
#pragma unroll 1
            for (int t = 0; t < count; ++t) step(t);
        }
        if constexpr (OUT) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int r = S::row(i, col.lane), ch = S::channel(i, col.lane);
                float y = fmaf(col.d[S::own(i)], float(x_now[i]), in[r][0][ch]);
                if (p.z) y *= float(z_now[i]) * sigmoid(float(z_now[i]));
                if (r < count && ch < col.count) static_cast<T*>(p.out)[(t0 + r) * p.channels + col.first + ch] = T(y);
            }
        }
    }
    if constexpr (OUT) {
        if (s.last_one) col.store_state(p, p.end + s.seq * size, h);
    } else {
        col.store_state(p, p.carry + slot * size, h);
        if (col.q == 0)
#pragma unroll
            for (int ch = 0; ch < 4; ++ch)
                if (col.at + ch < col.count) p.span[slot * p.channels + col.first + col.at + ch] = span[ch];
    }
}

// A thread to a state of a sequence with several segments: their own last states become the states before them, and (BACK) their own gradients
// the gradients behind them
template <bool BACK>
__global__ void __launch_bounds__(kThreads) join_kernel(Args p)
{
    const int64_t size = int64_t(p.channels) * p.states, blocks = (size + kThreads - 1) / kThreads, block = int64_t(p.first_block) + blockIdx.x;
    const int64_t seq = block / blocks, e = (block - seq * blocks) * kThreads + threadIdx.x;
    if (seq >= p.n || e >= size) return;
    int64_t first, past;
    rows_of(p, seq, first, past);
    const int64_t count = (past - first + p.segment - 1) / p.segment, slot = slot_of(p, seq, first);
    if (count < 2 || slot + count > p.slots) return;
    const float a = p.a[e] * kLog2e;
    const float* const span = p.span + e / p.states;
    float h = p.begin ? p.begin[seq * size + e] : 0.0f;
    for (int64_t k = slot; k < slot + count; ++k) {
        const float own = k + 1 < slot + count ? p.carry[k * size + e] : 0.0f;
        p.carry[k * size + e] = h;
        if (k + 1 < slot + count) h = fmaf(h, __builtin_amdgcn_exp2f(a * span[k * p.channels]), own);
    }
    if constexpr (BACK) {
        float g = p.grad_end ? p.grad_end[seq * size + e] : 0.0f;
        for (int64_t k = slot + count - 1; k >= slot; --k) {
            const float own = k > slot ? p.back[k * size + e] : 0.0f;
            p.back[k * size + e] = g;
            if (k > slot) g = fmaf(g, __builtin_amdgcn_exp2f(a * span[k * p.channels]), own);
        }
    }
}

// One token of each row: Q lanes to a channel, four states to a lane
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
    for (int k = 0; k < 4; ++k) {
        now[k] = fmaf(h.get(k), __builtin_amdgcn_exp2f(dt * (a.get(k) * kLog2e)), du * b.get(k));
        y = fmaf(c.get(k), now[k], y);
    }
    y = over_states<Q>(y);
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
    require(rows < (uint64_t(1) << 31) && n < (uint64_t(1) << 31) && channels < (uint64_t(1) << 24), "too many rows, channels or sequences");
    require(groups >= 1 && channels % groups == 0, "the channels are a multiple of the groups");
}

// Segments: as long as makes `most` waves over all rows, not shorter than four tiles
Plan plan_of(bool packed, int64_t rows, int64_t n, int64_t length, int channels, int states, int groups, bool back)
{
    Plan p;
    p.q = lanes_of(states);
    const int wide = 256 / p.q, tile = tile_rows(p.q);
    p.tiles = (channels / groups + wide - 1) / wide;
    const int64_t most = 4096, columns = int64_t(groups) * p.tiles;
    int64_t segment = (rows * columns + most - 1) / most;
    segment = (std::max<int64_t>(segment, 4 * tile) + tile - 1) / tile * tile;
    const int64_t longest = packed ? rows : length;
    p.several = longest > segment;
    p.segment = p.several ? segment : std::max<int64_t>((longest + tile - 1) / tile * tile, tile);
    p.per_sequence = packed ? 0 : std::max<int64_t>((length + p.segment - 1) / p.segment, 1);
    p.slots = n == 0 ? 0 : (packed ? rows / p.segment + n : n * p.per_sequence);
    return p;
}

void join_segments(const Args& p, bool back, hipStream_t stream)
{
    const int64_t blocks = (int64_t(p.channels) * p.states + kThreads - 1) / kThreads * p.n;
    if (back) launch_all(join_kernel<true>, blocks, kThreads, stream, p);
    else launch_all(join_kernel<false>, blocks, kThreads, stream, p);
}

}  // namespace selective
}  // namespace seqamd

using namespace seqamd;
using namespace seqamd::selective;

namespace {

uint64_t up(uint64_t bytes) { return (bytes + 255) / 256 * 256; }

uint64_t forward_workspace(const Plan& p, uint64_t channels, uint64_t states)
{
    return p.several ? up(uint64_t(p.slots) * channels * states * 4) + up(uint64_t(p.slots) * channels * 4) : 0;
}

}  // namespace

extern "C" {

__attribute__((visibility("default"))) uint64_t cusig_amd_selective_scan_workspace(bool packed, uint64_t sequences, uint64_t length, uint64_t rows, uint64_t channels,
                                                                                    uint64_t states, uint64_t groups) noexcept
{
    uint64_t bytes = 0;
    sigamd::guarded([&] {
        check_sizes(rows, sequences, channels, states, groups);
        bytes = forward_workspace(plan_of(packed, int64_t(rows), int64_t(sequences), int64_t(length), int(channels), int(states), int(groups), false), channels, states);
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
        require(offsets || sequences * length == rows, "rows are not sequences times length");
        if (sequences * channels == 0) return;
        require(a && final_state && (rows == 0 || (x && delta && b && c && y)), "a tensor is missing");
        const Plan plan = plan_of(offsets, int64_t(rows), int64_t(sequences), int64_t(length), int(channels), int(states), int(groups), false);
        check_workspace(workspace, workspace_bytes, forward_workspace(plan, channels, states));
        Args p{};
        p.x = x, p.delta = delta, p.a = a, p.b = b, p.c = c, p.d = d, p.z = z, p.bias = delta_bias, p.begin = initial_state, p.out = y, p.end = final_state;
        p.offsets = offsets, p.n = int64_t(sequences), p.length = int64_t(length), p.rows = int64_t(rows);
        p.channels = int(channels), p.states = int(states), p.groups = int(groups), p.per_group = int(channels / groups), p.tiles = plan.tiles;
        p.x_step = x_stride, p.delta_step = delta_stride, p.z_step = z_stride, p.b_step = b_stride, p.b_group = b_group, p.c_step = c_stride, p.c_group = c_group;
        p.softplus = softplus;
        p.segment = plan.segment, p.slots = plan.slots, p.per_sequence = plan.per_sequence, p.several = plan.several;
        p.carry = static_cast<float*>(workspace);
        p.span = reinterpret_cast<float*>(static_cast<char*>(workspace) + up(uint64_t(plan.slots) * channels * states * 4));
        const int64_t waves = p.slots * p.groups * p.tiles, blocks = (waves + kWaves - 1) / kWaves;
        const auto s = static_cast<hipStream_t>(stream);
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            with_lanes(plan.q, [&](auto q) {
                constexpr int Q = decltype(q)::value;
                if (p.several) {
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
