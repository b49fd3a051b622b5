// The selective scan's gradients.
//
// Mathematics.  Let gy_t be the gradient of the sum over states (that of y times the gate), k_t = exp(dt_t a), and G_t the gradient of h_t:
// G_t = gy_t c_t + k_{t+1} G_{t+1}, with that of the final state behind the last step.  Then for each channel (sums over states)
//   dx_t = dt_t sum G_t b_t + d gy_t,   d(dt_t) = sum (G_t k_t h_{t-1} a) + x_t sum G_t b_t,   dz_t = g_t y_t slope(z_t),
// for each state da = sum over rows of G_t k_t h_{t-1} dt_t, and for each row of a group (sums over its channels) db_t = sum G_t dt_t x_t,
// dc_t = sum gy_t h_t.  k_0 G_0 is the gradient of the initial state.  Nothing is taken from the forward pass: the states are formed again.
//
// Passes.  First every segment forward from a zero state: its state at each tile's first row, its own last state, and (where a
// sequence has several) the gradient of the state before it that its own rows make, as sum over t of (k_first ... k_t) gy_t c_t, so one
// exponential serves both.  Segments are joined; then each goes from its last tile to its first: the state before a tile is the stored one plus
// exp(a sum dt) times the segment's; half a tile's states are formed and kept in registers, and its rows gone back through.
// Sums over channels stay in a row's 64 lanes, then the block's waves, then the blocks, all in a fixed order.
//
// Bound: vector instructions, some fifteen and two and a half exponentials for each state and row.
#include "seq_selective.h"

#include <algorithm>
#include <type_traits>

namespace seqamd {
namespace selective {
namespace {

__device__ __forceinline__ float slope(float v)
{
    const float s = sigmoid(v);
    return s * fmaf(v, 1.0f - s, 1.0f);
}

// Every segment from a zero state: BACK: its own part of the gradients too
template <typename T, int Q, bool BACK>
__global__ void __launch_bounds__(kThreads, 2) states_kernel(Args p)
{
    using S = Shape<Q>;
    constexpr int R = S::kRows, E = S::kEach;
    __shared__ __attribute__((aligned(16))) float s_in[kWaves][R][BACK ? 3 : 2][S::kChannels];
    __shared__ __attribute__((aligned(16))) float s_bc[kWaves][R][2][S::kStates];
    const int wave = threadIdx.x / 64, columns = p.groups * p.tiles;
    const int64_t id = (int64_t(p.first_block) + blockIdx.x) * kWaves + wave, slot = id / columns;
    if (slot >= p.slots) return;
    const Segment s = segment_of(p, slot);
    if (!s.there || s.first >= s.past) return;
    Column<T, Q> col;
    col.init(p, int(id % columns) / p.tiles, int(id % columns) % p.tiles);
    const int64_t size = int64_t(p.channels) * p.states, tile0 = tile_of(slot, s, R);
    float h[4][4], span[4], decay[4][4], back[4][4];
#pragma unroll
    for (int ch = 0; ch < 4; ++ch) {
        span[ch] = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) h[ch][k] = back[ch][k] = 0.0f, decay[ch][k] = 1.0f;
    }
    auto& in = s_in[wave];
    auto& bc = s_bc[wave];
    T x[E], delta[E], z[E], g[E];
    Pack<T, 4> shared[S::kPacksEach];
    auto fetch = [&](int64_t t0) __attribute__((always_inline)) {
        col.load(p.x, p.x_step, t0, s.past, x);
        col.load(p.delta, p.delta_step, t0, s.past, delta);
        if (BACK && p.z) col.load(p.z, p.z_step, t0, s.past, z);
        if (BACK) col.load(p.grad, p.grad_step, t0, s.past, g);
        col.load_shared(p, t0, s.past, shared);
    };
    auto store_span = [&](float* to) __attribute__((always_inline)) {
        if (col.q == 0)
#pragma unroll
            for (int ch = 0; ch < 4; ++ch)
                if (col.at + ch < col.count) to[col.first + col.at + ch] = span[ch];
    };
    fetch(s.first);
    int64_t tile = tile0;
    for (int64_t t0 = s.first; t0 < s.past; t0 += R, ++tile) {
        if (t0 > s.first) {
            col.store_state(p, p.tile_state + tile * size, h);
            store_span(p.tile_span + tile * p.channels);
        }
        if (t0 + R >= s.past && s.last_one && (!BACK || s.first_one)) break;      // nobody asks for its own last state
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int r = S::row(i, col.lane), ch = S::channel(i, col.lane);
            const float raw = float(delta[i]) + col.bias[S::own(i)], dt = p.softplus ? softplus_of(raw) : raw;
            in[r][0][ch] = dt;
            in[r][1][ch] = dt * float(x[i]);
            if constexpr (BACK) in[r][2][ch] = p.z ? float(g[i]) * (float(z[i]) * sigmoid(float(z[i]))) : float(g[i]);
        }
        col.put_shared(shared, bc);
        if (t0 + R < s.past) fetch(t0 + R);
        auto step = [&](int t) __attribute__((always_inline)) {
            float dt[4], du[4], gy[4], b[4], c[4];
            read4(&in[t][0][col.at], dt);
            read4(&in[t][1][col.at], du);
            read4(&bc[t][0][4 * col.q], b);
            if constexpr (BACK) {
                read4(&in[t][2][col.at], gy);
                read4(&bc[t][1][4 * col.q], c);
            }
#pragma unroll
            for (int ch = 0; ch < 4; ++ch) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float e = __builtin_amdgcn_exp2f(dt[ch] * col.a[ch][k]);
                    h[ch][k] = fmaf(h[ch][k], e, du[ch] * b[k]);
                    if constexpr (BACK) {
                        decay[ch][k] *= e;
                        back[ch][k] = fmaf(decay[ch][k], gy[ch] * c[k], back[ch][k]);
                    }
                }
                span[ch] += dt[ch];
            }
        };
        const int count = s.past - t0 < R ? int(s.past - t0) : R;
        if (count == R) {
#pragma unroll 4
            for (int t = 0; t < R; ++t) step(t);
        } else {
#pragma unroll 1
            for (int t = 0; t < count; ++t) step(t);
        }
    }
    if (s.first_one && s.last_one) return;
    col.store_state(p, p.carry + slot * size, h);
    store_span(p.span + slot * p.channels);
    if constexpr (BACK) col.store_state(p, p.back + slot * size, back);
}

// the sum over the channels of a wave, for eight values: of lane l's four states n = 4 (l % Q) + k of b (v[0][k]) and of c (v[1][k]).  Returns
// two of them: lanes with l % 16 < Q hold those of states 4 q + 2 (row & 1) and the one behind, of b in rows 0 and 1 of 16 lanes, of c in rows 2 and 3
template <int Q>
__device__ __forceinline__ float2 over_channels(float (&v)[2][4])
{
    float u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[0][k]), __float_as_uint(v[1][k]), false, false);
        u[k] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    float w[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(u[k]), __float_as_uint(u[2 + k]), false, false);
        w[k] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        if constexpr (Q <= 8) w[k] += moved<0x128>(w[k]);       // rows turned by 8, 4, 2, 1
        if constexpr (Q <= 4) w[k] += moved<0x124>(w[k]);
        if constexpr (Q <= 2) w[k] += moved<0x122>(w[k]);
        if constexpr (Q <= 1) w[k] += moved<0x121>(w[k]);
    }
    return float2{w[0], w[1]};
}

// SOME: a wave may have fewer channels than there is room for.  What stands in their place takes no part in the sums over channels, not
// even as a product with zero: b and c may hold what is not finite.
template <typename T, int Q, bool SOME>
__global__ void __launch_bounds__(kThreads, 2) back_kernel(Args p)
{
    using S = Shape<Q>;
    constexpr int R = S::kRows, E = S::kEach, H = R < 8 ? R : 8, kParts = R / H;        // H: rows whose states are kept
    __shared__ __attribute__((aligned(16))) float s_in[kWaves][R][3][S::kChannels];
    __shared__ __attribute__((aligned(16))) float s_bc[kWaves][R][2][S::kStates];
    __shared__ __attribute__((aligned(16))) float s_part[kWaves][R][2][S::kStates];
    const int wave = threadIdx.x / 64, blocks = p.groups * p.group_blocks;
    const int64_t block = int64_t(p.first_block) + blockIdx.x;
    const int piece = int(block / blocks), group = int(block % blocks) / p.group_blocks, gb = int(block % blocks) % p.group_blocks;
    Column<T, Q> col;
    col.init(p, group, gb * p.waves + wave);
    const int64_t size = int64_t(p.channels) * p.states;
    auto& in = s_in[wave];
    auto& bc = s_bc[wave];
    float da[4][4], dd[S::kOwn], dbias[S::kOwn];
#pragma unroll
    for (int ch = 0; ch < 4; ++ch)
#pragma unroll
        for (int k = 0; k < 4; ++k) da[ch][k] = 0.0f;
#pragma unroll
    for (int i = 0; i < S::kOwn; ++i) dd[i] = dbias[i] = 0.0f;
    for (int64_t slot = piece; slot < p.slots; slot += p.pieces) {
        const Segment s = segment_of(p, slot);
        if (!s.there) continue;
        const bool alone = s.first_one && s.last_one;
        const float* const behind = alone ? (p.grad_end ? p.grad_end + s.seq * size : nullptr) : p.back + slot * size;
        const float* const before = alone ? (p.begin ? p.begin + s.seq * size : nullptr) : p.carry + slot * size;
        const int64_t tile0 = tile_of(slot, s, R);
        float back[4][4];
        col.load_state(p, behind, back);
        const int64_t tiles = (s.past - s.first + R - 1) / R;
        for (int64_t tile = tiles - 1; tile >= 0; --tile) {
            const int64_t t0 = s.first + tile * R;
            const int count = s.past - t0 < R ? int(s.past - t0) : R;
            {
                T x[E], delta[E], z[E], g[E];
                Pack<T, 4> shared[S::kPacksEach];
                col.load(p.x, p.x_step, t0, s.past, x);
                col.load(p.delta, p.delta_step, t0, s.past, delta);
                col.load(p.grad, p.grad_step, t0, s.past, g);
                if (p.z) col.load(p.z, p.z_step, t0, s.past, z);
                col.load_shared(p, t0, s.past, shared);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const int r = S::row(i, col.lane), ch = S::channel(i, col.lane);
                    const bool there = ch < col.count;
                    const float raw = float(delta[i]) + col.bias[S::own(i)], dt = p.softplus ? softplus_of(raw) : raw;
                    in[r][0][ch] = there ? dt : 0.0f;
                    in[r][1][ch] = there ? dt * float(x[i]) : 0.0f;
                    in[r][2][ch] = there ? (p.z ? float(g[i]) * (float(z[i]) * sigmoid(float(z[i]))) : float(g[i])) : 0.0f;
                }
                col.put_shared(shared, bc);
            }
            float h[4][4], y[4], dt[4], du[4], gy[4], b[4], c[4];
            auto forward = [&](int t) __attribute__((always_inline)) {
                read4(&in[t][0][col.at], dt);
                read4(&in[t][1][col.at], du);
                read4(&bc[t][0][4 * col.q], b);
#pragma unroll
                for (int ch = 0; ch < 4; ++ch)
#pragma unroll
                    for (int k = 0; k < 4; ++k) h[ch][k] = fmaf(h[ch][k], __builtin_amdgcn_exp2f(dt[ch] * col.a[ch][k]), du[ch] * b[k]);
            };
#pragma unroll 1
            for (int part = (count - 1) / H; part >= 0; --part) {
                // the state before the tile
                col.load_state(p, before, h);
                if (tile > 0) {
                    float own[4][4], span[4];
                    col.load_state(p, p.tile_state + (tile0 + tile) * size, own);
#pragma unroll
                    for (int ch = 0; ch < 4; ++ch) {
                        span[ch] = col.at + ch < col.count ? p.tile_span[(tile0 + tile) * p.channels + col.first + col.at + ch] : 0.0f;
#pragma unroll
                        for (int k = 0; k < 4; ++k) h[ch][k] = fmaf(h[ch][k], __builtin_amdgcn_exp2f(span[ch] * col.a[ch][k]), own[ch][k]);
                    }
                }
#pragma unroll 1
                for (int t = 0; t < part * H; ++t) forward(t);
                float start[4][4], kept_h[H][4][4];
#pragma unroll
                for (int ch = 0; ch < 4; ++ch)
#pragma unroll
                    for (int k = 0; k < 4; ++k) start[ch][k] = h[ch][k];
#pragma unroll
                for (int j = 0; j < H; ++j)
                    if (part * H + j < count) {
                        forward(part * H + j);
#pragma unroll
                        for (int ch = 0; ch < 4; ++ch)
#pragma unroll
                            for (int k = 0; k < 4; ++k) kept_h[j][ch][k] = h[ch][k];
                    }
#pragma unroll
                for (int j = H - 1; j >= 0; --j) {
                    const int t = part * H + j;
                    if (t >= count) continue;
                    read4(&in[t][0][col.at], dt);
                    read4(&in[t][1][col.at], du);
                    read4(&in[t][2][col.at], gy);
                    read4(&bc[t][0][4 * col.q], b);
                    read4(&bc[t][1][4 * col.q], c);
                    float sums[2][4], through[4], rate[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) sums[0][k] = sums[1][k] = 0.0f;
#pragma unroll
                    for (int ch = 0; ch < 4; ++ch) {
                        through[ch] = rate[ch] = y[ch] = 0.0f;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float now = fmaf(gy[ch], c[k], back[ch][k]);
                            const bool there = !SOME || col.at + ch < col.count;
                            sums[0][k] = fmaf(du[ch], there ? now : 0.0f, sums[0][k]);
                            sums[1][k] = fmaf(gy[ch], there ? kept_h[j][ch][k] : 0.0f, sums[1][k]);
                            y[ch] = fmaf(c[k], kept_h[j][ch][k], y[ch]);
                            through[ch] = fmaf(now, b[k], through[ch]);
                            back[ch][k] = now * __builtin_amdgcn_exp2f(dt[ch] * col.a[ch][k]);
                            const float r = back[ch][k] * (j ? kept_h[j ? j - 1 : 0][ch][k] : start[ch][k]);
                            rate[ch] = fmaf(r, col.a[ch][k], rate[ch]);
                            da[ch][k] = fmaf(r, dt[ch], da[ch][k]);
                        }
                        through[ch] = over_states<Q>(through[ch]);
                        rate[ch] = over_states<Q>(rate[ch]);
                        if (p.z) y[ch] = over_states<Q>(y[ch]);
                    }
                    *reinterpret_cast<float4*>(&in[t][0][col.at]) = float4{through[0], through[1], through[2], through[3]};
                    *reinterpret_cast<float4*>(&in[t][1][col.at]) = float4{rate[0], rate[1], rate[2], rate[3]};
                    if (p.z) *reinterpret_cast<float4*>(&in[t][2][col.at]) = float4{y[0], y[1], y[2], y[3]};
                    const float2 two = over_channels<Q>(sums);
                    const int row = col.lane / 16, q = col.lane % 16;
                    if (q < Q) *reinterpret_cast<float2*>(&s_part[wave][t][row / 2][4 * q + 2 * (row & 1)]) = two;
                }
            }
            // the channels' gradients of these rows
            {
                T x[E], delta[E], z[E], g[E];
                col.load(p.x, p.x_step, t0, s.past, x);
                col.load(p.delta, p.delta_step, t0, s.past, delta);
                col.load(p.grad, p.grad_step, t0, s.past, g);
                if (p.z) col.load(p.z, p.z_step, t0, s.past, z);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const int r = S::row(i, col.lane), ch = S::channel(i, col.lane), o = S::own(i);
                    if (r >= count || ch >= col.count) continue;
                    const float raw = float(delta[i]) + col.bias[o], dt = p.softplus ? softplus_of(raw) : raw, xv = float(x[i]), gv = float(g[i]);
                    const float through = in[r][0][ch], ddt = fmaf(in[r][1][ch], kLn2, through * xv), ddelta = p.softplus ? ddt * sigmoid(raw) : ddt;
                    const int64_t at = (t0 + r) * p.channels + col.first + ch;
                    float gy = gv;
                    if (p.z) {
                        const float zv = float(z[i]);
                        gy = gv * (zv * sigmoid(zv));
                        static_cast<T*>(p.dz)[at] = T(gv * fmaf(col.d[o], xv, in[r][2][ch]) * slope(zv));
                    }
                    static_cast<T*>(p.out)[at] = T(fmaf(through, dt, col.d[o] * gy));
                    static_cast<T*>(p.ddelta)[at] = T(ddelta);
                    dd[o] = fmaf(gy, xv, dd[o]);
                    dbias[o] += ddelta;
                }
            }
            // the block's sums over channels
            __syncthreads();
            float* const to = p.shared_parts + ((gb * p.rows + t0) * p.groups + group) * 2 * S::kStates;
            for (int e = threadIdx.x; e < count * 2 * S::kStates; e += blockDim.x) {
                const int t = e / (2 * S::kStates), n = e % (2 * S::kStates);
                float sum = 0.0f;
                for (int w = 0; w < p.waves; ++w) sum += (&s_part[w][t][0][0])[n];
                to[int64_t(t) * p.groups * 2 * S::kStates + n] = sum;
            }
            __syncthreads();
        }
        if (s.first_one && p.end) col.store_state(p, p.end + s.seq * size, back);
    }
    // the piece's sums over rows
    const int each = p.states + 2;
    float* const own = p.own_parts + int64_t(piece) * p.channels * each;
#pragma unroll
    for (int ch = 0; ch < 4; ++ch)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (col.at + ch < col.count && 4 * col.q + k < p.states) own[int64_t(col.first + col.at + ch) * each + 4 * col.q + k] = da[ch][k];
    // lanes with the same channels add up
#pragma unroll
    for (int i = 0; i < S::kOwn; ++i) {
        if constexpr (S::kChannels < 64)
#pragma unroll
            for (int m = S::kChannels; m < 64; m *= 2) dd[i] += __shfl_xor(dd[i], m), dbias[i] += __shfl_xor(dbias[i], m);
        const int ch = S::kChannels < 64 ? col.lane % S::kChannels : i * 64 + col.lane;
        if (ch < col.count && col.lane < S::kChannels) {
            own[int64_t(col.first + ch) * each + p.states] = dd[i];
            own[int64_t(col.first + ch) * each + p.states + 1] = dbias[i];
        }
    }
}

// the gradients of b and c: a thread to a value, over the blocks of its group
template <typename T>
__global__ void __launch_bounds__(kThreads) shared_kernel(Args p, int wide, T* db, T* dc)
{
    const int64_t e = (int64_t(p.first_block) + blockIdx.x) * kThreads + threadIdx.x, all = p.rows * p.groups * 2 * p.states;
    if (e >= all) return;
    const int64_t pair = e / (2 * p.states);            // row and group
    const int n = int(e - pair * 2 * p.states), dir = n / p.states, state = n % p.states;
    if (p.offsets) {
        const int64_t row = pair / p.groups, first = kept(p.offsets[0], 0, p.rows);
        if (row < first || row >= kept(p.offsets[p.n], first, p.rows)) return;
    }
    float sum = 0.0f;
    for (int g = 0; g < p.group_blocks; ++g) sum += p.shared_parts[((g * p.rows * p.groups + pair) * 2 + dir) * wide + state];
    (dir ? dc : db)[pair * p.states + state] = T(sum);
}

// those of a, d and bias: a thread to a value, over the pieces of the slots
__global__ void __launch_bounds__(kThreads) own_kernel(Args p, float* da, float* dd, float* dbias)
{
    const int each = p.states + 2;
    const int64_t e = int64_t(blockIdx.x) * kThreads + threadIdx.x, all = int64_t(p.channels) * each;
    if (e >= all) return;
    float sum = 0.0f;
    for (int n = 0; n < p.pieces; ++n) sum += p.own_parts[n * all + e];
    const int64_t ch = e / each;
    const int i = int(e - ch * each);
    if (i < p.states) da[ch * p.states + i] = sum;
    else if (i == p.states && dd) dd[ch] = sum;
    else if (i > p.states && dbias) dbias[ch] = sum;
}

uint64_t up(uint64_t bytes) { return (bytes + 255) / 256 * 256; }

struct Layout {
    Plan plan;
    int waves, group_blocks, pieces;
    uint64_t carry, back, span, tile_state, tile_span, shared_parts, own_parts, all;       // where they begin
};

Layout layout_of(bool packed, int64_t rows, int64_t n, int64_t length, int channels, int states, int groups)
{
    Layout l;
    l.plan = plan_of(packed, rows, n, length, channels, states, groups, true);
    const Plan& p = l.plan;
    l.waves = kWaves;
    while (p.tiles % l.waves) --l.waves;
    l.group_blocks = p.tiles / l.waves;
    // a piece of the slots to a block: enough of them for some waves to every SIMD
    const int64_t columns = int64_t(groups) * p.tiles, most = std::max<int64_t>(4096 / columns, 1);
    l.pieces = int(std::min(p.slots, most));
    const uint64_t size = uint64_t(channels) * states * 4, line = uint64_t(channels) * 4, tiles = uint64_t(rows / tile_rows(p.q) + p.slots), several = p.several ? p.slots : 0;
    uint64_t at = 0;
    auto take = [&](uint64_t& where, uint64_t bytes) { where = at, at += up(bytes); };
    take(l.carry, several * size);
    take(l.back, several * size);
    take(l.span, several * line);
    take(l.tile_state, tiles * size);
    take(l.tile_span, tiles * line);
    take(l.shared_parts, uint64_t(l.group_blocks) * rows * groups * 2 * 4 * p.q * 4);
    take(l.own_parts, uint64_t(l.pieces) * channels * (states + 2) * 4);
    l.all = at;
    return l;
}

}  // namespace
}  // namespace selective
}  // namespace seqamd

using namespace seqamd;
using namespace seqamd::selective;

extern "C" {

__attribute__((visibility("default"))) uint64_t cusig_amd_selective_scan_backprop_workspace(bool packed, uint64_t sequences, uint64_t length, uint64_t rows,
                                                                                             uint64_t channels, uint64_t states, uint64_t groups) noexcept
{
    uint64_t bytes = 0;
    sigamd::guarded([&] {
        check_sizes(rows, sequences, channels, states, groups);
        if (channels) bytes = layout_of(packed, int64_t(rows), int64_t(sequences), int64_t(length), int(channels), int(states), int(groups)).all;
    });
    return bytes;
}

__attribute__((visibility("default"))) int cusig_amd_selective_scan_backprop(
    int dtype, const void* grad_y, const void* x, const void* delta, const float* a, const void* b, const void* c, const float* d, const void* z,
    const float* delta_bias, const float* grad_final, const float* initial_state, void* grad_x, void* grad_delta, float* grad_a, void* grad_b, void* grad_c,
    float* grad_d, void* grad_z, float* grad_delta_bias, float* grad_initial, const int* offsets, uint64_t sequences, uint64_t length, uint64_t rows,
    uint64_t channels, uint64_t states, uint64_t groups, int64_t grad_stride, int64_t x_stride, int64_t delta_stride, int64_t z_stride, int64_t b_stride,
    int64_t b_group, int64_t c_stride, int64_t c_group, bool softplus, void* workspace, uint64_t workspace_bytes, void* stream) noexcept
{
    return sigamd::guarded([&] {
        check_sizes(rows, sequences, channels, states, groups);
        require(offsets || sequences * length == rows, "rows are not sequences times length");
        const auto s = static_cast<hipStream_t>(stream);
        Args p{};
        p.x = x, p.delta = delta, p.a = a, p.b = b, p.c = c, p.d = d, p.z = z, p.bias = delta_bias, p.grad = grad_y;
        p.begin = initial_state, p.grad_end = grad_final, p.end = grad_initial, p.out = grad_x, p.ddelta = grad_delta, p.dz = grad_z;
        p.offsets = offsets, p.n = int64_t(sequences), p.length = int64_t(length), p.rows = int64_t(rows);
        p.channels = int(channels), p.states = int(states), p.groups = int(groups), p.per_group = int(channels / groups);
        p.x_step = x_stride, p.delta_step = delta_stride, p.z_step = z_stride, p.grad_step = grad_stride;
        p.b_step = b_stride, p.b_group = b_group, p.c_step = c_stride, p.c_group = c_group;
        p.softplus = softplus;
        if (channels == 0) {
            require(rows == 0 || (grad_b && grad_c), "a tensor is missing");
            return;
        }
        require(a && grad_a && (sequences == 0 || grad_initial) && (!d || grad_d) && (!delta_bias || grad_delta_bias), "a tensor is missing");
        require(rows == 0 || (x && delta && b && c && grad_y && grad_x && grad_delta && grad_b && grad_c && (!z || grad_z)), "a tensor is missing");
        const Layout l = layout_of(offsets, p.rows, p.n, p.length, p.channels, p.states, p.groups);
        check_workspace(workspace, workspace_bytes, l.all);
        char* const w = static_cast<char*>(workspace);
        auto at = [&](uint64_t where) { return reinterpret_cast<float*>(w + where); };
        p.carry = at(l.carry), p.back = at(l.back), p.span = at(l.span), p.tile_state = at(l.tile_state), p.tile_span = at(l.tile_span);
        p.shared_parts = at(l.shared_parts), p.own_parts = at(l.own_parts);
        p.segment = l.plan.segment, p.slots = l.plan.slots, p.per_sequence = l.plan.per_sequence, p.several = l.plan.several, p.tiles = l.plan.tiles;
        p.waves = l.waves, p.group_blocks = l.group_blocks, p.pieces = l.pieces;
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            if (p.slots)
                with_lanes(l.plan.q, [&](auto q) {
                    constexpr int Q = decltype(q)::value;
                    const int64_t blocks = (p.slots * p.groups * p.tiles + kWaves - 1) / kWaves;
                    if (p.several) {
                        launch_all(states_kernel<T, Q, true>, blocks, kThreads, s, p);
                        join_segments(p, true, s);
                    } else {
                        launch_all(states_kernel<T, Q, false>, blocks, kThreads, s, p);
                    }
                    const int64_t work = int64_t(p.pieces) * p.groups * p.group_blocks;
                    if (p.per_group % Shape<Q>::kChannels) launch_all(back_kernel<T, Q, true>, work, 64 * p.waves, s, p);
                    else launch_all(back_kernel<T, Q, false>, work, 64 * p.waves, s, p);
                });
            if (p.rows)
                in_launches((p.rows * p.groups * 2 * p.states + kThreads - 1) / kThreads, kThreads, [&](unsigned first, dim3 grid) {
                    p.first_block = first;
                    hipLaunchKernelGGL(shared_kernel<T>, grid, dim3(kThreads), 0, s, p, 4 * l.plan.q, static_cast<T*>(grad_b), static_cast<T*>(grad_c));
                });
        });
        hipLaunchKernelGGL(own_kernel, dim3(unsigned((int64_t(p.channels) * (p.states + 2) + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, p, grad_a, grad_d, grad_delta_bias);
        SIG_HIP(hipGetLastError());
    });
}

}  // extern "C"
