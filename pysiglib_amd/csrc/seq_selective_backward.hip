// The selective scan's gradients.
//
// Mathematics.  Let gy_t be the gradient of the sum over states (that of y times the gate), k_t = exp(dt_t a), and G_t the gradient of h_t:
// G_t = gy_t c_t + k_{t+1} G_{t+1}, with that of the final state behind the last step.  Then for each channel (sums over states)
//   dx_t = dt_t sum G_t b_t + d gy_t,   d(dt_t) = sum (G_t k_t h_{t-1} a) + x_t sum G_t b_t,   dz_t = g_t y_t slope(z_t),
// for each state da = sum over rows of G_t k_t h_{t-1} dt_t, and for each row of a group (sums over its channels) db_t = sum G_t dt_t x_t,
// dc_t = sum gy_t h_t.  k_0 G_0 is the gradient of the initial state.  Nothing is taken from the forward pass: the states are formed again.
//
// Passes.  First every segment forward, the first of a sequence from its initial state, others from zero: the state before every eighth
// row, its own last state, and (where a sequence has several) the gradient of the state before it that its own rows make, as sum over t of
// (k_first ... k_t) gy_t c_t, so one exponential serves both.  Segments are joined; then each goes from its last rows to its
// first: the state before eight rows is the stored one plus exp(a sum dt) times the segment's; four rows' states are formed and kept in
// registers, and these rows gone back through.
// Sums over channels stay in a row's 64 lanes, then the block's waves, then the blocks, all in a fixed order.
//
// Bound: vector instructions, some twenty for each state and row.  Measured, 4 sequences of 2048 steps, 2048 channels of 16 states, bfloat16 (2.7e8 steps of states): states
// 111 us, joining 12, back 328, sums over blocks and pieces 7 and 8, each kernel by itself under a profiler.  Vector instructions take 61 % of back's cycles: two waves to a
// SIMD, which is what the kept states leave registers for, do not cover all of each other's waits, and their 256 registers do not hold everything that lives through a
// tile.  back_kernel keeps 56 (bfloat16, 64 states) to 192 registers (float32, up to four) in memory, 228 to 764 bytes to a lane, 444 in the case above; its
// loop over rows is free of that, but each tile of 16 rows stores some 20 words a lane there and loads 40, and the kernel writes 251 MB where its results and the partial
// sums are 119.  states_kernel<float> with the gradients' part keeps 3 to 51 with up to 32 states.
#include "seq_selective.h"

#include <algorithm>
#include <type_traits>

namespace seqamd {
namespace selective {
namespace {

// Every segment's own states; BACK: its own part of the gradients too
template <typename T, int Q, bool BACK>
__global__ void __launch_bounds__(kThreads, 2) states_kernel(Args p)
{
    using S = Shape<Q>;
    constexpr int R = S::kRows, E = S::kEach, G = S::kGroups, kSets = S::kSets, kSaved = S::kSaved;
    __shared__ __attribute__((aligned(16))) float s_in[kWaves][R][BACK ? 3 : 2][S::kChannels];
    __shared__ __attribute__((aligned(16))) float s_bc[kWaves][R][2][S::kStates];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), columns = p.groups * p.tiles;
    const int64_t id = (int64_t(p.first_block) + blockIdx.x) * kWaves + wave, slot = id / columns;
    if (slot >= p.slots) return;
    const Segment s = segment_of(p, slot);
    if (!s.there || s.first >= s.past) return;
    Column<T, Q> col;
    col.init(p, int(id % columns) / p.tiles, int(id % columns) % p.tiles);
    const int64_t size = int64_t(p.channels) * p.states;
    int64_t tile = tile_of(slot, s, kSaved);
    Four h[4], decay[4], back[4], span[kSets];
    col.load_state(p, s.first_one && p.begin ? p.begin + s.seq * size : nullptr, h);
#pragma unroll
    for (int u = 0; u < 4; ++u) back[u] = Four{}, decay[u] = Four{1.0f, 1.0f, 1.0f, 1.0f};
#pragma unroll
    for (int i = 0; i < kSets; ++i) span[i] = Four{};
    auto& in = s_in[wave];
    auto& bc = s_bc[wave];
    Pack<T, 2> x[E], delta[E], z[E], g[E];
    Pack<T, 4> shared[S::kPacksEach];
    auto fetch = [&](int64_t t0) __attribute__((always_inline)) {
        const int rows = s.past - t0 < R ? int(s.past - t0) : R;
        col.load(p.x, p.x_step, t0, rows, x);
        col.load(p.delta, p.delta_step, t0, rows, delta);
        if (BACK && p.z) col.load(p.z, p.z_step, t0, rows, z);
        if (BACK) col.load(p.grad, p.grad_step, t0, rows, g);
        col.load_shared(p, t0, rows, shared);
    };
    fetch(s.first);
    for (int64_t t0 = s.first; t0 < s.past; t0 += R) {
        const int rows = s.past - t0 < R ? int(s.past - t0) : R;
        {
            float v[E][2];
            col.steps(p, delta, v);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                auto& row = in[S::row(i, col.lane)];
                col.put(row[0], i, v[i][0], v[i][1]);
                col.put(row[1], i, v[i][0] * x[i].get(0), v[i][1] * x[i].get(1));
            }
            if constexpr (BACK) {
#pragma unroll
                for (int i = 0; i < E; ++i) v[i][0] = g[i].get(0), v[i][1] = g[i].get(1);
                if (p.z) col.gate(z, v);
#pragma unroll
                for (int i = 0; i < E; ++i) col.put(in[S::row(i, col.lane)][2], i, v[i][0], v[i][1]);
            }
        }
        col.put_shared(p, shared, bc);
        wave_sync();
        if (t0 + R < s.past) fetch(t0 + R);
        auto step = [&](int t) __attribute__((always_inline)) {
            float b[G], c[G];
            col.read_shared(bc[t][0], b);
            if constexpr (BACK) col.read_shared(bc[t][1], c);
#pragma unroll
            for (int i = 0; i < kSets; ++i) {
                const Four dt = *reinterpret_cast<const Four*>(&in[t][0][col.at + 4 * i]);
                const float du = in[t][1][col.at + 4 * i + col.j];
                Four gy{};
                if constexpr (BACK) gy = *reinterpret_cast<const Four*>(&in[t][2][col.at + 4 * i]);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const int u = i * G + g;
                    const Four e = decays(dt, col.a[u]);
                    h[u] = add_products(du, b[g], h[u] * e);
                    if constexpr (BACK) {
                        decay[u] *= e;
#pragma unroll
                        for (int k = 0; k < 4; ++k) back[u][k] = fmaf(decay[u][k], gy[k] * c[g], back[u][k]);
                    }
                }
                span[i] += dt;
            }
        };
#pragma unroll 1
        for (int t = 0; t < rows; t += kSaved, ++tile) {
            col.store_own(p, p.tile_state, tile, h);
            if (!s.first_one) col.store_line(p.tile_span + tile * p.channels, span);
            if (t + kSaved <= rows) {
#pragma unroll 4
                for (int k = 0; k < kSaved; ++k) step(t + k);
            } else {
#pragma unroll 1
                for (int k = t; k < rows; ++k) step(k);
            }
        }
        wave_sync();
    }
    if (s.first_one && s.last_one) return;
    col.store_own(p, p.carry, slot, h);
    col.store_line(p.span + slot * p.channels, span);
    if constexpr (BACK) {
        if (s.last_one && p.grad_end) {
            Four end[4];
            col.load_state(p, p.grad_end + s.seq * size, end);
            col.template over_copies<false>(p, end);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) back[u][k] = fmaf(decay[u][k], end[u][k], back[u][k]);
        }
        col.store_own(p, p.back, slot, back);
    }
}

// The sum over the channels of a wave of the lane's sums for b (v[0]) and c (v[1]).  Groups beside each other go to lanes with the lane's
// place in its quads: lanes 0 to 31 hold b's, 32 to 63 c's; with four groups rows of 16 lanes hold two each, with two one each.
template <int Q>
__device__ __forceinline__ float2 over_channels(const float (&v)[2][Shape<Q>::kGroups])
{
    constexpr int G = Shape<Q>::kGroups;
    float u[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[0][g]), __float_as_uint(v[1][g]), false, false);
        u[g] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    float w[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < (G == 4 ? 2 : 1); ++k) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(u[k]), __float_as_uint(u[G == 1 ? 0 : G / 2 + k]), false, false);
        w[k] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        if constexpr (Q <= 8) w[k] += moved<0x128>(w[k]);       // rows turned by 8 and 4
        if constexpr (Q <= 4) w[k] += moved<0x124>(w[k]);
    }
    return float2{w[0], w[1]};
}

// W waves to a block.  SOME: a wave may have fewer channels than there is room for.  What stands in their place is no
// number in particular, and takes no part in the sums over channels.  (Full waves without the selections: 16 sequences of 1000, 256 channels of 4, float32,
// forward and gradients 213 us, with them 234; 64 of 300, 256 of 8, float16, 180 and 194.)
template <typename T, int Q, int W, bool SOME>
__global__ void __launch_bounds__(64 * W, 2) back_kernel(Args p)
{
    using S = Shape<Q>;
    constexpr int R = S::kRows, E = S::kEach, G = S::kGroups, kSets = S::kSets, kSaved = S::kSaved, H = 4;      // H: rows whose states are kept
    __shared__ __attribute__((aligned(16))) float s_in[W][R][4][S::kChannels];
    __shared__ __attribute__((aligned(16))) float s_bc[W][R][2][S::kStates];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), blocks = p.groups * p.group_blocks;
    const int64_t block = int64_t(p.first_block) + blockIdx.x;
    const int piece = int(block / blocks), group = int(block % blocks) / p.group_blocks, gb = int(block % blocks) % p.group_blocks;
    Column<T, Q> col;
    col.init(p, group, gb * W + wave);
    const int64_t size = int64_t(p.channels) * p.states;
    auto& in = s_in[wave];
    auto& bc = s_bc[wave];
    Four da[4];
    float dd[S::kOwn][2], dbias[S::kOwn][2];
#pragma unroll
    for (int u = 0; u < 4; ++u) da[u] = Four{};
#pragma unroll
    for (int i = 0; i < S::kOwn; ++i) dd[i][0] = dd[i][1] = dbias[i][0] = dbias[i][1] = 0.0f;
    for (int64_t slot = piece; slot < p.slots; slot += p.pieces) {
        const Segment s = segment_of(p, slot);
        if (!s.there) continue;
        Four back[4];
        if (s.last_one) {
            col.load_state(p, p.grad_end ? p.grad_end + s.seq * size : nullptr, back);
            col.template over_copies<false>(p, back);
        } else {
            col.load_own(p, p.back, slot, back);
        }
        const int64_t tile0 = tile_of(slot, s, kSaved), tiles = (s.past - s.first + R - 1) / R;
        for (int64_t tile = tiles - 1; tile >= 0; --tile) {
            const int64_t t0 = s.first + tile * R;
            const int rows = s.past - t0 < R ? int(s.past - t0) : R;
            {
                Pack<T, 2> x[E], delta[E], z[E], g[E];
                Pack<T, 4> shared[S::kPacksEach];
                col.load(p.x, p.x_step, t0, rows, x);
                col.load(p.delta, p.delta_step, t0, rows, delta);
                col.load(p.grad, p.grad_step, t0, rows, g);
                if (p.z) col.load(p.z, p.z_step, t0, rows, z);
                col.load_shared(p, t0, rows, shared);
                float v[E][2];
                col.steps(p, delta, v);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    auto& row = in[S::row(i, col.lane)];
                    col.put(row[0], i, v[i][0], v[i][1]);
                    col.put(row[1], i, v[i][0] * x[i].get(0), v[i][1] * x[i].get(1));
                    col.put(row[3], i, v[i][0], v[i][1]);       // again: the first three are overwritten
                    v[i][0] = g[i].get(0), v[i][1] = g[i].get(1);
                }
                if (p.z) col.gate(z, v);
#pragma unroll
                for (int i = 0; i < E; ++i) col.put(in[S::row(i, col.lane)][2], i, v[i][0], v[i][1]);
                col.put_shared(p, shared, bc);
                wave_sync();
            }
            auto forward = [&](int t, Four (&h)[4]) __attribute__((always_inline)) {
                float b[G];
                col.read_shared(bc[t][0], b);
#pragma unroll
                for (int i = 0; i < kSets; ++i) {
                    const Four dt = *reinterpret_cast<const Four*>(&in[t][0][col.at + 4 * i]);
                    const float du = in[t][1][col.at + 4 * i + col.j];
#pragma unroll
                    for (int g = 0; g < G; ++g) h[i * G + g] = add_products(du, b[g], h[i * G + g] * decays(dt, col.a[i * G + g]));
                }
            };
            // back through up to four rows from `low` on, from the state before them
            auto reverse = [&](int low, const Four (&start)[4]) __attribute__((always_inline)) {
                Four kept_h[H][4];
#pragma unroll
                for (int k = 0; k < H; ++k)
                    if (low + k < rows) {
#pragma unroll
                        for (int u = 0; u < 4; ++u) kept_h[k][u] = k ? kept_h[k ? k - 1 : 0][u] : start[u];
                        forward(low + k, kept_h[k]);
                    }
#pragma unroll
                for (int k = H - 1; k >= 0; --k) {
                    const int t = low + k;
                    if (t >= rows) continue;
                    float b[G], c[G], sums[2][G];
                    col.read_shared(bc[t][0], b);
                    col.read_shared(bc[t][1], c);
#pragma unroll
                    for (int g = 0; g < G; ++g) sums[0][g] = sums[1][g] = 0.0f;
#pragma unroll
                    for (int i = 0; i < kSets; ++i) {
                        const int at = col.at + 4 * i;
                        const Four dt = *reinterpret_cast<const Four*>(&in[t][0][at]), du = *reinterpret_cast<const Four*>(&in[t][1][at]),
                                   gy = *reinterpret_cast<const Four*>(&in[t][2][at]);
                        const float gy_own = in[t][2][at + col.j];
                        Four through{}, rate{}, y{};
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            const int u = i * G + g;
                            const Four now = add_products(gy_own, c[g], back[u]), e = decays(dt, col.a[u]);
#pragma unroll
                            for (int n = 0; n < 4; ++n) {
                                const bool there = !SOME || at + n < col.count;
                                const float h = kept_h[k][u][n];
                                sums[0][g] = there ? fmaf(du[n], now[n], sums[0][g]) : sums[0][g];
                                sums[1][g] = there ? fmaf(gy[n], h, sums[1][g]) : sums[1][g];
                                y[n] = fmaf(c[g], h, y[n]);
                                through[n] = fmaf(now[n], b[g], through[n]);
                                back[u][n] = now[n] * e[n];
                                const float r = back[u][n] * (k ? kept_h[k ? k - 1 : 0][u][n] : start[u][n]);
                                rate[n] = fmaf(r, col.a[u][n], rate[n]);
                                da[u][n] = fmaf(r, dt[n], da[u][n]);
                            }
                        }
#pragma unroll
                        for (int n = 0; n < 4; ++n) through[n] = over_states<Q>(through[n]), rate[n] = over_states<Q>(rate[n]);
                        *reinterpret_cast<Four*>(&in[t][0][at]) = through;
                        *reinterpret_cast<Four*>(&in[t][1][at]) = rate;
                        if (p.z) {
#pragma unroll
                            for (int n = 0; n < 4; ++n) y[n] = over_states<Q>(y[n]);
                            *reinterpret_cast<Four*>(&in[t][2][at]) = y;
                        }
                    }
                    const float2 two = over_channels<Q>(sums);
                    const int row = col.lane / 16, l = col.lane % 16;       // of 16 lanes
                    if (l < 4 * S::kQuads) {
                        float* const to = &bc[t][row / 2][l / 4 * 16 + l % 4 * G];          // in the place of b and c, which this row has read
                        if constexpr (G == 4) *reinterpret_cast<float2*>(to + 2 * (row & 1)) = two;
                        else if constexpr (G == 2) to[row & 1] = two.x;
                        else to[0] = two.x;
                    }
                }
            };
#pragma unroll 1
            for (int low = (rows - 1) / kSaved * kSaved; low >= 0; low -= kSaved) {
                // the state before these rows
                Four h[4];
                const int64_t at = tile0 + tile * (R / kSaved) + low / kSaved;
                col.load_own(p, p.tile_state, at, h);
                if (!s.first_one) {
                    Four before[4], span[kSets];
                    col.load_own(p, p.carry, slot, before);
                    col.load_line(p.tile_span + at * p.channels, span);
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const Four e = decays(span[u / G], col.a[u]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) h[u][k] = fmaf(before[u][k], e[k], h[u][k]);
                    }
                }
                // its two halves, the second one first, in the same code
#pragma unroll 1
                for (int part = kSaved > H && low + H < rows ? 1 : 0; part >= 0; --part) {
                    Four start[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) start[u] = h[u];
                    if (part)
#pragma unroll
                        for (int k = 0; k < H; ++k) forward(low + k, start);
                    reverse(low + part * H, start);
                }
            }
            wave_sync();
            // the channels' gradients of these rows
            {
                Pack<T, 2> x[E], delta[E], z[E], g[E];
                col.load(p.x, p.x_step, t0, rows, x);
                col.load(p.delta, p.delta_step, t0, rows, delta);
                col.load(p.grad, p.grad_step, t0, rows, g);
                if (p.z) col.load(p.z, p.z_step, t0, rows, z);
                float dt[E][2], gy[E][2], v[E][2];
#pragma unroll
                for (int i = 0; i < E; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const auto& row = in[S::row(i, col.lane)];
                        const int ch = col.channel_of(i) + k;
                        dt[i][k] = row[3][ch];
                        gy[i][k] = g[i].get(k);
                        v[i][k] = fmaf(row[1][ch], kLn2, row[0][ch] * x[i].get(k));
                    }
                if (p.softplus)         // its slope: e^(raw - softplus(raw)), 1 where both are infinite (fminf takes the number; a raw NaN is in v already)
#pragma unroll
                    for (int i = 0; i < E; ++i)
#pragma unroll
                        for (int k = 0; k < 2; ++k) v[i][k] *= __builtin_amdgcn_exp2f(fminf(delta[i].get(k) + col.bias[i % S::kOwn][k] - dt[i][k], 0.0f) * kLog2e);
                col.store(p.ddelta, p.channels, t0, rows, v);
#pragma unroll
                for (int i = 0; i < E; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) dbias[i % S::kOwn][k] = S::row(i, col.lane) < rows ? dbias[i % S::kOwn][k] + v[i][k] : dbias[i % S::kOwn][k];
                if (p.z) {
#pragma unroll
                    for (int i = 0; i < E; ++i)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float gate = z[i].get(k), w = sigmoid(gate), y = fmaf(col.d[i % S::kOwn][k], x[i].get(k), in[S::row(i, col.lane)][2][col.channel_of(i) + k]);
                            v[i][k] = gy[i][k] * y * (w * fmaf(gate, 1.0f - w, 1.0f));
                            gy[i][k] *= gate * w;
                        }
                    col.store(p.dz, p.channels, t0, rows, v);
                }
#pragma unroll
                for (int i = 0; i < E; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        v[i][k] = fmaf(in[S::row(i, col.lane)][0][col.channel_of(i) + k], dt[i][k], col.d[i % S::kOwn][k] * gy[i][k]);
                        dd[i % S::kOwn][k] = S::row(i, col.lane) < rows ? fmaf(gy[i][k], x[i].get(k), dd[i % S::kOwn][k]) : dd[i % S::kOwn][k];
                    }
                col.store(p.out, p.channels, t0, rows, v);
            }
            // the block's sums over channels
            __syncthreads();
            float* const to = p.shared_parts + ((gb * p.rows + t0) * p.groups + group) * 2 * S::kStates;
            for (int e = threadIdx.x; e < rows * 2 * S::kStates; e += 64 * W) {
                const int t = e / (2 * S::kStates), n = e % (2 * S::kStates);
                float sum = 0.0f;
                for (int w = 0; w < W; ++w) sum += (&s_bc[w][t][0][0])[n];
                to[int64_t(t) * p.groups * 2 * S::kStates + n] = sum;
            }
            __syncthreads();
        }
        if (s.first_one && p.end) {
            col.template over_copies<true>(p, back);
            col.store_state(p, p.end + s.seq * size, back);
        }
    }
    col.template over_copies<true>(p, da);
    // the piece's sums over rows
    const int each = p.states + 2;
    float* const own = p.own_parts + int64_t(piece) * p.channels * each;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col.channel(u) + i < col.count && col.state(u) < p.states) own[int64_t(col.first + col.channel(u) + i) * each + col.state(u)] = da[u][i];
    // lanes with the same channels add up
#pragma unroll
    for (int i = 0; i < S::kOwn; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int m = S::kChannels / 2; m < 64; m *= 2) dd[i][k] += __shfl_xor(dd[i][k], m), dbias[i][k] += __shfl_xor(dbias[i][k], m);
            if (col.counts(i, k) && col.lane < S::kChannels / 2) {
                own[int64_t(col.first + col.channel_of(i) + k) * each + p.states] = dd[i][k];
                own[int64_t(col.first + col.channel_of(i) + k) * each + p.states + 1] = dbias[i][k];
            }
        }
}

// the gradients of b and c: a thread to a value, over the blocks of its group
template <typename T, int Q>
__global__ void __launch_bounds__(kThreads) shared_kernel(Args p, T* db, T* dc)
{
    using S = Shape<Q>;
    const int64_t e = (int64_t(p.first_block) + blockIdx.x) * kThreads + threadIdx.x, all = p.rows * p.groups * 2 * p.states;
    if (e >= all) return;
    const int64_t pair = e / (2 * p.states);            // row and group
    const int n = int(e - pair * 2 * p.states), dir = n / p.states, state = n % p.states;
    if (p.offsets) {
        const int64_t row = pair / p.groups, first = kept(p.offsets[0], 0, p.rows);
        if (row < first || row >= kept(p.offsets[p.n], first, p.rows)) return;
    }
    float sum = 0.0f;
    for (int g = 0; g < p.group_blocks; ++g) sum += p.shared_parts[((g * p.rows * p.groups + pair) * 2 + dir) * S::kStates + S::place(state)];
    if (!dir) sum *= copies_of(state, p.states, S::kStates);
    (dir ? dc : db)[pair * p.states + state] = T(sum);
}

// those of a, d and bias, over the pieces of the slots
__global__ void __launch_bounds__(kSumThreads) own_kernel(Args p, float* da, float* dd, float* dbias)
{
    const int each = p.states + 2;
    sum_pieces(p.own_parts, p.pieces, int64_t(p.channels) * each, p.first_block, [&](int64_t e, float sum) {
        const int64_t ch = e / each;
        const int i = int(e - ch * each);
        if (i < p.states) da[ch * p.states + i] = sum;
        else if (i == p.states && dd) dd[ch] = sum;
        else if (i > p.states && dbias) dbias[ch] = sum;
    });
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
    l.waves = p.waves;
    l.group_blocks = p.tiles / l.waves;
    // a piece of the slots to a block: enough of them for some waves to every SIMD
    const int64_t columns = int64_t(groups) * p.tiles, most = std::max<int64_t>(4096 / columns, 1);
    l.pieces = int(std::min(p.slots, most));
    const uint64_t size = uint64_t(groups) * p.tiles * 4096, line = uint64_t(channels) * 4, several = p.several ? p.slots : 0;
    const uint64_t tiles = uint64_t(rows / std::min(tile_rows(p.q), 8) + p.slots);
    uint64_t at = 0;
    auto take = [&](uint64_t& where, uint64_t bytes) { where = at, at += up(bytes); };
    take(l.carry, several * size);
    take(l.back, several * size);
    take(l.span, several * line);
    take(l.tile_state, tiles * size);
    take(l.tile_span, p.several ? tiles * line : 0);
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
        if (!offsets) check_rows(sequences, length, rows);
        check_strides({x_stride, delta_stride, z_stride, grad_stride});
        const auto s = static_cast<hipStream_t>(stream);
        Args p{};
        p.x = x, p.delta = delta, p.a = a, p.b = b, p.c = c, p.d = d, p.z = z, p.bias = delta_bias, p.grad = grad_y;
        p.begin = initial_state, p.grad_end = grad_final, p.end = grad_initial, p.out = grad_x, p.ddelta = grad_delta, p.dz = grad_z;
        p.offsets = offsets, p.n = int64_t(sequences), p.length = int64_t(length), p.rows = int64_t(rows);
        p.channels = int(channels), p.states = int(states), p.groups = int(groups), p.per_group = int(channels / groups);
        p.x_step = x_stride, p.delta_step = delta_stride, p.z_step = z_stride, p.grad_step = grad_stride;
        p.b_step = b_stride, p.b_group = b_group, p.c_step = c_stride, p.c_group = c_group;
        p.softplus = softplus;
        auto shared = [&](auto t, auto q) {
            using T = decltype(t);
            in_launches((p.rows * p.groups * 2 * p.states + kThreads - 1) / kThreads, kThreads, [&](unsigned first, dim3 grid) {
                Args more = p;
                more.first_block = first;
                hipLaunchKernelGGL((shared_kernel<T, decltype(q)::value>), grid, dim3(kThreads), 0, s, more, static_cast<T*>(grad_b), static_cast<T*>(grad_c));
            });
        };
        if (channels == 0) {            // sums over nothing
            require(rows == 0 || (grad_b && grad_c), "a tensor is missing");
            with_type(dtype, [&](auto t) { shared(t, std::integral_constant<int, 1>{}); });
            return;
        }
        require(a && grad_a && (sequences == 0 || grad_initial) && (!d || grad_d) && (!delta_bias || grad_delta_bias), "a tensor is missing");
        require(rows == 0 || (x && delta && b && c && grad_y && grad_x && grad_delta && grad_b && grad_c && (!z || grad_z)), "a tensor is missing");
        const Layout l = layout_of(offsets, p.rows, p.n, p.length, p.channels, p.states, p.groups);
        check_workspace(workspace, workspace_bytes, l.all);
        char* const w = static_cast<char*>(workspace);
        auto at = [&](uint64_t where) { return reinterpret_cast<float*>(w + where); };
        auto state_at = [&](uint64_t where) { return reinterpret_cast<Four*>(w + where); };
        p.carry = state_at(l.carry), p.back = state_at(l.back), p.span = at(l.span), p.tile_state = state_at(l.tile_state), p.tile_span = at(l.tile_span);
        p.shared_parts = at(l.shared_parts), p.own_parts = at(l.own_parts);
        p.segment = l.plan.segment, p.slots = l.plan.slots, p.per_sequence = l.plan.per_sequence, p.tiles = l.plan.tiles;
        p.group_blocks = l.group_blocks, p.pieces = l.pieces;
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            with_lanes(l.plan.q, [&](auto q) {
                constexpr int Q = decltype(q)::value;
                if (p.slots) {
                    const int64_t blocks = (p.slots * p.groups * p.tiles + kWaves - 1) / kWaves;
                    if (l.plan.several) {
                        launch_all(states_kernel<T, Q, true>, blocks, kThreads, s, p);
                        join_segments(p, true, s);
                    } else {
                        launch_all(states_kernel<T, Q, false>, blocks, kThreads, s, p);
                    }
                    const int64_t work = int64_t(p.pieces) * p.groups * p.group_blocks;
                    if (l.waves == kWaves) launch_all(back_kernel<T, Q, kWaves, false>, work, kThreads, s, p);
                    else if (p.per_group % Shape<Q>::kChannels) launch_all(back_kernel<T, Q, 1, true>, work, 64, s, p);
                    else launch_all(back_kernel<T, Q, 1, false>, work, 64, s, p);
                }
                shared(t, q);
            });
        });
        in_launches(sum_blocks(int64_t(p.channels) * (p.states + 2)), kSumThreads, [&](unsigned first, dim3 grid) {
            Args more = p;
            more.first_block = first;
            hipLaunchKernelGGL(own_kernel, grid, dim3(kSumThreads), 0, s, more, grad_a, grad_d, grad_delta_bias);
        });
    });
}

}  // extern "C"
