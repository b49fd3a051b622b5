// Root-mean-square norms of queries and keys for each head, and the rotation of channel pairs by the position, in one pass;
// and the gradients of both.
//
// Mathematics.  r = (mean x^2 + eps)^-1/2, y = R(position) (w . x r): the pairs (i, i + half) or (2 i, 2 i + 1) of the first
// `rotary` channels turn by the tables' angle, the others stay.  Backward, with g' = R^T g and u = w . g':
// dx = r (u - x r^2 mean(u . x)), dw = sum over tokens and heads of g' . x r.
//
// Bound: HBM.  A head belongs to a few lanes, each with whole pairs, so the only exchange between lanes is the sum of a row;
// a wave takes heads of one token, whose table rows it keeps in registers.  Everything between load and store is 32-bit.
// 16384 tokens, 40 heads of 128, bfloat16: 63 us, 5.3 TB/s; a call of few tokens is bound by the launch and the host (12 us).
// The sums of dw go by fixed pieces of the tokens, added up in a fixed order: the same inputs give the same bits.
#include "seq_common.h"

namespace seqamd {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kPieces = 1024;     // of the tokens at most, for the gradients of the weights

struct RotaryArgs {
    const void *q, *k;            // [tokens][heads][dim], rows of a head contiguous
    const void *gq, *gk;          // gradients of the outputs
    const float *qw, *kw, *cos, *sin;
    const int* positions;
    void *oq, *ok;                // outputs, or the gradients of q and k
    float* parts;                 // [pieces][2][dim]
    int64_t tokens, q_token, q_head, k_token, k_head, gq_token, gq_head, gk_token, gk_head, table;
    int heads, kv_heads, dim, rotary, split;
    float eps;
    bool past;                    // results go past the caches
    unsigned first_block;         // of a launch
};

// The U pairs of a lane: elements a[i] and b[i] are turned against each other (or stay, past the rotary part).
// `first` and `second`: where they are in the row; step 2 where neighbours are the pairs.
struct Place {
    int first, second, pairs;     // pairs: how many are there
    bool turns;
};

template <int U, bool NEAR>
__device__ __forceinline__ Place place_of(int unit, int dim, int rotary)
{
    const int half = rotary / 2, units = (half + U - 1) / U;
    Place p;
    if (unit < units) {
        const int at = unit * U;
        p.turns = true;
        p.pairs = half - at < U ? half - at : U;
        p.first = NEAR ? 2 * at : at;
        p.second = NEAR ? 2 * at + 1 : at + half;
        return p;
    }
    // the channels behind the rotary part, in runs of 2 U: the first U of a run against the others
    const int at = rotary + (unit - units) * 2 * U, left = dim - at;
    p.turns = false;
    p.first = at;
    if (NEAR) {
        p.second = at + 1;
        p.pairs = left <= 0 ? 0 : (left >= 2 * U ? U : left / 2);
    } else {
        const int n = left <= 0 ? 0 : (left >= 2 * U ? U : left / 2);
        p.second = at + n;
        p.pairs = n;
    }
    return p;
}

template <typename T, int U, bool NEAR>
__device__ __forceinline__ void load_pairs(const T* row, const Place& p, float* a, float* b)
{
    if constexpr (NEAR) {
        const Pack<T, 2 * U> x = load_some<T, 2 * U>(row + p.first, 2 * p.pairs);
#pragma unroll
        for (int i = 0; i < U; ++i) a[i] = x.get(2 * i), b[i] = x.get(2 * i + 1);
    } else {
        const Pack<T, U> x = load_some<T, U>(row + p.first, p.pairs), y = load_some<T, U>(row + p.second, p.pairs);
#pragma unroll
        for (int i = 0; i < U; ++i) a[i] = x.get(i), b[i] = y.get(i);
    }
}

template <typename T, int U, bool NEAR>
__device__ __forceinline__ void store_pairs(T* row, const Place& p, bool past, const float* a, const float* b)
{
    if constexpr (NEAR) {
        float x[2 * U];
#pragma unroll
        for (int i = 0; i < U; ++i) x[2 * i] = a[i], x[2 * i + 1] = b[i];
        Pack<T, 2 * U> o;
        o.set(x);
        if (past && p.pairs == U) store_past<T, 2 * U>(row + p.first, o);
        else store_some<T, 2 * U>(row + p.first, o, 2 * p.pairs);
    } else {
        Pack<T, U> x, y;
        x.set(a);
        y.set(b);
        if (past && p.pairs == U) {
            store_past<T, U>(row + p.first, x);
            store_past<T, U>(row + p.second, y);
        } else {
            store_some<T, U>(row + p.first, x, p.pairs);
            store_some<T, U>(row + p.second, y, p.pairs);
        }
    }
}

// the sum over the G lanes of a head
template <int G>
__device__ __forceinline__ float sum_of(float x)
{
#pragma unroll
    for (int m = 1; m < G; m *= 2) x += __shfl_xor(x, m);
    return x;
}

// A token's row of the tables; positions outside them give NaN
template <int U>
__device__ __forceinline__ void load_angle(const RotaryArgs& p, int64_t token, int unit, const Place& at, float* c, float* s)
{
    const int64_t pos = p.positions[token];
    const bool inside = pos >= 0 && pos < p.table;
    const int half = p.rotary / 2;
#pragma unroll
    for (int i = 0; i < U; ++i) c[i] = at.turns && inside ? 1.0f : (inside ? 1.0f : __builtin_nanf("")), s[i] = 0.0f;
    if (at.turns && inside) {
        const Pack<float, U> x = load_some<float, U>(p.cos + pos * half + unit * U, at.pairs), y = load_some<float, U>(p.sin + pos * half + unit * U, at.pairs);
#pragma unroll
        for (int i = 0; i < U; ++i) c[i] = x.get(i), s[i] = y.get(i);
    }
}

// G lanes to a head, U pairs to a lane.  A wave takes every (64 / G * split)-th head of one token.
template <typename T, int U, int G, bool NEAR>
__global__ void __launch_bounds__(kThreads) forward_kernel(RotaryArgs p)
{
    constexpr int kHeads = 64 / G;
    const int lane = threadIdx.x & 63, unit = lane % G;
    const int64_t wave = (int64_t(p.first_block) + blockIdx.x) * kWaves + (threadIdx.x >> 6);
    const int64_t token = wave / p.split;
    if (token >= p.tokens) return;
    const Place at = place_of<U, NEAR>(unit, p.dim, p.rotary);
    float wq[2][U], wk[2][U], c[U], s[U];
    load_pairs<float, U, NEAR>(p.qw, at, wq[0], wq[1]);
    load_pairs<float, U, NEAR>(p.kw, at, wk[0], wk[1]);
    load_angle<U>(p, token, unit, at, c, s);
    const int total = p.heads + p.kv_heads;
    const float inv = 1.0f / float(p.dim);
    for (int head = int(wave % p.split) * kHeads + lane / G; head < total; head += kHeads * p.split) {
        const bool key = head >= p.heads;
        const T* x = key ? static_cast<const T*>(p.k) + token * p.k_token + (head - p.heads) * p.k_head : static_cast<const T*>(p.q) + token * p.q_token + head * p.q_head;
        T* o = key ? static_cast<T*>(p.ok) + (token * p.kv_heads + head - p.heads) * p.dim : static_cast<T*>(p.oq) + (token * p.heads + head) * p.dim;
        float a[U], b[U], sum = 0.0f;
        load_pairs<T, U, NEAR>(x, at, a, b);
#pragma unroll
        for (int i = 0; i < U; ++i) sum = fmaf(a[i], a[i], fmaf(b[i], b[i], sum));
        const float r = rsqrtf(fmaf(sum_of<G>(sum), inv, p.eps));
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const float u = a[i] * r * (key ? wk[0][i] : wq[0][i]), v = b[i] * r * (key ? wk[1][i] : wq[1][i]);
            a[i] = u * c[i] - v * s[i];
            b[i] = u * s[i] + v * c[i];
        }
        store_pairs<T, U, NEAR>(o, at, p.past, a, b);
    }
}

template <typename T, int U, int G, bool NEAR>
__global__ void __launch_bounds__(kThreads) backward_kernel(RotaryArgs p)
{
    constexpr int kHeads = 64 / G;
    __shared__ float s_part[kThreads / G][2][2 * U * G];
    const int lane = threadIdx.x & 63, unit = lane % G, slot = threadIdx.x / G;
    const Place at = place_of<U, NEAR>(unit, p.dim, p.rotary);
    float wq[2][U], wk[2][U], dq[2][U], dk[2][U];
    load_pairs<float, U, NEAR>(p.qw, at, wq[0], wq[1]);
    load_pairs<float, U, NEAR>(p.kw, at, wk[0], wk[1]);
#pragma unroll
    for (int i = 0; i < U; ++i) dq[0][i] = dq[1][i] = dk[0][i] = dk[1][i] = 0.0f;
    const int total = p.heads + p.kv_heads;
    const float inv = 1.0f / float(p.dim);
    const int64_t waves = int64_t(gridDim.x) * kWaves;
    for (int64_t wave = int64_t(blockIdx.x) * kWaves + (threadIdx.x >> 6); wave < p.tokens * p.split; wave += waves) {
        const int64_t token = wave / p.split;
        float c[U], s[U];
        load_angle<U>(p, token, unit, at, c, s);
        for (int head = int(wave % p.split) * kHeads + lane / G; head < total; head += kHeads * p.split) {
            const bool key = head >= p.heads;
            const int h = key ? head - p.heads : head;
            const T* x = key ? static_cast<const T*>(p.k) + token * p.k_token + h * p.k_head : static_cast<const T*>(p.q) + token * p.q_token + h * p.q_head;
            const T* g = key ? static_cast<const T*>(p.gk) + token * p.gk_token + h * p.gk_head : static_cast<const T*>(p.gq) + token * p.gq_token + h * p.gq_head;
            T* o = key ? static_cast<T*>(p.ok) + (token * p.kv_heads + h) * p.dim : static_cast<T*>(p.oq) + (token * p.heads + h) * p.dim;
            float a[U], b[U], ga[U], gb[U], sum = 0.0f, dot = 0.0f;
            load_pairs<T, U, NEAR>(x, at, a, b);
            load_pairs<T, U, NEAR>(g, at, ga, gb);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const float u = ga[i] * c[i] + gb[i] * s[i], v = gb[i] * c[i] - ga[i] * s[i];
                sum = fmaf(a[i], a[i], fmaf(b[i], b[i], sum));
                ga[i] = u;
                gb[i] = v;
                dot = fmaf(u * (key ? wk[0][i] : wq[0][i]), a[i], fmaf(v * (key ? wk[1][i] : wq[1][i]), b[i], dot));
            }
            const float r = rsqrtf(fmaf(sum_of<G>(sum), inv, p.eps));
            const float back = sum_of<G>(dot) * inv * r * r;
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const float da = ga[i] * a[i] * r, db = gb[i] * b[i] * r;
                dq[0][i] += key ? 0.0f : da;
                dq[1][i] += key ? 0.0f : db;
                dk[0][i] += key ? da : 0.0f;
                dk[1][i] += key ? db : 0.0f;
                a[i] = r * (ga[i] * (key ? wk[0][i] : wq[0][i]) - a[i] * back);
                b[i] = r * (gb[i] * (key ? wk[1][i] : wq[1][i]) - b[i] * back);
            }
            store_pairs<T, U, NEAR>(o, at, p.past, a, b);
        }
    }
    // the block's piece of the weights' gradients
#pragma unroll
    for (int i = 0; i < U; ++i) {
        s_part[slot][0][unit * 2 * U + i] = dq[0][i];
        s_part[slot][0][unit * 2 * U + U + i] = dq[1][i];
        s_part[slot][1][unit * 2 * U + i] = dk[0][i];
        s_part[slot][1][unit * 2 * U + U + i] = dk[1][i];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * 2 * U * G; e += kThreads) {
        const int which = e / (2 * U * G), i = e % (2 * U * G);
        const Place to = place_of<U, NEAR>(i / (2 * U), p.dim, p.rotary);
        const int j = i % U;
        if (j >= to.pairs) continue;
        float sum = 0.0f;
        for (int n = 0; n < kThreads / G; ++n) sum += s_part[n][which][i];
        const int ch = (i % (2 * U) < U ? to.first : to.second) + (NEAR ? 2 * j : j);
        p.parts[(int64_t(blockIdx.x) * 2 + which) * p.dim + ch] = sum;
    }
}

// a block to 4 channels: 64 threads for each add up every 64th piece, then each other's sums
__global__ void __launch_bounds__(kThreads) weights_kernel(const float* parts, int pieces, int dim, float* dqw, float* dkw)
{
    __shared__ float s_sum[64][4];
    const int ch = threadIdx.x % 4, row = threadIdx.x / 4, e = blockIdx.x * 4 + ch;
    float sum = 0.0f;
    if (e < 2 * dim)
#pragma unroll
        for (int i = 0; i < kPieces / 64; ++i) {
            const int n = row + 64 * i;
            if (n < pieces) sum += parts[int64_t(n) * 2 * dim + e];
        }
    s_sum[row][ch] = sum;
    for (int half = 32; half; half /= 2) {
        __syncthreads();
        if (row < half) s_sum[row][ch] += s_sum[row + half][ch];
    }
    if (row == 0 && e < 2 * dim) (e < dim ? dqw : dkw)[e < dim ? e : e - dim] = s_sum[0][ch];
}

constexpr int kUnit = 4;

int lanes_for(int dim, int rotary)
{
    const int units = (rotary / 2 + kUnit - 1) / kUnit + (dim - rotary + 2 * kUnit - 1) / (2 * kUnit);
    int g = 4;
    while (g < units) g *= 2;
    return g;
}

// Few tokens: a token's heads are spread over more waves, until there are two for each SIMD or a head for each
int split_for(const RotaryArgs& p, int lanes)
{
    const int heads = 64 / lanes, most = (p.heads + p.kv_heads + heads - 1) / heads;
    int split = 1;
    while (split < most && p.tokens * split < 2048) split *= 2;
    return split < most ? split : most;
}

template <typename T, int G, bool NEAR>
void launch(RotaryArgs& p, bool back, float* dqw, float* dkw, hipStream_t stream)
{
    p.split = split_for(p, G);
    const int64_t blocks = (p.tokens * p.split + kWaves - 1) / kWaves;
    if (!back) {
        require(blocks < (int64_t(1) << 31), "too many tokens");
        launch_all(forward_kernel<T, kUnit, G, NEAR>, blocks, kThreads, stream, p);
        return;
    }
    // 32-bit loads fill the memory's queues with half the blocks, and fewer pieces are summed up sooner (8000 tokens, 20 heads of 128,
    // float32: 46 us, with all pieces 49; 16384, 40 heads of 128, bfloat16: 99 us, with half of them 129)
    const int most = sizeof(T) == 4 ? kPieces / 2 : kPieces, pieces = blocks < most ? int(blocks) : most;
    hipLaunchKernelGGL((backward_kernel<T, kUnit, G, NEAR>), dim3(pieces), dim3(kThreads), 0, stream, p);
    SIG_HIP(hipGetLastError());
    hipLaunchKernelGGL(weights_kernel, dim3((2 * p.dim + 3) / 4), dim3(kThreads), 0, stream, p.parts, pieces, p.dim, dqw, dkw);
    SIG_HIP(hipGetLastError());
}

template <typename T, bool NEAR>
void by_lanes(RotaryArgs& p, bool back, float* dqw, float* dkw, hipStream_t stream)
{
    switch (lanes_for(p.dim, p.rotary)) {
    case 4: return launch<T, 4, NEAR>(p, back, dqw, dkw, stream);
    case 8: return launch<T, 8, NEAR>(p, back, dqw, dkw, stream);
    case 16: return launch<T, 16, NEAR>(p, back, dqw, dkw, stream);
    case 32: return launch<T, 32, NEAR>(p, back, dqw, dkw, stream);
    default: return launch<T, 64, NEAR>(p, back, dqw, dkw, stream);       // 252 channels and more whose two parts both end inside a lane's
    }
}

void run(int dtype, RotaryArgs& p, bool interleaved, bool back, float* dqw, float* dkw, void* stream)
{
    require(p.dim >= 2 && p.dim % 2 == 0 && p.dim <= 256, "a head has 2 to 256 channels, an even number");
    require(p.rotary >= 0 && p.rotary % 2 == 0 && p.rotary <= p.dim, "the rotary part is an even number of a head's channels");
    require(p.heads >= 0 && p.kv_heads >= 0 && p.heads + p.kv_heads < (1 << 20) && p.tokens < (int64_t(1) << 31), "too many heads or tokens");
    require(!back || (dqw && dkw), "a tensor is missing");
    if (p.tokens == 0 || p.heads + p.kv_heads == 0) {
        if (back) {        // no pieces: zeros
            hipLaunchKernelGGL(weights_kernel, dim3((2 * p.dim + 3) / 4), dim3(kThreads), 0, static_cast<hipStream_t>(stream), p.parts, 0, p.dim, dqw, dkw);
            SIG_HIP(hipGetLastError());
        }
        return;
    }
    require(p.qw && p.kw && p.positions && (p.rotary == 0 || (p.cos && p.sin)), "a tensor is missing");
    require((p.heads == 0 || (p.q && p.oq && (!back || p.gq))) && (p.kv_heads == 0 || (p.k && p.ok && (!back || p.gk))), "a tensor is missing");
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        // (16384 tokens, 40 heads of 128 channels, bfloat16: 55 us, through the caches 70 us)
        p.past = goes_past(uint64_t(p.tokens) * (p.heads + p.kv_heads) * p.dim * sizeof(T), uint64_t(p.dim) * sizeof(T));
        if (interleaved) by_lanes<T, true>(p, back, dqw, dkw, static_cast<hipStream_t>(stream));
        else by_lanes<T, false>(p, back, dqw, dkw, static_cast<hipStream_t>(stream));
    });
}

}  // namespace
}  // namespace seqamd

using namespace seqamd;

extern "C" {

__attribute__((visibility("default"))) int cusig_amd_norm_rotary(
    int dtype, const void* q, const void* k, const float* q_weight, const float* k_weight, const float* cos, const float* sin, const int* positions, void* q_out,
    void* k_out, uint64_t tokens, uint64_t heads, uint64_t kv_heads, uint64_t dim, uint64_t rotary_dim, uint64_t table, int64_t q_token, int64_t q_head,
    int64_t k_token, int64_t k_head, float eps, bool interleaved, void* stream) noexcept
{
    return sigamd::guarded([&] {
        require(heads < (1u << 20) && kv_heads < (1u << 20) && dim <= 256 && rotary_dim <= dim && tokens < (uint64_t(1) << 31) && table < (uint64_t(1) << 31), "too many heads, channels or tokens");
        RotaryArgs p{};
        p.q = q, p.k = k, p.qw = q_weight, p.kw = k_weight, p.cos = cos, p.sin = sin, p.positions = positions, p.oq = q_out, p.ok = k_out;
        p.tokens = int64_t(tokens), p.heads = int(heads), p.kv_heads = int(kv_heads), p.dim = int(dim), p.rotary = int(rotary_dim), p.table = int64_t(table);
        p.q_token = q_token, p.q_head = q_head, p.k_token = k_token, p.k_head = k_head;
        p.eps = eps;
        run(dtype, p, interleaved, false, nullptr, nullptr, stream);
    });
}

__attribute__((visibility("default"))) uint64_t cusig_amd_norm_rotary_backprop_workspace(uint64_t dim) noexcept
{
    return uint64_t(kPieces) * 2 * dim * sizeof(float);
}

__attribute__((visibility("default"))) int cusig_amd_norm_rotary_backprop(
    int dtype, const void* grad_q, const void* grad_k, const void* q, const void* k, const float* q_weight, const float* k_weight, const float* cos,
    const float* sin, const int* positions, void* dq, void* dk, float* dq_weight, float* dk_weight, uint64_t tokens, uint64_t heads, uint64_t kv_heads,
    uint64_t dim, uint64_t rotary_dim, uint64_t table, int64_t q_token, int64_t q_head, int64_t k_token, int64_t k_head, int64_t grad_q_token,
    int64_t grad_q_head, int64_t grad_k_token, int64_t grad_k_head, float eps, bool interleaved, void* workspace, uint64_t workspace_bytes, void* stream) noexcept
{
    return sigamd::guarded([&] {
        require(heads < (1u << 20) && kv_heads < (1u << 20) && dim <= 256 && rotary_dim <= dim && tokens < (uint64_t(1) << 31) && table < (uint64_t(1) << 31), "too many heads, channels or tokens");
        check_workspace(workspace, workspace_bytes, cusig_amd_norm_rotary_backprop_workspace(dim));
        RotaryArgs p{};
        p.q = q, p.k = k, p.gq = grad_q, p.gk = grad_k, p.qw = q_weight, p.kw = k_weight, p.cos = cos, p.sin = sin, p.positions = positions, p.oq = dq, p.ok = dk;
        p.parts = static_cast<float*>(workspace);
        p.tokens = int64_t(tokens), p.heads = int(heads), p.kv_heads = int(kv_heads), p.dim = int(dim), p.rotary = int(rotary_dim), p.table = int64_t(table);
        p.q_token = q_token, p.q_head = q_head, p.k_token = k_token, p.k_head = k_head;
        p.gq_token = grad_q_token, p.gq_head = grad_q_head, p.gk_token = grad_k_token, p.gk_head = grad_k_head;
        p.eps = eps;
        run(dtype, p, interleaved, true, dq_weight, dk_weight, stream);
    });
}

}  // extern "C"
