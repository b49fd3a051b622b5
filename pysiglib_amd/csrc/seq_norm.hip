// The residual's addition and the root-mean-square norm of the sum, its gradients, and the same with an output in 8 bits.
//
// Mathematics.  s = x + residual as it is stored (in the residual's type), r = (mean s^2 + eps)^-1/2, out = s r w.  Backward, with
// u = g w: ds = r (u - s r^2 mean(u s)) + the gradient of s itself, dw = sum over rows of g s r.  The norm is of the stored sum, not
// of the sum before it is rounded: what the layers behind read and what the gradients are formed from is then what was normed.
//
// In 8 bits (float8_e4m3fn): q = out / scale with scale = max |out| / 448 of each row; 1 where the row is zero or holds NaN.
//
// Bound: HBM.  A row belongs to W waves, which hold it in registers between the sum of its squares and the output, so everything is
// read once and written once.  Everything between load and store is 32-bit; the sums of dw go by fixed pieces of the rows, added up in
// a fixed order: the same inputs give the same bits.
// Measured, inputs in turn: 16384 rows of 2048, bfloat16 with a residual in float32, 79 us (403 MB, 5.1 TB/s), gradients 108 us (537 MB, 5.0 TB/s) and 5 us for
// the weight's sums; 16384 rows of 4096, bfloat16, into 8 bits 87 us (470 MB, 5.4 TB/s, a part of it found in the last cache); 32 rows of 4096 4.1 us.
#include "seq_common.h"

#include <type_traits>

namespace seqamd {
namespace {

constexpr int kThreads = 256;
// Of the rows at most, for the gradient of the weight: 16384 rows of 2048 channels, bfloat16, both directions 109 us, with 512 pieces 112, with 2048 115
constexpr int kPieces = 1024;

// From how many bytes of results on they are stored past the caches, in MiB; of those that may be, which the 8-bit output is not.  Kept and past, us, inputs in
// turn.  Forward, 2048 channels, bfloat16: 120 MiB 46 and 47, 136 51 and 53, 152 60 and 58, 200 79 and 76; with a copy that reads the results 136 98 and 104,
// 152 117 and 115; forward and gradients 136 95 and 98, 168 115 and 117, 184 132 and 126; the sum in float32 136 136 and 123, 152 149 and 136.  Into 8 bits, 4096 channels,
// where the layer behind reads the 8 bits and not the sum: 88 MiB of sums 63 and 58, 120 84 and 79; with a copy that reads the sum 88 90 and 99, 104 115 and 116, 120 132 and 130.
constexpr uint64_t kPast = uint64_t(144) << 20, kPastEight = uint64_t(112) << 20;

struct NormArgs {
    const void *x, *residual;       // residual null: the sum is x, and not written
    const void *grad, *grad_total;  // of the outputs; grad_total may be null
    const float* weight;
    void *out, *total;              // outputs; backward: total is read
    void *dx, *dresidual;           // dresidual null: as dx
    float* scales;
    float* parts;                   // [pieces][channels]
    int64_t rows, x_step, residual_step, grad_step, grad_total_step;
    int channels;
    float eps;
    bool past;                      // results go past the caches
    unsigned first_block;
};

// adds the V values of a pack to / forms them from floats
template <typename T, int V>
__device__ __forceinline__ void widen(const Pack<T, V>& p, float* to)
{
#pragma unroll
    for (int i = 0; i < V; ++i) to[i] = p.get(i);
}

template <typename T, int V>
__device__ __forceinline__ void put(T* to, const float* from, int count, bool past)
{
    Pack<T, V> o;
    o.set(from);
    if (past && count >= V) store_past<T, V>(to, o);
    else store_some<T, V>(to, o, count);
}

// The sum (or, of absolute values' bits, the largest) over the W waves of a row; `room` takes W words and is not written
// again before every wave has read it, which the caller sees to by taking turns between two of them.
template <int W, typename X, typename F>
__device__ __forceinline__ X over_row(X v, X* room, F&& both)
{
#pragma unroll
    for (int m = 1; m < 64; m *= 2) v = both(v, __shfl_xor(v, m));
    if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = v;
        __syncthreads();
        v = room[0];
#pragma unroll
        for (int w = 1; w < W; ++w) v = both(v, room[w]);
    }
    return v;
}

// T: type of x, R: of the residual and the sum.  W waves to a row, K packs of V elements to a lane.
template <typename T, typename R, int W, int K, bool EIGHT>
__global__ void __launch_bounds__(W > 4 ? 64 * W : kThreads) norm_kernel(NormArgs p)
{
    constexpr int V = 16 / sizeof(T), kBlock = W > 4 ? 64 * W : kThreads, kRows = kBlock / (64 * W);
    __shared__ float s_sum[W > 1 ? W : 1];
    __shared__ unsigned s_top[W > 1 ? W : 1];
    const int64_t row = (int64_t(p.first_block) + blockIdx.x) * kRows + (W > 1 ? 0 : threadIdx.x / 64);
    if (row >= p.rows) return;              // a whole wave, and with W > 1 a whole block
    const int lane = W > 1 ? threadIdx.x : threadIdx.x % 64, channels = p.channels;
    const T* const x = static_cast<const T*>(p.x) + row * p.x_step;
    const R* const add = p.residual ? static_cast<const R*>(p.residual) + row * p.residual_step : nullptr;
    Pack<T, V> in[K];
    Pack<R, V> more[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int at = (k * W * 64 + lane) * V;
        if (at < channels) in[k] = load_some<T, V>(x + at, channels - at);
        if (at < channels && add) more[k] = load_some<R, V>(add + at, channels - at);
    }
    float s[K][V], sum = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int at = (k * W * 64 + lane) * V;
        if (at >= channels) {
#pragma unroll
            for (int i = 0; i < V; ++i) s[k][i] = 0.0f;
            continue;
        }
        widen<T, V>(in[k], s[k]);
        if (add) {
            Pack<R, V> total;
#pragma unroll
            for (int i = 0; i < V; ++i) s[k][i] += more[k].get(i);
            total.set(s[k]);
            R* const to = static_cast<R*>(p.total) + row * channels + at;
            if (p.past && channels - at >= V) store_past<R, V>(to, total);
            else store_some<R, V>(to, total, channels - at);
            widen<R, V>(total, s[k]);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) sum = fmaf(s[k][i], s[k][i], sum);
    }
    sum = over_row<W>(sum, s_sum, [](float a, float b) { return a + b; });
    const float r = rsqrtf(fmaf(sum, 1.0f / float(channels), p.eps));
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int at = (k * W * 64 + lane) * V;
        if (at >= channels) continue;
        const Pack<float, V> w = load_some<float, V>(p.weight + at, channels - at);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            s[k][i] = s[k][i] * r * w.get(i);
            if constexpr (EIGHT) top = max(top, __float_as_uint(s[k][i]) & 0x7fffffffu);
        }
        if constexpr (!EIGHT) put<T, V>(static_cast<T*>(p.out) + row * channels + at, s[k], channels - at, p.past);
    }
    if constexpr (EIGHT) {
        // NaN has larger bits than every number: one in the row makes the scale 1
        top = over_row<W>(top, s_top, [](unsigned a, unsigned b) { return max(a, b); });
        const float ratio = __uint_as_float(top) / 448.0f, scale = ratio > 0.0f ? ratio : 1.0f;       // of 3e-43 and less it is zero
        if (lane == 0) p.scales[row] = scale;
        // out / scale by the reciprocal and one correction from the remainder: the quotient's rounding, and not three, decides between two
        // neighbours of eight bits.  The reciprocal of a scale below 2^-64 may be beyond the numbers: both move.  An infinite scale has the reciprocal
        // zero, and a remainder from zero instead of from itself: finite outputs are then zero, infinite ones NaN, as out / scale is.
        const float move = scale < 5.421010862e-20f ? 7.922816251e28f : 1.0f, inverse = 1.0f / (scale * move), divisor = inverse > 0.0f ? scale * move : 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int at = (k * W * 64 + lane) * V;
            if (at >= channels) continue;
            unsigned char* const to = static_cast<unsigned char*>(p.out) + row * channels + at;
            unsigned q[V / 4];
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float whole = s[k][i + j] * move, near = whole * inverse, y = fmaf(fmaf(-near, divisor, whole), inverse, near);
                    v[j] = y > 448.0f ? 448.0f : (y < -448.0f ? -448.0f : y);       // NaN stays
                }
                int two = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
                q[i / 4] = unsigned(__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], two, true));
            }
            if (channels - at >= V) __builtin_memcpy(to, q, V);
            else
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (i < channels - at) to[i] = static_cast<unsigned char>(q[i / 4] >> (8 * (i % 4)));
        }
    }
}

// Gradients.  Blocks go through the rows; a lane keeps its channels' sums of g s r.  W = 1: the block's waves have rows of
// their own and add up at the end.
template <typename T, typename R, int W, int K>
__global__ void __launch_bounds__(W > 4 ? 64 * W : kThreads) norm_back_kernel(NormArgs p)
{
    constexpr int V = 16 / sizeof(T), kBlock = W > 4 ? 64 * W : kThreads, kRows = kBlock / (64 * W);
    __shared__ float s_two[2][2][W > 1 ? W : 1];
    __shared__ float s_dw[W > 1 ? 1 : kRows][W > 1 ? 1 : 64 * K * V];
    const int lane = W > 1 ? threadIdx.x : threadIdx.x % 64, own = W > 1 ? 0 : threadIdx.x / 64, channels = p.channels;
    const float inv = 1.0f / float(channels);
    float dw[K][V], w[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int at = (k * W * 64 + lane) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] = 0.0f;
        if (at < channels) widen<float, V>(load_some<float, V>(p.weight + at, channels - at), w[k]);
    }
    int side = 0;
    for (int64_t row = int64_t(blockIdx.x) * kRows + own; row < p.rows; row += int64_t(gridDim.x) * kRows) {
        Pack<R, V> total[K], after[K];
        Pack<T, V> grad[K];
        const R* const ap = p.grad_total ? static_cast<const R*>(p.grad_total) + row * p.grad_total_step : nullptr;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int at = (k * W * 64 + lane) * V;
            if (at >= channels) continue;
            total[k] = load_some<R, V>(static_cast<const R*>(p.total) + row * p.x_step + at, channels - at);
            grad[k] = load_some<T, V>(static_cast<const T*>(p.grad) + row * p.grad_step + at, channels - at);
            if (ap) after[k] = load_some<R, V>(ap + at, channels - at);
        }
        float sum = 0.0f, dot = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int at = (k * W * 64 + lane) * V;
            if (at >= channels) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float s = total[k].get(i);
                sum = fmaf(s, s, sum);
                dot = fmaf(grad[k].get(i) * w[k][i], s, dot);
            }
        }
#pragma unroll
        for (int m = 1; m < 64; m *= 2) sum += __shfl_xor(sum, m), dot += __shfl_xor(dot, m);
        if constexpr (W > 1) {          // two rooms in turn: a wave that is a row ahead writes into the other
            if ((threadIdx.x & 63) == 0) s_two[side][0][threadIdx.x >> 6] = sum, s_two[side][1][threadIdx.x >> 6] = dot;
            __syncthreads();
            sum = dot = 0.0f;
#pragma unroll
            for (int i = 0; i < W; ++i) sum += s_two[side][0][i], dot += s_two[side][1][i];
            side ^= 1;
        }
        const float r = rsqrtf(fmaf(sum, inv, p.eps)), back = dot * inv * r * r;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int at = (k * W * 64 + lane) * V;
            if (at >= channels) continue;
            float ds[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float s = total[k].get(i), g = grad[k].get(i);
                dw[k][i] = fmaf(g * s, r, dw[k][i]);
                ds[i] = r * (g * w[k][i] - s * back);
                if (ap) ds[i] += after[k].get(i);
            }
            put<T, V>(static_cast<T*>(p.dx) + row * channels + at, ds, channels - at, p.past);
            if constexpr (!std::is_same_v<T, R>) put<R, V>(static_cast<R*>(p.dresidual) + row * channels + at, ds, channels - at, p.past);
        }
    }
    float* const part = p.parts + int64_t(blockIdx.x) * channels;
    if constexpr (W > 1) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int at = (k * W * 64 + lane) * V;
            if (at < channels) put<float, V>(part + at, dw[k], channels - at, false);
        }
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) s_dw[own][(k * 64 + lane) * V + i] = dw[k][i];
        __syncthreads();
        for (int e = threadIdx.x; e < channels; e += kThreads) {
            float sum = 0.0f;
#pragma unroll
            for (int n = 0; n < kRows; ++n) sum += s_dw[n][e];
            part[e] = sum;
        }
    }
}

__global__ void __launch_bounds__(kSumThreads) norm_weight_kernel(const float* parts, int pieces, int channels, float* dw)
{
    sum_pieces(parts, pieces, channels, 0, [&](int64_t e, float sum) { dw[e] = sum; });
}

// Waves to a row and packs to a lane: a wave holds up to two packs a lane, four waves up to eight, and eight waves what float32
// rows have beyond that.  (32768 rows of 1024 channels, bfloat16, two packs to a lane of one wave 49 us, one pack to a lane of four 57;
// gradients as well 107 and 115; 64 to 4096 rows alike.)
struct NormPlan {
    int waves, packs;
};

constexpr int kMost = 16384;        // channels

template <typename T>
NormPlan plan_of(int channels)
{
    const int packs = (channels + 16 / int(sizeof(T)) - 1) / (16 / int(sizeof(T)));
    NormPlan p;
    p.waves = packs <= 128 ? 1 : (packs <= 2048 ? 4 : 8);
    const int each = (packs + 64 * p.waves - 1) / (64 * p.waves);
    p.packs = 1;
    while (p.packs < each) p.packs *= 2;
    return p;
}

// calls body with the plan's numbers as types
template <typename T, typename F>
void by_plan(const NormPlan& p, F&& body)
{
    using std::integral_constant;
    if (p.waves == 1) return p.packs == 1 ? body(integral_constant<int, 1>{}, integral_constant<int, 1>{}) : body(integral_constant<int, 1>{}, integral_constant<int, 2>{});
    if (p.waves == 4) {
        switch (p.packs) {
        case 1: return body(integral_constant<int, 4>{}, integral_constant<int, 1>{});
        case 2: return body(integral_constant<int, 4>{}, integral_constant<int, 2>{});
        case 4: return body(integral_constant<int, 4>{}, integral_constant<int, 4>{});
        default: return body(integral_constant<int, 4>{}, integral_constant<int, 8>{});
        }
    }
    if constexpr (sizeof(T) == 4) return body(integral_constant<int, 8>{}, integral_constant<int, 8>{});
}

// calls body(T{}, R{}): the residual has x's type or is float32
template <typename F>
void with_types(int dtype, int residual, F&& body)
{
    require(residual == dtype || residual == kF32, "the residual has the type of x or float32");
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (residual == dtype) body(t, t);
        else if constexpr (sizeof(T) == 2) body(t, float{});
    });
}

void check(uint64_t rows, uint64_t channels)
{
    require(rows < (uint64_t(1) << 31) && channels >= 1 && channels <= kMost, "a row has 1 to 16384 channels");
}

template <bool EIGHT>
void forward(int dtype, int residual, NormArgs& p, hipStream_t stream)
{
    if (p.rows == 0) return;
    require(p.x && p.weight && p.out && (!p.residual || p.total) && (!EIGHT || p.scales), "a tensor is missing");
    with_types(dtype, residual, [&](auto t, auto u) {
        using T = decltype(t);
        using R = decltype(u);
        const uint64_t cells = uint64_t(p.rows) * p.channels;
        p.past = goes_past(cells * ((EIGHT ? 0 : sizeof(T)) + (p.residual ? sizeof(R) : 0)), uint64_t(p.channels) * sizeof(T), EIGHT ? kPastEight : kPast);
        by_plan<T>(plan_of<T>(p.channels), [&](auto w, auto k) {
            constexpr int W = decltype(w)::value, K = decltype(k)::value, kBlock = W > 4 ? 64 * W : kThreads, kRows = kBlock / (64 * W);
            launch_all(norm_kernel<T, R, W, K, EIGHT>, (p.rows + kRows - 1) / kRows, kBlock, stream, p);
        });
    });
}

void backward(int dtype, int residual, NormArgs& p, float* dw, hipStream_t stream)
{
    require(dw, "a tensor is missing");
    int pieces = 0;
    if (p.rows) {
        require(p.total && p.grad && p.weight && p.dx && (residual == dtype || p.dresidual), "a tensor is missing");
        with_types(dtype, residual, [&](auto t, auto u) {
            using T = decltype(t);
            using R = decltype(u);
            const uint64_t cells = uint64_t(p.rows) * p.channels;
            p.past = goes_past(cells * (sizeof(T) + (std::is_same_v<T, R> ? 0 : sizeof(R))), uint64_t(p.channels) * sizeof(T), kPast);
            by_plan<T>(plan_of<T>(p.channels), [&](auto w, auto k) {
                constexpr int W = decltype(w)::value, K = decltype(k)::value, kBlock = W > 4 ? 64 * W : kThreads, kRows = kBlock / (64 * W);
                const int64_t blocks = (p.rows + kRows - 1) / kRows;
                pieces = int(blocks < kPieces ? blocks : kPieces);
                hipLaunchKernelGGL((norm_back_kernel<T, R, W, K>), dim3(pieces), dim3(kBlock), 0, stream, p);
                SIG_HIP(hipGetLastError());
            });
        });
    }
    hipLaunchKernelGGL(norm_weight_kernel, dim3(unsigned(sum_blocks(p.channels))), dim3(kSumThreads), 0, stream, p.parts, pieces, p.channels, dw);
    SIG_HIP(hipGetLastError());
}

}  // namespace
}  // namespace seqamd

using namespace seqamd;

extern "C" {

__attribute__((visibility("default"))) int cusig_amd_norm_residual(
    int dtype, int residual_dtype, const void* x, const void* residual, const float* weight, void* out, void* total, float* scales, uint64_t rows,
    uint64_t channels, int64_t x_stride, int64_t residual_stride, float eps, void* stream) noexcept
{
    return sigamd::guarded([&] {
        check(rows, channels);
        NormArgs p{};
        p.x = x, p.residual = residual, p.weight = weight, p.out = out, p.total = total, p.scales = scales;
        p.rows = int64_t(rows), p.channels = int(channels), p.x_step = x_stride, p.residual_step = residual_stride;
        p.eps = eps;
        if (scales) forward<true>(dtype, residual_dtype, p, static_cast<hipStream_t>(stream));
        else forward<false>(dtype, residual_dtype, p, static_cast<hipStream_t>(stream));
    });
}

__attribute__((visibility("default"))) uint64_t cusig_amd_norm_residual_backprop_workspace(uint64_t channels) noexcept
{
    return uint64_t(kPieces) * channels * sizeof(float);
}

__attribute__((visibility("default"))) int cusig_amd_norm_residual_backprop(
    int dtype, int residual_dtype, const void* grad_out, const void* grad_total, const void* total, const float* weight, void* dx, void* dresidual,
    float* dweight, uint64_t rows, uint64_t channels, int64_t grad_out_stride, int64_t grad_total_stride, int64_t total_stride, float eps, void* workspace,
    uint64_t workspace_bytes, void* stream) noexcept
{
    return sigamd::guarded([&] {
        check(rows, channels);
        check_workspace(workspace, workspace_bytes, cusig_amd_norm_residual_backprop_workspace(channels));
        NormArgs p{};
        p.grad = grad_out, p.grad_total = grad_total, p.total = const_cast<void*>(total), p.weight = weight, p.dx = dx, p.dresidual = dresidual;
        p.parts = static_cast<float*>(workspace);
        p.rows = int64_t(rows), p.channels = int(channels);
        p.grad_step = grad_out_stride, p.grad_total_step = grad_total_stride, p.x_step = total_stride;
        p.eps = eps;
        backward(dtype, residual_dtype, p, dweight, static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
