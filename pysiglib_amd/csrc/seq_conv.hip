// Short causal convolution of each channel over sequences of any length, with an activation, its gradients, and one step of it
// against the rows that are kept.
//
// Mathematics.  Position p of a sequence is its p-th row; positions -(W - 1) to -1 are the rows of its initial state.
// v_p = bias + sum_k w_k x_{p - W + 1 + k}, y = v sigmoid(v) or v.  Backward, with e = g times the activation's slope at v:
// dx_p = sum_j w_{W - 1 - j} e_{p + j} over the positions p + j of the sequence, plus the gradient of the final state where p is one of the
// last W - 1 positions; for p < 0 that is the gradient of the initial state.  dw_k = sum_p e_p x_{p - W + 1 + k}, dbias = sum_p e_p.
//
// Bound: HBM.  A thread takes a run of R rows of a few channels with all its loads on their way at once and keeps the window of the last
// W - 1 rows in registers; the W - 1 rows before (backward: and behind) its run it reads again, from the caches.  Sums are 32-bit;
// those of dw go by fixed pieces of the rows, added up in a fixed order: the same inputs give the same bits.
#include "seq_common.h"

#include <type_traits>

namespace seqamd {
namespace {

constexpr int kThreads = 256;
constexpr int kWidest = 8;

struct ConvArgs {
    const void* x;              // [rows][channels], rows x_step apart
    const void* grad;           // of y, backward
    const void* begin;          // initial states [n][W - 1][channels] or null
    const void* grad_end;       // gradients of the final states or null, backward
    const float *w, *bias;      // [channels][W]; bias may be null
    void* out;                  // y; backward: dx
    void* end;                  // final states; backward: gradients of the initial states
    float* parts;               // backward: [pieces][W + 1][channels]
    const int* offsets;         // [n + 1] rows where sequences begin, or null: n sequences of `length` rows
    int64_t rows, x_step, grad_step, length, n;
    int channels, lanes, channel_blocks, pieces;
    int64_t runs, blocks, idle; // blocks with runs; `idle` ones behind them serve sequences without rows
    bool silu, past;
    unsigned first_block;
};

// The rows [first, past) of a sequence, kept inside the tensors whatever the offsets hold
__device__ __forceinline__ void rows_of(const ConvArgs& p, int64_t i, int64_t& first, int64_t& past)
{
    if (p.offsets) {
        first = kept(p.offsets[i], 0, p.rows);
        past = kept(p.offsets[i + 1], first, p.rows);
    } else {
        first = i * p.length;
        past = first + p.length;
    }
}

// the first sequence that ends behind row t
__device__ __forceinline__ int64_t sequence_at(const ConvArgs& p, int64_t t)
{
    if (!p.offsets) return t / p.length;
    int64_t lo = 0, hi = p.n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (p.offsets[mid + 1] <= t) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896341f)); }

__device__ __forceinline__ float slope(float v)
{
    const float s = sigmoid(v);
    return s * fmaf(v, 1.0f - s, 1.0f);
}

// A thread's V channels.  Where the last ones would be behind the row, it takes the last V of the row instead: what two lanes form, they form
// alike.  PART: a row has fewer than V.
template <typename T, int V, bool PART>
struct Lane {
    int ch, count;
    __device__ __forceinline__ Lane(int at, int channels) : ch(PART ? at : min(at, channels - V)), count(PART ? max(0, min(channels - at, V)) : V) {}
    template <typename X>
    __device__ __forceinline__ Pack<X, V> load(const void* from) const
    {
        if constexpr (PART) return load_some<X, V>(static_cast<const X*>(from) + ch, count);
        else return load_pack<X, V>(static_cast<const X*>(from) + ch);
    }
    template <typename X>
    __device__ __forceinline__ void store(void* to, const float* v, bool past) const
    {
        Pack<X, V> o;
        o.set(v);
        X* const at = static_cast<X*>(to) + ch;
        if constexpr (PART) store_some<X, V>(at, o, count);
        else if (past) store_past<X, V>(at, o);
        else store_pack<X, V>(at, o);
    }
};

// a row at position p of sequence i that begins at row `first`, as floats
template <typename T, int V, int W, bool PART>
__device__ __forceinline__ void row_at(const ConvArgs& a, const Lane<T, V, PART>& lane, int64_t i, int64_t first, int64_t p, float* to)
{
    if (p >= 0) {
        const Pack<T, V> x = lane.template load<T>(static_cast<const T*>(a.x) + (first + p) * a.x_step);
#pragma unroll
        for (int v = 0; v < V; ++v) to[v] = x.get(v);
    } else if (a.begin) {
        const Pack<T, V> x = lane.template load<T>(static_cast<const T*>(a.begin) + (i * (W - 1) + (W - 1 + p)) * a.channels);
#pragma unroll
        for (int v = 0; v < V; ++v) to[v] = x.get(v);
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) to[v] = 0.0f;
    }
}

template <typename T, int V, int W, bool PART>
__device__ __forceinline__ void weights_of(const ConvArgs& a, const Lane<T, V, PART>& lane, float (&w)[W][V], float* bias)
{
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const bool there = v < lane.count;
#pragma unroll
        for (int k = 0; k < W; ++k) w[k][v] = there ? a.w[int64_t(lane.ch + v) * W + k] : 0.0f;
        bias[v] = there && a.bias ? a.bias[lane.ch + v] : 0.0f;
    }
}

// sequences without rows: the state (or its gradient) behind no rows is the one before them
template <typename T, int W>
__device__ void without_rows(const ConvArgs& a, const void* from, void* to)
{
    const int64_t each = int64_t(W - 1) * a.channels, first_block = int64_t(a.first_block) + blockIdx.x - a.blocks, more = a.n * each;
    for (int64_t e = first_block * kThreads + threadIdx.x; e < more; e += a.idle * kThreads) {
        int64_t first, past;
        rows_of(a, e / each, first, past);
        if (first == past) static_cast<T*>(to)[e] = from ? static_cast<const T*>(from)[e] : T(0.0f);
    }
}

template <typename T, int V, int W, int R, bool PART>
__global__ void __launch_bounds__(kThreads) conv_kernel(ConvArgs a)
{
    const int64_t block = int64_t(a.first_block) + blockIdx.x;
    if (block >= a.blocks) return without_rows<T, W>(a, a.begin, a.end);
    const int groups = kThreads / a.lanes;
    const Lane<T, V, PART> lane((int(block % a.channel_blocks) * a.lanes + int(threadIdx.x) % a.lanes) * V, a.channels);
    const int64_t t0 = (block / a.channel_blocks * groups + threadIdx.x / a.lanes) * R;
    if (t0 >= a.rows) return;
    const T* const x = static_cast<const T*>(a.x);
    Pack<T, V> in[R];
#pragma unroll
    for (int r = 0; r < R; ++r) in[r] = lane.template load<T>(x + (t0 + r < a.rows ? t0 + r : a.rows - 1) * a.x_step);
    float w[W][V], bias[V], win[W][V];
    weights_of<T, V, W, PART>(a, lane, w, bias);
    int64_t i = sequence_at(a, t0), first = 0, past = 0;
    if (i < a.n) rows_of(a, i, first, past);
    // the window before row t
    auto fill = [&](int64_t t) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) row_at<T, V, W, PART>(a, lane, i, first, t - first - (W - 1) + k, win[k]);
    };
    auto one = [&](int r, int64_t t) __attribute__((always_inline)) {
        float y[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            win[W - 1][v] = in[r].get(v);
            float sum = bias[v];
#pragma unroll
            for (int k = 0; k < W; ++k) sum = fmaf(w[k][v], win[k][v], sum);
            y[v] = a.silu ? sum * sigmoid(sum) : sum;
#pragma unroll
            for (int k = 0; k < W - 1; ++k) win[k][v] = win[k + 1][v];
        }
        lane.template store<T>(static_cast<T*>(a.out) + t * a.channels, y, a.past);
    };
    auto finish = [&] __attribute__((always_inline)) {
        if (a.end)
#pragma unroll
            for (int k = 0; k < W - 1; ++k) lane.template store<T>(static_cast<T*>(a.end) + (i * (W - 1) + k) * a.channels, win[k], false);
    };
    if (i < a.n && t0 >= first && t0 + R <= past) {
        fill(t0);
#pragma unroll
        for (int r = 0; r < R; ++r) one(r, t0 + r);
        if (t0 + R == past) finish();
        return;
    }
    // sequences begin or end among these rows
    bool filled = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t t = t0 + r;
        while (i < a.n && t >= past) {
            if (++i < a.n) rows_of(a, i, first, past);
            filled = false;
        }
        if (i >= a.n || t < first) continue;
        if (!filled) fill(t);
        filled = true;
        one(r, t);
        if (t + 1 == past) finish();
    }
}

// Gradients: a block goes through runs of R rows, a thread walks each from its last row to its first with the window of the W - 1 values e
// behind the row and that of the W rows of x up to it.
template <typename T, int V, int W, int R, bool PART>
__global__ void __launch_bounds__(kThreads) conv_back_kernel(ConvArgs a)
{
    const int64_t block = int64_t(a.first_block) + blockIdx.x;
    if (block >= a.blocks) return without_rows<T, W>(a, a.grad_end, a.end);
    __shared__ float s_sum[kThreads][V + 1];
    const int groups = kThreads / a.lanes, cb = int(block % a.channel_blocks), piece = int(block / a.channel_blocks), group = int(threadIdx.x) / a.lanes;
    const Lane<T, V, PART> lane((cb * a.lanes + int(threadIdx.x) % a.lanes) * V, a.channels);
    const T *const x = static_cast<const T*>(a.x), *const grad = static_cast<const T*>(a.grad);
    float w[W][V], bias[V], dw[W][V], db[V];
    weights_of<T, V, W, PART>(a, lane, w, bias);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        db[v] = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) dw[k][v] = 0.0f;
    }
    float e[W][V];              // e[j]: of the row j behind
    // row t with the rows of x up to it: e, and where the row is the run's own its part of the sums and dx
    auto value = [&](const float (&xs)[W][V], const float* g, bool own) __attribute__((always_inline)) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float sum = bias[v];
#pragma unroll
            for (int k = 0; k < W; ++k) sum = fmaf(w[k][v], xs[k][v], sum);
            e[0][v] = a.silu ? g[v] * slope(sum) : g[v];
            if (own) {
                db[v] += e[0][v];
#pragma unroll
                for (int k = 0; k < W; ++k) dw[k][v] = fmaf(e[0][v], xs[k][v], dw[k][v]);
            }
        }
    };
    auto derivative = [&](float* d) __attribute__((always_inline)) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            d[v] = 0.0f;
#pragma unroll
            for (int j = 0; j < W; ++j) d[v] = fmaf(w[W - 1 - j][v], e[j][v], d[v]);
        }
    };
    auto shift = [&] __attribute__((always_inline)) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int j = W - 1; j > 0; --j) e[j][v] = e[j - 1][v];
    };
    auto clear = [&] __attribute__((always_inline)) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int j = 0; j < W; ++j) e[j][v] = 0.0f;
    };
    for (int64_t run = int64_t(piece) * groups + group; run < a.runs; run += int64_t(a.pieces) * groups) {
        const int64_t t0 = run * R, t1 = t0 + R < a.rows ? t0 + R : a.rows;
        int64_t i = sequence_at(a, t0), first = 0, past = 0;
        if (i >= a.n) continue;
        rows_of(a, i, first, past);
        if (t0 - (W - 1) >= first && t0 + R + W - 1 <= past) {
            // nothing but rows of one sequence that are neither its first nor its last ones
            constexpr int kX = R + 2 * (W - 1), kG = R + W - 1;
            Pack<T, V> xs[kX], gs[kG];
#pragma unroll
            for (int r = 0; r < kX; ++r) xs[r] = lane.template load<T>(x + (t0 - (W - 1) + r) * a.x_step);
#pragma unroll
            for (int r = 0; r < kG; ++r) gs[r] = lane.template load<T>(grad + (t0 + r) * a.grad_step);
            clear();
#pragma unroll
            for (int r = kG - 1; r >= 0; --r) {
                float taps[W][V], g[V], d[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    g[v] = gs[r].get(v);
#pragma unroll
                    for (int k = 0; k < W; ++k) taps[k][v] = xs[r + k].get(v);
                }
                value(taps, g, r < R);
                if (r < R) {
                    derivative(d);
                    lane.template store<T>(static_cast<T*>(a.out) + (t0 + r) * a.channels, d, a.past);
                }
                shift();
            }
            continue;
        }
        for (; i < a.n; ++i) {
            rows_of(a, i, first, past);
            if (first >= t1) break;
            const int64_t low = t0 > first ? t0 : first, high = t1 < past ? t1 : past;
            if (low >= high) continue;
            clear();
            const int64_t len = past - first;
            int64_t t = high + W - 2 < past - 1 ? high + W - 2 : past - 1;
            float taps[W][V];
#pragma unroll
            for (int k = 1; k < W; ++k) row_at<T, V, W, PART>(a, lane, i, first, t - first - (W - 1) + k, taps[k - 1]);
            // down to the sequence's first row, and from there through the positions of the initial state
            const int64_t lowest = low == first ? first - (W - 1) : low;
            for (; t >= lowest; --t) {
                const int64_t p = t - first;
                float d[V];
                if (p >= 0) {
                    const Pack<T, V> gp = lane.template load<T>(grad + t * a.grad_step);
                    float g[V];
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        g[v] = gp.get(v);
#pragma unroll
                        for (int k = W - 1; k > 0; --k) taps[k][v] = taps[k - 1][v];
                    }
                    row_at<T, V, W, PART>(a, lane, i, first, p - (W - 1), taps[0]);
                    value(taps, g, t < high);
                } else {
#pragma unroll
                    for (int v = 0; v < V; ++v) e[0][v] = 0.0f;
                }
                if (t < high) {
                    derivative(d);
                    if (a.grad_end && p >= len - (W - 1)) {
                        const Pack<T, V> more = lane.template load<T>(static_cast<const T*>(a.grad_end) + (i * (W - 1) + p - (len - (W - 1))) * a.channels);
#pragma unroll
                        for (int v = 0; v < V; ++v) d[v] += more.get(v);
                    }
                    if (p >= 0) lane.template store<T>(static_cast<T*>(a.out) + t * a.channels, d, a.past);
                    else lane.template store<T>(static_cast<T*>(a.end) + (i * (W - 1) + (W - 1) + p) * a.channels, d, false);
                }
                shift();
            }
        }
    }
    // the block's piece of the weights' gradients, a tap after the other
#pragma unroll
    for (int k = 0; k <= W; ++k) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) s_sum[threadIdx.x][v] = k < W ? dw[k < W ? k : 0][v] : db[v];
        __syncthreads();
        if (group == 0)
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v < lane.count) {
                    float sum = 0.0f;
                    for (int n = 0; n < groups; ++n) sum += s_sum[n * a.lanes + threadIdx.x][v];
                    a.parts[(int64_t(piece) * (W + 1) + k) * a.channels + lane.ch + v] = sum;
                }
    }
}

__global__ void __launch_bounds__(kSumThreads) conv_weight_kernel(const float* parts, int pieces, int channels, int width, float* dw, float* db)
{
    sum_pieces(parts, pieces, int64_t(width + 1) * channels, [&](int64_t e, float sum) {
        const int k = int(e / channels), ch = int(e % channels);
        if (k < width) dw[int64_t(ch) * width + k] = sum;
        else if (db) db[ch] = sum;
    });
}

template <typename T, int V, int W>
__global__ void __launch_bounds__(kThreads) conv_step_kernel(ConvArgs a)
{
    const int packs = (a.channels + V - 1) / V;
    const int64_t e = (int64_t(a.first_block) + blockIdx.x) * kThreads + threadIdx.x;
    if (e >= a.rows * packs) return;
    const int64_t row = e / packs;
    const Lane<T, V, true> lane(int(e - row * packs) * V, a.channels);
    float w[W][V], bias[V], xs[W][V], y[V];
    T* const state = static_cast<T*>(a.end) + row * (W - 1) * a.channels;
#pragma unroll
    for (int k = 0; k < W; ++k) {
        const Pack<T, V> x = lane.template load<T>(k < W - 1 ? state + int64_t(k) * a.channels : static_cast<const T*>(a.x) + row * a.x_step);
#pragma unroll
        for (int v = 0; v < V; ++v) xs[k][v] = x.get(v);
    }
    weights_of<T, V, W, true>(a, lane, w, bias);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float sum = bias[v];
#pragma unroll
        for (int k = 0; k < W; ++k) sum = fmaf(w[k][v], xs[k][v], sum);
        y[v] = a.silu ? sum * sigmoid(sum) : sum;
    }
    lane.template store<T>(static_cast<T*>(a.out) + row * a.channels, y, false);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) lane.template store<T>(state + int64_t(k) * a.channels, xs[k + 1], false);
}

template <typename F>
void with_width(uint64_t width, F&& body)
{
    using std::integral_constant;
    switch (width) {
    case 1: return body(integral_constant<int, 1>{});
    case 2: return body(integral_constant<int, 2>{});
    case 3: return body(integral_constant<int, 3>{});
    case 4: return body(integral_constant<int, 4>{});
    case 5: return body(integral_constant<int, 5>{});
    case 6: return body(integral_constant<int, 6>{});
    case 7: return body(integral_constant<int, 7>{});
    case 8: return body(integral_constant<int, 8>{});
    default: throw std::invalid_argument("a convolution has 1 to 8 taps");
    }
}

constexpr int kForwardRows = 16, kBackwardRows = 16;        // of a run
constexpr int kBackwardBlocks = 1024;

// lanes to a row: a power of two, at most a wave
int lanes_for(int packs)
{
    int lanes = 8;
    while (lanes < packs && lanes < 64) lanes *= 2;
    return lanes;
}

void place(ConvArgs& a, int v, int rows)
{
    const int packs = (a.channels + v - 1) / v;
    a.lanes = lanes_for(packs);
    a.channel_blocks = (packs + a.lanes - 1) / a.lanes;
    a.runs = (a.rows + rows - 1) / rows;
    const int64_t groups = kThreads / a.lanes;
    a.pieces = int((a.runs + groups - 1) / groups);
}

int64_t idle_blocks(const ConvArgs& a, int width)
{
    if (!a.offsets && a.length) return 0;
    const int64_t blocks = (a.n * (width - 1) * a.channels + kThreads - 1) / kThreads;
    return blocks < 256 ? blocks : 256;
}

// pieces of the rows in the gradients' sums: enough blocks to fill the chip some times over
int pieces_of(int64_t rows, int channels)
{
    ConvArgs a{};
    a.rows = rows, a.channels = channels;
    place(a, 4, kBackwardRows);
    const int most = kBackwardBlocks / a.channel_blocks > 0 ? kBackwardBlocks / a.channel_blocks : 1;
    return a.pieces < most ? a.pieces : most;
}

void check(const ConvArgs& a, uint64_t width, uint64_t rows, uint64_t channels, uint64_t n, uint64_t length)
{
    require(width >= 1 && width <= kWidest, "a convolution has 1 to 8 taps");
    require(channels < (uint64_t(1) << 27) && rows < (uint64_t(1) << 31) && n < (uint64_t(1) << 31), "too many rows, channels or sequences");
    require(a.offsets || n * length == rows, "rows are not sequences times length");
}

ConvArgs args_of(const void* x, const float* w, const float* bias, const int* offsets, uint64_t n, uint64_t length, uint64_t rows, uint64_t channels, int64_t x_step, bool silu)
{
    ConvArgs a{};
    a.x = x, a.w = w, a.bias = bias, a.offsets = offsets;
    a.n = int64_t(n), a.length = int64_t(length), a.rows = int64_t(rows), a.channels = int(channels), a.x_step = x_step;
    a.silu = silu;
    return a;
}

}  // namespace
}  // namespace seqamd

using namespace seqamd;

extern "C" {

__attribute__((visibility("default"))) int cusig_amd_causal_conv(
    int dtype, const void* x, const float* weight, const float* bias, const void* initial_state, void* y, void* final_state, const int* offsets,
    uint64_t sequences, uint64_t length, uint64_t rows, uint64_t channels, uint64_t width, int64_t x_stride, bool silu, void* stream) noexcept
{
    return sigamd::guarded([&] {
        ConvArgs a = args_of(x, weight, bias, offsets, sequences, length, rows, channels, x_stride, silu);
        check(a, width, rows, channels, sequences, length);
        a.begin = initial_state, a.out = y, a.end = final_state;
        if (a.channels == 0 || a.n == 0) return;
        require((weight || width * channels == 0) && (final_state || width == 1) && (rows == 0 || (x && y)), "a tensor is missing");
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            constexpr int V = 16 / sizeof(T);
            with_width(width, [&](auto w) {
                constexpr int W = decltype(w)::value;
                place(a, V, kForwardRows);
                a.blocks = int64_t(a.pieces) * a.channel_blocks;
                a.past = goes_past(uint64_t(a.rows) * a.channels * sizeof(T), uint64_t(a.channels) * sizeof(T));
                a.idle = idle_blocks(a, W);
                const int64_t blocks = a.blocks + a.idle;
                if (a.channels < V) launch_all(conv_kernel<T, V, W, kForwardRows, true>, blocks, kThreads, static_cast<hipStream_t>(stream), a);
                else launch_all(conv_kernel<T, V, W, kForwardRows, false>, blocks, kThreads, static_cast<hipStream_t>(stream), a);
            });
        });
    });
}

__attribute__((visibility("default"))) uint64_t cusig_amd_causal_conv_backprop_workspace(uint64_t rows, uint64_t channels, uint64_t width) noexcept
{
    uint64_t bytes = 0;
    sigamd::guarded([&] {
        ConvArgs a{};
        check(a, width, rows, channels, 0, 0);
    });
    if (width >= 1 && width <= kWidest && channels < (uint64_t(1) << 27) && rows < (uint64_t(1) << 31) && rows && channels)
        bytes = uint64_t(pieces_of(int64_t(rows), int(channels))) * (width + 1) * channels * sizeof(float);
    return bytes;
}

__attribute__((visibility("default"))) int cusig_amd_causal_conv_backprop(
    int dtype, const void* grad_y, const void* x, const float* weight, const float* bias, const void* initial_state, const void* grad_final, void* grad_x,
    float* grad_weight, float* grad_bias, void* grad_initial, const int* offsets, uint64_t sequences, uint64_t length, uint64_t rows, uint64_t channels,
    uint64_t width, int64_t grad_stride, int64_t x_stride, bool silu, void* workspace, uint64_t workspace_bytes, void* stream) noexcept
{
    return sigamd::guarded([&] {
        ConvArgs a = args_of(x, weight, bias, offsets, sequences, length, rows, channels, x_stride, silu);
        check(a, width, rows, channels, sequences, length);
        a.grad = grad_y, a.begin = initial_state, a.grad_end = grad_final, a.out = grad_x, a.end = grad_initial;
        a.grad_step = grad_stride;
        if (a.channels == 0) return;
        require(weight && grad_weight && (a.n == 0 || grad_initial || width == 1) && (rows == 0 || (x && grad_y && grad_x)), "a tensor is missing");
        check_workspace(workspace, workspace_bytes, cusig_amd_causal_conv_backprop_workspace(rows, channels, width));
        a.parts = static_cast<float*>(workspace);
        int pieces = 0;
        if (a.n)
            with_type(dtype, [&](auto t) {
                using T = decltype(t);
                constexpr int V = 4;
                with_width(width, [&](auto w) {
                    // windows of more than four taps leave registers for half the rows
                    constexpr int W = decltype(w)::value, R = W > 4 ? kBackwardRows / 2 : kBackwardRows;
                    place(a, V, R);
                    pieces = a.rows ? pieces_of(a.rows, a.channels) : 0;
                    a.pieces = pieces;
                    a.blocks = int64_t(a.pieces) * a.channel_blocks;
                    a.past = goes_past(uint64_t(a.rows) * a.channels * sizeof(T), uint64_t(a.channels) * sizeof(T));
                    a.idle = idle_blocks(a, W);
                    const int64_t blocks = a.blocks + a.idle;
                    if (a.channels < V) launch_all(conv_back_kernel<T, V, W, R, true>, blocks, kThreads, static_cast<hipStream_t>(stream), a);
                    else launch_all(conv_back_kernel<T, V, W, R, false>, blocks, kThreads, static_cast<hipStream_t>(stream), a);
                });
            });
        hipLaunchKernelGGL(conv_weight_kernel, sum_blocks(int64_t(width + 1) * a.channels), dim3(kSumThreads), 0, static_cast<hipStream_t>(stream), a.parts, pieces,
                           a.channels, int(width), grad_weight, grad_bias);
        SIG_HIP(hipGetLastError());
    });
}

__attribute__((visibility("default"))) int cusig_amd_causal_conv_step(
    int dtype, const void* x, void* state, const float* weight, const float* bias, void* y, uint64_t rows, uint64_t channels, uint64_t width,
    int64_t x_stride, bool silu, void* stream) noexcept
{
    return sigamd::guarded([&] {
        ConvArgs a = args_of(x, weight, bias, nullptr, rows, 1, rows, channels, x_stride, silu);
        check(a, width, rows, channels, rows, 1);
        a.out = y, a.end = state;
        if (rows * channels == 0) return;
        require(x && weight && y && (state || width == 1), "a tensor is missing");
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            constexpr int V = 4;
            with_width(width, [&](auto w) {
                launch_all(conv_step_kernel<T, V, decltype(w)::value>, (a.rows * ((a.channels + V - 1) / V) + kThreads - 1) / kThreads, kThreads, static_cast<hipStream_t>(stream), a);
            });
        });
    });
}

}  // extern "C"
