// Short causal convolution of each channel over sequences of any length, with an activation, its gradients, and one step of it
// against the rows that are kept.
//
// Mathematics.  Position p of a sequence is its p-th row; positions -(W - 1) to -1 are the rows of its initial state.
// v_p = bias + sum_k w_k x_{p - W + 1 + k}, y = v sigmoid(v) or v.  Backward, with e = g times the activation's slope at v:
// dx_p = sum_j w_{W - 1 - j} e_{p + j} over the positions p + j of the sequence, plus the gradient of the final state where p is one of the
// last W - 1 positions; for p < 0 that is the gradient of the initial state.  dw_k = sum_p e_p x_{p - W + 1 + k}, dbias = sum_p e_p.
//
// Bound: forward HBM and the loads that are on their way, backward those and vector instructions (47 and 57 % of the cycles): a load's row is cut to the tensor and multiplied
// in 64 bits, and short runs read their weights and the rows before them again.  A thread takes a run of R rows of a few channels with all its loads on their way at once and keeps the window of the last
// W - 1 rows in registers; the W - 1 rows before (backward: and behind) its run it reads again, from the caches.  Sums are 32-bit;
// those of dw go by fixed pieces of the rows, added up in a fixed order: the same inputs give the same bits.
// Measured, 8 sequences of 2048, 2048 channels, 4 taps, bfloat16, inputs in turn: forward 38 us (134 MB, 3.5 TB/s), gradients 71 us (201 MB, 2.8 TB/s: the loads
// of three or four blocks of a compute unit at once, and three times the forward's arithmetic) and 4.6 us for the weights' sums; one token of 64 streams of 4096
// channels 3.9 us.  In memory instead of registers are the rows of float32's gradients (48 to 128 bytes a lane with 2 to 8 taps: the edges' path takes them by a pointer) and, forward, those of
// fewer channels than a pack has (272 bytes).
#include "seq_common.h"

#include <type_traits>

namespace seqamd {
namespace {

constexpr int kThreads = 256;
constexpr int kWidest = 8;
// Rows that a thread takes at once, backward.  8 sequences of 2048, 2048 channels, bfloat16, both directions: 111 us, with 2 rows 128, with 8 109, but in float32, 1024
// channels, whose rows the compiler keeps in memory, 100 and 128.
constexpr int kAtOnce = 4;

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
    int64_t run, blocks, idle;  // backward: rows of a thread; blocks with rows; `idle` ones behind them serve sequences without rows
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

// Gradients: a thread walks a run of rows from its last to its first, U at a time, with the window of the W - 1 values e behind them; the next
// rows are on their way meanwhile.  The W - 1 rows behind its own it goes through first, for their e.
template <typename T, int V, int W, bool PART>
__global__ void __launch_bounds__(kThreads) conv_back_kernel(ConvArgs a)
{
    const int64_t block = int64_t(a.first_block) + blockIdx.x;
    if (block >= a.blocks) return without_rows<T, W>(a, a.grad_end, a.end);
    constexpr int U = kAtOnce, kX = U + W - 1;
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
    // row t with the rows of x up to it: e, and where the row is the run's own its part of the sums
    auto value = [&](const float (&xs)[W][V], const Pack<T, V>& g, bool own) __attribute__((always_inline)) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float sum = bias[v];
#pragma unroll
            for (int k = 0; k < W; ++k) sum = fmaf(w[k][v], xs[k][v], sum);
            e[0][v] = a.silu ? g.get(v) * slope(sum) : g.get(v);
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
    auto load = [&](const T* from, int64_t step, int64_t t) __attribute__((always_inline)) {
        return lane.template load<T>(from + (t < 0 ? 0 : (t < a.rows ? t : a.rows - 1)) * step);
    };
    const int64_t t0 = (int64_t(piece) * groups + group) * a.run, t1 = t0 + a.run < a.rows ? t0 + a.run : a.rows;
    if (t0 < t1) {
        int64_t i = -1, first = 0, past = 0;        // the sequence that the walk is in: none
        // the gradient of the final state, which the last W - 1 positions have
        auto add_end = [&](int64_t p, float* d) __attribute__((always_inline)) {
            const int64_t place = p - (past - first - (W - 1));
            if (!a.grad_end || place < 0) return;
            const Pack<T, V> more = lane.template load<T>(static_cast<const T*>(a.grad_end) + (i * (W - 1) + place) * a.channels);
#pragma unroll
            for (int v = 0; v < V; ++v) d[v] += more.get(v);
        };
        // a row near a sequence's first or last one; xs: the rows of memory up to it
        auto one = [&](const Pack<T, V>* xs, const Pack<T, V>& g, int64_t t, bool own) __attribute__((always_inline)) {
            if (i < 0 || t < first) {
                i = sequence_at(a, t);
                if (i < a.n) rows_of(a, i, first, past);
                if (i >= a.n || t < first || t >= past) {       // of none
                    i = -1;
                    return;
                }
                clear();
            } else if (t == past - 1) {
                clear();
            }
            const int64_t p = t - first;
            float taps[W][V], d[V];
#pragma unroll
            for (int k = 0; k < W; ++k) {
                if (p - (W - 1) + k >= 0)
#pragma unroll
                    for (int v = 0; v < V; ++v) taps[k][v] = xs[k].get(v);
                else row_at<T, V, W, PART>(a, lane, i, first, p - (W - 1) + k, taps[k]);
            }
            value(taps, g, own);
            if (own) {
                derivative(d);
                add_end(p, d);
                lane.template store<T>(static_cast<T*>(a.out) + t * a.channels, d, a.past);
            }
            shift();
            if (own && p == 0) {            // on through the positions of the initial state
#pragma unroll
                for (int k = 1; k < W; ++k) {
#pragma unroll
                    for (int v = 0; v < V; ++v) e[0][v] = 0.0f;
                    derivative(d);
                    add_end(-k, d);
                    lane.template store<T>(static_cast<T*>(a.end) + (i * (W - 1) + (W - 1) - k) * a.channels, d, false);
                    shift();
                }
            }
        };
        clear();
        if constexpr (W > 1) {
            // the rows behind the run, as far as the sequence of its last row goes
            Pack<T, V> xs[2 * (W - 1)], gs[W - 1];
#pragma unroll
            for (int k = 0; k < 2 * (W - 1); ++k) xs[k] = load(x, a.x_step, t1 - (W - 1) + k);
#pragma unroll
            for (int k = 0; k < W - 1; ++k) gs[k] = load(grad, a.grad_step, t1 + k);
            i = sequence_at(a, t1 - 1);
            if (i < a.n) rows_of(a, i, first, past);
            if (i >= a.n || t1 - 1 < first || t1 - 1 >= past) i = -1;
            else
#pragma unroll
                for (int k = W - 2; k >= 0; --k)
                    if (t1 + k < past) one(xs + k, gs[k], t1 + k, false);
        }
        // x[k]: row t - (U - 1) - (W - 1) + k
        Pack<T, V> xs[kX], gs[U], xn[U], gn[U];
        int64_t t = t1 - 1;
#pragma unroll
        for (int k = 0; k < kX; ++k) xs[k] = load(x, a.x_step, t - (U - 1) - (W - 1) + k);
#pragma unroll
        for (int k = 0; k < U; ++k) gs[k] = load(grad, a.grad_step, t - (U - 1) + k);
        for (; t >= t0; t -= U) {
            if (t - U >= t0) {
#pragma unroll
                for (int k = 0; k < U; ++k) xn[k] = load(x, a.x_step, t - U - (U - 1) - (W - 1) + k);
#pragma unroll
                for (int k = 0; k < U; ++k) gn[k] = load(grad, a.grad_step, t - U - (U - 1) + k);
            }
            if (i >= 0 && t - (U - 1) >= t0 && t - (U - 1) - (W - 1) >= first && t < past - W) {
                // nothing but rows of one sequence that are neither its first nor its last ones
#pragma unroll
                for (int r = 0; r < U; ++r) {
                    float taps[W][V], d[V];
#pragma unroll
                    for (int v = 0; v < V; ++v)
#pragma unroll
                        for (int k = 0; k < W; ++k) taps[k][v] = xs[U - 1 - r + k].get(v);
                    value(taps, gs[U - 1 - r], true);
                    derivative(d);
                    lane.template store<T>(static_cast<T*>(a.out) + (t - r) * a.channels, d, a.past);
                    shift();
                }
            } else {
#pragma unroll
                for (int r = 0; r < U; ++r)
                    if (t - r >= t0) one(xs + U - 1 - r, gs[U - 1 - r], t - r, true);
            }
#pragma unroll
            for (int k = W - 2; k >= 0; --k) xs[U + k] = xs[k];
#pragma unroll
            for (int k = 0; k < U; ++k) xs[k] = xn[k], gs[k] = gn[k];
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

__global__ void __launch_bounds__(kSumThreads) conv_weight_kernel(const float* parts, int pieces, int channels, int width, float* dw, float* db, unsigned first_block)
{
    sum_pieces(parts, pieces, int64_t(width + 1) * channels, first_block, [&](int64_t e, float sum) {
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

// Rows of a thread, of 16 bytes each.  8 sequences of 2048, 2048 channels, bfloat16: 38 us, with 8 rows 41, with 24 40; 37 of up to 1500, 997 channels, float16:
// 30, 28 and 29; the first of 1024 channels, float32: 30, 28 and 28.
constexpr int kForwardRows = 16;

// lanes to a row: a power of two, at most a wave
int lanes_for(int packs)
{
    int lanes = 8;
    while (lanes < packs && lanes < 64) lanes *= 2;
    return lanes;
}

// how a row's packs of v channels go to lanes and blocks
void place(ConvArgs& a, int v)
{
    const int packs = (a.channels + v - 1) / v;
    a.lanes = lanes_for(packs);
    a.channel_blocks = (packs + a.lanes - 1) / a.lanes;
}

int64_t idle_blocks(const ConvArgs& a, int width)
{
    if (!a.offsets && a.length) return 0;
    const int64_t blocks = (a.n * (width - 1) * a.channels + kThreads - 1) / kThreads;
    return blocks < 256 ? blocks : 256;
}

// Backward: runs as long as make 4096 waves, of 16 rows at least.  A thread has v = 8 bytes of a row: 8 sequences of 2048, 1024 channels, float32, forward
// and gradients 101 us, with 16 bytes, whose windows leave registers for fewer waves, 132.  Results past the caches from 128 MB on: 8 of 2048, 4096 channels,
// bfloat16, both directions 190 us, kept 205; 2048 channels, float32, 178 and 175; forward alone, 8 of 4096, 4096 channels, bfloat16, 114 and 122.
void place_back(ConvArgs& a, int v)
{
    place(a, v);
    const int64_t groups = kThreads / a.lanes, most = a.channel_blocks < 1024 ? 1024 / a.channel_blocks * groups : groups;
    a.run = (a.rows + most - 1) / most;
    a.run = ((a.run > 16 ? a.run : 16) + kAtOnce - 1) / kAtOnce * kAtOnce;
    a.pieces = int((a.rows + a.run * groups - 1) / (a.run * groups));
}

// no fewer than those of any type
int most_pieces(int64_t rows, int channels)
{
    int most = 0;
    for (int v = 2; v <= 4; v += 2) {
        ConvArgs a{};
        a.rows = rows, a.channels = channels;
        place_back(a, v);
        most = a.pieces > most ? a.pieces : most;
    }
    return most;
}

void check_sizes(uint64_t width, uint64_t rows, uint64_t channels, uint64_t n)
{
    require(width >= 1 && width <= kWidest, "a convolution has 1 to 8 taps");
    require(channels < (uint64_t(1) << 27) && rows < (uint64_t(1) << 31) && n < (uint64_t(1) << 31), "too many rows, channels or sequences");
}

void check(const ConvArgs& a, uint64_t width, uint64_t rows, uint64_t channels, uint64_t n, uint64_t length)
{
    check_sizes(width, rows, channels, n);
    if (!a.offsets) check_rows(n, length, rows);
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
                place(a, V);
                const int64_t each = int64_t(kForwardRows) * (kThreads / a.lanes);
                a.blocks = (a.rows + each - 1) / each * a.channel_blocks;
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
        check_sizes(width, rows, channels, 0);
        if (rows && channels) bytes = uint64_t(most_pieces(int64_t(rows), int(channels))) * (width + 1) * channels * sizeof(float);
    });
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
                constexpr int V = 8 / sizeof(T);
                with_width(width, [&](auto w) {
                    constexpr int W = decltype(w)::value;
                    place_back(a, V);
                    pieces = a.pieces;
                    a.blocks = int64_t(pieces) * a.channel_blocks;
                    a.past = goes_past(uint64_t(a.rows) * a.channels * sizeof(T), uint64_t(a.channels) * sizeof(T));
                    a.idle = idle_blocks(a, W);
                    const int64_t blocks = a.blocks + a.idle;
                    if (a.channels < V) launch_all(conv_back_kernel<T, V, W, true>, blocks, kThreads, static_cast<hipStream_t>(stream), a);
                    else launch_all(conv_back_kernel<T, V, W, false>, blocks, kThreads, static_cast<hipStream_t>(stream), a);
                });
            });
        in_launches(sum_blocks(int64_t(width + 1) * a.channels), kSumThreads, [&](unsigned first, dim3 grid) {
            hipLaunchKernelGGL(conv_weight_kernel, grid, dim3(kSumThreads), 0, static_cast<hipStream_t>(stream), a.parts, pieces, a.channels, int(width), grad_weight,
                               grad_bias, first);
        });
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
