// Gated linear recurrence h_t = exp(g_t) h_{t-1} + x_t for each channel, over sequences of any length, forward and
// backward, and one step of it against a kept state.
//
// Mathematics.  A run of steps maps the state before it to the state behind it by h -> A h + B with A the product of its
// decays; two runs behind each other compose to (A1 A2, A2 B1 + B2).  Sequences packed behind each other are one run whose
// decays are zero where a sequence begins.  Backward, c_t = exp(g_t) (G_t + c_{t+1}) is the same kind of recurrence from
// the other end: dx_t = G_t + c_{t+1}, dg_t = c_t h_{t-1}, and c at a sequence's first step is the gradient of its initial
// state.
//
// Bound: HBM.  Every element is read once and written once: a block holds a chunk of steps of its channels in registers,
// publishes the chunk's (A, B), collects those of the chunks before it back to one that is the state itself, and only then
// walks its steps.  States, products and sums are 32-bit whatever the element type.
#include "seq_common.h"

#include <type_traits>

namespace seqamd {
namespace {

constexpr int kThreads = 256;
constexpr int kWindow = 32;      // chunks that a block looks back at once

struct ScanArgs {
    const void* gate;        // log decays
    const void* in;          // forward: x; backward: gradients of h
    const void* h;           // backward: the states of the forward
    void* out;               // forward: h; backward: dx
    void* out2;              // backward: dg
    const float* begin;      // forward: initial states [n][channels] or null; backward: gradients of the final states or null
    const float* init;       // backward: initial states or null
    float* end;              // forward: final states; backward: gradients of the initial states
    const int* offsets;      // [n + 1] rows where sequences begin, or null: n sequences of `length` rows
    unsigned long long* words;   // [chunks][channels] what the chunks publish, zero at the start
    unsigned* ticket;        // zero at the start
    int64_t rows, gate_stride, in_stride;
    int64_t length, n;
    int channels, channel_blocks, chunks;
};

// A chunk's word for a channel: B in the low half, A in the high half with its sign bit set (A is a product of
// exponentials).  Zero: not there yet.  A word whose A is zero holds the state itself.  Both halves travel in one 64-bit
// access, so no order between accesses is needed.
__device__ __forceinline__ void publish(unsigned long long* w, float a, float b)
{
    const unsigned long long v = (static_cast<unsigned long long>(__float_as_uint(a) | 0x80000000u) << 32) | __float_as_uint(b);
    __hip_atomic_store(w, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The word, waited for.  The wait ends: a block takes its chunk from a counter when it starts to run, so the chunk waited
// for is held by a block that already runs, and a block publishes its word before it waits for any other.
__device__ __forceinline__ unsigned long long collect(const unsigned long long* w)
{
    unsigned long long v;
    while (!((v = __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) >> 63)) __builtin_amdgcn_s_sleep(1);
    return v;
}

__device__ __forceinline__ float word_a(unsigned long long v) { return __uint_as_float(static_cast<unsigned>(v >> 32) & 0x7fffffffu); }
__device__ __forceinline__ float word_b(unsigned long long v) { return __uint_as_float(static_cast<unsigned>(v)); }

// A product that overflowed to infinity takes nothing from a state of zero, one of zero nothing from any state
__device__ __forceinline__ float apply(float a, float b, float h) { return h == 0.0f || a == 0.0f ? b : fmaf(a, h, b); }

// A run whose product is zero forgets whatever came before it, also after a product that overflowed
__device__ __forceinline__ float chain(float a1, float a2) { return a1 == 0.0f || a2 == 0.0f ? 0.0f : a1 * a2; }

// 16-bit gates carry at most 11 bits: the hardware exponential of the scaled argument is far below their rounding
template <typename T>
__device__ __forceinline__ float decay(float g)
{
    if constexpr (sizeof(T) == 4) return expf(g);
    else return __expf(g);
}

// Rows [t0, t0 + ROWS) of the packed rows: at[r] = the sequence that begins (forward) or ends (backward) at row t0 + r,
// ends[r] = the sequence that ends (forward) or begins (backward) there, -1: none.  Returns whether there is any.
template <int ROWS, bool BACK>
__device__ bool find_edges(const ScanArgs& p, int64_t t0, int* at, int* ends)
{
    const int tid = threadIdx.x;
    for (int r = tid; r < ROWS; r += kThreads) at[r] = ends[r] = -1;
    __syncthreads();
    int found = 0;
    auto mark = [&](int64_t i, int64_t first, int64_t last) {
        if (first >= t0 && first < t0 + ROWS) {
            (BACK ? ends : at)[first - t0] = int(i);
            found = 1;
        }
        if (last >= t0 && last < t0 + ROWS) {
            (BACK ? at : ends)[last - t0] = int(i);
            found = 1;
        }
    };
    if (p.offsets) {
        // many sequences: the first that can touch these rows, by bisection (the offsets ascend)
        int64_t lo = 0, hi = p.n;
        if (p.n > 4 * kThreads)
            while (lo < hi) {
                const int64_t mid = (lo + hi) / 2;
                if (p.offsets[mid + 1] <= t0) lo = mid + 1;
                else hi = mid;
            }
        else
            lo = 0;
        for (int64_t base = lo; base < p.n; base += kThreads) {
            const int64_t i = base + tid;
            int64_t first = t0 + ROWS;
            if (i < p.n) {
                first = p.offsets[i];
                const int64_t past = p.offsets[i + 1];
                if (first >= 0 && past > first && past <= p.rows) mark(i, first, past - 1);
            }
            if (__syncthreads_and(first >= t0 + ROWS)) break;
        }
    } else {
        for (int r = tid; r < ROWS; r += kThreads) {
            const int64_t t = t0 + r, i = t / p.length, s = t - i * p.length;
            if (t >= 0 && t < p.rows && (s == 0 || s == p.length - 1)) mark(i, s == 0 ? t : -1, s == p.length - 1 ? t : -1);
        }
    }
    return __syncthreads_or(found) != 0;
}

// A block: ROWS = R * kThreads / LC rows of LC * V channels; a thread walks R rows of V channels.
// Backward mirrors the rows: "row r" of a block is the r-th from the end.
template <typename T, int V, int R, int LC, bool BACK>
__global__ void __launch_bounds__(kThreads) scan_kernel(ScanArgs p)
{
    constexpr int kGroups = kThreads / LC, kRows = R * kGroups, kEach = kWindow / kGroups;
    using P = Pack<T, V>;
    __shared__ int s_at[kRows], s_ends[kRows];
    __shared__ float s_a[kGroups][LC * V], s_b[kGroups][LC * V];
    __shared__ unsigned long long s_words[kWindow][LC * V];
    __shared__ float s_carry[LC * V];
    __shared__ unsigned s_ticket;
    const int tid = threadIdx.x, lane = tid % LC, group = tid / LC;
    if (tid == 0) s_ticket = atomicAdd(p.ticket, 1u);
    __syncthreads();
    const int chunk = s_ticket / p.channel_blocks, cb = s_ticket % p.channel_blocks;
    const int ch0 = cb * LC * V + lane * V;
    const int count = p.channels - ch0 < 0 ? 0 : (p.channels - ch0 > V ? V : p.channels - ch0);
    // first row in memory of the chunk; mirrored, chunk 0 holds the last rows
    const int64_t t0 = BACK ? p.rows - int64_t(chunk + 1) * kRows : int64_t(chunk) * kRows;
    auto row_of = [&](int r) { return BACK ? t0 + kRows - 1 - r : t0 + r; };

    P gate[R], in[R], prev[BACK ? R : 1];
    const T* gp = static_cast<const T*>(p.gate) + ch0;
    const T* ip = static_cast<const T*>(p.in) + ch0;
    const T* hp = static_cast<const T*>(p.h) + ch0;
    const bool whole = t0 >= (BACK ? 1 : 0) && t0 + kRows <= p.rows && (cb + 1) * LC * V <= p.channels;
    if (whole) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t t = row_of(group * R + r);
            gate[r] = load_pack<T, V>(gp + t * p.gate_stride);
            in[r] = load_pack<T, V>(ip + t * p.in_stride);
            if constexpr (BACK) prev[r] = load_pack<T, V>(hp + (t - 1) * int64_t(p.channels));
        }
    } else {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t t = row_of(group * R + r);
            const int have = t >= 0 && t < p.rows ? count : 0;
            gate[r] = load_some<T, V>(gp + t * p.gate_stride, have);
            in[r] = load_some<T, V>(ip + t * p.in_stride, have);
            if constexpr (BACK) prev[r] = load_some<T, V>(hp + (t - 1) * int64_t(p.channels), t >= 1 && t < p.rows ? count : 0);
        }
    }
    const bool edges = find_edges<kRows, BACK>(p, t0, s_at, s_ends);
    auto at_of = [&](int r) { return s_at[BACK ? kRows - 1 - r : r]; };
    auto ends_of = [&](int r) { return s_ends[BACK ? kRows - 1 - r : r]; };
    auto state_at = [&](const float* s, int64_t seq, int v) { return s && v < count ? s[seq * p.channels + ch0 + v] : 0.0f; };

    // the thread's rows as one map
    float a[V], b[V];
#pragma unroll
    for (int v = 0; v < V; ++v) a[v] = 1.0f, b[v] = 0.0f;
    auto fold = [&](auto all) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (edges) {
                const int seq = at_of(group * R + r);
                if (seq >= 0)
#pragma unroll
                    for (int v = 0; v < V; ++v) a[v] = 0.0f, b[v] = state_at(p.begin, seq, v);
            }
            const int64_t t = row_of(group * R + r);
            if (!decltype(all)::value && (t < 0 || t >= p.rows)) continue;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float d = decay<T>(gate[r].get(v)), x = in[r].get(v);
                a[v] *= d;
                b[v] = BACK ? d * (b[v] + x) : fmaf(d, b[v], x);
            }
        }
    };
    if (whole) fold(std::true_type{});
    else fold(std::false_type{});
#pragma unroll
    for (int v = 0; v < V; ++v) {
        s_a[group][lane * V + v] = a[v];
        s_b[group][lane * V + v] = b[v];
    }
    __syncthreads();
    // what the groups before this one do to the state, and (for the last group) the chunk as a whole
    float before_a[V], before_b[V];
#pragma unroll
    for (int v = 0; v < V; ++v) before_a[v] = 1.0f, before_b[v] = 0.0f;
    for (int g = 0; g < group; ++g)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float ga = s_a[g][lane * V + v];
            before_b[v] = apply(ga, s_b[g][lane * V + v], before_b[v]);
            before_a[v] = chain(before_a[v], ga);
        }
    unsigned long long* const words = p.words + ch0;
    if (group == kGroups - 1 && p.chunks > 1)
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v < count) publish(words + int64_t(chunk) * p.channels + v, chunk ? chain(before_a[v], a[v]) : 0.0f, apply(a[v], b[v], before_b[v]));
    // the chunks before this one, back to the nearest that holds the state, then forward from it one after the other: the
    // same products and sums in the same order wherever it was found, so the same inputs give the same bits
    float carry[V];
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = 0.0f;
    if (chunk) {
        unsigned long long got[kEach][V];
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int c = chunk - 1 - group * kEach - k;
#pragma unroll
            for (int v = 0; v < V; ++v)
                got[k][v] = c >= 0 && v < count ? __hip_atomic_load(words + int64_t(c) * p.channels + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 1ull << 63;
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int c = chunk - 1 - group * kEach - k;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (!(got[k][v] >> 63)) got[k][v] = collect(words + int64_t(c) * p.channels + v);
                s_words[group * kEach + k][v * LC + lane] = got[k][v];
            }
        }
        __syncthreads();
        for (int e = tid; e < LC * V; e += kThreads) {
            int k = 0;
            while (k < kWindow && word_a(s_words[k][e]) != 0.0f) ++k;
            float h;
            if (k < kWindow) {
                h = word_b(s_words[k][e]);
            } else {
                // none of them: the oldest turns into the state once the ones before it have
                k = kWindow - 1;
                const unsigned long long* w = p.words + int64_t(chunk - kWindow) * p.channels + cb * LC * V + (e % LC) * V + e / LC;
                unsigned long long got;
                while (word_a(got = collect(w)) != 0.0f) __builtin_amdgcn_s_sleep(1);
                h = word_b(got);
            }
            while (--k >= 0) h = apply(word_a(s_words[k][e]), word_b(s_words[k][e]), h);
            s_carry[e] = h;
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = s_carry[v * LC + lane];
    }
    if (group == kGroups - 1 && chunk && chunk + 1 < p.chunks)
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v < count)
                publish(words + int64_t(chunk) * p.channels + v, 0.0f, apply(chain(before_a[v], a[v]), apply(a[v], b[v], before_b[v]), carry[v]));

    float state[V];
#pragma unroll
    for (int v = 0; v < V; ++v) state[v] = apply(before_a[v], before_b[v], carry[v]);
    T* op = static_cast<T*>(p.out) + ch0;
    T* op2 = static_cast<T*>(p.out2) + ch0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        gate[r].renew();
        in[r].renew();
    }
    auto walk = [&](auto all) {
        constexpr bool kAll = decltype(all)::value;
        auto put = [&](T* q, const P& o) {
            if constexpr (kAll) store_pack<T, V>(q, o);
            else store_some<T, V>(q, o, count);
        };
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t t = row_of(group * R + r);
            if (!kAll && (t < 0 || t >= p.rows)) continue;
            int last = -1;
            if (edges) {
                const int seq = at_of(group * R + r);
                last = ends_of(group * R + r);
                if (seq >= 0)
#pragma unroll
                    for (int v = 0; v < V; ++v) state[v] = state_at(p.begin, seq, v);
            }
            P o;
            if constexpr (!BACK) {
#pragma unroll
                for (int v = 0; v < V; ++v) state[v] = fmaf(decay<T>(gate[r].get(v)), state[v], in[r].get(v));
                o.set(state);
                put(op + t * p.channels, o);
            } else {
                float e[V], dg[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    e[v] = state[v] + in[r].get(v);
                    state[v] = decay<T>(gate[r].get(v)) * e[v];
                    dg[v] = state[v] * (last >= 0 ? state_at(p.init, last, v) : prev[r].get(v));
                }
                o.set(e);
                put(op + t * p.channels, o);
                o.set(dg);
                put(op2 + t * p.channels, o);
            }
            if (last >= 0)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (v < count) p.end[int64_t(last) * p.channels + ch0 + v] = state[v];
        }
    };
    if (whole) walk(std::true_type{});
    else walk(std::false_type{});
}

__global__ void __launch_bounds__(kThreads) prepare_kernel(unsigned long long* words, int64_t count, unsigned* ticket, const float* begin, float* end,
                                                           const int* offsets, int64_t n, int64_t length, int64_t rows, int channels)
{
    const int64_t step = int64_t(gridDim.x) * kThreads, first = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    for (int64_t i = first; i < count; i += step) words[i] = 0;
    if (first == 0) *ticket = 0;
    // sequences without steps: the state behind them is the state before them
    if (offsets || length == 0)
        for (int64_t i = first; i < n * channels; i += step) {
            const int64_t s = i / channels;
            if (length == 0 || offsets[s] >= offsets[s + 1]) end[i] = begin ? begin[i] : 0.0f;
        }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) step_kernel(const T* x, const T* gate, float* state, T* out, int64_t n, int channels, int64_t x_stride, int64_t gate_stride, int packs)
{
    const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= n * packs) return;
    const int64_t row = i / packs;
    const int ch = int(i - row * packs) * V, count = channels - ch > V ? V : channels - ch;
    const Pack<T, V> a = load_some<T, V>(gate + row * gate_stride + ch, count), b = load_some<T, V>(x + row * x_stride + ch, count);
    Pack<float, V> s = load_some<float, V>(state + row * channels + ch, count);
    Pack<T, V> o;
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = fmaf(decay<T>(a.get(v)), s.get(v), b.get(v));
    s.set(h);
    o.set(h);
    store_some<float, V>(state + row * channels + ch, s, count);
    store_some<T, V>(out + row * channels + ch, o, count);
}

// A chunk holds 128 rows of 256 bytes where there are channels enough, 512 rows of 64 bytes where there are few
template <typename T>
struct Shape {
    static constexpr int V = 8 / sizeof(T), R = 16, kWide = 32, kNarrow = 8;
};

struct Plan {
    int rows, lanes, chunks, channel_blocks;
};

template <typename T>
Plan plan_of(int64_t rows, int channels)
{
    using S = Shape<T>;
    Plan p;
    p.lanes = channels <= S::kNarrow * S::V ? S::kNarrow : S::kWide;
    p.rows = S::R * kThreads / p.lanes;
    const int64_t chunks = (rows + p.rows - 1) / p.rows, blocks = (channels + p.lanes * S::V - 1) / (p.lanes * S::V);
    require(chunks * blocks < (int64_t(1) << 31), "the sequences are too long");
    p.chunks = int(chunks);
    p.channel_blocks = int(blocks);
    return p;
}

constexpr size_t kTicketBytes = 256;

template <typename T>
size_t scan_workspace(int64_t rows, int channels)
{
    const Plan p = plan_of<T>(rows, channels);
    return kTicketBytes + (p.chunks > 1 ? size_t(p.chunks) * channels * sizeof(unsigned long long) : 0);
}

template <typename T, bool BACK>
void scan(ScanArgs p, void* workspace, size_t bytes, hipStream_t stream)
{
    using S = Shape<T>;
    if (p.n * p.channels == 0) return;
    const Plan plan = plan_of<T>(p.rows, p.channels);
    require(bytes >= scan_workspace<T>(p.rows, p.channels) && workspace, "the workspace is too small");
    p.ticket = static_cast<unsigned*>(workspace);
    p.words = reinterpret_cast<unsigned long long*>(static_cast<char*>(workspace) + kTicketBytes);
    p.chunks = plan.chunks;
    p.channel_blocks = plan.channel_blocks;
    const int64_t words = plan.chunks > 1 ? int64_t(plan.chunks) * p.channels : 0;
    const int64_t todo = words > p.n * p.channels ? words : p.n * p.channels;
    const int64_t blocks = (todo + kThreads - 1) / kThreads;
    hipLaunchKernelGGL(prepare_kernel, dim3(blocks > 1024 ? 1024 : unsigned(blocks)), dim3(kThreads), 0, stream, p.words, words, p.ticket, p.begin, p.end,
                       p.offsets, p.n, p.length, p.rows, p.channels);
    SIG_HIP(hipGetLastError());
    if (p.rows == 0) return;
    const dim3 grid(unsigned(plan.chunks) * unsigned(plan.channel_blocks));
    if (plan.lanes == S::kWide)
        hipLaunchKernelGGL((scan_kernel<T, S::V, S::R, S::kWide, BACK>), grid, dim3(kThreads), 0, stream, p);
    else
        hipLaunchKernelGGL((scan_kernel<T, S::V, S::R, S::kNarrow, BACK>), grid, dim3(kThreads), 0, stream, p);
    SIG_HIP(hipGetLastError());
}

void check_scan(uint64_t rows, uint64_t channels, uint64_t n, uint64_t length, const int* offsets)
{
    require(channels < (uint64_t(1) << 31) && rows < (uint64_t(1) << 31) && n < (uint64_t(1) << 31), "too many rows, channels or sequences");
    require(channels == 0 || rows < (uint64_t(1) << 60) / channels, "the sequences are too long");
    require(offsets || n * length == rows, "rows are not sequences times length");
}

}  // namespace
}  // namespace seqamd

using namespace seqamd;

extern "C" {

__attribute__((visibility("default"))) uint64_t cusig_amd_linear_recurrence_workspace(int dtype, uint64_t rows, uint64_t channels) noexcept
{
    uint64_t bytes = 0;
    sigamd::guarded([&] {
        check_scan(rows, channels, 0, 0, reinterpret_cast<const int*>(1));
        with_type(dtype, [&](auto t) { bytes = scan_workspace<decltype(t)>(int64_t(rows), int(channels)); });
    });
    return bytes;
}

__attribute__((visibility("default"))) int cusig_amd_linear_recurrence(
    int dtype, const void* x, const void* log_decay, const float* initial_state, void* h, float* final_state, const int* offsets, uint64_t sequences,
    uint64_t length, uint64_t rows, uint64_t channels, int64_t x_stride, int64_t log_decay_stride, void* workspace, uint64_t workspace_bytes, void* stream) noexcept
{
    return sigamd::guarded([&] {
        check_scan(rows, channels, sequences, length, offsets);
        ScanArgs p{};
        p.gate = log_decay;
        p.in = x;
        p.out = h;
        p.begin = initial_state;
        p.end = final_state;
        p.offsets = offsets;
        p.rows = int64_t(rows);
        p.gate_stride = log_decay_stride;
        p.in_stride = x_stride;
        p.length = int64_t(length);
        p.n = int64_t(sequences);
        p.channels = int(channels);
        with_type(dtype, [&](auto t) { scan<decltype(t), false>(p, workspace, workspace_bytes, static_cast<hipStream_t>(stream)); });
    });
}

__attribute__((visibility("default"))) int cusig_amd_linear_recurrence_backprop(
    int dtype, const void* h, const void* log_decay, const void* grad_h, const float* grad_final, const float* initial_state, void* grad_x,
    void* grad_log_decay, float* grad_initial, const int* offsets, uint64_t sequences, uint64_t length, uint64_t rows, uint64_t channels,
    int64_t log_decay_stride, int64_t grad_stride, void* workspace, uint64_t workspace_bytes, void* stream) noexcept
{
    return sigamd::guarded([&] {
        check_scan(rows, channels, sequences, length, offsets);
        ScanArgs p{};
        p.gate = log_decay;
        p.in = grad_h;
        p.h = h;
        p.out = grad_x;
        p.out2 = grad_log_decay;
        p.begin = grad_final;
        p.init = initial_state;
        p.end = grad_initial;
        p.offsets = offsets;
        p.rows = int64_t(rows);
        p.gate_stride = log_decay_stride;
        p.in_stride = grad_stride;
        p.length = int64_t(length);
        p.n = int64_t(sequences);
        p.channels = int(channels);
        with_type(dtype, [&](auto t) { scan<decltype(t), true>(p, workspace, workspace_bytes, static_cast<hipStream_t>(stream)); });
    });
}

__attribute__((visibility("default"))) int cusig_amd_linear_recurrence_step(
    int dtype, const void* x, const void* log_decay, float* state, void* h, uint64_t rows, uint64_t channels, int64_t x_stride, int64_t log_decay_stride,
    void* stream) noexcept
{
    return sigamd::guarded([&] {
        check_scan(rows, channels, rows, 1, nullptr);
        if (rows * channels == 0) return;
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            constexpr int V = 4;
            const uint64_t packs = (channels + V - 1) / V, blocks = (rows * packs + kThreads - 1) / kThreads;
            require(blocks < (uint64_t(1) << 31), "too many rows and channels");
            hipLaunchKernelGGL((step_kernel<T, V>), dim3(unsigned(blocks)), dim3(kThreads), 0, static_cast<hipStream_t>(stream), static_cast<const T*>(x),
                               static_cast<const T*>(log_decay), state, static_cast<T*>(h), int64_t(rows), int(channels), x_stride, log_decay_stride, int(packs));
            SIG_HIP(hipGetLastError());
        });
    });
}

}  // extern "C"
