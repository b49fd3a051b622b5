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
// walks its steps.  States, products and sums are 32-bit whatever the element type.  One sequence of 100003 steps of 384 channels,
// float32: 110 us, 4.2 TB/s; forward and gradients of 8 of 2048 steps of 2048 channels, bfloat16: 147 us, 3.7 TB/s.  Odd rows of
// 16 bits lie across the words that lanes load: 37 of up to 1500 steps of 997 channels, float16, 146 us, 2.5 TB/s.
#include "seq_common.h"

#include <type_traits>

namespace seqamd {
namespace {

constexpr int kThreads = 256;
constexpr int kTicketStep = 64;  // words between the counters of two channel blocks

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
    unsigned* ticket;        // [channel_blocks][kTicketStep] zero at the start
    int64_t rows, gate_stride, in_stride;
    int64_t length, n;
    int channels, channel_blocks, chunks;
    bool past;               // results go past the caches
    unsigned first_block;    // of a launch
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

// A decay that is zero forgets whatever came before it, also what is not finite, and a run's product is zero where it has one or a
// sequence begins in it.  Other products stop at the smallest positive number, so that a state that is not finite goes through them
// wherever in a chunk their steps lie; to a finite one that adds at most 5e-7.
__device__ __forceinline__ float at_least(float a) { return a < 1.401298464e-45f ? 1.401298464e-45f : a; }

__device__ __forceinline__ float chain(float a1, float a2) { return a1 == 0.0f || a2 == 0.0f ? 0.0f : at_least(a1 * a2); }

// The hardware's exponential of the scaled argument: off by |g| 2^-24 of its size from the scaling and one rounding
__device__ __forceinline__ float decay(float g) { return __builtin_amdgcn_exp2f(g * 1.44269504088896341f); }

// The rows [first, past) of a packed sequence, kept inside the tensors whatever the offsets hold
__device__ __forceinline__ void rows_of(const int* offsets, int64_t i, int64_t rows, int64_t& first, int64_t& past)
{
    first = kept(offsets[i], 0, rows);
    past = kept(offsets[i + 1], first, rows);
}

// a step: a product with a decay of zero is zero, whatever the state
__device__ __forceinline__ float next_state(float d, float h, float x) { return weighed(d, h) + x; }

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
            int64_t first = t0 + ROWS, past;
            if (i < p.n) {
                rows_of(p.offsets, i, p.rows, first, past);
                if (past > first) mark(i, first, past - 1);
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
// A lane whose channels would end behind the last takes the last V instead: what several lanes form, they form alike.  Rows
// behind the end are loaded from the last one; nothing follows them, and they are not stored.  PART: fewer than V channels.
template <typename T, int V, int R, int LC, bool BACK, bool PART, bool PAST>
__global__ void __launch_bounds__(kThreads, PART ? 1 : (BACK || R > 16 ? 3 : 4)) scan_kernel(ScanArgs p)
{
    constexpr int kGroups = kThreads / LC, kRows = R * kGroups, kWindow = kGroups < 16 ? 16 : kGroups, kEach = kWindow / kGroups;
    using P = Pack<T, V>;
    __shared__ int s_at[kRows], s_ends[kRows];
    __shared__ float s_a[kGroups][LC * V], s_b[kGroups][LC * V];
    __shared__ unsigned long long s_words[kWindow][LC * V];
    __shared__ float s_carry[LC * V];
    __shared__ unsigned s_ticket;
    const int tid = threadIdx.x, lane = tid % LC, group = tid / LC;
    // The chunks of a channel block are counted by a number of its own: 2048 blocks on a single one took 18 ns each, one after
    // the other, a third of the call.
    const int cb = (p.first_block + blockIdx.x) % p.channel_blocks;
    if (tid == 0) s_ticket = atomicAdd(p.ticket + cb * kTicketStep, 1u);
    __syncthreads();
    const int chunk = s_ticket;
    const int ch0 = PART ? lane * V : min(cb * LC * V + lane * V, p.channels - V);
    const int count = PART ? max(0, min(p.channels - ch0, V)) : V;
    // first row in memory of the chunk; mirrored, chunk 0 holds the last rows
    const int64_t t0 = BACK ? p.rows - int64_t(chunk + 1) * kRows : int64_t(chunk) * kRows;
    auto row_of = [&](int r) { return BACK ? t0 + kRows - 1 - r : t0 + r; };
    // rows of sequences: those before and behind them are not written
    int first_row = 0, past_row = int(p.rows);
    if (p.offsets) {
        first_row = __builtin_amdgcn_readfirstlane(int(kept(p.offsets[0], 0, p.rows)));
        past_row = __builtin_amdgcn_readfirstlane(int(kept(p.offsets[p.n], first_row, p.rows)));
    }

    P gate[R], in[R], prev[BACK ? R : 1];
    const bool whole = t0 >= (BACK ? 1 : 0) && t0 + kRows <= p.rows;
    // a row of the first group at an address that is the same for all lanes, the lane's place at an offset from it
    auto load = [&](P* to, const void* from, int64_t stride, int back) __attribute__((always_inline)) {
        const T* const base = static_cast<const T*>(from);
        if (whole && !PART) {
            const int64_t first = BACK ? t0 + R - 1 - back : t0;
            const int at = (BACK ? kGroups - 1 - group : group) * R * int(stride) + ch0;
#pragma unroll
            for (int r = 0; r < R; ++r) to[r] = load_pack<T, V>(base + (BACK ? first - r : first + r) * stride + unsigned(at));
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t t = row_of(group * R + r) - back, row = t < 0 ? 0 : (t >= p.rows ? p.rows - 1 : t);
                to[r] = PART ? load_some<T, V>(base + row * stride + ch0, count) : load_pack<T, V>(base + row * stride + ch0);
            }
        }
    };
    load(gate, p.gate, p.gate_stride, 0);
    load(in, p.in, p.in_stride, 0);
    if constexpr (BACK) load(prev, p.h, p.channels, 1);
    const bool edges = find_edges<kRows, BACK>(p, t0, s_at, s_ends);
    auto at_of = [&](int r) { return s_at[BACK ? kRows - 1 - r : r]; };
    auto ends_of = [&](int r) { return s_ends[BACK ? kRows - 1 - r : r]; };
    auto state_at = [&](const float* s, int64_t seq, int v) { return s && v < count ? s[seq * p.channels + ch0 + v] : 0.0f; };

    // the thread's rows as one map
    float a[V], b[V], least[V];         // least: the smallest decay, zero where a sequence begins
#pragma unroll
    for (int v = 0; v < V; ++v) a[v] = least[v] = 1.0f, b[v] = 0.0f;
    {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (edges) {
                const int seq = at_of(group * R + r);
                if (seq >= 0)       // a too: with no need of its own, but rows whose work is apart spill registers
#pragma unroll
                    for (int v = 0; v < V; ++v) a[v] = least[v] = 0.0f, b[v] = state_at(p.begin, seq, v);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float d = decay(gate[r].get(v)), x = in[r].get(v);
                a[v] *= d;
                least[v] = fminf(least[v], d);
                b[v] = BACK ? weighed(d, b[v] + x) : next_state(d, b[v], x);
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) a[v] = least[v] == 0.0f ? 0.0f : at_least(a[v]);
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
                const unsigned long long* w = p.words + int64_t(chunk - kWindow) * p.channels + (PART ? (e % LC) * V : min(cb * LC * V + (e % LC) * V, p.channels - V)) + e / LC;
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
    auto walk = [&](auto all) __attribute__((always_inline)) {
        constexpr bool kAll = decltype(all)::value;
        auto put = [&](T* q, const P& o) __attribute__((always_inline)) {
            if constexpr (PART) store_some<T, V>(q, o, count);
            else if constexpr (kAll && PAST) store_past<T, V>(q, o);
            else store_pack<T, V>(q, o);
        };
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t t = row_of(group * R + r);
            if (!kAll && (t < first_row || t >= past_row)) continue;
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
                for (int v = 0; v < V; ++v) state[v] = next_state(decay(gate[r].get(v)), state[v], in[r].get(v));
                o.set(state);
                put(op + t * p.channels, o);
            } else {
                float e[V], dg[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    e[v] = state[v] + in[r].get(v);
                    state[v] = weighed(decay(gate[r].get(v)), e[v]);
                    float h = prev[r].get(v);
                    if (last >= 0) h = state_at(p.init, last, v);
                    dg[v] = weighed(state[v], h);
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
    if (whole && !PART && t0 >= first_row && t0 + kRows <= past_row) walk(std::true_type{});
    else walk(std::false_type{});
}

// Many sequences or channels: a block walks the whole of a sequence for LC * V channels, a chunk of kRows rows after the other, with
// the next chunk's rows on their way meanwhile.  Nothing is published and nothing waited for.  A wave's lanes are 64 / LC pieces of
// R rows each; their maps meet in a scan over the lanes, those of the four waves in shared memory.
template <typename T, int V, int R, int LC, bool BACK>
__global__ void __launch_bounds__(kThreads, 2) column_kernel(ScanArgs p)
{
    constexpr int kPieces = 64 / LC, kWaves = kThreads / 64, kRows = R * kPieces * kWaves;
    using P = Pack<T, V>;
    __shared__ float s_a[2][kWaves][LC * V], s_b[2][kWaves][LC * V];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, channel_lane = lane % LC, piece = lane / LC;
    // Blocks go around the eight dies: each die takes neighbouring channel blocks, which share cache lines, a sequence's all together (37
    // of up to 1500 steps, 997 channels, float16, gradients: 90 us, an eighth of every sequence to a die 97, the longest first
    // besides 82; but of equal lengths 68, 84 and 86).
    const unsigned all = unsigned(p.n) * unsigned(p.channel_blocks), block = p.first_block + blockIdx.x, die = block % 8, each = all / 8, more = all % 8;
    const unsigned id = die * each + min(die, more) + block / 8;
    const int seq = id / p.channel_blocks, cb = id % p.channel_blocks;
    int64_t begin = int64_t(seq) * p.length, rows = p.length;
    if (p.offsets) {
        rows_of(p.offsets, seq, p.rows, begin, rows);
        rows -= begin;
    }
    begin = __builtin_amdgcn_readfirstlane(int(begin));
    rows = __builtin_amdgcn_readfirstlane(int(rows));
    const int ch0 = min(cb * LC * V + channel_lane * V, p.channels - V);
    const int own = (wave * kPieces + piece) * R;              // the thread's first row of a chunk, from the sequence's begin (backward: its end)
    float carry[V];
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = p.begin ? p.begin[int64_t(seq) * p.channels + ch0 + v] : 0.0f;

    if (rows <= 0) {                            // the state behind no steps is the state before them
        if (wave + piece == 0)
#pragma unroll
            for (int v = 0; v < V; ++v) p.end[int64_t(seq) * p.channels + ch0 + v] = carry[v];
        return;
    }
    const int64_t chunks = (rows + kRows - 1) / kRows;
    // a chunk's r-th row of the piece that is first in memory, the same for all lanes; the others' at a distance from it
    auto place = [&](int64_t chunk, int r) { return BACK ? begin + rows - 1 - chunk * kRows - (kRows - R) - r : begin + chunk * kRows + r; };
    const int apart = BACK ? kRows - R - own : own;

    P next_gate[R], next_in[R], next_prev[BACK ? R : 1];
    auto load = [&](P* to, const void* from, int64_t stride, int64_t chunk, int back) __attribute__((always_inline)) {
        const T* const base = static_cast<const T*>(from);
        if (chunk + 1 < chunks) {
            const unsigned at = unsigned(apart * int(stride) + ch0);
#pragma unroll
            for (int r = 0; r < R; ++r) to[r] = load_pack<T, V>(base + (place(chunk, r) - back) * stride + at);
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r) {       // rows past the sequence's end: the last one in their place
                const int64_t t = min(chunk * kRows + own + r, rows - 1), row = BACK ? max(begin + rows - 1 - t - back, int64_t(0)) : begin + t;
                to[r] = load_pack<T, V>(base + row * stride + ch0);
            }
        }
    };
    auto fetch = [&](int64_t chunk) __attribute__((always_inline)) {
        load(next_gate, p.gate, p.gate_stride, chunk, 0);
        load(next_in, p.in, p.in_stride, chunk, 0);
        if constexpr (BACK) load(next_prev, p.h, p.channels, chunk, 1);
    };
    fetch(0);
    for (int64_t chunk = 0; chunk < chunks; ++chunk) {
        P gate[R], in[R], prev[BACK ? R : 1];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            gate[r] = next_gate[r];
            in[r] = next_in[r];
            if constexpr (BACK) prev[r] = next_prev[r];
        }
        if (chunk + 1 < chunks) fetch(chunk + 1);
        float a[V], b[V], least[V];
#pragma unroll
        for (int v = 0; v < V; ++v) a[v] = least[v] = 1.0f, b[v] = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float d = decay(gate[r].get(v)), x = in[r].get(v);
                a[v] *= d;
                least[v] = fminf(least[v], d);
                b[v] = BACK ? weighed(d, b[v] + x) : next_state(d, b[v], x);
            }
#pragma unroll
        for (int v = 0; v < V; ++v) a[v] = least[v] == 0.0f ? 0.0f : at_least(a[v]);
        // inclusive over the pieces before it in the wave, then the one before
#pragma unroll
        for (int m = LC; m < 64; m *= 2)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float pa = __shfl_up(a[v], m), pb = __shfl_up(b[v], m);
                if (lane >= m) {
                    b[v] = apply(a[v], b[v], pb);
                    a[v] = chain(pa, a[v]);
                }
            }
        const int side = chunk & 1;
        if (piece == kPieces - 1)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                s_a[side][wave][channel_lane * V + v] = a[v];
                s_b[side][wave][channel_lane * V + v] = b[v];
            }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float pa = __shfl_up(a[v], LC), pb = __shfl_up(b[v], LC);
            a[v] = piece ? pa : 1.0f;
            b[v] = piece ? pb : 0.0f;
        }
        __syncthreads();
        float state[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            state[v] = carry[v];
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float now = apply(s_a[side][w][channel_lane * V + v], s_b[side][w][channel_lane * V + v], carry[v]);
                carry[v] = now;
                if (w + 1 == wave) state[v] = now;
            }
            state[v] = apply(a[v], b[v], state[v]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            gate[r].renew();
            in[r].renew();
        }
        const unsigned there = unsigned(apart * p.channels + ch0);
        auto walk = [&](auto all_there, auto past) __attribute__((always_inline)) {
            auto put = [](T* q, const P& o) __attribute__((always_inline)) {
                if constexpr (decltype(past)::value) store_past<T, V>(q, o);
                else store_pack<T, V>(q, o);
            };
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t t = chunk * kRows + own + r;
                if (!decltype(all_there)::value && t >= rows) break;
                T* const op = static_cast<T*>(p.out) + place(chunk, r) * p.channels;
                T* const op2 = static_cast<T*>(p.out2) + place(chunk, r) * p.channels;
                P o;
                if constexpr (!BACK) {
#pragma unroll
                    for (int v = 0; v < V; ++v) state[v] = next_state(decay(gate[r].get(v)), state[v], in[r].get(v));
                    o.set(state);
                    put(op + there, o);
                } else {
                    float e[V], dg[V];
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        e[v] = state[v] + in[r].get(v);
                        state[v] = weighed(decay(gate[r].get(v)), e[v]);
                        float h = prev[r].get(v);
                        if (!decltype(all_there)::value && t == rows - 1) h = p.init ? p.init[int64_t(seq) * p.channels + ch0 + v] : 0.0f;
                        dg[v] = weighed(state[v], h);
                    }
                    o.set(e);
                    put(op + there, o);
                    o.set(dg);
                    put(op2 + there, o);
                }
                if (!decltype(all_there)::value && t == rows - 1)
#pragma unroll
                    for (int v = 0; v < V; ++v) p.end[int64_t(seq) * p.channels + ch0 + v] = state[v];
            }
        };
        if (chunk + 1 == chunks) walk(std::false_type{}, std::false_type{});
        else if (p.past) walk(std::true_type{}, std::true_type{});
        else walk(std::true_type{}, std::false_type{});
    }
}

__global__ void __launch_bounds__(kThreads) prepare_kernel(unsigned long long* words, int64_t count, unsigned* ticket, int tickets, const float* begin, float* end,
                                                           const int* offsets, int64_t n, int64_t length, int64_t rows, int channels)
{
    const int64_t step = int64_t(gridDim.x) * kThreads, first = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    for (int64_t i = first; i < count; i += step) words[i] = 0;
    for (int64_t i = first; i < tickets; i += step) ticket[i * kTicketStep] = 0;
    // sequences without steps: the state behind them is the state before them
    if (offsets || length == 0)
        for (int64_t i = first; i < n * channels; i += step) {
            const int64_t s = i / channels;
            int64_t first = 0, past = length;
            if (offsets) rows_of(offsets, s, rows, first, past);
            if (first == past) end[i] = begin ? begin[i] : 0.0f;
        }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) step_kernel(const T* x, const T* gate, float* state, T* out, int64_t n, int channels, int64_t x_stride, int64_t gate_stride, int packs,
                                                        unsigned first_block)
{
    const int64_t i = (int64_t(first_block) + blockIdx.x) * kThreads + threadIdx.x;
    if (i >= n * packs) return;
    const int64_t row = i / packs;
    const int ch = int(i - row * packs) * V, count = channels - ch > V ? V : channels - ch;
    const Pack<T, V> a = load_some<T, V>(gate + row * gate_stride + ch, count), b = load_some<T, V>(x + row * x_stride + ch, count);
    Pack<float, V> s = load_some<float, V>(state + row * channels + ch, count);
    Pack<T, V> o;
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = next_state(decay(a.get(v)), s.get(v), b.get(v));
    s.set(h);
    o.set(h);
    store_some<float, V>(state + row * channels + ch, s, count);
    store_some<T, V>(out + row * channels + ch, o, count);
}

// Lanes take eight bytes of a row.  Where blocks publish, a chunk has kWide lanes to a row and 256 rows forward (100003 steps of 384
// channels, float32: 107 us, with 128 rows 128 us, with 64 178 us) and 128 backward (registers), with few channels kNarrow lanes and 512 rows.
// Where a block has its sequence to itself, kNarrow lanes, 256 rows forward and 128 backward, or 128 for short sequences.
template <typename T>
struct Shape {
    static constexpr int V = 8 / sizeof(T), kWide = 32, kNarrow = 8, kForward = 32, kBackward = 16, kFew = 16;
};

struct Plan {
    int lanes, chunks, channel_blocks;
    bool columns;
};

// A block to a sequence and 64 bytes of channels where these are blocks enough, or the sequences short, on average: the lengths are
// not known here.  (A sequence of 100000 steps beside 199 of 30, 64 channels, bfloat16, is walked by two blocks, 1.2 ms; alone it
// publishes, 76 us.)  When it was chosen, 8 sequences of 2048, 2048 channels, bfloat16: 42 us forward and 65 us backward, publishing 83 and 123; 4 of 512, 1024 channels, float32: 10 and 12, publishing 14
// and 17; but one of 4096, 4096 channels: 54 and 82, publishing 42 and 57; 2 of 4000, 64 channels: 32 and 53, publishing 15 and 17.
template <typename T, bool BACK>
Plan plan_of(int64_t rows, int64_t n, int channels)
{
    using S = Shape<T>;
    Plan p;
    const int64_t narrow = (channels + S::kNarrow * S::V - 1) / (S::kNarrow * S::V);
    p.columns = channels >= S::V && (n * narrow >= 192 || rows <= 1024 * n);
    if (p.columns) {
        p.lanes = S::kNarrow;
        p.chunks = 0;
        p.channel_blocks = int(narrow);
        require(n * narrow < (int64_t(1) << 31), "too many sequences and channels");
        return p;
    }
    p.lanes = channels <= S::kNarrow * S::V ? S::kNarrow : S::kWide;
    const int64_t size = (p.lanes == S::kNarrow ? S::kFew : (BACK ? S::kBackward : S::kForward)) * kThreads / p.lanes;
    const int64_t chunks = (rows + size - 1) / size, blocks = (channels + p.lanes * S::V - 1) / (p.lanes * S::V);
    require(chunks * blocks < (int64_t(1) << 31), "the sequences are too long");
    p.chunks = int(chunks);
    p.channel_blocks = int(blocks);
    return p;
}

size_t ticket_bytes(const Plan& p) { return size_t(p.channel_blocks) * kTicketStep * sizeof(unsigned); }

template <typename T, bool BACK>
size_t scan_workspace(int64_t rows, int64_t n, int channels)
{
    const Plan p = plan_of<T, BACK>(rows, n, channels);
    if (p.columns) return 0;
    return ticket_bytes(p) + (p.chunks > 1 ? size_t(p.chunks) * channels * sizeof(unsigned long long) : 0);
}

template <typename T, bool BACK>
void scan(ScanArgs p, void* workspace, size_t bytes, hipStream_t stream)
{
    using S = Shape<T>;
    if (p.n * p.channels == 0) return;
    require(p.end && (p.rows == 0 || (p.gate && p.in && p.out && (!BACK || (p.h && p.out2)))), "a tensor is missing");
    const Plan plan = plan_of<T, BACK>(p.rows, p.n, p.channels);
    const size_t need = scan_workspace<T, BACK>(p.rows, p.n, p.channels);
    const int64_t widest = p.gate_stride > p.in_stride ? p.gate_stride : p.in_stride;
    require(p.gate_stride >= 0 && p.in_stride >= 0 && (widest > p.channels ? widest : p.channels) <= (int64_t(1) << 20),
            "rows are at most 2^20 elements long and apart");
    check_workspace(workspace, bytes, need);
    p.chunks = plan.chunks;
    p.channel_blocks = plan.channel_blocks;
    // (gradients of 8 sequences of 2048 steps, 2048 channels, bfloat16, alone: 65 us, through the caches 96 us)
    p.past = goes_past(uint64_t(p.rows) * p.channels * sizeof(T) * (BACK ? 2 : 1), uint64_t(p.channels) * sizeof(T));
    if (plan.columns) {
        require(p.n * p.channel_blocks < (int64_t(1) << 31), "too many sequences and channels");
        if (p.rows <= 128 * p.n) return launch_all(column_kernel<T, S::V, 4, S::kNarrow, BACK>, p.n * p.channel_blocks, kThreads, stream, p);
        return launch_all(column_kernel<T, S::V, BACK ? 4 : 8, S::kNarrow, BACK>, p.n * p.channel_blocks, kThreads, stream, p);
    }
    p.ticket = static_cast<unsigned*>(workspace);
    p.words = reinterpret_cast<unsigned long long*>(static_cast<char*>(workspace) + ticket_bytes(plan));
    const int64_t words = plan.chunks > 1 ? int64_t(plan.chunks) * p.channels : 0;
    const int64_t todo = words > p.n * p.channels ? words : p.n * p.channels;
    const int64_t blocks = (todo + kThreads - 1) / kThreads;
    hipLaunchKernelGGL(prepare_kernel, dim3(blocks > 1024 ? 1024 : unsigned(blocks)), dim3(kThreads), 0, stream, p.words, words, p.ticket, p.channel_blocks, p.begin, p.end,
                       p.offsets, p.n, p.length, p.rows, p.channels);
    SIG_HIP(hipGetLastError());
    if (p.rows == 0) return;
    const int64_t grid = int64_t(plan.chunks) * plan.channel_blocks;
    if (p.channels < S::V) launch_all(scan_kernel<T, S::V, S::kFew, S::kNarrow, BACK, true, false>, grid, kThreads, stream, p);
    else if (plan.lanes == S::kWide && p.past) launch_all(scan_kernel<T, S::V, BACK ? S::kBackward : S::kForward, S::kWide, BACK, false, true>, grid, kThreads, stream, p);
    else if (plan.lanes == S::kWide) launch_all(scan_kernel<T, S::V, BACK ? S::kBackward : S::kForward, S::kWide, BACK, false, false>, grid, kThreads, stream, p);
    else launch_all(scan_kernel<T, S::V, S::kFew, S::kNarrow, BACK, false, false>, grid, kThreads, stream, p);
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

__attribute__((visibility("default"))) uint64_t cusig_amd_linear_recurrence_workspace(int dtype, uint64_t rows, uint64_t sequences, uint64_t channels) noexcept
{
    uint64_t bytes = 0;
    sigamd::guarded([&] {
        check_scan(rows, channels, sequences, 0, reinterpret_cast<const int*>(1));
        with_type(dtype, [&](auto t) { bytes = scan_workspace<decltype(t), true>(int64_t(rows), int64_t(sequences), int(channels)); });       // no less than forward
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
        require(x && log_decay && state && h, "a tensor is missing");
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            constexpr int V = 4;
            const uint64_t packs = (channels + V - 1) / V, blocks = (rows * packs + kThreads - 1) / kThreads;
            require(blocks < (uint64_t(1) << 31), "too many rows and channels");
            in_launches(int64_t(blocks), kThreads, [&](unsigned first, dim3 grid) {
                hipLaunchKernelGGL((step_kernel<T, V>), grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream), static_cast<const T*>(x),
                                   static_cast<const T*>(log_decay), state, static_cast<T*>(h), int64_t(rows), int(channels), x_stride, log_decay_stride, int(packs), first);
            });
        });
    });
}

}  // extern "C"
