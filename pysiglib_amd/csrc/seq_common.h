// Shared by the operators on token sequences (seq_*.hip): element types, vector loads and stores, sequences packed behind
// each other, argument checks.  These operators take their scratch from the caller and only enqueue on the caller's stream.
#pragma once
#include "sig_host.h"
#include "../../include/cusig_amd.h"

#include <cstdint>

namespace seqamd {

using bf16 = __bf16;
using f16 = _Float16;

// element types of the C ABI
enum : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

// V elements as the words they come in: kept like that, two 16-bit elements share a register until they are used
template <typename T, int V>
struct Pack {
    static_assert(sizeof(T) * V % 4 == 0, "whole words");
    static constexpr int kWords = sizeof(T) * V / 4;
    unsigned w[kWords];

    __device__ __forceinline__ float get(int i) const
    {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else if constexpr (__is_same(T, bf16)) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        else return static_cast<float>(__builtin_bit_cast(f16, static_cast<unsigned short>(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu)));
    }
    // one element into words that are zero
    __device__ __forceinline__ void put(int i, T x)
    {
        if constexpr (sizeof(T) == 4) w[i] = __builtin_bit_cast(unsigned, x);
        else w[i / 2] |= static_cast<unsigned>(__builtin_bit_cast(unsigned short, x)) << (i & 1 ? 16 : 0);
    }
    // rounds to nearest, ties to even
    __device__ __forceinline__ void set(const float* x)
    {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = __float_as_uint(x[i]);
        } else {
            typedef T Two __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int i = 0; i < V; i += 2) w[i / 2] = __builtin_bit_cast(unsigned, Two{T(x[i]), T(x[i + 1])});
        }
    }
    // the values as they were, but unknown to the compiler: what was formed from them before is formed again, not kept
    __device__ __forceinline__ void renew()
    {
#pragma unroll
        for (int i = 0; i < kWords; ++i) asm volatile("" : "+v"(w[i]));
    }
};

// V elements from an address that need only be aligned to one: gfx950 loads dwords at any byte address
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p)
{
    Pack<T, V> r;
    __builtin_memcpy(r.w, p, sizeof r.w);
    return r;
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& r)
{
    __builtin_memcpy(p, r.w, sizeof r.w);
}

// the same past the caches, in whole lines: for results that would leave them unread
template <typename T, int V>
__device__ __forceinline__ void store_past(T* p, const Pack<T, V>& r)
{
    typedef unsigned Words __attribute__((ext_vector_type(Pack<T, V>::kWords), aligned(4)));
    Words x;
#pragma unroll
    for (int i = 0; i < Pack<T, V>::kWords; ++i) x[i] = r.w[i];
    __builtin_nontemporal_store(x, reinterpret_cast<Words*>(p));
}

// the first `count` of V elements, the others zero
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_some(const T* p, int count)
{
    if (count >= V) return load_pack<T, V>(p);
    Pack<T, V> r;
#pragma unroll
    for (int i = 0; i < Pack<T, V>::kWords; ++i) r.w[i] = 0;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < count) {
            if constexpr (sizeof(T) == 4) r.w[i] = __builtin_bit_cast(unsigned, p[i]);
            else r.w[i / 2] |= static_cast<unsigned>(__builtin_bit_cast(unsigned short, p[i])) << (i & 1 ? 16 : 0);
        }
    return r;
}

template <typename T, int V>
__device__ __forceinline__ void store_some(T* p, const Pack<T, V>& r, int count)
{
    if (count >= V) return store_pack<T, V>(p, r);
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < count) {
            if constexpr (sizeof(T) == 4) p[i] = __builtin_bit_cast(T, r.w[i]);
            else p[i] = __builtin_bit_cast(T, static_cast<unsigned short>(r.w[i / 2] >> (i & 1 ? 16 : 0)));
        }
}

// Whether results of so many bytes, in rows of `row` bytes, are stored past the caches.  Those of less than half of the last one's 256 MB
// stay there for the call that reads them.  8 sequences, 2048 channels, bfloat16, forward and gradients in turn over three sets of
// inputs, the gradients' results kept and past the caches: of 96 MB 108 us both, of 120 MB 141 and 137, of 128 MB (2048 steps) 157 and 148,
// of 256 MB 333 and 311; with 2048 steps and the forward's 64 MB past the caches too 160.  Lines that are written in pieces are kept:
// gradients of 23000 steps of 997 channels in float16 took 126 us instead of 89.
inline bool goes_past(uint64_t bytes, uint64_t row, uint64_t from = uint64_t(128) << 20) { return bytes >= from && row % 128 == 0; }

// A weight times what it weighs: zero where it has no weight, also of what is not finite (v_mul_legacy_f32)
extern "C" __device__ __attribute__((const)) float weighed(float weight, float x) __asm("llvm.amdgcn.fmul.legacy");

__device__ __forceinline__ int64_t kept(int64_t x, int64_t low, int64_t high) { return x < low ? low : (x > high ? high : x); }

inline void require(bool ok, const char* what)
{
    if (!ok) throw std::invalid_argument(what);
}

// n sequences of `length` rows: the product may be beyond 64 bits
inline void check_rows(uint64_t n, uint64_t length, uint64_t rows)
{
    require(n == 0 ? rows == 0 : rows % n == 0 && rows / n == length, "rows are not sequences times length");
}

inline void check_workspace(const void* workspace, uint64_t bytes, uint64_t need)
{
    require(bytes >= need && (workspace || need == 0), "the workspace is too small");
    require(reinterpret_cast<uintptr_t>(workspace) % 256 == 0 || need == 0, "the workspace is not aligned to 256 bytes");
}

// A launch numbers its threads with 32 bits: more blocks go in several, each of which tells its kernel what its first one is.
// Multiples of eight: a block stays on its die.
template <typename Launch>
void in_launches(int64_t blocks, int threads, Launch&& launch)
{
    const int64_t most = ((int64_t(1) << 32) / threads - 1) / 8 * 8;
    for (int64_t first = 0; first < blocks; first += most) {
        launch(unsigned(first), dim3(static_cast<unsigned>(blocks - first < most ? blocks - first : most)));
        SIG_HIP(hipGetLastError());
    }
}

// Sums over pieces: parts [pieces][columns], each column's sum goes to put(column, sum).  A block to 32 columns; 32 threads for each add up
// every 32nd piece, then each other's sums: the order is fixed.
constexpr int kSumThreads = 1024;

template <typename F>
__device__ __forceinline__ void sum_pieces(const float* parts, int pieces, int64_t columns, unsigned first_block, F&& put)
{
    __shared__ float s_sum[32][33];
    const int lane = threadIdx.x % 32, row = threadIdx.x / 32;
    const int64_t at = (int64_t(first_block) + blockIdx.x) * 32, e = at + lane;
    float sum = 0.0f;
    if (e < columns)
#pragma unroll 8
        for (int n = row; n < pieces; n += 32) sum += parts[n * columns + e];
    s_sum[row][lane] = sum;
    __syncthreads();
    // turned: a half wave to a column
    sum = s_sum[lane][row];
#pragma unroll
    for (int m = 16; m; m /= 2) sum += __shfl_xor(sum, m);
    if (lane == 0 && at + row < columns) put(at + row, sum);
}

inline int64_t sum_blocks(int64_t columns) { return (columns + 31) / 32; }

template <typename Args>
void launch_all(void (*kernel)(Args), int64_t blocks, int threads, hipStream_t stream, Args p)
{
    in_launches(blocks, threads, [&](unsigned first, dim3 grid) {
        p.first_block = first;
        hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, stream, p);
    });
}

// calls body(T{}) with the element type of `dtype`
template <typename F>
void with_type(int dtype, F&& body)
{
    switch (dtype) {
    case kF32: body(float{}); break;
    case kBF16: body(bf16{}); break;
    case kF16: body(f16{}); break;
    default: throw std::invalid_argument("unknown element type");
    }
}

}  // namespace seqamd
