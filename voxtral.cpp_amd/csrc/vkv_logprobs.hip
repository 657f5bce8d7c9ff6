// Log probabilities of rows of logits on gfx950: maximum, sum and weighted sum
// of the exponentials, and the largest few values, in one read of the row.
//
// k_logprobs_part: a work group takes a chunk of a row into registers, finds
// the chunk's maximum, sums exp(x - max) and (x - max) exp(x - max), and picks
// its n_top largest elements.  k_logprobs_join: a work group per row joins the
// chunks.
#include <hip/hip_runtime.h>

#include <cfloat>

#include "vkv_serve.h"

namespace vkv {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// Values in order as unsigned numbers: NaN above all, -0 beside 0.  An
// element's key is its value's number above its index counted down, so keys
// are distinct and equal values rank by rising index.  0 is no element.
__device__ __forceinline__ unsigned order_of(float x) {
    if (x != x) return 0xffffffffu;
    const unsigned b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned o) {
    if (o == 0xffffffffu) return __builtin_nanf("");
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ u64 key_of(float x, unsigned index) { return (u64)order_of(x) << 32 | (0xffffffffu - index); }

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

// A number T that at least n of the wave's 64 keys reach, as large as such a
// number can be: bit by bit from the top, until exactly n reach it.
__device__ __forceinline__ u64 nth_key(u64 key, int n) {
    u64 t = 0;
    for (int bit = 63; bit >= 0; --bit) {
        const u64 up = t | 1ull << bit;
        const int c = __popcll(__ballot(key >= up));
        if (c >= n) t = up;
        if (c == n) break;
    }
    return t;
}

// The n largest of the work group's keys (PER per thread, 0 = none; distinct),
// in falling order at out[0, n), 0 where there are fewer.  best: the thread's
// largest key.  The n-th largest of a wave's 64 best keys is reached by n keys
// at least, so nothing below the largest such number of the four waves can be
// among the n; what is not below it stands in at most n threads per wave, so
// the list holds it.
template <int PER, typename Key>
__device__ __forceinline__ void select(u64 best, Key key, int n, u64 *list, int capacity, u64 *wave_t, int *count,
                                       u64 *out) {
    const int tid = threadIdx.x;
    const u64 t = nth_key(best, n);
    if (tid == 0) *count = 0;
    if ((tid & 63) == 0) wave_t[tid >> 6] = t;
    __syncthreads();
    u64 least = 1;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) least = wave_t[w] > least ? wave_t[w] : least;
    if (best >= least) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const u64 k = key(i);
            if (k >= least) {
                const int at = atomicAdd(count, 1);
                if (at < capacity) list[at] = k;
            }
        }
    }
    __syncthreads();
    const int c = min(*count, capacity);
    for (int i = tid; i < c; i += kThreads) {
        const u64 k = list[i];
        int above = 0;
        for (int j = 0; j < c && above < n; ++j) above += list[j] > k;
        if (above < n) out[above] = k;
    }
    for (int i = c + tid; i < n; i += kThreads) out[i] = 0;
}

template <typename T, int BLOCKS> struct Chunk {
    static constexpr int per_block = 16 / (int)sizeof(T);      // elements of a 16-byte block
    static constexpr int per_thread = BLOCKS * per_block;
    static constexpr int elements = kThreads * per_thread;
};

// A chunk: BLOCKS blocks of 16 bytes per thread, counted from the 16-byte
// boundary at or below the row's first element.
template <typename T, int BLOCKS>
__global__ __launch_bounds__(kThreads) void k_logprobs_part(LogprobsArgs a) {
    constexpr int EB = Chunk<T, BLOCKS>::per_block, PER = Chunk<T, BLOCKS>::per_thread;
    constexpr int CAP = kLogprobsMaxTop * PER;    // of a wave; the threshold is the same for all
    __shared__ u64 list[kWaves * CAP > 4096 ? 4096 : kWaves * CAP];
    __shared__ u64 wave_t[kWaves];
    __shared__ float red[kWaves][2];
    __shared__ int count;
    const int tid = threadIdx.x, chunk = blockIdx.x, row = blockIdx.y;
    const T *x = (const T *)a.logits + (int64_t)row * a.row_stride;
    const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const T *blocks = x - shift;

    float v[PER];
    int index[BLOCKS];      // of a block's first element; may be below 0 or beyond the row
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
        const int64_t e = ((int64_t)(chunk * BLOCKS + b) * kThreads + tid) * EB - shift;
        index[b] = (int)(e < a.n_vocab ? e : a.n_vocab);
        if (e >= 0 && e + EB <= a.n_vocab) {
            T y[EB] __attribute__((aligned(16)));
            *(uint4 *)y = *(const uint4 *)(blocks + e + shift);
#pragma unroll
            for (int i = 0; i < EB; ++i) v[b * EB + i] = (float)y[i];
        } else {
#pragma unroll
            for (int i = 0; i < EB; ++i) v[b * EB + i] = e + i >= 0 && e + i < a.n_vocab ? (float)x[e + i] : -INFINITY;
        }
    }
    float m = v[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) m = fmaxf(m, v[i]);
    m = wave_max(m);
    if ((tid & 63) == 0) red[tid >> 6][0] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0]));
    const float ref = m > -INFINITY ? m : 0.0f;
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const float d = v[i] - ref, e = expf(d);
        s += e;
        // a probability of 0 adds nothing to the entropy, whatever its logarithm
        t += e != 0.0f ? e * d : 0.0f;
    }
    s = wave_sum(s);
    t = wave_sum(t);
    __syncthreads();
    if ((tid & 63) == 0) {
        red[tid >> 6][0] = s;
        red[tid >> 6][1] = t;
    }
    __syncthreads();
    if (tid == 0) {
        float *st = a.stats + ((int64_t)row * a.n_chunks + chunk) * 4;
        st[0] = m;
        st[1] = red[0][0] + red[1][0] + red[2][0] + red[3][0];
        st[2] = red[0][1] + red[1][1] + red[2][1] + red[3][1];
    }
    if (a.n_top == 0) return;
    auto key = [&](int i) -> u64 {
        const int at = index[i / EB] + i % EB;
        return at >= 0 && at < a.n_vocab ? key_of(v[i], (unsigned)at) : 0;
    };
    u64 best = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const u64 k = key(i);
        best = k > best ? k : best;
    }
    select<PER>(best, key, a.n_top, list, (int)(sizeof(list) / sizeof(u64)), wave_t, &count,
                a.keys + ((int64_t)row * a.n_chunks + chunk) * a.n_top);
}

constexpr int kJoinPer = 8;      // candidates per thread and turn

template <typename T>
__global__ __launch_bounds__(kThreads) void k_logprobs_join(LogprobsArgs a) {
    __shared__ u64 list[kWaves * kLogprobsMaxTop * kJoinPer];
    __shared__ u64 wave_t[kWaves];
    __shared__ u64 top[kLogprobsMaxTop];
    __shared__ float red[kWaves][2];
    __shared__ int count;
    const int tid = threadIdx.x, row = blockIdx.x;
    const float *st = a.stats + (int64_t)row * a.n_chunks * 4;
    float m = -INFINITY;
    for (int i = tid; i < a.n_chunks; i += kThreads) m = fmaxf(m, st[4 * i]);
    m = wave_max(m);
    if ((tid & 63) == 0) red[tid >> 6][0] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0]));
    const float ref = m > -INFINITY ? m : 0.0f;
    float s = 0.0f, t = 0.0f;
    for (int i = tid; i < a.n_chunks; i += kThreads) {
        const float d = (st[4 * i] > -INFINITY ? st[4 * i] : 0.0f) - ref, f = expf(d);
        // the chunk's terms move from its own maximum to the row's
        s += st[4 * i + 1] != 0.0f ? f * st[4 * i + 1] : 0.0f;
        t += st[4 * i + 1] != 0.0f && f != 0.0f ? f * (st[4 * i + 2] + d * st[4 * i + 1]) : 0.0f;
    }
    s = wave_sum(s);
    t = wave_sum(t);
    __syncthreads();
    if ((tid & 63) == 0) {
        red[tid >> 6][0] = s;
        red[tid >> 6][1] = t;
    }
    __syncthreads();
    s = red[0][0] + red[1][0] + red[2][0] + red[3][0];
    t = red[0][1] + red[1][1] + red[2][1] + red[3][1];
    // a row of -inf alone: no sum
    const bool none = s == 0.0f;
    const float log_s = none ? 0.0f : logf(s);
    auto logprob = [&](float x) { return none ? -INFINITY : (x - ref) - log_s; };
    if (tid == 0) {
        if (a.entropy) a.entropy[row] = none ? 0.0f : log_s - t / s;
        if (a.tokens) {
            const int token = a.tokens[row];
            float lp = token == -1 ? 0.0f : __builtin_nanf("");
            if (token >= 0 && token < a.n_vocab) lp = logprob((float)((const T *)a.logits)[row * a.row_stride + token]);
            a.logprob[row] = lp;
        }
    }
    if (a.n_top == 0) return;
    // the chunks' lists, a turn's worth at a time, joined with the largest so
    // far; n_top of them at least are there after the first turn
    const u64 *keys = a.keys + (int64_t)row * a.n_chunks * a.n_top;
    const int64_t n_keys = (int64_t)a.n_chunks * a.n_top;
    if (tid < kLogprobsMaxTop) top[tid] = 0;
    __syncthreads();
    for (int64_t base = 0; base < n_keys; base += kThreads * kJoinPer - kThreads) {
        u64 mine[kJoinPer];
        u64 best = 0;
#pragma unroll
        for (int i = 0; i < kJoinPer; ++i) {
            // the last place of a thread is for the largest so far
            const int64_t at = base + i * kThreads + tid;
            mine[i] = i < kJoinPer - 1 ? (at < n_keys ? keys[at] : 0) : tid < a.n_top ? top[tid] : 0;
            best = mine[i] > best ? mine[i] : best;
        }
        __syncthreads();
        select<kJoinPer>(best, [&](int i) { return mine[i]; }, a.n_top, list, (int)(sizeof(list) / sizeof(u64)), wave_t,
                         &count, top);
        __syncthreads();
    }
    if (tid < a.n_top) {
        const u64 k = top[tid];
        a.top_ids[(int64_t)row * a.n_top + tid] = (int32_t)(0xffffffffu - (unsigned)k);
        a.top_logprobs[(int64_t)row * a.n_top + tid] = logprob(value_of((unsigned)(k >> 32)));
    }
}

template <typename T> hipError_t run(const LogprobsArgs &a, int blocks, hipStream_t st) {
    const dim3 grid((unsigned)a.n_chunks, (unsigned)a.n_rows);
    if (blocks == 2)
        k_logprobs_part<T, 2><<<grid, kThreads, 0, st>>>(a);
    else
        k_logprobs_part<T, sizeof(T) == 4 ? 8 : 4><<<grid, kThreads, 0, st>>>(a);
    k_logprobs_join<T><<<(unsigned)a.n_rows, kThreads, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace

int logprobs_blocks(int n_rows, int64_t n_vocab, int elem_bytes) {
    const int64_t small = n_rows * ((n_vocab * elem_bytes / 16 + 1) / (2 * kThreads) + 1);
    return small <= 1024 ? 2 : elem_bytes == 4 ? 8 : 4;
}

hipError_t launch_logprobs(int dtype, const LogprobsArgs &a, hipStream_t st) {
    const int blocks = logprobs_blocks(a.n_rows, a.n_vocab, dtype == VKV_DTYPE_F32 ? 4 : 2);
    if (dtype == VKV_DTYPE_F16) return run<_Float16>(a, blocks, st);
    if (dtype == VKV_DTYPE_BF16) return run<__bf16>(a, blocks, st);
    return run<float>(a, blocks, st);
}

}  // namespace vkv
