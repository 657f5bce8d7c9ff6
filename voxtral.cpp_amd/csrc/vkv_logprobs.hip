// Log probabilities of rows of logits on gfx950: maximum, sum and weighted sum
// of the exponentials, and the largest few values, in one read of the row.
//
// k_logprobs_part: a work group takes a chunk of a row into registers; each of
// its waves sums exp(x - max) and (x - max) exp(x - max) against its own
// maximum, and the work group picks its n_top largest elements.
// k_logprobs_join: a work group per row joins the waves' sums and the chunks'
// lists.
#include <hip/hip_runtime.h>

#include <cfloat>

#include "vkv_serve.h"

namespace vkv {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr float kLog2e = 1.44269504088896340736f;

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

// over the wave: rotations within rows of 16 lanes, then the rows
template <typename F> __device__ __forceinline__ float wave_reduce(float x, F f) {
    auto turn = [](float v, auto by) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + decltype(by)::value, 0xf, 0xf, false));
    };
    x = f(x, turn(x, std::integral_constant<int, 8>{}));
    x = f(x, turn(x, std::integral_constant<int, 4>{}));
    x = f(x, turn(x, std::integral_constant<int, 2>{}));
    x = f(x, turn(x, std::integral_constant<int, 1>{}));
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float wave_max(float x) {
    return wave_reduce(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float x) {
    return wave_reduce(x, [](float a, float b) { return a + b; });
}

// A number that n of the wave's 64 numbers reach, and few more (0 where n are
// not above 0): bit by bit from the top.
template <typename N> __device__ __forceinline__ N nth_of_wave(N x, int n) {
    N t = 0;
    for (int bit = 8 * (int)sizeof(N) - 1; bit >= 0; --bit) {
        const N up = t | (N)1 << bit;
        const int c = __popcll(__ballot(x >= up));
        if (c >= n) t = up;
        if (c >= n && c <= n + 6) break;
    }
    return t;
}

constexpr int kListMax = 1024;

// The list's n largest in falling order at out[0, n), 0 where there are fewer;
// keys of a list are distinct.  The list has room for seven more.
__device__ __forceinline__ void rank(const u64 *list, int c, int n, u64 *out) {
    for (int i = threadIdx.x; i < c; i += kThreads) {
        const u64 k = list[i];
        int above = 0;
        for (int j = 0; j < c; j += 8) {
            u64 x[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) x[q] = list[j + q];
#pragma unroll
            for (int q = 0; q < 8; ++q) above += j + q < c && x[q] > k;
        }
        if (above < n) out[above] = k;
    }
    for (int i = c + threadIdx.x; i < n; i += kThreads) out[i] = 0;
}

// The n largest keys one after the other, each the largest below the last: for
// chunks with so many equal values, or NaN, that a list does not hold them.
template <int PER, typename Key> __device__ __forceinline__ void pick(Key key, int n, u64 *wave_best, u64 *out) {
    u64 last = ~0ull;
    for (int r = 0; r < n; ++r) {
        u64 best = 0;
#pragma unroll 4
        for (int i = 0; i < PER; ++i) {
            const u64 k = key(i);
            if (k < last && k > best) best = k;
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            const u64 o = __shfl_xor(best, d);
            best = o > best ? o : best;
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 0) wave_best[threadIdx.x >> 6] = best;
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) best = wave_best[w] > best ? wave_best[w] : best;
        if (threadIdx.x == 0) out[r] = best;
        last = best;
    }
}

template <typename T, int BLOCKS> struct Chunk {
    static constexpr int per_block = 16 / (int)sizeof(T);      // elements of a 16-byte block
    static constexpr int per_thread = BLOCKS * per_block;
};

// A chunk: BLOCKS blocks of 16 bytes per thread, counted from the 16-byte
// boundary at or below the row's first element.
//
// The n-th largest of a wave's 64 lane maxima is reached by n elements at
// least, so nothing below the largest such value of the four waves is among
// the chunk's n largest; what is not below it, a few more than n elements as a
// rule, goes to a list that is ranked by counting.
template <typename T, int BLOCKS>
__global__ __launch_bounds__(kThreads) void k_logprobs_part(LogprobsArgs a) {
    constexpr int EB = Chunk<T, BLOCKS>::per_block, PER = Chunk<T, BLOCKS>::per_thread;
    __shared__ u64 list[kListMax + 7];
    __shared__ u64 wave_best[kWaves];
    __shared__ unsigned wave_t[kWaves];
    __shared__ int count, wave_odd[kWaves];
    const int tid = threadIdx.x, chunk = blockIdx.x, row = blockIdx.y;
    const T *x = (const T *)a.logits + (int64_t)row * a.row_stride;
    const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    if (tid == 0) count = 0;

    // element i of block b is the row's element first + b kThreads EB + i
    const int64_t first = ((int64_t)chunk * BLOCKS * kThreads + tid) * EB - shift;
    const int64_t chunk0 = (int64_t)chunk * BLOCKS * kThreads * EB - shift;
    float v[PER];
    if (chunk0 >= 0 && chunk0 + (int64_t)BLOCKS * kThreads * EB <= a.n_vocab) {
        uint4 y[BLOCKS];
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) y[b] = *(const uint4 *)(x + first + b * kThreads * EB);
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
            for (int i = 0; i < EB; ++i) v[b * EB + i] = (float)((const T *)&y[b])[i];
    } else {
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            const int64_t e = first + b * kThreads * EB;
            if (e >= 0 && e + EB <= a.n_vocab) {
                const uint4 y = *(const uint4 *)(x + e);
#pragma unroll
                for (int i = 0; i < EB; ++i) v[b * EB + i] = (float)((const T *)&y)[i];
            } else {
#pragma unroll
                for (int i = 0; i < EB; ++i) v[b * EB + i] = e + i >= 0 && e + i < a.n_vocab ? (float)x[e + i] : -INFINITY;
            }
        }
    }
    float mine = v[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) mine = fmaxf(mine, v[i]);
    const float m = wave_max(mine);
    const float ref = m > -INFINITY ? m : 0.0f;
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const float d = v[i] - ref, e = __builtin_amdgcn_exp2f(d * kLog2e);
        s += e;
        // (below -200 the exponential is 0: no infinity times 0)
        t = fmaf(e, fmaxf(d, -200.0f), t);
    }
    s = wave_sum(s);
    t = wave_sum(t);
    if ((tid & 63) == 0) {
        float *st = a.stats + (((int64_t)row * a.n_chunks + chunk) * kWaves + (tid >> 6)) * 4;
        st[0] = m;
        st[1] = s;
        st[2] = t;
        wave_odd[tid >> 6] = s != s;     // NaN, or +inf
    }
    if (a.n_top == 0) return;
    const unsigned nth = nth_of_wave(order_of(mine), a.n_top);
    if ((tid & 63) == 0) wave_t[tid >> 6] = nth;
    __syncthreads();
    unsigned least = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) least = wave_t[w] > least ? wave_t[w] : least;
    const float limit = value_of(least);
    const int64_t left = a.n_vocab - first;
    auto at = [&](int i) { return (i / EB) * kThreads * EB + i % EB; };      // from first
    if (limit > -INFINITY) {
        if (mine >= limit) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (v[i] >= limit) {
                    const int p = atomicAdd(&count, 1);
                    if (p < kListMax) list[p] = key_of(v[i], (unsigned)(first + at(i)));
                }
        }
    } else {
        // fewer than n above -inf: they, and the first n of the chunk for those of -inf that rank
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if ((v[i] > -INFINITY || first + at(i) - max(chunk0, (int64_t)0) < a.n_top) && first + at(i) >= 0 && at(i) < left) {
                const int p = atomicAdd(&count, 1);
                if (p < kListMax) list[p] = key_of(v[i], (unsigned)(first + at(i)));
            }
    }
    __syncthreads();
    u64 *out = a.keys + ((int64_t)row * a.n_chunks + chunk) * a.n_top;
    if (wave_odd[0] | wave_odd[1] | wave_odd[2] | wave_odd[3] || count > kListMax)
        pick<PER>([&](int i) -> u64 { return first + at(i) >= 0 && at(i) < left ? key_of(v[i], (unsigned)(first + at(i))) : 0; },
                  a.n_top, wave_best, out);
    else
        rank(list, count, a.n_top, out);
}

constexpr int kJoinPer = 4;      // keys of the chunks' lists per thread and turn

// A work group per row.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_logprobs_join(LogprobsArgs a) {
    __shared__ u64 list[kThreads * kJoinPer + kLogprobsMaxTop + 7];
    __shared__ u64 wave_t[kWaves];
    __shared__ u64 top[kLogprobsMaxTop];
    __shared__ float red[kWaves][4];
    __shared__ int count;
    const int tid = threadIdx.x, row = blockIdx.x;
    const float4 *st = (const float4 *)a.stats + (int64_t)row * a.n_chunks * kWaves;
    const int n_stats = a.n_chunks * kWaves;
    const u64 *keys = a.keys + (int64_t)row * a.n_chunks * a.n_top;
    const int n_keys = a.n_chunks * a.n_top;

    // everything the row needs is asked for at once
    u64 k[kJoinPer];
#pragma unroll
    for (int i = 0; i < kJoinPer; ++i) k[i] = i * kThreads + tid < n_keys ? keys[i * kThreads + tid] : 0;
    const int token = a.tokens ? a.tokens[row] : -1;
    const bool is_token = token >= 0 && token < a.n_vocab;
    const float at_token = is_token ? (float)((const T *)a.logits)[row * a.row_stride + token] : 0.0f;
    float m = -INFINITY, s = 0.0f, t = 0.0f;
    for (int i = tid; i < n_stats; i += kThreads) {
        const float4 x = st[i];
        const float to = fmaxf(m, x.x), ref = to > -INFINITY ? to : 0.0f;
        const float dm = (m > -INFINITY ? m : 0.0f) - ref, dx = (x.x > -INFINITY ? x.x : 0.0f) - ref;
        const float fm = expf(dm), fx = expf(dx);
        // both sums move to the larger maximum; what has no term, or weighs nothing, adds nothing
        t = (s != 0.0f && fm != 0.0f ? fm * (t + dm * s) : 0.0f) + (x.y != 0.0f && fx != 0.0f ? fx * (x.z + dx * x.y) : 0.0f);
        s = (s != 0.0f ? fm * s : 0.0f) + (x.y != 0.0f ? fx * x.y : 0.0f);
        m = to;
    }
    const float wm = wave_max(m);
    if ((tid & 63) == 0) red[tid >> 6][0] = wm;
    __syncthreads();
    const float top_m = fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0]));
    const float ref = top_m > -INFINITY ? top_m : 0.0f;
    {
        const float d = (m > -INFINITY ? m : 0.0f) - ref, f = expf(d);
        t = s != 0.0f && f != 0.0f ? f * (t + d * s) : 0.0f;
        s = s != 0.0f ? f * s : 0.0f;
    }
    s = wave_sum(s);
    t = wave_sum(t);
    if ((tid & 63) == 0) {
        red[tid >> 6][1] = s;
        red[tid >> 6][2] = t;
    }

    // the n largest keys: as in a chunk, a turn's worth of keys at a time,
    // joined with the largest so far
    if (tid < kLogprobsMaxTop) top[tid] = 0;
    for (int base = 0; base < n_keys; base += kThreads * kJoinPer) {
        if (base)
#pragma unroll
            for (int i = 0; i < kJoinPer; ++i) {
                const int at = base + i * kThreads + tid;
                k[i] = at < n_keys ? keys[at] : 0;
            }
        u64 best = 0;
#pragma unroll
        for (int i = 0; i < kJoinPer; ++i) best = k[i] > best ? k[i] : best;
        const u64 nth = nth_of_wave(best, a.n_top);
        __syncthreads();
        if (tid == 0) count = 0;
        if ((tid & 63) == 0) wave_t[tid >> 6] = nth;
        __syncthreads();
        u64 least = 1;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) least = wave_t[w] > least ? wave_t[w] : least;
#pragma unroll
        for (int i = 0; i < kJoinPer; ++i)
            if (k[i] >= least) list[atomicAdd(&count, 1)] = k[i];
        if (base && tid < a.n_top && top[tid]) list[atomicAdd(&count, 1)] = top[tid];
        __syncthreads();
        rank(list, count, a.n_top, top);
    }
    __syncthreads();
    s = red[0][1] + red[1][1] + red[2][1] + red[3][1];
    t = red[0][2] + red[1][2] + red[2][2] + red[3][2];
    // a row of -inf alone: no sum
    const bool none = s == 0.0f;
    const float log_s = none ? 0.0f : logf(s);
    auto logprob = [&](float x) { return none ? -INFINITY : (x - ref) - log_s; };
    if (tid < a.n_top) {
        const u64 key = top[tid];
        a.top_ids[(int64_t)row * a.n_top + tid] = (int32_t)(0xffffffffu - (unsigned)key);
        a.top_logprobs[(int64_t)row * a.n_top + tid] = logprob(value_of((unsigned)(key >> 32)));
    }
    if (tid == kThreads - 1) {
        if (a.entropy) a.entropy[row] = none ? 0.0f : log_s - t / s;
        if (a.tokens) a.logprob[row] = is_token ? logprob(at_token) : token == -1 ? 0.0f : __builtin_nanf("");
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
