// A paged 8-bit K/V cache on gfx950: the page map built from request lengths,
// the quantizing append and the single-query attention over the pages.
//
// Page layout (codes, one byte each; S tokens, D dims): K is [S][D]; V is
// stored by blocks of 16 tokens with the token innermost, token 4 g + j and
// dim 16 t + r of a block at ((r * 4 + g) * (D / 16) + t) * 4 + j.  That is
// the order in which the lanes of v_mfma_f32_16x16x32_f16 take the transposed
// V: lane (r, g) reads D / 4 contiguous bytes of a block, and no byte moves
// between lanes.
#include <hip/hip_runtime.h>

#include <cfloat>

#include "vkv_serve.h"
#include "vkv_wave.h"

namespace vkv {
namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;

// ---------------------------------------------------------------------------
// Page map
// ---------------------------------------------------------------------------

constexpr int kMapThreads = 1024;

__device__ __forceinline__ int pages_of(int len, int page) { return (int)(((int64_t)len + page - 1) / page); }

struct MapReq {
    int old_len, new_len, held, want;
    __device__ int ret() const { return held > want ? held - want : 0; }
    __device__ int take() const { return want > held ? want - held : 0; }
    __device__ int grow() const { return new_len > old_len ? new_len - old_len : 0; }
};

__device__ __forceinline__ MapReq map_req(const MapArgs &a, int r) {
    MapReq q{0, 0, 0, 0};
    if (r < a.n_req) {
        q.old_len = a.len_old[r];
        q.new_len = a.len_new[r];
        q.held = pages_of(q.old_len, a.page_size);
        q.want = pages_of(q.new_len, a.page_size);
    }
    return q;
}

// inclusive sum over the work group; every thread's total in *total.  LDS:
// one word per wave.
__device__ __forceinline__ int block_scan(int x, int *lds, int *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = x;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kMapThreads / 64; ++w) {
        const int s = lds[w];
        if (w < wave) before += s;
        all += s;
    }
    *total = all;
    return x + before;
}

// first index i in [0, n) with p[i] > x (p rising), n if none
__device__ __forceinline__ int upper_bound(const int *p, int n, int x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p[mid] > x) hi = mid; else lo = mid + 1;
    }
    return lo;
}

// slot and position of packed token t of request r
__device__ __forceinline__ void map_token(const MapArgs &a, int t, int r, int pos) {
    const int page = a.table[(int64_t)r * a.table_stride + pos / a.page_size];
    a.slots[t] = page * a.page_size + pos % a.page_size;
    a.positions[t] = pos;
}

// Any number of requests.  One work group: the free stack is one list, and a
// step's lengths are a few KB.  Pass 1 sums what the step moves and checks it;
// nothing is written before the whole step is known to fit.  Pass 2 pushes the
// returned pages, pass 3 pops the taken ones; both spread the moved pages (not
// the requests) over the threads, by a search in the scanned counts.  Bound by
// the latency of its passes' loads and barriers (1000 requests 13.1 us).
// NOTOKENS: the tokens' slots are left to k_map_tokens.
template <bool NOTOKENS>
__global__ __launch_bounds__(kMapThreads) void k_page_map(MapArgs a) {
    __shared__ int wave_sum[kMapThreads / 64];
    __shared__ int upto[kMapThreads];
    __shared__ int first[kMapThreads];
    __shared__ unsigned long long sum64[3];
    __shared__ int bad;
    const int tid = threadIdx.x;
    const int n_free = *a.n_free;
    const int64_t cap = (int64_t)a.table_stride * a.page_size;
    if (tid < 3) sum64[tid] = 0;
    if (tid == 0) bad = n_free < 0 || n_free > a.n_pages;
    __syncthreads();

    // pass 1: totals, in 64 bits (any lengths may stand there)
    unsigned long long ret = 0, take = 0, grow = 0;
    bool wrong = false;
    for (int r = tid; r < a.n_req; r += kMapThreads) {
        const MapReq q = map_req(a, r);
        wrong |= q.old_len < 0 || q.new_len < 0 || q.old_len > cap || q.new_len > cap;
        ret += (unsigned)q.ret();
        take += (unsigned)q.take();
        grow += (unsigned)q.grow();
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        ret += __shfl_xor(ret, d);
        take += __shfl_xor(take, d);
        grow += __shfl_xor(grow, d);
    }
    if ((tid & 63) == 0) {
        atomicAdd(&sum64[0], ret);
        atomicAdd(&sum64[1], take);
        atomicAdd(&sum64[2], grow);
    }
    if (wrong) bad = 1;
    __syncthreads();
    if (tid == 0 && ((int64_t)sum64[0] > (int64_t)a.n_pages - n_free || sum64[2] > (unsigned long long)a.max_tokens))
        bad = 1;
    __syncthreads();
    const int n_ret = bad ? 0 : (int)sum64[0];

    // the ids to be returned are checked before one of them is pushed
    if (n_ret) {
        for (int base = 0; base < a.n_req; base += kMapThreads) {
            const MapReq q = map_req(a, base + tid);
            int total;
            const int up = block_scan(q.ret(), wave_sum, &total);
            upto[tid] = up;
            first[tid] = q.want - (up - q.ret());
            __syncthreads();
            for (int j = tid; j < total; j += kMapThreads) {
                const int r = upper_bound(upto, kMapThreads, j);
                const int id = a.table[(int64_t)(base + r) * a.table_stride + first[r] + j];
                if (id < 0 || id >= a.n_pages) bad = 1;
            }
            __syncthreads();
        }
    }
    const int status = bad ? 2 : (int64_t)sum64[1] > (int64_t)n_free + n_ret ? 1 : 0;

    if (status) {   // nothing moves
        for (int r = tid; r <= a.n_req; r += kMapThreads) {
            a.cu_new[r] = 0;
            if (r < a.n_req) a.len_out[r] = a.len_old[r];
        }
        if (!NOTOKENS)
            for (int t = tid; t < a.max_tokens; t += kMapThreads) a.slots[t] = a.positions[t] = -1;
        if (tid == 0) {
            *a.n_free_out = n_free;
            *a.status = status;
        }
        return;
    }

    // pass 2: returned pages onto the stack
    if (n_ret) {
        for (int base = 0, done = 0; base < a.n_req; base += kMapThreads) {
            const MapReq q = map_req(a, base + tid);
            int total;
            const int up = block_scan(q.ret(), wave_sum, &total);
            upto[tid] = up;
            first[tid] = q.want - (up - q.ret());
            __syncthreads();
            for (int j = tid; j < total; j += kMapThreads) {
                const int r = upper_bound(upto, kMapThreads, j);
                a.free_pages[n_free + done + j] =
                    a.table[(int64_t)(base + r) * a.table_stride + first[r] + j];
            }
            done += total;
            __syncthreads();
        }
    }
    const int top = n_free + n_ret;

    // pass 3: taken pages off the stack's top; lengths, offsets, tokens
    int taken = 0, grown = 0;
    for (int base = 0; base < a.n_req; base += kMapThreads) {
        const int rr = base + tid;
        const MapReq q = map_req(a, rr);
        int total;
        int up = block_scan(q.take(), wave_sum, &total);
        upto[tid] = up;
        first[tid] = q.held - (up - q.take());
        __syncthreads();
        for (int j = tid; j < total; j += kMapThreads) {
            const int r = upper_bound(upto, kMapThreads, j);
            a.table[(int64_t)(base + r) * a.table_stride + first[r] + j] = a.free_pages[top - 1 - taken - j];
        }
        taken += total;
        __syncthreads();
        up = block_scan(q.grow(), wave_sum, &total);
        if (rr < a.n_req) {
            a.cu_new[rr] = grown + up - q.grow();
            a.len_out[rr] = q.new_len;
        }
        if (!NOTOKENS) {
            upto[tid] = up;
            first[tid] = q.old_len - (up - q.grow());
            __syncthreads();
            for (int j = tid; j < total; j += kMapThreads) {
                const int r = upper_bound(upto, kMapThreads, j);
                map_token(a, grown + j, base + r, first[r] + j);
            }
        }
        grown += total;
        __syncthreads();
    }
    if (!NOTOKENS)
        for (int t = grown + tid; t < a.max_tokens; t += kMapThreads) a.slots[t] = a.positions[t] = -1;
    if (tid == 0) {
        a.cu_new[a.n_req] = grown;
        *a.n_free_out = top - taken;
        *a.status = 0;
    }
}

// inclusive sum over the wave
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);      // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);     // row_bcast 15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);     // row_bcast 31 into rows 2 and 3
    return x;
}

// The same as k_page_map for as many requests as threads: a request is a
// thread's from the first load to the last store, the three sums are scanned
// together, and a step of single tokens (the usual one) needs no search and
// two trips to memory, lengths and then pages.  The time is latency, so the
// fewest threads are the fastest: 32 requests 4.0 us with 64 threads, 5.9 with
// 1024, 11.1 by k_page_map; 200 requests 4.7 us with 256, 5.9 with 1024; 1000
// requests 6.6 us, 13.1 by k_page_map.
template <int THREADS, bool NOTOKENS>
__global__ __launch_bounds__(THREADS) void k_page_map_small(MapArgs a) {
    constexpr int WAVES = THREADS / 64;
    __shared__ int upto[3][THREADS];        // inclusive sums: returned, taken, grown
    __shared__ int from[3][THREADS];        // a request's first entry or position, less the sum before it
    __shared__ int held_of[THREADS];
    __shared__ __attribute__((aligned(16))) int of_wave[WAVES][4];
    __shared__ float rough[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n_free = *a.n_free;
    const int shift = __builtin_ctz((unsigned)a.page_size);
    const int64_t cap = (int64_t)a.table_stride << shift;
    const bool mine = tid < a.n_req;
    const int old_len = mine ? a.len_old[tid] : 0, new_len = mine ? a.len_new[tid] : 0;
    const bool wrong = old_len < 0 || new_len < 0 || old_len > cap || new_len > cap;
    const int round = a.page_size - 1;
    const int held = (int)(((int64_t)old_len + round) >> shift), want = (int)(((int64_t)new_len + round) >> shift);
    const int ret = max(held - want, 0), take = max(want - held, 0), grow = wrong ? 0 : max(new_len - old_len, 0);
    int up[3] = {wave_scan(wrong ? 0 : ret), wave_scan(wrong ? 0 : take), wave_scan(grow)};
    // the sums wrap only beyond what any step may move, and a rough sum tells
    float r = wrong ? 0.0f : (float)ret + (float)take + (float)grow;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) r += __shfl_xor(r, d);
    const bool many = __any(take > 1 || grow > 1);
    if (lane == 63) {
        of_wave[wave][0] = up[0];
        of_wave[wave][1] = up[1];
        of_wave[wave][2] = up[2];
    }
    const bool any_wrong = __any(wrong);
    if (lane == 0) {
        of_wave[wave][3] = (any_wrong ? 1 : 0) | (many ? 2 : 0);
        rough[wave] = r;
    }
    __syncthreads();
    int total[3] = {0, 0, 0}, flags = 0;
    r = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const int4 x = *(const int4 *)of_wave[w];
        if (w < wave) {
            up[0] += x.x;
            up[1] += x.y;
            up[2] += x.z;
        }
        total[0] += x.x;
        total[1] += x.y;
        total[2] += x.z;
        flags |= x.w;
        r += rough[w];
    }
    // (max_tokens < 2^30, pages < 2^27 by the checks of the call)
    bool bad = (flags & 1) || r > 1.5e9f || n_free < 0 || n_free > a.n_pages || total[0] > a.n_pages - n_free ||
               total[2] > a.max_tokens;
    const int n_ret = bad ? 0 : total[0];
    const bool spread = (flags & 2) != 0 && !bad;
    if (n_ret > 0 || spread) {
        upto[0][tid] = up[0];
        upto[1][tid] = up[1];
        upto[2][tid] = up[2];
        from[0][tid] = want - (up[0] - ret);
        from[1][tid] = held - (up[1] - take);
        from[2][tid] = old_len - (up[2] - grow);
        held_of[tid] = held;
        __syncthreads();
    }
    auto returned = [&](int j) {
        const int q = upper_bound(upto[0], THREADS, j);
        return a.table[(int64_t)q * a.table_stride + from[0][q] + j];
    };
    if (n_ret > 0) {    // the ids to be returned are checked before one of them is pushed
        bool strange = false;
        for (int j = tid; j < n_ret; j += THREADS) {
            const int id = returned(j);
            strange |= id < 0 || id >= a.n_pages;
        }
        bad = __syncthreads_or(strange);
    }
    const int status = bad ? 2 : total[1] > n_free + n_ret ? 1 : 0;
    if (status) {       // nothing moves
        if (mine) a.len_out[tid] = old_len;
        for (int i = tid; i <= a.n_req; i += THREADS) a.cu_new[i] = 0;
        if (!NOTOKENS)
            for (int t = tid; t < a.max_tokens; t += THREADS) a.slots[t] = a.positions[t] = -1;
        if (tid == 0) {
            *a.n_free_out = n_free;
            *a.status = status;
        }
        return;
    }
    if (n_ret > 0) {
        for (int j = tid; j < n_ret; j += THREADS) a.free_pages[n_free + j] = returned(j);
        __syncthreads();
    }
    const int top = n_free + n_ret, n_take = total[1], n_grow = total[2];
    if (!spread) {
        int page = -1;
        if (take) page = a.free_pages[top - up[1]];
        const int entry = old_len >> shift;
        if (grow && !NOTOKENS) {
            const int p = take ? page : a.table[(int64_t)tid * a.table_stride + entry];
            a.slots[up[2] - 1] = (p << shift) + (old_len & round);
            a.positions[up[2] - 1] = old_len;
        }
        if (take) a.table[(int64_t)tid * a.table_stride + held] = page;
    } else {
        for (int j = tid; j < n_take; j += THREADS) {
            const int q = upper_bound(upto[1], THREADS, j);
            a.table[(int64_t)q * a.table_stride + from[1][q] + j] = a.free_pages[top - 1 - j];
        }
        if (!NOTOKENS)
            for (int t = tid; t < n_grow; t += THREADS) {
                const int q = upper_bound(upto[2], THREADS, t), pos = from[2][q] + t, entry = pos >> shift;
                // a new page's id straight from the stack
                const int p = entry >= held_of[q] ? a.free_pages[top - 1 - (entry - from[1][q])]
                                                  : a.table[(int64_t)q * a.table_stride + entry];
                a.slots[t] = (p << shift) + (pos & round);
                a.positions[t] = pos;
            }
    }
    if (mine) {
        a.cu_new[tid] = up[2] - grow;
        a.len_out[tid] = new_len;
    }
    if (!NOTOKENS)
        for (int t = n_grow + tid; t < a.max_tokens; t += THREADS) a.slots[t] = a.positions[t] = -1;
    if (tid == 0) {
        a.cu_new[a.n_req] = n_grow;
        *a.n_free_out = top - n_take;
        *a.status = 0;
    }
}

// The map's own work group does the tokens too where they are so many turns of
// its threads at the most (32 requests, 64 tokens: 4.0 us, 5.3 with a second
// launch; 401 of up to 4000: 8.5 and 9.8; 64 of up to 1800, 28 turns: 18.5 and
// 7.2).
constexpr int kMapInlineTurns = 4;
constexpr int kMapOffsets = 4096;    // that k_map_tokens keeps in LDS

// Slots and positions of many tokens, after the map itself, by a search in
// the offsets, which stay in LDS where they fit (65536 places for 401 requests
// 3.6 us: latency).
__global__ __launch_bounds__(256) void k_map_tokens(MapArgs a) {
    __shared__ int cu[kMapOffsets];
    const int n = a.n_req;
    const int *offsets = a.cu_new;
    if (n < kMapOffsets) {
        for (int i = threadIdx.x; i <= n; i += 256) cu[i] = a.cu_new[i];
        __syncthreads();
        offsets = cu;
    }
    const int total = offsets[n];
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < a.max_tokens; t += (int64_t)gridDim.x * 256) {
        if (t >= total) {
            a.slots[t] = a.positions[t] = -1;
            continue;
        }
        // cu_new[0] = 0: the request is the last with cu_new <= t
        const int r = upper_bound(offsets, n + 1, (int)t) - 1;
        map_token(a, (int)t, r, a.len_out[r] - offsets[r + 1] + (int)t);
    }
}

// ---------------------------------------------------------------------------
// Codes and scales
// ---------------------------------------------------------------------------

// FMT below: VKV_DTYPE_E4M3 or VKV_DTYPE_I8
constexpr int kScaleMin = -100, kScaleMax = 120;   // exponents of a scale

__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
__device__ __forceinline__ int exponent_of(float scale) {
    const int e = (int)((__float_as_uint(scale) >> 23) & 255) - 127;
    return min(max(e, kScaleMin), kScaleMax);
}

// Least e with amax <= largest code * 2^e.  The largest codes are 448 =
// 1.75 * 2^8 and 127 = 1.984375 * 2^6, so e is the exponent of amax less 8 or
// 6, and one more where the mantissa is larger.  A power of two, so that a
// value in units of the scale is exact and only its rounding to a code loses
// anything, and so that codes move to a larger scale without a second error
// but for what falls below the smallest step.
template <int FMT> __device__ __forceinline__ int scale_exponent(float amax) {
    const unsigned b = __float_as_uint(amax);
    const int x = (int)(b >> 23) - 127, m = (int)(b & 0x7fffff);
    const int e = FMT == VKV_DTYPE_E4M3 ? x - 8 + (m > 0x600000) : x - 6 + (m > 0x7e0000);
    return min(max(e, kScaleMin), kScaleMax);
}

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) <= FLT_MAX; }

// Four values in units of the scale to four codes (nearest, ties to even).
// FINE: all are finite.  An int8 code is the low byte of x + 1.5 * 2^23, whose
// step is 1.
template <int FMT, bool FINE> __device__ __forceinline__ unsigned pack4(float a, float b, float c, float d) {
    if constexpr (FMT == VKV_DTYPE_E4M3) {
        if constexpr (!FINE) {
            const float nan = __builtin_nanf("");
            a = is_finite(a) ? a : nan;
            b = is_finite(b) ? b : nan;
            c = is_finite(c) ? c : nan;
            d = is_finite(d) ? d : nan;
        }
        unsigned r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    } else {
        auto one = [](float x) -> unsigned {
            if (!FINE) x = x == x ? x : 0.0f;
            return __float_as_uint(__builtin_amdgcn_fmed3f(x, -127.0f, 127.0f) + 12582912.0f);
        };
        return __builtin_amdgcn_perm(one(b), one(a), 0x0c0c0400u) | __builtin_amdgcn_perm(one(d), one(c), 0x04000c0cu);
    }
}

template <int FMT> __device__ __forceinline__ void unpack4(unsigned w, float v[4]) {
    if constexpr (FMT == VKV_DTYPE_E4M3) {
        v[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0);
        v[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
        v[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2);
        v[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
    } else {
        v[0] = (float)(int8_t)(w & 255);
        v[1] = (float)(int8_t)(w >> 8 & 255);
        v[2] = (float)(int8_t)(w >> 16 & 255);
        v[3] = (float)(int8_t)(w >> 24);
    }
}

// codes at a scale 2^k times smaller than the new one, k > 0
template <int FMT> __device__ __forceinline__ unsigned rescale4(unsigned w, float down) {
    float v[4];
    unpack4<FMT>(w, v);
    return pack4<FMT, false>(v[0] * down, v[1] * down, v[2] * down, v[3] * down);
}

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------

template <typename T> __device__ __forceinline__ float to_f32(T x) { return (float)x; }

// Eight (or four) neighbouring values of a row, as they are stored.
template <typename T, int N> struct Raw {
    uint4 w[(N * sizeof(T) + 15) / 16];
    __device__ void load(const T *p) {
        if constexpr (N * sizeof(T) >= 16) {
#pragma unroll
            for (int i = 0; i < (int)(N * sizeof(T) / 16); ++i) w[i] = ((const uint4 *)p)[i];
        } else {
            const uint2 x = *(const uint2 *)p;
            w[0].x = x.x;
            w[0].y = x.y;
        }
    }
    __device__ float operator[](int i) const { return to_f32(((const T *)w)[i]); }
};

// code = round(x 2^-e), e the least exponent that holds the page's largest
// magnitude.  The run of tokens that a page's rows come in: the work group of
// the run's first token does it all; `looks` tokens are a work group's to look
// at for first ones.
//
// A wave owns one 16-token block of one (page, K or V, head), so a block's
// rows are read once and stay in registers between the search for the largest
// magnitude and the rounding; S / 16 waves share a page and meet in LDS.  Lane
// (g, c) has rows 4 g + j and dims [c D/16, (c + 1) D/16): four tokens of a
// dim are a word of V's stored order.
//
// Few tokens are bound by latency: slots, rows, and the page's waves' meeting
// (32 of 8 x 128 f32 values 4.6 us, 2.5 of them an empty launch's).  4099
// tokens of prompts, bf16 to int8 pages of 64: 12.6 us for 25 MB, 2.0 TB/s: the
// search for the runs ends after 5 us, the rows are there after 9.  Finite rows
// are told by one maximum of their bits and rounded without a test for each
// value (14.0 us with one).
template <typename T, int FMT, int D>
__global__ __launch_bounds__(1024) void k_pages_append(AppendPagesArgs a) {
    constexpr int N = D / 16;
    __shared__ int win[16][16];     // a wave's: last token of the run for each slot of its block, -1: none
    __shared__ float top[16];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int S = a.page_size, blocks = S / 16, units = (int)blockDim.x / 64 / blocks;
    const int unit = blockIdx.y * units + wave / blocks, b = wave % blocks;
    const bool busy = unit < 2 * a.n_kv_heads;
    const bool is_v = unit >= a.n_kv_heads;
    const int head = busy ? is_v ? unit - a.n_kv_heads : unit : 0;
    const int g = lane >> 4, c = lane & 15;
    auto slot_at = [&](int t) { return t >= 0 && t < a.n_tokens ? a.slots[t] : -1; };
    auto page_of = [&](int s) { return s >= 0 && s < a.n_slots ? s / S : -1; };
    // first tokens of their page among those this work group looks at
    const int t0 = blockIdx.x * a.looks;
    const int slot0 = slot_at(t0 + lane), before0 = slot_at(t0 + lane - 1);
    const int page0 = page_of(slot0);
    unsigned long long firsts = __ballot(lane < a.looks && page0 >= 0 && page0 != page_of(before0));
    for (; firsts; firsts &= firsts - 1) {
        const int bit = __ffsll(firsts) - 1, t = t0 + bit;
        const int page = __builtin_amdgcn_readlane(page0, bit);
        // the run, which ends at the first token of another page: each wave
        // for its own block
        if (lane < 16) win[wave][lane] = -1;
        bool fresh = false;      // a page begins with its slot 0: what it held before does not count
        for (int i = t + lane, slot = bit == 0 ? slot0 : slot_at(i);;) {
            const unsigned long long out = __ballot(page_of(slot) != page);
            const int n = out ? __ffsll(out) - 1 : 64;
            const int offset = slot - page * S;
            fresh |= __any(lane < n && offset == 0);
            if (lane < n && offset >> 4 == b) atomicMax(&win[wave][offset & 15], i);
            if (out) break;
            i += 64;
            slot = slot_at(i);
        }
        const int64_t ph = (int64_t)page * a.n_kv_heads + head;
        uint8_t *codes = (is_v ? a.v_codes : a.k_codes) + ph * ((int64_t)S * D) + b * (16 * D);
        float *scale = (is_v ? a.v_scale : a.k_scale) + ph;
        const float scale_old = *scale;
        int rows[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) rows[j] = busy ? win[wave][4 * g + j] : -1;
        const T *src = (const T *)(is_v ? a.v : a.k) + head * D + c * N;
        Raw<T, N> x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (rows[j] >= 0) x[j].load(src + (int64_t)rows[j] * a.row_stride);
        // words of the block as it is: K by row, V by dim, for what is kept of them
        unsigned old[4][N / 4];
        const bool whole = rows[0] >= 0 && rows[1] >= 0 && rows[2] >= 0 && rows[3] >= 0;
        if (busy && !whole) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                old[i / (N / 4)][i % (N / 4)] =
                    is_v ? ((const unsigned *)codes)[(((c * N + i) % 16) * 4 + g) * N + (c * N + i) / 16]
                         : ((const unsigned *)(codes + (4 * g + i / (N / 4)) * D + c * N))[i % (N / 4)];
        }
        unsigned most = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (rows[j] >= 0)
#pragma unroll
                for (int n = 0; n < N; ++n) most = max(most, __float_as_uint(x[j][n]) & 0x7fffffffu);
        const bool fine = !__any(most >= 0x7f800000u);
        float amax = __uint_as_float(most);
        if (!fine) {
            amax = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (rows[j] >= 0)
#pragma unroll
                    for (int n = 0; n < N; ++n) amax = fmaxf(amax, is_finite(x[j][n]) ? fabsf(x[j][n]) : 0.0f);
        }
        amax = wave_max(amax);
        if (blocks > 1) {
            __syncthreads();
            if (lane == 0) top[wave] = amax;
            __syncthreads();
            for (int i = 0; i < blocks; ++i) amax = fmaxf(amax, top[wave - b + i]);
        }
        if (!busy) continue;
        int e = scale_exponent<FMT>(amax);
        float down = 1.0f;
        if (!fresh) {
            const int before = exponent_of(scale_old);
            if (e > before) down = exp2_int(max(before - e, -126)); else e = before;
        }
        const bool grown = down != 1.0f;
        const float inv = exp2_int(-e);
        if (b == 0 && lane == 0) *scale = exp2_int(e);
        auto store = [&](auto is_fine) {
            constexpr bool FINE = decltype(is_fine)::value;
            if (!is_v) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (rows[j] >= 0 || grown) {
                        unsigned w[N / 4];
#pragma unroll
                        for (int n = 0; n < N / 4; ++n)
                            w[n] = rows[j] >= 0 ? pack4<FMT, FINE>(x[j][4 * n] * inv, x[j][4 * n + 1] * inv, x[j][4 * n + 2] * inv,
                                                             x[j][4 * n + 3] * inv)
                                                : rescale4<FMT>(old[j][n], down);
                        unsigned *dst = (unsigned *)(codes + (4 * g + j) * D + c * N);
                        if constexpr (N == 8)
                            *(uint2 *)dst = uint2{w[0], w[1]};
                        else
                            *dst = w[0];
                    }
            } else {
                unsigned mask = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) mask |= rows[j] >= 0 ? 255u << 8 * j : 0u;
                if (mask != 0 || grown)
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        unsigned y = pack4<FMT, FINE>(rows[0] >= 0 ? x[0][n] * inv : 0.0f, rows[1] >= 0 ? x[1][n] * inv : 0.0f,
                                                rows[2] >= 0 ? x[2][n] * inv : 0.0f, rows[3] >= 0 ? x[3][n] * inv : 0.0f);
                        if (!whole) {
                            unsigned w = old[n / (N / 4)][n % (N / 4)];
                            if (grown) w = rescale4<FMT>(w, down);
                            y = (w & ~mask) | (y & mask);
                        }
                        ((unsigned *)codes)[(((c * N + n) % 16) * 4 + g) * N + (c * N + n) / 16] = y;
                    }
            }
        };
        if (fine) store(std::true_type{}); else store(std::false_type{});
    }
}

// ---------------------------------------------------------------------------
// Single-query attention
// ---------------------------------------------------------------------------

// four codes to f16, exactly
template <int FMT> __device__ __forceinline__ void codes_f16(unsigned w, half2_t &lo, half2_t &hi) {
    if constexpr (FMT == VKV_DTYPE_E4M3) {
        lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
        hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
    } else {
        // 0x6400 | u is 1024 + u in f16, with u = code + 128
        const unsigned u = w ^ 0x80808080u;
        const unsigned a = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
        const unsigned b = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
        const half2_t off = {(_Float16)1152.0f, (_Float16)1152.0f};
        lo = __builtin_bit_cast(half2_t, a) - off;
        hi = __builtin_bit_cast(half2_t, b) - off;
    }
}

template <int FMT> __device__ __forceinline__ half8_t codes8(unsigned w0, unsigned w1) {
    half2_t a, b, c, d;
    codes_f16<FMT>(w0, a, b);
    codes_f16<FMT>(w1, c, d);
    return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ float lane_value(float x, int lane) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane));
}

// What a row attends to: keys [lo, len), none where len <= 0.
struct Span {
    int lo, len;
    bool bad;     // a length that the call's bounds or the table do not hold
};
__device__ __forceinline__ Span row_span(const PagedAttnArgs &a, int row) {
    Span s;
    s.len = a.lens[row];
    s.bad = s.len > a.max_len;
    s.lo = a.window > 0 && s.len > a.window ? s.len - a.window : 0;
    return s;
}

template <typename T> __device__ __forceinline__ T from_f32(float x) { return (T)x; }

constexpr int kXcds = 8;

// A 16-token block of codes (16 D bytes) into LDS without registers: whole
// lines, past the caches' order (one work group reads them).  Its 16-byte
// pieces are shuffled within each row of D bytes, piece c of row r to c ^ (r
// over the rows of a 256-byte stretch), so that the 16 lanes that read one
// column's pieces of 16 rows at a time meet no bank twice.
template <int D> struct Block {
    static constexpr int pieces = D / 16, bytes = 16 * D;
    static __device__ __forceinline__ int shuffled(int row, int piece) { return piece ^ (row / (256 / D) & (pieces - 1)); }
    // byte of a block that lane's part of load q is to bring
    static __device__ __forceinline__ int source(int q, int lane) {
        const int at = q * 64 + lane, row = at / pieces;
        return (row * pieces + shuffled(row, at % pieces)) * 16;
    }
    static __device__ __forceinline__ int place(int row, int piece) { return row * D + shuffled(row, piece) * 16; }
    static __device__ __forceinline__ void load(const uint8_t *src, uint8_t *dst, const int (&from)[D / 64]) {
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)src, 0, bytes, 0x00020000);
#pragma unroll
        for (int q = 0; q < D / 64; ++q)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void *)(dst + q * 1024), 16,
                                                     from[q], 0, 0, 2 /* non-temporal */);
    }
};

template <int N> __device__ __forceinline__ void wait_loads() {     // at most N vector loads under way
    __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14);
}

// This lane's pieces of two neighbouring blocks at k, row n, and the wait for
// them, after which their place may be written.  Written out because the
// compiler has each LDS read wait for every load into LDS that it cannot tell
// apart; which loads must have arrived is counted by hand (wait_loads).
template <int D> __device__ __forceinline__ void read_blocks(const uint8_t *k, int n, int piece0, int piece1, uint4 (&w)[2][D / 64]) {
    const unsigned base = (unsigned)(size_t)(const __attribute__((address_space(3))) uint8_t *)k;
    const unsigned a0 = base + Block<D>::place(n, piece0), a1 = base + Block<D>::place(n, piece1);
    if constexpr (D == 128)
        asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %4 offset:2048\n\t"
                     "ds_read_b128 %3, %5 offset:2048\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(w[0][0]), "=&v"(w[0][D / 64 - 1]), "=&v"(w[1][0]), "=&v"(w[1][D / 64 - 1])
                     : "v"(a0), "v"(a1)
                     : "memory");
    else
        asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:1024\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(w[0][0]), "=&v"(w[1][0])
                     : "v"(a0)
                     : "memory");
}

// A wave's state: Q's column, the output's, maximum and sum so far.
template <int D> struct AttnState {
    half8_t q[D / 32];
    floatx4 o[D / 16];
    float m, l, factor;
};

// A work group's chunk of keys [begin, hi), of which [lo, hi) count: its
// 16-key blocks' places and scales, a lane each.
template <int D> struct Chunk {
    const uint8_t *k_codes, *v_codes;
    int blk, begin, lo, hi;
    float ks, vs;
    int from[D / 64];
    // the two blocks at key s (the last one again behind it) on their way to `to`
    __device__ __forceinline__ void load(const uint8_t *codes, int s, uint8_t *to) const {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int at = min((s - begin) / 16 + b, (hi - 1 - begin) / 16);
            Block<D>::load(codes + (int64_t)__builtin_amdgcn_readlane(blk, at) * (16 * D), to + b * Block<D>::bytes, from);
        }
    }
};

// The 32 keys at s, of which k and v hold the codes; once they have been read,
// those at s_next take their places.
template <int FMT, int D>
__device__ __forceinline__ void attn_step(uint8_t *k, uint8_t *v, const Chunk<D> &c, int s, int s_next, AttnState<D> &st) {
    constexpr int NL = D / 64, NT = D / 16;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int at = (s - c.begin) / 16;
    floatx4 sc[2];
    uint4 w[2][NL];
    read_blocks<D>(k, n, g, 4 + g, w);
    c.load(c.k_codes, s_next, k);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        floatx4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<FMT>(w[b][i].x, w[b][i].y), st.q[2 * i], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<FMT>(w[b][i].z, w[b][i].w), st.q[2 * i + 1], acc, 0, 0, 0);
        }
        const float f = st.factor * lane_value(c.ks, at + b);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = acc[i], y = row_turn<8>(x);
            sc[b][i] = ((n < 8 ? x : y) + (n < 8 ? y : x) * (1.0f / 2048.0f)) * f;
        }
    }
    unsigned keep[2] = {~0u, ~0u};
    const bool edge = s < c.lo || s + 32 > c.hi;
    if (edge) {
        // the first and the last step: keys outside the span weigh nothing,
        // and their V codes (which may be anything) become 0
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            keep[b] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = s + 16 * b + 4 * g + i;
                const bool in = key >= c.lo && key < c.hi;
                sc[b][i] = in ? sc[b][i] : -INFINITY;
                keep[b] |= in ? 255u << 8 * i : 0u;
            }
        }
    }
    float mx = sc[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, sc[i / 4][i % 4]);
    mx = rows_max(mx);
    // the running maximum moves only when it is passed by 2^8: p <= 256
    if (__any(mx > st.m + 8.0f)) {
        const float m_new = fmaxf(st.m, mx);
        const float f = m_new > -INFINITY ? __builtin_amdgcn_exp2f(st.m - m_new) : 1.0f;
        st.l *= f;
#pragma unroll
        for (int t = 0; t < NT; ++t) st.o[t] *= f;
        st.m = m_new;
    }
    const float m_use = st.m > -INFINITY ? st.m : 0.0f;
    half8_t p8;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const float w = lane_value(c.vs, at + b);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = __builtin_amdgcn_exp2f(sc[b][i] - m_use);
            st.l += p;
            const float x = p * w;
            const _Float16 hi16 = (_Float16)x;
            p8[4 * b + i] = n < 8 ? hi16 : (_Float16)((x - (float)hi16) * 2048.0f);
        }
    }
    wait_loads<3 * 2 * NL>();
    read_blocks<D>(v, n, NL * g, NL * g + 1, w);
    c.load(c.v_codes, s_next, v);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        uint4 a = w[0][i], b = w[1][i];
        if (edge) {
            a.x &= keep[0]; a.y &= keep[0]; a.z &= keep[0]; a.w &= keep[0];
            b.x &= keep[1]; b.y &= keep[1]; b.z &= keep[1]; b.w &= keep[1];
        }
        st.o[4 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<FMT>(a.x, b.x), p8, st.o[4 * i], 0, 0, 0);
        st.o[4 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<FMT>(a.y, b.y), p8, st.o[4 * i + 1], 0, 0, 0);
        st.o[4 * i + 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<FMT>(a.z, b.z), p8, st.o[4 * i + 2], 0, 0, 0);
        st.o[4 * i + 3] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<FMT>(a.w, b.w), p8, st.o[4 * i + 3], 0, 0, 0);
    }
}

// All of a wave's steps: two at a time over two places for K and two for V.
// The first two steps' codes are asked for before Q is put into its form.
template <typename T, int FMT, int D, int WAVES>
__device__ __forceinline__ void attn_steps(uint8_t *k0, uint8_t *k1, uint8_t *v0, uint8_t *v1, Chunk<D> &c, bool mine, int first,
                                           const Raw<T, 8> (&q)[D / 32], float scale, float &vref, AttnState<D> &st) {
    constexpr int STEP = 32 * WAVES, LOADS = 2 * (D / 64), NM = D / 32;
    const int n = threadIdx.x & 15;
    c.load(c.k_codes, first, k0);
    c.load(c.v_codes, first, v0);
    c.load(c.k_codes, first + STEP, k1);
    c.load(c.v_codes, first + STEP, v1);
    float qmax = 0.0f;
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int i = 0; i < 8; ++i) qmax = fmaxf(qmax, fabsf(q[m][i]));
    qmax = rows_max(qmax);
    const int eq = qmax > 0.0f && is_finite(qmax) ? max((int)(__float_as_uint(qmax) >> 23) - 127, -126) : 0;
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = ldexpf(q[m][i], -eq);
            const _Float16 hi = (_Float16)x;
            st.q[m][i] = n < 8 ? hi : (_Float16)((x - (float)hi) * 2048.0f);
        }
    st.factor = ldexpf(scale * kLog2e, eq);
    // V's codes are weighted by their scale over the chunk's largest: powers
    // of two, so nothing is rounded
    c.vs = mine ? c.vs : 0.0f;
    vref = wave_max(c.vs);
    c.vs *= vref > 0.0f ? 1.0f / vref : 0.0f;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) st.o[t] = floatx4{0, 0, 0, 0};
    st.m = -INFINITY;
    st.l = 0.0f;
    // (waited for here: at the loop's head a wait would take in the codes)
    asm volatile("" : "+v"(c.ks), "+v"(c.blk));
    for (int s = first; s < c.hi; s += 2 * STEP) {
        wait_loads<3 * LOADS>();
        attn_step<FMT, D>(k0, v0, c, s, s + 2 * STEP, st);
        if (s + STEP >= c.hi) break;
        wait_loads<3 * LOADS>();
        attn_step<FMT, D>(k1, v1, c, s + STEP, s + 3 * STEP, st);
    }
}

// out = sum_j 2^(s_j - m) V_j / sum_j 2^(s_j - m), s_j = scale log2 e q . K_j,
// in one pass over the keys with a running maximum m.  A work group takes a
// chunk of a row's keys for up to 8 query heads of a kv head, its waves 32 keys
// at a time in turn; DIRECT: one chunk is the row.  Both products are
// v_mfma_f32_16x16x32_f16: codes are exact in f16; q and the weights take two
// columns each, the value in f16 and what that leaves (times 2^11), so that the
// 16 columns are 8 heads and nothing is multiplied twice.  A V scale is a power
// of two and goes into the weights.
//
// Bound by the codes' way from HBM (32 flop for a byte: the matrix cores are
// busy for less than a tenth of the time).  Codes go into LDS without registers, two steps
// ahead (32 KiB per wave in flight for D 128), past the caches' order, by whole
// lines.  64 ragged requests of up to 8192 tokens (8 kv heads of 128, 575 MB)
// 116 us, 5.0 TB/s; 64 x 8192 tokens 5.1 to 5.9 TB/s; 131 rows of 32 heads of
// 64 in a window of 750 68 us, 4.6 TB/s; one row of 8192 tokens (17 MB) 8.7 us,
// a launch, the table, and two steps' latency.  A copy of 1 GiB runs at 5.06
// TB/s, reads alone at 5.8 to 6.7.
template <typename T, int FMT, int D, int WAVES, bool DIRECT>
__global__ __launch_bounds__(64 * WAVES) void k_paged_attn(PagedAttnArgs a) {
    constexpr int NM = D / 32, NT = D / 16;
    constexpr int RING = 8 * Block<D>::bytes;       // of a wave: two steps' K, then V
    // the waves' codes on their way, and at the end their parts of the output
    __shared__ __attribute__((aligned(16))) uint8_t lds[WAVES * RING];
    __shared__ float lds_ml[WAVES][8][2];
    float(*lds_o)[8][D] = (float(*)[8][D])lds;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int group = a.n_q_heads / a.n_kv_heads, tiles = (group + 7) / 8;
    // Work group i runs on XCD i mod 8.  The heads of a (row, chunk) follow
    // each other on one XCD: a page's heads lie side by side in memory, and
    // their scales in one line.
    const int per = a.n_kv_heads * tiles, turn = blockIdx.x / kXcds;
    const int unit = turn / per * kXcds + blockIdx.x % kXcds;
    if (unit >= a.n_rows * a.n_chunks) return;
    const int kvh = turn % per % a.n_kv_heads, tile = turn % per / a.n_kv_heads;
    const int row = unit % a.n_rows, chunk = unit / a.n_rows;
    const int heads = min(group - 8 * tile, 8);
    const int head0 = kvh * group + 8 * tile;

    // this lane's column of Q: dims 64 i + 16 g + 8 m + [0, 8) of MFMA 2 i + m
    // (before the codes: loads return in order)
    Raw<T, 8> qv[NM];
    {
        const int col_head = head0 + min(n & 7, heads - 1);
        const T *q = (const T *)a.q + (int64_t)row * a.q_stride + (int64_t)col_head * D;
#pragma unroll
        for (int m = 0; m < NM; ++m) qv[m].load(q + 64 * (m / 2) + 16 * g + 8 * (m % 2));
    }

    // The chunk's 16-key blocks, one per lane (chunk <= 1024): their pages.
    // Without a window the chunk's place does not depend on the length, and
    // the table holds max_len tokens: both are read at once.
    auto page_at = [&](int kb) { return a.table[(int64_t)row * a.table_stride + kb / a.page_size]; };
    int id = 0;
    if (a.window == 0 && chunk * a.chunk + 16 * lane < a.max_len) id = page_at(chunk * a.chunk + 16 * lane);
    const Span sp = row_span(a, row);
    const int begin = (sp.lo & ~31) + chunk * a.chunk;
    if (sp.bad || begin >= sp.len) {
        if (DIRECT) {
            T *out = (T *)a.out + (int64_t)row * a.out_stride + (int64_t)head0 * D;
            const float v = sp.bad ? __builtin_nanf("") : 0.0f;
            for (int i = tid; i < heads * D; i += 64 * WAVES) out[i] = from_f32<T>(v);
        }
        return;
    }
    const int end = min(sp.len, begin + a.chunk);
    const int kb = begin + 16 * lane;
    const bool mine = kb < end;
    if (a.window > 0 && mine) id = page_at(kb);
    const bool off = id < 0 || id >= a.n_pages;
    if (off || !mine) id = 0;
    const bool bad_page = __any(mine && off);
    // the blocks' places in the layer, and their pages' scales
    const int ph = id * a.n_kv_heads + kvh;
    const int blk = ph * (a.page_size / 16) + kb % a.page_size / 16;

    Chunk<D> c{a.k_codes, a.v_codes, blk, begin, sp.lo, end, a.k_scale[ph], a.v_scale[ph], {}};
    asm volatile("" ::: "memory");      // (those loads before the codes)
#pragma unroll
    for (int q = 0; q < D / 64; ++q) c.from[q] = Block<D>::source(q, lane);
    uint8_t *ring = lds + wave * RING;
    AttnState<D> st;
    float vref;
    attn_steps<T, FMT, D, WAVES>(ring, ring + 2 * Block<D>::bytes, ring + 4 * Block<D>::bytes, ring + 6 * Block<D>::bytes, c, mine,
                          begin + 32 * wave, qv, a.scale, vref, st);

    // the waves' parts meet in LDS, where no codes are on their way any more
    wait_loads<0>();
    __syncthreads();
    const float l = rows_sum(st.l);
    if (n < 8 && g == 0) {
        lds_ml[wave][n][0] = st.m;
        lds_ml[wave][n][1] = l;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = st.o[t][i], y = row_turn<8>(x);
            if (n < 8) lds_o[wave][n][16 * t + 4 * g + i] = (x + y * (1.0f / 2048.0f)) * vref;
        }
    __syncthreads();
    for (int i = tid; i < heads * D; i += 64 * WAVES) {
        const int h = i / D, d = i % D;
        float m = lds_ml[0][h][0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) m = fmaxf(m, lds_ml[w][h][0]);
        float sum = 0.0f, acc = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = lds_ml[w][h][0] > -INFINITY ? __builtin_amdgcn_exp2f(lds_ml[w][h][0] - m) : 0.0f;
            sum += f * lds_ml[w][h][1];
            acc += f * lds_o[w][h][d];
        }
        if (bad_page) acc = sum = __builtin_nanf("");
        if (DIRECT) {
            T *out = (T *)a.out + (int64_t)row * a.out_stride + (int64_t)head0 * D;
            out[i] = from_f32<T>(sum != 0.0f ? acc / sum : 0.0f);
        } else {
            const int64_t part = ((int64_t)row * a.n_q_heads + head0 + h) * a.n_chunks + chunk;
            a.part_o[part * D + d] = acc;
            if (d == 0) {
                a.part_ml[part * 2] = m;
                a.part_ml[part * 2 + 1] = sum;
            }
        }
    }
}

// Joins the chunks of a (row, query head): a wave's lanes read the chunks'
// maxima and sums, 64 at a time, then 16 of their parts of the output at once.
// Latency: 32 chunks of 32 heads 4.0 us, as 2 or 3 trips to memory take.
template <typename T, int D>
__global__ __launch_bounds__(64) void k_paged_merge(PagedAttnArgs a) {
    constexpr int V = D / 64;       // dims per lane
    typedef float vec __attribute__((ext_vector_type(V)));
    const int head = blockIdx.x % a.n_q_heads, row = blockIdx.x / a.n_q_heads;
    const int lane = threadIdx.x;
    T *out = (T *)a.out + (int64_t)row * a.out_stride + (int64_t)head * D + lane * V;
    const int64_t part = (int64_t)blockIdx.x * a.n_chunks;
    const float2 *ml = (const float2 *)a.part_ml + part;
    // (of chunks that do not exist there is room, and nothing is used)
    float2 first = ml[min(lane, a.n_chunks - 1)];
    const Span sp = row_span(a, row);
    if (sp.bad || sp.len <= 0) {
        for (int i = 0; i < V; ++i) out[i] = from_f32<T>(sp.bad ? __builtin_nanf("") : 0.0f);
        return;
    }
    const int n = min(a.n_chunks, (sp.len - (sp.lo & ~31) + a.chunk - 1) / a.chunk);
    float m = -INFINITY, sum = 0.0f;
    vec acc = {};
    for (int c0 = 0; c0 < n; c0 += 64) {
        if (c0) first = ml[min(c0 + lane, n - 1)];
        const bool on = c0 + lane < n;
        const float m_new = fmaxf(m, wave_max(on ? first.x : -INFINITY));
        const float before = m > -INFINITY ? exp2f(m - m_new) : 0.0f;
        // (a maximum of -inf: nothing in the chunk, or NaN, which its sum keeps)
        const float f = on ? first.x > -INFINITY ? exp2f(first.x - m_new) : 0.0f : 0.0f;
        float s = on ? f * first.y : 0.0f;
        s = wave_sum(s);
        sum = sum * before + s;
        acc *= before;
        m = m_new;
        const float *o = a.part_o + (part + c0) * D + lane * V;
        const int k = min(n - c0, 64);
        for (int i = 0; i < k; i += 16) {
            vec x[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = *(const vec *)(o + (int64_t)min(i + j, k - 1) * D);
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (i + j < k) acc += lane_value(f, i + j) * x[j];
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = from_f32<T>(sum != 0.0f ? acc[i] / sum : 0.0f);
}

// Up to so many work groups (two per CU) a chunk is four waves', else two
// waves': four work groups of two fill a CU's LDS and hide each other's starts
// and ends (64 ragged requests of up to 8192 tokens 132 -> 120 us, 4 x 8192
// tokens 24.6 -> 19.5 us), but where all run at once the shorter chunk of a
// wave is faster (1 x 8192 tokens 11.5 against 12.3 us, merge included).
constexpr int64_t kAttnFew = 512;

template <typename T, int FMT, int D> hipError_t attn_launch(const PagedAttnArgs &a, hipStream_t st) {
    const int tiles = (a.n_q_heads / a.n_kv_heads + 7) / 8;
    const int64_t units = ((int64_t)a.n_rows * a.n_chunks + kXcds - 1) / kXcds * kXcds;
    const unsigned grid = (unsigned)(units * a.n_kv_heads * tiles);
    const bool few = (int64_t)a.n_rows * a.n_chunks * a.n_kv_heads * tiles <= kAttnFew;
    if (a.n_chunks == 1) {
        few ? k_paged_attn<T, FMT, D, 4, true><<<grid, 256, 0, st>>>(a) : k_paged_attn<T, FMT, D, 2, true><<<grid, 128, 0, st>>>(a);
    } else {
        few ? k_paged_attn<T, FMT, D, 4, false><<<grid, 256, 0, st>>>(a) : k_paged_attn<T, FMT, D, 2, false><<<grid, 128, 0, st>>>(a);
        k_paged_merge<T, D><<<(unsigned)(a.n_rows * a.n_q_heads), 64, 0, st>>>(a);
    }
    return hipGetLastError();
}

// A work group looks at as few tokens as leave this many work groups: each of
// its first tokens is a chain of loads (1000 requests of one token each 15.5
// us, 36 where a work group looks at 16; 512 tokens of prompts in pages of 64
// 10.0 us, 15.3 where it looks at one, 10.5 with half the work groups), and a
// page's worth of tokens at the most (4099 tokens as above 13.9 us, 15.0 where
// it looks at 32, 49 where it looks at one).
constexpr int64_t kAppendGroups = 2048;

template <typename T, int FMT, int D> hipError_t append_launch(AppendPagesArgs a, hipStream_t st) {
    const int waves = a.page_size / 16 > 4 ? a.page_size / 16 : 4, units = waves / (a.page_size / 16);
    const int64_t heads = (2 * a.n_kv_heads + units - 1) / units;
    for (a.looks = 1; a.looks < 64 && a.looks < a.page_size && heads * a.n_tokens > kAppendGroups * a.looks;) a.looks *= 2;
    const dim3 grid((unsigned)((a.n_tokens + a.looks - 1) / a.looks), (unsigned)heads);
    k_pages_append<T, FMT, D><<<grid, 64 * waves, 0, st>>>(a);
    return hipGetLastError();
}

// f(type tag, format constant, head dim constant) for a call's types
template <typename F> hipError_t by_types(int dtype, int code, int head_dim, F f) {
    auto dim = [&](auto t, auto c) {
        if (head_dim == 64) return f(t, c, std::integral_constant<int, 64>{});
        return f(t, c, std::integral_constant<int, 128>{});
    };
    auto fmt = [&](auto t) {
        if (code == VKV_DTYPE_I8) return dim(t, std::integral_constant<int, VKV_DTYPE_I8>{});
        return dim(t, std::integral_constant<int, VKV_DTYPE_E4M3>{});
    };
    if (dtype == VKV_DTYPE_F16) return fmt((_Float16)0);
    if (dtype == VKV_DTYPE_BF16) return fmt((__bf16)0.0f);
    return fmt(0.0f);
}

}  // namespace

hipError_t launch_page_map(const MapArgs &a, hipStream_t st) {
    const int threads = a.n_req <= 64 ? 64 : a.n_req <= 256 ? 256 : 1024;
    const bool inl = a.max_tokens <= kMapInlineTurns * threads;
    if (a.n_req <= 64)
        inl ? k_page_map_small<64, false><<<1, 64, 0, st>>>(a) : k_page_map_small<64, true><<<1, 64, 0, st>>>(a);
    else if (a.n_req <= 256)
        inl ? k_page_map_small<256, false><<<1, 256, 0, st>>>(a) : k_page_map_small<256, true><<<1, 256, 0, st>>>(a);
    else if (a.n_req <= 1024)
        inl ? k_page_map_small<1024, false><<<1, 1024, 0, st>>>(a) : k_page_map_small<1024, true><<<1, 1024, 0, st>>>(a);
    else
        inl ? k_page_map<false><<<1, kMapThreads, 0, st>>>(a) : k_page_map<true><<<1, kMapThreads, 0, st>>>(a);
    if (!inl) {
        const int64_t wgs = ((int64_t)a.max_tokens + 255) / 256;
        k_map_tokens<<<(unsigned)(wgs < 65536 ? wgs : 65536), 256, 0, st>>>(a);
    }
    return hipGetLastError();
}

hipError_t launch_pages_append(int dtype, int code, int head_dim, const AppendPagesArgs &a, hipStream_t st) {
    return by_types(dtype, code, head_dim, [&](auto t, auto c, auto d) {
        return append_launch<decltype(t), decltype(c)::value, decltype(d)::value>(a, st);
    });
}

hipError_t launch_paged_attn(int dtype, int code, int head_dim, const PagedAttnArgs &a, hipStream_t st) {
    return by_types(dtype, code, head_dim, [&](auto t, auto c, auto d) {
        return attn_launch<decltype(t), decltype(c)::value, decltype(d)::value>(a, st);
    });
}

}  // namespace vkv
