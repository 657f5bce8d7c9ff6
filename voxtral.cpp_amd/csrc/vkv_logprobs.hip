// Log probabilities of rows of logits on gfx950: maximum, sum and weighted sum
// of the exponentials, and the largest few values, in one read of the row.
//
// k_logprobs_part: a work group takes a chunk of a row into registers; each of
// its waves sums exp(x - max) and (x - max) exp(x - max) against its own
// maximum (whose own terms it counts), and the work group picks its n_top largest elements.
// k_logprobs_join: a work group per row joins the waves' sums and the chunks'
// lists.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>

#include "vkv_serve.h"
#include "vkv_wave.h"

namespace vkv {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 256;
// Pieces: 2 blocks per thread where that makes few work groups (a row or a
// few: the time is latency) whose lists k_logprobs_join takes in one turn (a
// row in f32, n_top 5: 9.8 us, 11.0 with the larger pieces; n_top 20, two turns:
// 16.0 us, 11.7 with the larger pieces; 32 rows, n_top 5, beyond kFewGroups:
// 14.9 us, 12.1 with them), else 32 elements per thread, as many pieces per
// work group as leave kManyGroups of them, which run at the same time (rows of
// 131072 logits in bf16, n_top 20, both launches: 251 rows 23.4 us, 29.1 with
// twice the work groups, 29.1 with 3/4; 512 rows 32.4 us, 35.7 where a work
// group takes 4 pieces at the most, 32.5 where it takes 16).
constexpr int kBlocksFew = 2;
constexpr int64_t kFewGroups = 1024, kManyGroups = 1024, kTurnsMost = 8;
// A chunk that may list more elements than this looks for its limit twice (251
// rows as above 25.4 -> 23.4 us; n_top 5, where it lists 20, 21.1 -> 22.1 us).
constexpr int kFewKeys = 48;
constexpr int kWaves = kThreads / 64;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

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

// A number that n of the work group's numbers (one per thread) reach, and few
// more (0 where n are not above 0): bit by bit from the top.  One wave looks
// for it: the steps are the scalar unit's, which all waves of a CU share.
struct Search {
    unsigned x[kThreads], found;
};
__device__ __forceinline__ void search_nth(Search &at, int n) {
    if (threadIdx.x >= 64) return;
    unsigned mine[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mine[w] = at.x[w * 64 + threadIdx.x];
    unsigned t = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const unsigned up = t | 1u << bit;
        int c = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) c += __popcll(__ballot(mine[w] >= up));
        if (c >= n) t = up;
        if (c >= n && c <= n + n / 4) break;
    }
    if (threadIdx.x == 0) at.found = t;
}

// Keys of a few elements, a piece of the list for each wave; a few words
// behind a piece are read, not used.
constexpr int kPiece = 256;
struct List {
    u64 key[kWaves][kPiece];
    u64 more[4];
    __attribute__((aligned(16))) int count[kWaves];
};

// how many of the lanes below this one are in the set
__device__ __forceinline__ int lanes_below(u64 set) {
    return __builtin_amdgcn_mbcnt_hi((unsigned)(set >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)set, 0));
}

// The wave's elements for which `take` holds go to its piece, as far as it has
// room; `kept` counts them all.
template <typename Take, typename Key> __device__ __forceinline__ void put(List &list, int &kept, Take take, Key key) {
    const u64 on = __ballot(take);
    if (on == 0) return;
    const int at = kept + lanes_below(on);
    if (take && at < kPiece) list.key[threadIdx.x >> 6][at] = key();
    kept += __popcll(on);
}

// Blocks with elements that are not below a limit, a piece for each wave.
constexpr int kHot = 128;
struct Hot {
    uint4 block[kWaves][kHot];
    int first[kWaves][kHot];
};

// The list's n largest in falling order at out[0, n), 0 where there are fewer;
// its keys are distinct.  A barrier is between the list's writing and this.
__device__ __forceinline__ void rank(const List &list, int n, u64 *out) {
    const int4 c = *(const int4 *)list.count;
    const int to1 = c.x, to2 = to1 + c.y, to3 = to2 + c.z, total = to3 + c.w;
    for (int i = threadIdx.x; i < total; i += kThreads) {
        const int w = (i >= to1) + (i >= to2) + (i >= to3);
        const u64 k = list.key[w][i - (w == 0 ? 0 : w == 1 ? to1 : w == 2 ? to2 : to3)];
        int above = 0;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) {
            const int of_v = v == 0 ? c.x : v == 1 ? c.y : v == 2 ? c.z : c.w;
            for (int j = 0; j < of_v; j += 4) {
                u64 x[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) x[q] = list.key[v][j + q];
#pragma unroll
                for (int q = 0; q < 4; ++q) above += j + q < of_v && x[q] > k;
            }
        }
        if (above < n) out[above] = k;
    }
    for (int i = total + threadIdx.x; i < n; i += kThreads) out[i] = 0;
}

// The n largest of the row's elements [from, to) one after the other, each the
// largest below the last: for chunks with more elements above the limit than a
// list holds (they rise, and the limit is the first piece's), NaN or +inf.
template <typename T> __device__ __noinline__ void pick(const T *x, int64_t from, int64_t to, int n, u64 *wave_best, u64 *out) {
    u64 last = ~0ull;
    for (int r = 0; r < n; ++r) {
        u64 best = 0;
        for (int64_t i = from + threadIdx.x; i < to; i += kThreads) {
            const u64 k = key_of((float)x[i], (unsigned)i);
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

// log p_t = x_t - m - log s, entropy = log s - t / s with s = sum exp(x - m), t =
// sum (x - m) exp(x - m).  A work group takes `turns` pieces of BLOCKS 16-byte
// blocks per thread, counted from the 16-byte boundary at or below the row's
// first element; the next piece is on its way while one is worked on.
//
// A value that n of the 256 threads' maxima reach is reached by n elements at
// least, so nothing below it is among the n largest.  Found once, in the first
// piece, by one wave while the others sum, it is the limit for all.  The blocks
// with elements that are not below it, a few more than n per piece as a rule,
// are set aside whole, one test for a block; at the end their elements go to a
// list that is ranked by counting.  Equal values rank by rising index, so of
// those that equal the limit (masked logits of the type's lowest value, a row
// of zeros) each wave keeps its first n (251 rows of zeros as below 34 us).
//
// Bound by the vector units beside the loads, about 8 instructions and one
// exponential for an element: 251 rows of 131072 logits in bf16 with 20
// alternatives 21.7 us, 3.0 TB/s (12 us without alternatives), 2 of them for the
// maximum's terms kept apart.  One f32 row 5.3 us: a launch, a load, a search
// and a ranking.
template <typename T, int BLOCKS>
__global__ __launch_bounds__(kThreads) void k_logprobs_part(LogprobsArgs a) {
    constexpr int EB = 16 / (int)sizeof(T);     // elements of a block
    constexpr int PER = BLOCKS * EB;            // of a thread and piece
    constexpr int PIECE = kThreads * PER;
    __shared__ List list;
    __shared__ Hot hot;
    __shared__ Search search;
    __shared__ u64 wave_best[kWaves];
    __shared__ int wave_odd[kWaves];
    const int tid = threadIdx.x, chunk = blockIdx.x, row = blockIdx.y;
    const T *x = (const T *)a.logits + (int64_t)row * a.row_stride;
    const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const int vocab = a.n_vocab;
    const int chunk0 = (int)((int64_t)chunk * a.turns * PIECE - shift);
    const int begin = max(chunk0, 0), end = (int)min((int64_t)chunk0 + (int64_t)a.turns * PIECE, (int64_t)vocab);
    // (the first element of block b of a piece: piece + (b kThreads + tid) EB)
    auto load = [&](int piece, uint4 *y) {
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            const int e = piece + (b * kThreads + tid) * EB;
            if (e >= 0 && e + EB <= vocab) y[b] = *(const uint4 *)(x + e);
        }
    };
    uint4 next[BLOCKS];
    load(chunk0, next);
    float m = -INFINITY, s = 0.0f, t = 0.0f, n = 0.0f, limit = -INFINITY, largest = -INFINITY;
    int kept = 0, set_aside = 0, even_blocks = 0;
    for (int piece = chunk0; piece < end; piece += PIECE) {
        float v[PER];
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
            for (int i = 0; i < EB; ++i) v[b * EB + i] = (float)((const T *)&next[b])[i];
        if (piece < 0 || piece + PIECE > vocab) {
            // the row's ends: blocks that are not all its own, element by element
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
                const int e = piece + (b * kThreads + tid) * EB;
                if (!(e >= 0 && e + EB <= vocab))
#pragma unroll
                    for (int i = 0; i < EB; ++i) v[b * EB + i] = e + i >= 0 && e + i < vocab ? (float)x[e + i] : -INFINITY;
            }
        }
        if (piece + PIECE < end) load(piece + PIECE, next);
        float of_block[BLOCKS], mine = -INFINITY;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            of_block[b] = v[b * EB];
#pragma unroll
            for (int i = 1; i < EB; ++i) of_block[b] = fmaxf(of_block[b], v[b * EB + i]);
            mine = fmaxf(mine, of_block[b]);
        }
        largest = fmaxf(largest, mine);
        const bool looks = a.n_top && !(limit > -INFINITY);
        if (looks) {
            __syncthreads();        // (the value before is read)
            search.x[tid] = order_of(mine);
            __syncthreads();
            search_nth(search, a.n_top);
        }
        const float m_new = fmaxf(m, wave_max(mine));
        const float ref = m_new > -INFINITY ? m_new : 0.0f;
        // the sums so far move to the new maximum (without a term: none)
        if (m_new > m && s + n != 0.0f) {
            const float d = (m - ref) * kLog2e, f = __builtin_amdgcn_exp2f(d);
            t = f != 0.0f ? f * fmaf(d, s + n, t) : 0.0f;
            s = (s + n) * f;
            n = 0.0f;
        }
        m = m_new;
        // exp(x - ref) = 2^d, d = x log2 e - c in one rounding; what c's own
        // lacks is the same for every term and comes off the sums
        const float c = ref * kLog2e, top = fabsf(m) <= FLT_MAX ? m : __builtin_nanf("");
        float lack = fmaf(ref, kLog2e, -c), s1 = 0.0f, t1 = 0.0f, n1 = 0.0f;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            if (__any(of_block[b] == top)) {
#pragma unroll
                for (int i = 0; i < EB; ++i) {
                    const float x = v[b * EB + i], d = fmaf(x, kLog2e, -c), e = __builtin_amdgcn_exp2f(d);
                    s1 += x == top ? 0.0f : e;
                    t1 = fmaf(x == top ? 0.0f : e, d, t1);
                    n1 += x == top ? 1.0f : 0.0f;
                }
            } else {
#pragma unroll
                for (int i = 0; i < EB; ++i) {
                    const float d = fmaf(v[b * EB + i], kLog2e, -c), e = __builtin_amdgcn_exp2f(d);
                    s1 += e;
                    t1 = fmaf(e, d, t1);
                }
            }
        }
        if (__any(!(fabsf(t1) <= FLT_MAX && fabsf(lack) <= 1.0f))) {
            // a logit of -inf (0 times the logarithm of 0 is 0), or one so
            // large that c lacks whole powers of two: d from the difference
            lack = s1 = t1 = n1 = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float d = (v[i] - ref) * kLog2e, e = v[i] == top ? 0.0f : __builtin_amdgcn_exp2f(d);
                s1 += e;
                t1 = fmaf(e, fmaxf(d, -200.0f), t1);
                n1 += v[i] == top ? 1.0f : 0.0f;
            }
        }
        t1 = fmaf(-lack, s1, t1);
        lack = __builtin_amdgcn_exp2f(-lack);
        s = fmaf(s1, lack, s);
        t = fmaf(t1, lack, t);          // in log2 units
        n += n1;
        if (a.n_top == 0) continue;
        if (looks) {
            __syncthreads();
            limit = value_of(search.found);
        }
        if (limit > -INFINITY) {
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
                bool take = of_block[b] >= limit;
                u64 on = __ballot(take);
                if (on == 0) continue;
                if (set_aside + __popcll(on) > kHot / 2) {
                    // many: of the blocks that only reach the limit the wave's next n are enough
                    const u64 even = __ballot(of_block[b] == limit);
                    take = take && (of_block[b] > limit || even_blocks + lanes_below(even) < a.n_top);
                    even_blocks += __popcll(even);
                    on = __ballot(take);
                }
                const int at = set_aside + lanes_below(on);
                if (take && at < kHot) {
                    T y[EB] __attribute__((aligned(16)));
#pragma unroll
                    for (int i = 0; i < EB; ++i) y[i] = (T)v[b * EB + i];
                    hot.block[tid >> 6][at] = *(const uint4 *)y;
                    hot.first[tid >> 6][at] = piece + (b * kThreads + tid) * EB;
                }
                set_aside += __popcll(on);
            }
        } else {
            // fewer than n above -inf: they, and the chunk's first n for those of -inf that rank
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int e = piece + ((i / EB) * kThreads + tid) * EB + i % EB;
                put(list, kept, e >= 0 && e < vocab && (v[i] > -INFINITY || e - begin < a.n_top),
                    [&] { return key_of(v[i], (unsigned)e); });
            }
        }
    }
    s = wave_sum(s);
    t = wave_sum(t);
    n = wave_sum(n);
    if (limit > -INFINITY && a.turns * a.n_top > kFewKeys) {
        // the limit again, from all pieces: a list of few is ranked sooner
        __syncthreads();
        search.x[tid] = order_of(largest);
        __syncthreads();
        search_nth(search, a.n_top);
        __syncthreads();
        limit = fmaxf(limit, value_of(search.found));
    }
    int even_before = 0;
    for (int i = tid & 63; i - (tid & 63) < min(set_aside, kHot); i += 64) {
        const bool in = i < min(set_aside, kHot);
        const uint4 y = hot.block[tid >> 6][min(i, kHot - 1)];
        const int first = hot.first[tid >> 6][min(i, kHot - 1)];
        // (and of the elements, in their order)
        float z[EB];
        int even = even_before;
#pragma unroll
        for (int q = 0; q < EB; ++q) {
            z[q] = in ? (float)((const T *)&y)[q] : -INFINITY;
            const u64 on = __ballot(z[q] == limit);
            even += lanes_below(on);
            even_before += __popcll(on);
        }
#pragma unroll
        for (int q = 0; q < EB; ++q) {
            put(list, kept, z[q] > limit || (z[q] == limit && even < a.n_top), [&] { return key_of(z[q], (unsigned)(first + q)); });
            even += z[q] == limit;
        }
    }
    if ((tid & 63) == 0) {
        *((float4 *)a.stats + ((int64_t)row * a.n_chunks + chunk) * kWaves + (tid >> 6)) = float4{m, s, t * kLn2, n};
        list.count[tid >> 6] = min(kept, kPiece);
        wave_odd[tid >> 6] = s != s || kept > kPiece || set_aside > kHot;   // NaN or +inf, or a full list
    }
    if (a.n_top == 0) return;
    __syncthreads();
    u64 *out = a.keys + ((int64_t)row * a.n_chunks + chunk) * a.n_top;
    if (wave_odd[0] | wave_odd[1] | wave_odd[2] | wave_odd[3])
        pick(x, begin, end, a.n_top, wave_best, out);
    else
        rank(list, a.n_top, out);
}

// keys of the chunks' lists per thread and turn: with the largest so far, a
// wave's fit its piece
constexpr int kJoinPer = 3;
// up to so many keys go to the list all together, without a limit (160 keys of
// a bf16 row 12.1 us, 10.2 with one; 80 of 251 rows 25.4 us, 25.8 with one)
constexpr int kJoinAll = 128;

// A wave's, or several waves', elements: the maximum m, how many there are of
// it, and of the others the sums of exp(x - m) and (x - m) exp(x - m).  The
// maximum's own terms are kept apart because in a row that is sure of its
// token they are all but the whole sum: log(n + s) = log n + log1p(s / n) then
// has the others' part in full.
struct Sums {
    float m, s, t, n;
    // to the maximum `to`, which is not below m; what has no term, or weighs
    // nothing, adds nothing
    __device__ __forceinline__ void bring(float to) {
        if (m == to) return;
        const float d = m - to, f = expf(d), all = s + n;
        t = all != 0.0f && f != 0.0f ? f * (t + d * all) : 0.0f;
        s = all != 0.0f ? f * all : 0.0f;
        n = 0.0f;
        m = to;
    }
};

// A work group per row.  Latency: statistics and lists, the token's logit, a
// search and a ranking (one row 4.7 us, 251 rows with 20 alternatives 5.2 us).
template <typename T>
__global__ __launch_bounds__(kThreads) void k_logprobs_join(LogprobsArgs a) {
    __shared__ List list;
    __shared__ Search search;
    __shared__ u64 top[kLogprobsMaxTop];
    __shared__ float red[kWaves][4];
    const int tid = threadIdx.x, row = blockIdx.x;
    const float4 *st = (const float4 *)a.stats + (int64_t)row * a.n_chunks * kWaves;
    const int n_stats = a.n_chunks * kWaves;
    const u64 *keys = a.keys + (int64_t)row * a.n_chunks * a.n_top;
    const int n_keys = a.n_chunks * a.n_top;

    // everything the row needs is asked for at once; the waves take turns at
    // the keys, so that few of them are shared out evenly
    const int mine = (tid & 63) * kWaves + (tid >> 6);
    u64 k[kJoinPer];
#pragma unroll
    for (int i = 0; i < kJoinPer; ++i) k[i] = i * kThreads + mine < n_keys ? keys[i * kThreads + mine] : 0;
    const int token = a.tokens ? a.tokens[row] : -1;
    const bool is_token = token >= 0 && token < a.n_vocab;
    const float at_token = is_token ? (float)((const T *)a.logits)[row * a.row_stride + token] : 0.0f;
    Sums sums{-INFINITY, 0.0f, 0.0f, 0.0f};
    for (int i = tid; i < n_stats; i += kThreads) {
        const float4 y = st[i];
        Sums more{y.x, y.y, y.z, y.w};
        const float to = fmaxf(sums.m, more.m);
        sums.bring(to);
        more.bring(to);
        sums.s += more.s;
        sums.t += more.t;
        sums.n += more.n;
    }
    const float wm = wave_max(sums.m);
    if ((tid & 63) == 0) red[tid >> 6][0] = wm;
    __syncthreads();
    const float ref = fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0]));
    sums.bring(ref);
    const float ws = wave_sum(sums.s), wt = wave_sum(sums.t), wn = wave_sum(sums.n);
    if ((tid & 63) == 0) {
        red[tid >> 6][1] = ws;
        red[tid >> 6][2] = wt;
        red[tid >> 6][3] = wn;
    }

    // the n largest keys: as in a chunk, a turn's worth of keys at a time,
    // joined with the largest so far
    if (tid < kLogprobsMaxTop) top[tid] = 0;
    for (int base = 0; base < n_keys; base += kThreads * kJoinPer) {
        if (base)
#pragma unroll
            for (int i = 0; i < kJoinPer; ++i) {
                const int at = base + i * kThreads + mine;
                k[i] = at < n_keys ? keys[at] : 0;
            }
        u64 best = 0;
#pragma unroll
        for (int i = 0; i < kJoinPer; ++i) best = k[i] > best ? k[i] : best;
        u64 least = 1;
        __syncthreads();
        if (n_keys > kJoinAll) {
            search.x[tid] = (unsigned)(best >> 32);
            __syncthreads();
            search_nth(search, a.n_top);
            __syncthreads();
            least = max((u64)search.found << 32, (u64)1);
        }
        int kept = 0;
#pragma unroll
        for (int i = 0; i < kJoinPer; ++i) put(list, kept, k[i] >= least, [&] { return k[i]; });
        if (base) put(list, kept, tid < a.n_top && top[tid] >= least, [&] { return top[tid]; });
        if ((tid & 63) == 0) list.count[tid >> 6] = kept;
        __syncthreads();
        rank(list, a.n_top, top);
    }
    __syncthreads();
    const float s = red[0][1] + red[1][1] + red[2][1] + red[3][1];
    const float t = red[0][2] + red[1][2] + red[2][2] + red[3][2];
    const float n = red[0][3] + red[1][3] + red[2][3] + red[3][3];
    // a row of -inf alone: no sum
    const bool none = n == 0.0f && s == 0.0f;
    const float log_s = none ? 0.0f : logf(n) + log1pf(s / n);
    auto logprob = [&](float x) { return none ? -INFINITY : (x - ref) - log_s; };
    if (tid < a.n_top) {
        const u64 key = top[tid];
        a.top_ids[(int64_t)row * a.n_top + tid] = (int32_t)(0xffffffffu - (unsigned)key);
        a.top_logprobs[(int64_t)row * a.n_top + tid] = logprob(value_of((unsigned)(key >> 32)));
    }
    if (tid == kThreads - 1) {
        if (a.entropy) a.entropy[row] = none ? 0.0f : log_s - t / (n + s);
        if (a.tokens) a.logprob[row] = is_token ? logprob(at_token) : token == -1 ? 0.0f : __builtin_nanf("");
    }
}

template <typename T> hipError_t run(const LogprobsArgs &a, int blocks, hipStream_t st) {
    const dim3 grid((unsigned)a.n_chunks, (unsigned)a.n_rows);
    if (blocks == kBlocksFew)
        k_logprobs_part<T, kBlocksFew><<<grid, kThreads, 0, st>>>(a);
    else
        k_logprobs_part<T, sizeof(T) == 4 ? 8 : 4><<<grid, kThreads, 0, st>>>(a);
    k_logprobs_join<T><<<(unsigned)a.n_rows, kThreads, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace

LogprobsPlan logprobs_plan(int n_rows, int64_t n_vocab, int elem_bytes, int n_top, bool rows_aligned) {
    // blocks of a row, wherever in a block it begins
    const int64_t per = 16 / elem_bytes, blocks = (n_vocab + (rows_aligned ? 1 : 2) * (per - 1)) / per;
    LogprobsPlan p;
    const int64_t small = (blocks + kBlocksFew * kThreads - 1) / (kBlocksFew * kThreads);
    p.blocks = n_rows * small <= kFewGroups && small * n_top <= kThreads * kJoinPer ? kBlocksFew : elem_bytes == 4 ? 8 : 4;
    const int64_t pieces = (blocks + p.blocks * kThreads - 1) / (p.blocks * kThreads);
    p.turns = (int32_t)std::min<int64_t>((n_rows * pieces + kManyGroups - 1) / kManyGroups, std::min<int64_t>(pieces, kTurnsMost));
    p.chunks = (int32_t)((pieces + p.turns - 1) / p.turns);
    return p;
}

int64_t logprobs_chunks_most(int64_t n_rows, int64_t n_vocab) {
    int64_t most = 0;
    for (int per : {4, 8}) {
        const int64_t blocks = (n_vocab + 2 * (per - 1)) / per;
        const int64_t small = (blocks + kBlocksFew * kThreads - 1) / (kBlocksFew * kThreads);
        const int64_t large = (blocks + 32 / per * kThreads - 1) / (32 / per * kThreads);
        // a chunk of `turns` pieces: turns is 1, its most, or at least what leaves kManyGroups chunks
        const int64_t many = std::max(n_rows * ((large + kTurnsMost - 1) / kTurnsMost), std::min(n_rows * large, kManyGroups + n_rows));
        most = std::max(most, std::max(std::min(n_rows * small, kFewGroups), many));
    }
    return most;
}

hipError_t launch_logprobs(int dtype, const LogprobsArgs &a, int blocks, hipStream_t st) {
    if (dtype == VKV_DTYPE_F16) return run<_Float16>(a, blocks, st);
    if (dtype == VKV_DTYPE_BF16) return run<__bf16>(a, blocks, st);
    return run<float>(a, blocks, st);
}

}  // namespace vkv
