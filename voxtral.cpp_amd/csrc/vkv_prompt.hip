// Causal attention of packed prompts on gfx950.
//
// Two launches.  k_prompt_pack turns each prompt's K and V, a tile of 64 or 32
// keys of one kv head at a time, into the operands of v_mfma_f32_32x32x16: 1
// KiB pieces of 16 bytes per lane, V transposed.  Every query tile of the prompt
// reads them again, so the transposition, the split of f32 rows and the search
// for the largest value are paid once per key instead of once per (key, query
// tile).
// k_prompt_attn then streams them into LDS unchanged and keeps everything
// else in registers.
//
// f32 rows are multiplied as hi + lo with both in f16 (x hi, lo = x - hi;
// three products, the fourth is below f32's own rounding): the matrix cores'
// f32 form runs at 1/16 of the f16 rate, the three f16 products at 1/3.  q is
// scaled by a power of two per row, K and V per tile, to a largest magnitude
// in [2^13, 2^14), so that lo keeps its 11 bits down to 2^-15 of it.
#include <hip/hip_runtime.h>

#include <cfloat>

#include "vkv_serve.h"

namespace vkv {
namespace {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kTopExp = 13;     // scaled rows have their largest magnitude in [2^13, 2^14)
constexpr int kPExp = 6;        // p <= 2^8 is scaled to <= 2^14

// T: type of the rows; F32 rows become two f16 planes
template <typename T> struct Operand {
    typedef _Float16 elem;
    static constexpr int planes = 1;
};
template <> struct Operand<float> {
    typedef _Float16 elem;
    static constexpr int planes = 2;
};
template <> struct Operand<__bf16> {
    typedef __bf16 elem;
    static constexpr int planes = 1;
};

// keys of a tile: two tiles take half of a CU's LDS at the most
template <typename T, int D> constexpr int tile_keys() { return prompt_keys(Operand<T>::planes, D); }

template <typename E> __device__ __forceinline__ floatx16 mfma(uint4 a, uint4 b, floatx16 c) {
    if constexpr (std::is_same<E, __bf16>::value)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8_t, a), __builtin_bit_cast(bf8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

template <typename E> struct Vec8 { typedef E type __attribute__((ext_vector_type(8))); };

// eight values rounded to the operand type
template <typename E> __device__ __forceinline__ uint4 round8(const float *x) {
    typename Vec8<E>::type r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (E)x[i];
    return __builtin_bit_cast(uint4, r);
}

// and what that leaves of them; CHECK: nothing of what is not finite
template <bool CHECK> __device__ __forceinline__ uint4 rest8(const float *x) {
    half8_t r;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float hi = (float)(_Float16)x[i];
        r[i] = (_Float16)(!CHECK || fabsf(hi) <= FLT_MAX ? x[i] - hi : 0.0f);
    }
    return __builtin_bit_cast(uint4, r);
}

template <typename T> __device__ __forceinline__ void load8(const T *p, float *x) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *(const float4 *)p, b = *(const float4 *)(p + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const auto v = __builtin_bit_cast(typename Vec8<T>::type, *(const uint4 *)p);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
    }
}

__device__ __forceinline__ float finite_abs(float x) {
    x = fabsf(x);
    return x <= FLT_MAX ? x : 0.0f;
}

__device__ __forceinline__ int exponent(float amax) {
    return amax > 0.0f ? max((int)(__float_as_uint(amax) >> 23) - 127, -100) : 0;
}

// the two halves of a wave
__device__ __forceinline__ float halves_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

struct Prompt {
    int seq, start, n, local;    // local: the slot's number among the prompt's own
};

// Prompt i's slots of `per` units begin at floor(cu[i] * mul / per) + i: at
// least ceil(n_i * mul / per) of them lie before prompt i + 1's, so the place
// of every slot follows from the offsets alone, without a sum over the
// prompts.  Offsets are held to [0, n_tokens], whatever they are.
__device__ __forceinline__ int offset_of(const PromptArgs &a, int i) {
    return min(max(((const __attribute__((address_space(4))) int32_t *)a.cu)[i], 0), a.n_tokens);
}
__device__ __forceinline__ bool find_prompt(const PromptArgs &a, int64_t slot, int mul, int per, Prompt &p) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = a.n_seq;
    for (;;) {   // a 64th of the range is left at each turn
        const int step = (hi - lo + 63) / 64;
        const int i = lo + lane * step;
        const bool le = i < hi && (int64_t)offset_of(a, min(i, a.n_seq)) * mul / per + i <= slot;
        const int c = __popcll(__ballot(le));
        if (c == 0) return false;
        lo += (c - 1) * step;
        hi = min(hi, lo + step);
        if (step == 1) break;
    }
    p.seq = __builtin_amdgcn_readfirstlane(lo);
    p.start = offset_of(a, p.seq);
    p.n = max(offset_of(a, p.seq + 1) - p.start, 0);
    p.local = (int)(slot - ((int64_t)p.start * mul / per + p.seq));
    return true;
}

// What k_prompt_pack says of a tile: the exponents of K and V and whether V
// holds what is not finite, in one word.
struct TileInfo {
    int word;
    __device__ int ek() const { return (word & 1023) - 512; }
    __device__ int ev() const { return (word >> 10 & 1023) - 512; }
    __device__ int odd() const { return word >> 20; }
};

// A tile's operands: K, planes x [blocks of 32 keys][D/16][64 lanes] 16 bytes:
// lane (r, h) has key 32 kb + r, dims 16 m + 8 h + [0, 8).  V, planes x
// [D/32][blocks of 16 keys][64 lanes]: lane (r, h) has dim 32 dt + r, keys
// 16 u + 4 h + [0, 4) and 16 u + 8 + 4 h + [0, 4), the keys whose scores a
// lane of half h holds.
template <typename T, int D> constexpr int tile_bytes() { return Operand<T>::planes * 2 * tile_keys<T, D>() * D * 2; }

// A work group per (tile, kv head).  K rows go from memory to their lanes as
// they are; V passes through LDS, by rows in and by columns out.  Bound by
// memory: 8192 tokens of 8 x 128 bf16, 67 MB in and out, 15.3 us, 4.4 TB/s; 6539
// tokens of f32 in 13 prompts, 107 MB, 25 us, 4.3 TB/s; 38 tokens 4.7 us, a
// launch and its loads' latency.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_prompt_pack(PromptArgs a) {
    typedef typename Operand<T>::elem E;
    constexpr int NP = Operand<T>::planes, kTile = tile_keys<T, D>(), U = kTile / 16;
    constexpr int NS = kTile * D / 8 / 256;     // 16-byte pieces per thread, K or V
    __shared__ float vt[kTile][D];
    __shared__ float red[4][2];
    __shared__ int odd;
    const int tid = threadIdx.x;
    const int head = blockIdx.y;
    Prompt p;
    if (!find_prompt(a, blockIdx.x, 1, kTile, p)) return;
    const int key0 = p.local * kTile;
    if (key0 >= p.n) return;
    if (tid == 0) odd = 0;
    __syncthreads();
    const int64_t tile = (int64_t)head * a.n_tiles + blockIdx.x;

    float kx[NS][8];
    float kmax = 0.0f, vmax = 0.0f;
    bool strange = false;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int piece = tid + 256 * s, l = piece & 63, m = (piece >> 6) % (D / 16), kb = (piece >> 6) / (D / 16);
        const int key = key0 + 32 * kb + (l & 31);
        if (key < p.n)
            load8((const T *)a.k + (p.start + key) * a.k_stride + head * D + 16 * m + 8 * (l >> 5), kx[s]);
        else
            for (int i = 0; i < 8; ++i) kx[s][i] = 0.0f;
        // V by rows into LDS
        const int row = piece / (D / 8), d = piece % (D / 8) * 8;
        float x[8];
        if (key0 + row < p.n)
            load8((const T *)a.v + (p.start + key0 + row) * a.v_stride + head * D + d, x);
        else
            for (int i = 0; i < 8; ++i) x[i] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // a key without weight must not reach the output, and 0 times
            // what is not finite would: such values are left to k_prompt_attn
            const bool fine = fabsf(x[i]) <= FLT_MAX;
            strange |= !fine;
            vt[row][d + i] = fine ? x[i] : 0.0f;
            kmax = fmaxf(kmax, finite_abs(kx[s][i]));
            vmax = fmaxf(vmax, finite_abs(x[i]));
        }
    }
    if (strange) odd = 1;
    int ek = kTopExp, ev = kTopExp;
    if constexpr (NP == 2) {
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            kmax = fmaxf(kmax, __shfl_xor(kmax, d));
            vmax = fmaxf(vmax, __shfl_xor(vmax, d));
        }
        if ((tid & 63) == 0) {
            red[tid >> 6][0] = kmax;
            red[tid >> 6][1] = vmax;
        }
        __syncthreads();
        ek = exponent(fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0])));
        ev = exponent(fmaxf(fmaxf(red[0][1], red[1][1]), fmaxf(red[2][1], red[3][1])));
    } else {
        __syncthreads();
    }
    uint4 *out = (uint4 *)(a.data + tile * tile_bytes<T, D>());
    constexpr int PLANE = kTile * D / 8;        // 16-byte pieces of a plane
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int piece = tid + 256 * s;
        if constexpr (NP == 2) {
            for (int i = 0; i < 8; ++i) kx[s][i] = ldexpf(kx[s][i], kTopExp - ek);
            out[PLANE + piece] = rest8<true>(kx[s]);
        }
        out[piece] = round8<E>(kx[s]);
        const int l = piece & 63, u = (piece >> 6) % U, dt = (piece >> 6) / U;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int key = 16 * u + (i >= 4 ? 8 : 0) + 4 * (l >> 5) + (i & 3);
            x[i] = vt[key][32 * dt + (l & 31)];
            if constexpr (NP == 2) x[i] = ldexpf(x[i], kTopExp - ev);
        }
        if constexpr (NP == 2) out[3 * PLANE + piece] = rest8<true>(x);
        out[NP * PLANE + piece] = round8<E>(x);
    }
    if (tid == 0) a.info[tile] = (ek + 512) | (ev + 512) << 10 | odd << 20;
}

constexpr int kPromptThreads = 2 * kPromptRows;

// Half a tile (K or V) into LDS without registers; buffer loads, beside which
// the waits for LDS reads stay counted.
template <int BYTES> __device__ __forceinline__ void fetch(const uint8_t *src, uint8_t *dst, int wave) {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)src, 0, BYTES, 0x00020000);
#pragma unroll
    for (int i = 0; i < BYTES / (kPromptThreads * 16); ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rsrc, (__attribute__((address_space(3))) void *)(dst + i * (kPromptThreads * 16) + wave * 1024), 16,
            threadIdx.x * 16, i * (kPromptThreads * 16), 0, 0);
}

__device__ __forceinline__ void wait_for_memory() { __builtin_amdgcn_s_waitcnt(0x0f70); }   // vmcnt(0)

// none of the wave's LDS reads are under way, and the others are as far
__device__ __forceinline__ void meet() {
    __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0)
    asm volatile("s_barrier" ::: "memory");
}

// A wave's 32 rows: their columns of Q and of O^T; the scores of a tile, then
// its weights; the running maximum (in log2 units) and the sum of each column,
// every lane its own half of the keys; the factor of the scores; the exponent
// that O's weights are scaled by.
template <typename T, int D> struct Rows {
    static constexpr int keys = tile_keys<T, D>();
    uint4 q[Operand<T>::planes][D / 16], p[Operand<T>::planes][keys / 16];
    floatx16 o[D / 32], s[keys / 32];
    float factor, m, l;
    int ev_ref, large;
    int token, t_first, t_last;
    int first_tile, last_tile;      // of those the wave sees
};

// S^T of the tile whose K is at k
template <typename T, int D> __device__ __forceinline__ void scores(Rows<T, D> &r, const uint8_t *k) {
    typedef typename Operand<T>::elem E;
    constexpr int NP = Operand<T>::planes, NM = D / 16, KB = Rows<T, D>::keys / 32, PLANE = KB * 32 * D * 2;
    k += (threadIdx.x & 63) * 16;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) r.s[kb][i] = 0.0f;
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const uint4 hi = *(const uint4 *)(k + (kb * NM + m) * 1024);
            r.s[kb] = mfma<E>(hi, r.q[0][m], r.s[kb]);
            if constexpr (NP == 2) {
                const uint4 lo = *(const uint4 *)(k + PLANE + (kb * NM + m) * 1024);
                r.s[kb] = mfma<E>(hi, r.q[1][m], r.s[kb]);
                r.s[kb] = mfma<E>(lo, r.q[0][m], r.s[kb]);
            }
        }
}

// V's values that are not finite, left out of the product: the rows that see
// their key take them as they are.
template <typename T, int D>
__device__ __forceinline__ void strange_values(const PromptArgs &a, const Prompt &p, int head, int kt, Rows<T, D> &r) {
    constexpr int KEYS = Rows<T, D>::keys;
#pragma unroll 1
    for (int key = kt * KEYS; key < (kt + 1) * KEYS && key < p.n; ++key) {
        const bool in = key <= r.token && (a.window <= 0 || key > r.token - a.window);
        const T *x = (const T *)a.v + (p.start + key) * a.v_stride + head * D + 4 * (int)((threadIdx.x & 63) >> 5);
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float y = (float)x[32 * t + 8 * (i >> 2) + (i & 3)];
                if (in && !(fabsf(y) <= FLT_MAX)) r.o[t][i] += y;
            }
    }
}

// The matrix cores' half of a tile: O^T += V^T P^T for the tile whose weights
// are at hand, and the scores of the next.  The next tile's operands are
// fetched into the other places on the way: the four are restrict, or each
// read would wait for the loads.  LAST: there is no next.
template <typename T, int D, bool LAST>
__device__ __forceinline__ void products(const PromptArgs &a, const Prompt &p, int head, int kt, int odd, int wave,
                                         const uint8_t *k_src, const uint8_t *v_src, const uint8_t *__restrict__ k_cur,
                                         uint8_t *__restrict__ k_next, const uint8_t *__restrict__ v_cur,
                                         uint8_t *__restrict__ v_next, Rows<T, D> &r) {
    typedef typename Operand<T>::elem E;
    constexpr int NP = Operand<T>::planes, NM = D / 16, ND = D / 32, KEYS = Rows<T, D>::keys, U = KEYS / 16;
    constexpr int HALF = tile_bytes<T, D>() / 2, PLANE = KEYS * D * 2;
    const int lane = threadIdx.x & 63;
    if constexpr (!LAST) {
        fetch<HALF>(k_src, k_next, wave);
        fetch<HALF>(v_src, v_next, wave);
    }
    if (kt + 1 < r.first_tile || kt > r.last_tile) return;
    const uint8_t *v = v_cur + lane * 16;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int t = 0; t < ND; ++t) {
            const uint4 vh = *(const uint4 *)(v + (t * U + u) * 1024);
            r.o[t] = mfma<E>(vh, r.p[0][u], r.o[t]);
            if constexpr (NP == 2) {
                r.o[t] = mfma<E>(vh, r.p[1][u], r.o[t]);
                r.o[t] = mfma<E>(*(const uint4 *)(v + PLANE + (t * U + u) * 1024), r.p[0][u], r.o[t]);
            }
        }
    if constexpr (!LAST) scores(r, k_cur);
    // a few operands are read ahead of the products
    constexpr int AHEAD = NP == 2 ? 2 : 6, PAIRS = U * ND + (LAST ? 0 : KEYS / 32 * NM);
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * NP, 0);
#pragma unroll
    for (int i = 0; i < PAIRS - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, NP == 2 ? 3 : 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, NP, 0);
    }
    if (odd) strange_values(a, p, head, kt, r);
}

// The vector units' half: the scores of tile kt become weights, and the sums
// so far are brought to the new maximum.
template <typename T, int D>
__device__ __forceinline__ void weights(const PromptArgs &a, int kt, TileInfo info, Rows<T, D> &r) {
    typedef typename Operand<T>::elem E;
    constexpr int NP = Operand<T>::planes, ND = D / 32, KEYS = Rows<T, D>::keys, U = KEYS / 16;
    if (kt < r.first_tile || kt > r.last_tile) {
#pragma unroll
        for (int n = 0; n < NP; ++n)
#pragma unroll
            for (int u = 0; u < U; ++u) r.p[n][u] = uint4{0, 0, 0, 0};
        return;
    }
    const float f = fmaxf(NP == 2 ? ldexpf(r.factor, info.ek() - kTopExp) : r.factor, FLT_MIN);
    const int key0 = kt * KEYS;
    if (key0 + KEYS - 1 > r.t_first || (a.window > 0 && key0 <= r.t_last - a.window)) {
        // keys [low, high], counted from this lane's first
        const int high = r.token - key0 - 4 * (int)((threadIdx.x & 63) >> 5);
        const int low = a.window > 0 ? high - a.window + 1 : INT32_MIN;
#pragma unroll
        for (int i = 0; i < KEYS / 2; ++i) {
            const int j = 32 * (i >> 4) + 8 * (i >> 2 & 3) + (i & 3);
            r.s[i >> 4][i & 15] = j <= high && j >= low ? r.s[i >> 4][i & 15] : -INFINITY;
        }
    }
    float mx = r.s[0][0];
#pragma unroll
    for (int i = 1; i < KEYS / 2; ++i) mx = fmaxf(mx, r.s[i >> 4][i & 15]);
    mx = halves_max(mx) * f;
    // the running maximum moves only when it is passed by 2^8
    if (__any(mx > r.m + 8.0f)) {
        const float m_new = fmaxf(r.m, mx);
        const float g = m_new > -INFINITY ? __builtin_amdgcn_exp2f(r.m - m_new) : 1.0f;
        r.l *= g;
#pragma unroll
        for (int t = 0; t < ND; ++t) r.o[t] *= g;
        r.m = m_new;
        r.large = __any(m_new > -INFINITY && fabsf(m_new) > 0x1p20f);
    }
    float pfac = 1.0f;
    if constexpr (NP == 2) {
        const int ev = info.ev();
        if (ev > r.ev_ref) {
            const float g = ldexpf(1.0f, max(r.ev_ref - ev, -300));
#pragma unroll
            for (int t = 0; t < ND; ++t) r.o[t] *= g;
            r.ev_ref = ev;
        }
        pfac = ldexpf(1.0f, kPExp + ev - r.ev_ref);
    }
    float by = f, from = r.m > -INFINITY ? -r.m : 0.0f;
    if (r.large) {
        // the maximum's own rounding would show in the largest weights: every
        // score is rounded as it was
#pragma clang fp contract(off)
#pragma unroll
        for (int i = 0; i < KEYS / 2; ++i) {
            const float x = r.s[i >> 4][i & 15] * f;
            r.s[i >> 4][i & 15] = x + from;
        }
        by = 1.0f;
        from = 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float e = __builtin_amdgcn_exp2f(fmaf(r.s[u >> 1][(u & 1) * 8 + i], by, from));
            r.l += e;
            x[i] = NP == 2 ? e * pfac : e;
        }
        r.p[0][u] = round8<E>(x);
        if constexpr (NP == 2) r.p[1][u] = rest8<false>(x);
    }
}

// The wave's 32 rows at wrow: their places, the tiles that they see, and this
// lane's column of Q (dims 16 m + 8 half + [0, 8)) on its way to x; the row's
// query head of the kv head is returned.
template <typename T, int D>
__device__ __forceinline__ int take_rows(const PromptArgs &a, const Prompt &p, int head, unsigned wrow, unsigned rows, Rows<T, D> &r,
                                         float (&x)[D / 16][8]) {
    constexpr int KEYS = Rows<T, D>::keys;
    const int lane = threadIdx.x & 63, group = a.n_q_heads / a.n_kv_heads;
    const unsigned row = min(wrow + (lane & 31), rows - 1);
    r.token = (int)(row / (unsigned)group);
    const int hq = (int)(row - (unsigned)r.token * (unsigned)group);
    r.t_first = __builtin_amdgcn_readlane(r.token, 0);
    r.t_last = __builtin_amdgcn_readlane(r.token, 31);
    r.first_tile = a.window > 0 && r.t_first >= a.window ? (r.t_first - a.window + 1) / KEYS : 0;
    r.last_tile = wrow < rows ? r.t_last / KEYS : -2;      // a wave without rows sees no key
    const T *q = (const T *)a.q + (p.start + r.token) * a.q_stride + (head * group + hq) * D + 8 * (lane >> 5);
#pragma unroll
    for (int m = 0; m < D / 16; ++m) load8(q + 16 * m, x[m]);
    return hq;
}

// Q in its form, and nothing summed so far.
template <typename T, int D>
__device__ __forceinline__ void start_rows(const PromptArgs &a, float (&x)[D / 16][8], Rows<T, D> &r) {
    typedef typename Operand<T>::elem E;
    constexpr int NP = Operand<T>::planes, NM = D / 16, ND = D / 32;
    r.factor = fabsf(a.scale) * kLog2e;
    float by = a.scale < 0.0f ? -1.0f : 1.0f;
    bool fine = true;       // the largest value's exponent is that of finite ones
    if constexpr (NP == 2) {
        unsigned top = 0;
#pragma unroll
        for (int m = 0; m < NM; ++m)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[m][i]) & 0x7fffffffu);
        fine = !__any(top >= 0x7f800000u);
        if (!fine) {
            top = 0;
#pragma unroll
            for (int m = 0; m < NM; ++m)
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(finite_abs(x[m][i])));
        }
        const int e = exponent(halves_max(__uint_as_float(top)));
        r.factor = ldexpf(r.factor, e - kTopExp);
        by = ldexpf(by, kTopExp - e);
    }
#pragma unroll
    for (int m = 0; m < NM; ++m) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[m][i] *= by;
        r.q[0][m] = round8<E>(x[m]);
        if constexpr (NP == 2) r.q[1][m] = rest8<false>(x[m]);
    }
    if (!fine)
#pragma unroll
        for (int m = 0; m < NM; ++m)
            if constexpr (NP == 2) r.q[1][m] = rest8<true>(x[m]);
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) r.o[t][i] = 0.0f;
    r.m = -INFINITY;
    r.l = 0.0f;
    r.ev_ref = -1000;
    r.large = 0;
}

// A work group: 4 waves on 128 rows of one (prompt, kv head), a row being
// (token, query head of the kv head), so the heads that share K and V read one
// copy of them in LDS.  Wave w owns rows 32 w + [0, 32) as the columns of S^T =
// K Q^T and O^T = V^T P^T; a lane's scores are the keys it supplies to the
// second product, so P stays in its registers.
//
// The products of a tile and the softmax of a tile take about as long, on
// units that can work at the same time: the registers and the LDS of a work
// group leave room for a second one on the CU, and each SIMD's two waves, of
// two work groups that never wait for each other, fill each other's gaps (13
// prompts of up to 1021 tokens, f32: 168 us, 180 with one work group of two
// halves that take turns; 38 tokens 9.5 and 15 us).  Operands of tile kt's turn
// (its V, the K of tile kt + 1) are in LDS at its start; those of the next come
// in meanwhile.
//
// Bound by the matrix cores at the clock that they leave: 8192 tokens of 32
// heads of 128 in bf16, 550 Gflop, 508 to 540 us with the card, 1.02 to 1.08
// Pflop/s, where a product of two 8192 x 8192 matrices runs at 1.14; f32, three
// products, 1.3 ms, 1.26 Pflop/s of f16 products.  13 prompts as above: 153 us,
// 0.75 Pflop/s: work groups of 11 tiles on average, whose first loads and
// last stores no work of their own hides.
template <typename T, int D>
__global__ __launch_bounds__(kPromptThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_prompt_attn(PromptArgs a) {
    constexpr int NP = Operand<T>::planes;
    constexpr int NM = D / 16, ND = D / 32, KEYS = Rows<T, D>::keys;
    constexpr int BYTES = tile_bytes<T, D>(), HALF = BYTES / 2;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * BYTES];   // K, K, V, V

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = lane >> 5;
    const int group = a.n_q_heads / a.n_kv_heads;
    const int head = blockIdx.x % a.n_kv_heads;
    // the later tiles of a prompt have the most keys: they go first
    const int64_t slot = a.n_slots - 1 - blockIdx.x / a.n_kv_heads;
    Prompt p;
    if (!find_prompt(a, slot, group, kPromptRows, p)) return;
    // a call's rows are fewer than 2^31
    const unsigned rows = (unsigned)p.n * (unsigned)group;
    const unsigned row0 = (unsigned)p.local * kPromptRows;
    if (row0 >= rows) return;

    Rows<T, D> r;
    float x[NM][8];
    const unsigned wrow = row0 + 32 * wave, row = wrow + (lane & 31);
    const int hq = take_rows(a, p, head, wrow, rows, r, x);
    const int wg_first = (int)(row0 / (unsigned)group);
    const int wg_last = (int)(min(row0 + kPromptRows, rows) - 1) / group;
    const int kt0 = a.window > 0 && wg_first >= a.window ? (wg_first - a.window + 1) / KEYS : 0;
    const int kt1 = wg_last / KEYS;
    const int64_t tile0 = (int64_t)head * a.n_tiles + p.start / KEYS + p.seq;
    const uint8_t *data = a.data + tile0 * BYTES;
    // the words of 64 tiles, a lane each: a load for every tile would have the
    // waits for it cover the operands that are on their way
    auto tile_words = [&](int kt) { return a.info[tile0 + min(kt + lane, kt1)]; };
    int words = tile_words(kt0);
    // K of the first tile where the turn before the first has it, then the first turn's operands
    fetch<HALF>(data + (int64_t)kt0 * BYTES, lds + HALF, wave);
    fetch<HALF>(data + (int64_t)min(kt0 + 1, kt1) * BYTES, lds, wave);
    fetch<HALF>(data + (int64_t)kt0 * BYTES + HALF, lds + 2 * HALF, wave);

    start_rows(a, x, r);
    wait_for_memory();
    meet();
    scores(r, lds + HALF);
    TileInfo info{__builtin_amdgcn_readlane(words, 0)};
    weights(a, kt0, info, r);
    meet();
    int cur = 0;
    for (int kt = kt0; kt < kt1; ++kt, cur = HALF - cur) {
        const int next = HALF - cur;
        products<T, D, false>(a, p, head, kt, info.odd(), wave, data + (int64_t)min(kt + 2, kt1) * BYTES,
                              data + (int64_t)(kt + 1) * BYTES + HALF, lds + cur, lds + next, lds + 2 * HALF + cur,
                              lds + 2 * HALF + next, r);
        if (((kt + 1 - kt0) & 63) == 0) {
            words = tile_words(kt + 1);
            asm volatile("" : "+v"(words));     // waited for here, not at every tile
        }
        info.word = __builtin_amdgcn_readlane(words, (kt + 1 - kt0) & 63);
        weights(a, kt + 1, info, r);
        wait_for_memory();
        meet();
    }
    products<T, D, true>(a, p, head, kt1, info.odd(), wave, nullptr, nullptr, nullptr, nullptr, lds + 2 * HALF + cur, nullptr, r);

    const float l = halves_sum(r.l);
    if (row < rows) {
        float g = l != 0.0f ? 1.0f / l : 0.0f;
        if constexpr (NP == 2) g = ldexpf(g, r.ev_ref - kTopExp - kPExp);
        T *out = (T *)a.out + (p.start + r.token) * a.out_stride + (head * group + hq) * D + 4 * half;
#pragma unroll
        for (int t = 0; t < ND; ++t)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                T y[4] __attribute__((aligned(16)));
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = (T)(r.o[t][4 * b + i] * g);
                if constexpr (sizeof(T) == 4)
                    *(float4 *)(out + 32 * t + 8 * b) = *(const float4 *)y;
                else
                    *(uint2 *)(out + 32 * t + 8 * b) = *(const uint2 *)y;
            }
    }
}

// The same where there are few rows: a work group's 4 waves share 32 rows and
// take the key tiles in turn, and their parts meet in LDS.  No two waves read
// the same operands, so they come straight into registers: V's while the
// scores are made, the next K while they become weights.  Bound by those
// loads' latency: f32, 32 heads over 8 of 128, 200 tokens 15.8 us with the
// launch of k_prompt_pack, 21.0 by k_prompt_attn.
template <typename T, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void k_prompt_attn_few(PromptArgs a) {
    typedef typename Operand<T>::elem E;
    constexpr int NP = Operand<T>::planes, NM = D / 16, ND = D / 32, KEYS = Rows<T, D>::keys, KB = KEYS / 32, U = KEYS / 16;
    constexpr int BYTES = tile_bytes<T, D>(), HALF = BYTES / 2, PIECES = HALF / 1024, PLANE = PIECES / NP;
    constexpr int OWN = 2 * ND;             // of half of O's 16 ND values per lane, a wave's to join
    __shared__ float parts[4][4 * OWN][64];
    __shared__ float lds_m[4][64], lds_l[4][64];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int group = a.n_q_heads / a.n_kv_heads;
    const int head = blockIdx.x % a.n_kv_heads;
    Prompt p;
    if (!find_prompt(a, a.n_slots - 1 - blockIdx.x / a.n_kv_heads, group, kPromptRowsFew, p)) return;
    const unsigned rows = (unsigned)p.n * (unsigned)group;
    const unsigned row0 = (unsigned)p.local * kPromptRowsFew, row = row0 + (lane & 31);
    if (row0 >= rows) return;
    Rows<T, D> r;
    float x[NM][8];
    const int hq = take_rows(a, p, head, row0, rows, r, x);
    const int kt0 = r.first_tile, kt1 = r.last_tile;
    const int64_t tile0 = (int64_t)head * a.n_tiles + p.start / KEYS + p.seq;
    const uint8_t *data = a.data + tile0 * BYTES + lane * 16;
    int words_at = kt0, words = a.info[tile0 + min(kt0 + lane, kt1)];
    uint4 k[PIECES], v[PIECES];
    auto load = [&](uint4 (&to)[PIECES], const uint8_t *from) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) to[i] = *(const uint4 *)(from + i * 1024);
    };
    load(k, data + (int64_t)min(kt0 + wave, kt1) * BYTES);
    start_rows(a, x, r);
    for (int kt = kt0 + wave; kt <= kt1; kt += 4) {
        load(v, data + (int64_t)kt * BYTES + HALF);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) r.s[kb][i] = 0.0f;
#pragma unroll
        for (int m = 0; m < NM; ++m)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                r.s[kb] = mfma<E>(k[kb * NM + m], r.q[0][m], r.s[kb]);
                if constexpr (NP == 2) {
                    r.s[kb] = mfma<E>(k[kb * NM + m], r.q[1][m], r.s[kb]);
                    r.s[kb] = mfma<E>(k[PLANE + kb * NM + m], r.q[0][m], r.s[kb]);
                }
            }
        load(k, data + (int64_t)min(kt + 4, kt1) * BYTES);
        if (kt - words_at >= 64) {
            words_at += 64;
            words = a.info[tile0 + min(words_at + lane, kt1)];
        }
        const TileInfo info{__builtin_amdgcn_readlane(words, kt - words_at)};
        weights(a, kt, info, r);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < ND; ++t) {
                r.o[t] = mfma<E>(v[t * U + u], r.p[0][u], r.o[t]);
                if constexpr (NP == 2) {
                    r.o[t] = mfma<E>(v[t * U + u], r.p[1][u], r.o[t]);
                    r.o[t] = mfma<E>(v[PLANE + t * U + u], r.p[0][u], r.o[t]);
                }
            }
        if (info.odd()) strange_values(a, p, head, kt, r);
    }

    // the waves' parts, to one maximum
    const float l = halves_sum(r.l);
    lds_m[wave][lane] = r.m;
    lds_l[wave][lane] = l;
    __syncthreads();
    float m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, lds_m[w][lane]);
    // (a maximum of -inf: no key, or NaN, which the sum keeps)
    auto by = [&](float of) { return of > -INFINITY ? __builtin_amdgcn_exp2f(of - m) : 1.0f; };
#pragma unroll
    for (int w = 0; w < 4; ++w) sum += lds_l[w][lane] * by(lds_m[w][lane]);
    float f = l != 0.0f ? by(r.m) : 0.0f;
    if constexpr (NP == 2) f = l != 0.0f ? ldexpf(f, r.ev_ref - kTopExp - kPExp) : 0.0f;
    const float g = sum != 0.0f ? 1.0f / sum : 0.0f;
    T *out = (T *)a.out + (p.start + r.token) * a.out_stride + (head * group + hq) * D + 4 * (lane >> 5);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4 * OWN; ++i) parts[wave][i][lane] = r.o[h * ND / 2 + i / 16][i % 16] * f;
        __syncthreads();
        if (row < rows)
#pragma unroll
            for (int b = 0; b < OWN / 4; ++b) {
                const int at = wave * OWN + 4 * b, t = h * ND / 2 + at / 16;
                T y[4] __attribute__((aligned(16)));
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    y[i] = (T)((parts[0][at + i][lane] + parts[1][at + i][lane] + parts[2][at + i][lane] + parts[3][at + i][lane]) * g);
                T *to = out + 32 * t + 8 * (at % 16 / 4);
                if constexpr (sizeof(T) == 4)
                    *(float4 *)to = *(const float4 *)y;
                else
                    *(uint2 *)to = *(const uint2 *)y;
            }
    }
}

template <typename T, int D> hipError_t prompt_launch(const PromptArgs &a, hipStream_t st) {
    k_prompt_pack<T, D><<<dim3((unsigned)a.n_tiles, (unsigned)a.n_kv_heads), 256, 0, st>>>(a);
    const unsigned groups = (unsigned)(a.n_slots * a.n_kv_heads);
    a.rows == kPromptRows ? k_prompt_attn<T, D><<<groups, kPromptThreads, 0, st>>>(a) : k_prompt_attn_few<T, D><<<groups, 256, 0, st>>>(a);
    return hipGetLastError();
}

template <typename T> hipError_t prompt_dim(int head_dim, const PromptArgs &a, hipStream_t st) {
    return head_dim == 64 ? prompt_launch<T, 64>(a, st) : prompt_launch<T, 128>(a, st);
}

}  // namespace

hipError_t launch_prompt_attn(int dtype, int head_dim, const PromptArgs &a, hipStream_t st) {
    if (dtype == VKV_DTYPE_F16) return prompt_dim<_Float16>(head_dim, a, st);
    if (dtype == VKV_DTYPE_BF16) return prompt_dim<__bf16>(head_dim, a, st);
    return prompt_dim<float>(head_dim, a, st);
}

}  // namespace vkv
