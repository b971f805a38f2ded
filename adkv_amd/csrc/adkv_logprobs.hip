// Log probabilities of given tokens from rows of logits, the rows' entropy and their likeliest tokens, in one pass over the logits.
//
//   M = max x, d_i = x_i - M, S = sum e^(d_i) over all but one of the largest, T = sum e^(d_i) d_i over the same
//   log p_token = d_token - log(1 + S),   entropy = log(1 + S) - T / (1 + S)
// The largest is left out of the sums, so that log(1 + S) keeps its digits where one token is nearly certain, and T is a sum of numbers of one sign.
// A lane holds back the largest it has seen, adds the smaller of it and the next one, and sums relative to a reference r of its own, the largest of its
// first logits (replaced where a logit is more than FAR larger); the difference is taken before anything else, so that logits of any size keep theirs.
// Logits beyond +-MOST count as that beside others.  The last steps, once a row, are in 64 bits.  NaN and infinities are looked for beside it: v_max drops a NaN.
//
// The likeliest: a key is the logit's bits in the order of numbers with the index, backwards, behind them, so that all keys differ and equal logits
// come lowest index first.  The lanes' maxima of the first step, 64 groups of them, give a bound that at least `top` keys reach; what reaches it goes to a
// list in the LDS, some 1.2 to 1.7 times `top` per step, and a list of more than REFINE keys raises the bound the same way.  At the end each key of
// the list counts the larger ones.  Rows whose keys overrun the list (ascending logits) or that have a NaN are searched a key at a time instead.
//
// A workgroup per row.  Bound by memory where rows are many; see the launcher for the size of the workgroups.
#include <math.h>

#include <algorithm>

#include "adkv_device.h"

#include "../../include/adkv_hip.h"

#pragma clang fp contract(off)

namespace adkv_logprobs {
using adkv::check_launch;
using adkv::cu_count;

typedef uint32_t u4v __attribute__((ext_vector_type(4)));
#define GLOBAL __attribute__((address_space(1)))

constexpr int F32 = ADKV_DT_F32, F16 = ADKV_DT_F16, BF16 = ADKV_DT_BF16;
constexpr int STEP = 4;                 // vectors of 16 bytes of a lane's step
constexpr int CAP = 1024, REFINE = 256; // keys of a list; above which it is looked through
constexpr int TOP = 32;
constexpr float L2E = 1.44269504088896340736f;
constexpr float MOST = 1.7e38f;         // stands for everything above it, -MOST for everything below: differences are finite
constexpr float NONE = -3.0e38f;        // a reference before there is one
constexpr float FAR = 40.0f;

struct Args {
    const char *x;
    long s0, s1; // bytes
    const int64_t *tokens;
    int n1, V, top;
    float *logprobs, *entropy, *top_logprobs;
    int64_t *top_tokens;
};

struct Sums {
    float big, s, t, r; // the largest so far, which is not in the sums; sum e^d, sum e^d d, d = x - r
};

__device__ __forceinline__ float within(float x) { return __builtin_amdgcn_fmed3f(x, -MOST, MOST); }

__device__ __forceinline__ void add(Sums &a, float x)
{
    const float d = fminf(x, a.big) - a.r, e = __builtin_amdgcn_exp2f(d * L2E);
    a.big = fmaxf(a.big, x);
    a.s += e;
    a.t = __builtin_fmaf(e, d, a.t);
}

__device__ __forceinline__ void refer(Sums &a, float r)
{
    const float shift = a.r - r, e = __builtin_amdgcn_exp2f(shift * L2E);
    a.t = e == 0.0f ? 0.0f : e * __builtin_fmaf(shift, a.s, a.t); // the difference of a lowest value may be infinite
    a.s *= e;
    a.r = r;
}

__device__ __forceinline__ void merge(Sums &a, Sums b)
{
    const float r = fmaxf(a.r, b.r);
    refer(a, r);
    refer(b, r);
    a.s += b.s;
    a.t += b.t;
    const float smaller = fminf(a.big, b.big);
    a.big = fmaxf(a.big, b.big);
    if (smaller == -INFINITY) // one of them has seen nothing
        return;
    const float d = smaller - r, e = __builtin_amdgcn_exp2f(d * L2E);
    a.s += e;
    a.t = __builtin_fmaf(e, d, a.t);
}

__device__ __forceinline__ uint64_t key(float x, int i)
{
    const uint32_t u = __float_as_uint(x + 0.0f); // no negative zero
    const uint32_t order = x != x ? 0xFFFFFFFFu : (int)u < 0 ? ~u : u | 0x80000000u;
    return (uint64_t)order << 32 | (0xFFFFFFFFu - (uint32_t)i);
}
__device__ __forceinline__ float number(uint64_t k)
{
    const uint32_t o = (uint32_t)(k >> 32);
    return o == 0xFFFFFFFFu ? NAN : __uint_as_float((int)o < 0 ? o & 0x7FFFFFFFu : ~o);
}

template <int TYPE> struct Piece {
    static constexpr int SIZE = TYPE == F32 ? 4 : 2, N = 16 / SIZE;
    static __device__ __forceinline__ float one(const char *row, int i)
    {
        if constexpr (TYPE == F32)
            return *(const GLOBAL float *)(row + (long)i * 4);
        else if constexpr (TYPE == BF16)
            return __uint_as_float((uint32_t)*(const GLOBAL uint16_t *)(row + (long)i * 2) << 16);
        else
            return (float)*(const GLOBAL _Float16 *)(row + (long)i * 2);
    }
    static __device__ __forceinline__ void open(u4v w, float *x)
    {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (TYPE == F32) {
                x[i] = __uint_as_float(w[i]);
            } else if constexpr (TYPE == BF16) {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            } else {
                typedef _Float16 h2v __attribute__((ext_vector_type(2)));
                const uint32_t u = w[i]; // a bit cast of an element of a vector is one of its first
                const h2v h = __builtin_bit_cast(h2v, u);
                x[2 * i] = (float)h.x;
                x[2 * i + 1] = (float)h.y;
            }
        }
    }
    static constexpr uint32_t LOW = TYPE == F32 ? 0xFF800000u : TYPE == BF16 ? 0xFF80FF80u : 0xFC00FC00u; // minus infinities
};

struct List {
    uint64_t keys[2][CAP];
    uint64_t groups[64];
    uint64_t bound;
    int n[2], overrun;
};

// The top-th largest of the groups' largest keys: at least `top` keys reach it.  0 where fewer groups have any.  A wave's work.
__device__ __forceinline__ uint64_t bound_of(uint64_t mine, int top)
{
    int larger = 0;
    for (int i = 0; i < 64; i++) {
        const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)mine, i);
        larger += other > mine;
    }
    const uint64_t is = __ballot(larger == top - 1 && mine != 0);
    if (is == 0)
        return 0;
    const int at = __builtin_ctzll(is);
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), at) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)mine, at);
}

// Leaves those of the list `from` in the other one that reach a bound found from its groups; all threads of the workgroup
template <int NT>
__device__ void refine(List &l, int from, int top)
{
    const int n = min(l.n[from], CAP);
    if (threadIdx.x < 64)
        l.groups[threadIdx.x] = 0;
    if (threadIdx.x == 0)
        l.n[from ^ 1] = 0;
    __syncthreads();
    uint64_t most = 0;
    for (int i = threadIdx.x; i < n; i += NT)
        most = std::max(most, l.keys[from][i]);
    if (most)
        atomicMax((unsigned long long *)&l.groups[threadIdx.x & 63], (unsigned long long)most);
    __syncthreads();
    if (threadIdx.x < 64) {
        const uint64_t b = bound_of(l.groups[threadIdx.x], top);
        if (threadIdx.x == 0)
            l.bound = b;
    }
    __syncthreads();
    const uint64_t bound = l.bound;
    for (int i = threadIdx.x; i < n; i += NT)
        if (l.keys[from][i] >= bound)
            l.keys[from ^ 1][atomicAdd(&l.n[from ^ 1], 1)] = l.keys[from][i];
    __syncthreads();
}

template <int TYPE, int NT, bool WITH_TOP>
__global__ __launch_bounds__(NT) void logprobs_kernel(const Args a)
{
    using P = Piece<TYPE>;
    __shared__ List list[1];
    __shared__ Sums left[NT / 64];
    __shared__ int strange;
    __shared__ double result[2]; // M, log(1 + S)
    __shared__ uint64_t best;
    const int tid = threadIdx.x, lane = tid & 63;
    const long r = blockIdx.x;
    const char *row = a.x + r / a.n1 * a.s0 + r % a.n1 * a.s1;
    if (tid == 0)
        strange = 0;
    if constexpr (WITH_TOP)
        if (tid == 0) {
            list->n[0] = list->n[1] = 0;
            list->overrun = 0;
        }
    // whole vectors between the first and the last aligned one; single logits in front of and behind them
    const int head = std::min(a.V, (int)((16 - ((uintptr_t)row & 15)) & 15) / P::SIZE), vectors = (a.V - head) / P::N, tail = a.V - head - vectors * P::N;
    const char *body = row + (long)head * P::SIZE;
    const int lone = tid < head ? tid : tid >= NT - tail ? a.V - (NT - tid) : -1; // NT > 14
    const float single = lone >= 0 ? P::one(row, lone) : -INFINITY;
    u4v now[STEP], next[STEP];
    const auto load = [&](int v0, u4v *to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < STEP; i++) {
            const int v = v0 + i * NT + tid;
            to[i] = (u4v){P::LOW, P::LOW, P::LOW, P::LOW};
            if (v < vectors)
                to[i] = *(const GLOBAL u4v *)(body + (long)v * 16);
        }
    };
    load(0, now);
    Sums sums = {-INFINITY, 0.0f, 0.0f, NONE};
    bool first = true, nan = single != single;
    uint64_t bound = 0;
    float bound_value = -INFINITY;
    int from = 0;
    const auto take = [&](float x, int i) __attribute__((always_inline)) {
        if constexpr (WITH_TOP) {
            const uint64_t k = key(x, i);
            if (k >= bound) {
                const int at = atomicAdd(&list->n[from], 1);
                if (at < CAP)
                    list->keys[from][at] = k;
                else
                    list->overrun = 1;
            }
        }
    };
    for (int v0 = 0; first || v0 < vectors; v0 += STEP * NT) {
        load(v0 + STEP * NT, next);
        float x[STEP][P::N], most[STEP];
#pragma unroll
        for (int i = 0; i < STEP; i++) {
            P::open(now[i], x[i]);
            most[i] = x[i][0];
#pragma unroll
            for (int e = 1; e < P::N; e++)
                most[i] = fmaxf(most[i], x[i][e]);
        }
        if (WITH_TOP && first) {
            // the lane's largest key
            uint64_t mine = lone >= 0 ? key(single, lone) : 0;
#pragma unroll
            for (int i = 0; i < STEP; i++)
#pragma unroll
                for (int e = 0; e < P::N; e++) {
                    const int v = v0 + i * NT + tid;
                    if (v < vectors)
                        mine = std::max(mine, key(x[i][e], head + v * P::N + e));
                }
            if (tid < 64)
                list->groups[tid] = 0;
            __syncthreads();
            if (mine)
                atomicMax((unsigned long long *)&list->groups[lane], (unsigned long long)mine);
            __syncthreads();
            bound = bound_of(list->groups[lane], a.top);
            bound_value = bound ? number(bound) : -INFINITY;
            if (lone >= 0)
                take(single, lone);
        }
        if constexpr (WITH_TOP) {
#pragma unroll
            for (int i = 0; i < STEP; i++)
                if (__any(most[i] >= bound_value)) {
#pragma unroll
                    for (int e = 0; e < P::N; e++) {
                        const int v = v0 + i * NT + tid;
                        if (x[i][e] >= bound_value && v < vectors)
                            take(x[i][e], head + v * P::N + e);
                    }
                }
        }
        if (first) {
            if (lone >= 0) {
                sums.big = sums.r = within(single);
            }
            first = false;
        }
#pragma unroll
        for (int i = 0; i < STEP; i++) {
            const float top = within(most[i]);
            if (__any(top > sums.r + FAR)) {
                if (top > sums.r + FAR)
                    refer(sums, top);
            }
            const int v = v0 + i * NT + tid;
            if (v < vectors) {
#pragma unroll
                for (int e = 0; e < P::N; e++) {
                    nan |= x[i][e] != x[i][e];
                    const float y = within(x[i][e]);
                    if (e == 0 && sums.big == -INFINITY)
                        sums.big = y; // the lane's first
                    else
                        add(sums, y);
                }
            }
        }
        if constexpr (WITH_TOP) {
            __syncthreads();
            if (list->n[from] > REFINE) {
                refine<NT>(*list, from, a.top);
                from ^= 1;
                bound = std::max(bound, list->bound);
                bound_value = bound ? number(bound) : -INFINITY;
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < STEP; i++)
            now[i] = next[i];
    }
    if (__any(nan) && lane == 0)
        strange = 1;
    for (int d = 32; d; d >>= 1) {
        Sums o;
        o.big = __shfl_xor(sums.big, d);
        o.s = __shfl_xor(sums.s, d);
        o.t = __shfl_xor(sums.t, d);
        o.r = __shfl_xor(sums.r, d);
        merge(sums, o);
    }
    if (lane == 0)
        left[tid / 64] = sums;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < NT / 64; w++)
            merge(sums, left[w]);
        left[0] = sums;
    }
    __syncthreads();
    sums = left[0];
    float M = sums.big;
    if (fabsf(M) >= MOST) {
        // nothing but what may be minus infinity, or plus infinity
        M = -INFINITY;
        for (int i = tid; i < a.V; i += NT)
            M = fmaxf(M, P::one(row, i));
        for (int d = 32; d; d >>= 1)
            M = fmaxf(M, __shfl_xor(M, d));
        __syncthreads();
        if (lane == 0)
            left[tid / 64].big = M;
        __syncthreads();
        for (int w = 0; w < NT / 64; w++)
            M = fmaxf(M, left[w].big);
        if (tid == 0 && fabsf(M) == INFINITY)
            strange |= 2;
    }
    if (tid == 0) {
        const double shift = (double)sums.r - (double)sums.big, scale = exp(shift), S = scale * sums.s, T = scale * ((double)sums.t + shift * sums.s);
        const double log1 = strange ? (double)NAN : log1p(S);
        result[0] = M;
        result[1] = log1;
        const int64_t token = a.tokens[r];
        a.logprobs[r] = token < 0 ? 0.0f : token < a.V ? (float)((double)P::one(row, (int)token) - M - log1) : NAN;
        a.entropy[r] = (float)(log1 - T / (1.0 + S));
    }
    if constexpr (WITH_TOP) {
        __syncthreads();
        const auto put = [&](int rank, uint64_t k) {
            const float x = number(k);
            a.top_tokens[r * a.top + rank] = (int64_t)(0xFFFFFFFFu - (uint32_t)k);
            a.top_logprobs[r * a.top + rank] = (float)((double)x - result[0] - result[1]);
        };
        if (!(strange & 1) && !list->overrun) {
            if (list->n[from] > 2 * TOP) {
                refine<NT>(*list, from, a.top);
                from ^= 1;
            }
            const int n = list->n[from];
            for (int i = tid; i < n; i += NT) {
                const uint64_t k = list->keys[from][i];
                int rank = 0;
                for (int j = 0; j < n; j++)
                    rank += list->keys[from][j] > k;
                if (rank < a.top)
                    put(rank, k);
            }
            return;
        }
        uint64_t last = ~0ull;
        for (int rank = 0; rank < a.top; rank++) {
            if (tid == 0)
                best = 0;
            __syncthreads();
            uint64_t mine = 0;
            for (int i = tid; i < a.V; i += NT) {
                const uint64_t k = key(P::one(row, i), i);
                if ((rank == 0 || k < last) && k > mine)
                    mine = k;
            }
            atomicMax((unsigned long long *)&best, (unsigned long long)mine);
            __syncthreads();
            last = best;
            if (tid == 0)
                put(rank, last);
            __syncthreads();
        }
    }
}

template <int TYPE> static auto kernel_of(int threads, bool top)
{
    if (threads == 256)
        return top ? logprobs_kernel<TYPE, 256, true> : logprobs_kernel<TYPE, 256, false>;
    return top ? logprobs_kernel<TYPE, 1024, true> : logprobs_kernel<TYPE, 1024, false>;
}

} // namespace adkv_logprobs

extern "C" int adkv_token_logprobs(const void *logits, int64_t stride0, int64_t stride1, const int64_t *tokens, int n0, int n1, int V, int dtype,
                                   int top, float *logprobs, float *entropy, float *top_logprobs, int64_t *top_tokens, void *stream)
{
    using namespace adkv_logprobs;
    if (!logits || !tokens || !logprobs || !entropy || (top > 0 && (!top_logprobs || !top_tokens)))
        return ADKV_E_NULL;
    if (n0 <= 0 || n1 <= 0 || V <= 0 || top < 0 || top > TOP || top > V || stride0 < 0 || stride1 < 0 || V > INT32_MAX - 65536)
        return ADKV_E_SHAPE;
    if (dtype != F32 && dtype != F16 && dtype != BF16)
        return ADKV_E_UNSUPPORTED;
    const int64_t rows = (int64_t)n0 * n1;
    if (rows >= 1 << 22) // a grid is 2^32 threads at most
        return ADKV_E_SHAPE;
    const int size = dtype == F32 ? 4 : 2;
    if ((uint64_t)logits & (size - 1))
        return ADKV_E_ALIGN;
    if (((uint64_t)logprobs | (uint64_t)entropy | (uint64_t)top_logprobs) & 3 || ((uint64_t)tokens | (uint64_t)top_tokens) & 7)
        return ADKV_E_ALIGN;
    Args a = {(const char *)logits, (long)stride0 * size, (long)stride1 * size, tokens, n1, V, top, logprobs, entropy, top_logprobs, top_tokens};
    const int threads = rows >= 4ll * cu_count() ? 256 : 1024;
    const auto kernel = dtype == F32 ? kernel_of<F32>(threads, top > 0) : dtype == F16 ? kernel_of<F16>(threads, top > 0) : kernel_of<BF16>(threads, top > 0);
    hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(threads), 0, (hipStream_t)stream, a);
    return check_launch();
}
