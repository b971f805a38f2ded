// Log probabilities of given tokens from rows of logits, the rows' entropy and their likeliest tokens, in one pass over the logits.
//
//   M = max x, d_i = x_i - M, S = sum e^(d_i) over all but one of the largest, T = sum e^(d_i) d_i over the same
//   log p_token = d_token - log(1 + S),   entropy = log(1 + S) - T / (1 + S)
// The largest is left out of the sums, so that log(1 + S) keeps its digits where one token is nearly certain, and T is a sum of numbers of one sign.
// A lane holds back the largest it has seen, adds the smaller of it and the next one, and sums relative to a reference r of its own, the largest of its
// first logits (replaced where a logit is more than 2^FAR larger), all in powers of two: x log2(e) - r is one multiply-add, and r log2(e) - M log2(e) another
// at the end, so that neither r nor log2(e) need be exact.  References are within +-FLOOR, where r is off by 2^-4 at most (one of 10^10 would be off by 2^9, and
// 2^d infinite).  Logits below FLOOR, minus infinity and what else stands for hidden tokens among them, weigh nothing; rows whose
// largest is not within half of +-FLOOR are gone through again.  NaN is looked for beside it: v_med3 and v_max drop it.
//
// The likeliest: a key is the logit's bits in the order of numbers with the index, backwards, behind them, so that all keys differ and equal logits
// come lowest index first.  The lanes' maxima of the first step, 64 groups of them, give a bound that at least `top` keys reach; what reaches it goes to a
// list in the LDS, some 1.2 to 1.7 times `top` per step, and after one, two, four.. steps a list of more than REFINE keys raises the bound the same way.  At
// the end each key of the list counts the larger ones.  Rows whose keys overrun the list (ascending logits) or that have a NaN are searched a key at a time instead.
//
// A workgroup per row; the launcher says how large.  MI355X: 4096 rows of 32000 bf16 logits 55 us, 4.7 TB/s, 1000 rows of 128001 fp32 ones 94, 5.4 TB/s: memory (a
// copy runs at 5.15, reads alone faster).  Alternatives cost the bound in front and the ranks behind, some 4 us of few rows and more of many that are in step: four rows
// of 32000 10.6 us where they are 6.2 without; 1000 rows of 128001 fp16 ones with 20 of them, all resident at once, 69 where they are 50.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "adkv_device.h"

#include "../../include/adkv_hip.h"

#pragma clang fp contract(off)

namespace adkv_logprobs {
using adkv::check_launch;
using adkv::cu_count;

typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
#define GLOBAL __attribute__((address_space(1)))

constexpr int F32 = ADKV_DT_F32, F16 = ADKV_DT_F16, BF16 = ADKV_DT_BF16;
constexpr int CAP = 1024, REFINE = 128; // keys of a list; above which it is looked through
constexpr int TOP = 32;
constexpr float L2E = 1.44269504088896340736f;
constexpr float FLOOR = -0x1p20f; // times log2(e) it is exact, and its difference from itself zero
constexpr float FAR = 60.0f;

struct Args {
    const char *x;
    long s0, s1; // bytes
    const int64_t *tokens;
    int n1, V, top;
    float *logprobs, *entropy, *top_logprobs;
    int64_t *top_tokens;
};

struct Sums {
    float big, s, t, r; // the largest so far, which is not in the sums; sum 2^d, sum 2^d d, d = x log2(e) - r
};

__device__ __forceinline__ void add(Sums &a, float x)
{
    const float d = __builtin_fmaf(__builtin_amdgcn_fmed3f(x, FLOOR, a.big), L2E, -a.r), e = __builtin_amdgcn_exp2f(d);
    a.big = fmaxf(a.big, x);
    a.s += e;
    a.t = __builtin_fmaf(e, d, a.t);
}

__device__ __forceinline__ void refer(Sums &a, float r)
{
    // in two steps: what is up to 2^FAR above its reference is not lost before it is 2^-126 of the new one
    const float shift = a.r - r, e = __builtin_amdgcn_exp2f(0.5f * shift);
    a.t = __builtin_fmaf(shift, a.s, a.t) * e * e;
    a.s = a.s * e * e;
    a.r = r;
}

// Over a wave, in all of its lanes: within four lanes, eight, sixteen, then between rows of sixteen
template <typename F>
__device__ __forceinline__ uint32_t fold(uint32_t v, F f)
{
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));  // lane ^ 1
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));  // lane ^ 2
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false)); // 7 - lane of eight
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false)); // 15 - lane of sixteen
#pragma unroll
    for (int i = 0; i < 2; i++) {
        unsigned x = v, y = v;
        asm volatile("" : "+v"(y)); // two copies: the compiler folds a swap of a register with itself
        const u2v r = i ? __builtin_amdgcn_permlane32_swap(x, y, false, false) : __builtin_amdgcn_permlane16_swap(x, y, false, false);
        x = r.x;
        y = r.y;
        asm volatile("" : "+v"(x), "+v"(y));
        v = f(x, y);
    }
    return v;
}
__device__ __forceinline__ float largest(float v)
{
    return __uint_as_float(fold(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
__device__ __forceinline__ float sum(float v)
{
    return __uint_as_float(fold(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
__device__ __forceinline__ uint32_t smallest(uint32_t v)
{
    return fold(v, [](uint32_t a, uint32_t b) { return std::min(a, b); });
}

// The sums of all lanes, in all of them; one that has seen nothing has FLOOR for its largest
__device__ __forceinline__ void together(Sums &a, int lane)
{
    refer(a, largest(a.r));
    const float big = largest(a.big);
    const uint64_t holders = __ballot(a.big == big);
    if (lane != __builtin_ctzll(holders)) { // what others held back is not the largest, or not the one of them that is left out
        const float d = __builtin_fmaf(a.big, L2E, -a.r), e = __builtin_amdgcn_exp2f(d);
        a.s += e;
        a.t = __builtin_fmaf(e, d, a.t);
    }
    a.big = big;
    a.s = sum(a.s);
    a.t = sum(a.t);
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
    uint64_t keys[CAP];
    uint64_t raised;
    int n, overrun;
};

__device__ __forceinline__ uint64_t of_lane(uint64_t k, int i)
{
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)k, i);
}

// A bound that at least `top` of all keys reach, from the largest keys of 2 * top or more groups of lanes (0: none): the least of those that hold the
// top-th largest value of them.  0 where fewer groups have any.
__device__ __forceinline__ uint64_t bound_of(uint64_t mine, int top)
{
    // 16 groups of four lanes for up to 8, 32 of two for up to 16: what reaches the bound is 1.1 to 1.4 times `top` then
    for (int d = 32; d >= 16 && top * 4 <= 2 * d; d /= 2) {
        const uint64_t other = (uint64_t)(uint32_t)__shfl_xor((int)(mine >> 32), d) << 32 | (uint32_t)__shfl_xor((int)mine, d);
        mine = std::max(mine, other);
    }
    const int groups = top <= 8 ? 16 : top <= 16 ? 32 : 64;
    const uint32_t value = (uint32_t)(mine >> 32);
    int larger = 0;
    for (int i = 0; i < groups; i += 16)
#pragma unroll
        for (int j = 0; j < 16; j++)
            larger += (uint32_t)__builtin_amdgcn_readlane((int)value, i + j) > value;
    const bool among = larger < top && mine != 0;
    if (__popcll(__ballot(among)) * groups < top * 64)
        return 0;
    const uint32_t least = smallest(among ? value : ~0u);
    return (uint64_t)least << 32 | smallest(among && value == least ? (uint32_t)mine : ~0u);
}

// A wave's work: of the list's n keys those that reach a bound found from them stay
__device__ __forceinline__ uint64_t refine(List &l, int &n, int top, int lane)
{
    uint64_t most = 0;
    for (int i = lane; i < n; i += 64)
        most = std::max(most, l.keys[i]);
    const uint64_t bound = bound_of(most, top);
    int kept = 0;
    for (int i = lane; __any(i < n); i += 64) {
        const uint64_t k = i < n ? l.keys[i] : 0;
        const uint64_t stay = __ballot(i < n && k >= bound);
        if (i < n && k >= bound)
            l.keys[kept + __popcll(stay & ((1ull << lane) - 1))] = k;
        kept += __popcll(stay);
    }
    n = kept;
    return bound;
}

template <int TYPE, int NT, bool WITH_TOP>
__global__ __launch_bounds__(NT, WITH_TOP ? 6 : 8) void logprobs_kernel(const Args a)
{
    using P = Piece<TYPE>;
    constexpr int NW = NT / 64;
    constexpr int STEP = WITH_TOP && NT == 256 ? 4 : 2; // vectors of 16 bytes of a lane's step
    __shared__ List list[1];
    __shared__ uint64_t first[NT];
    __shared__ Sums left[NW];
    __shared__ bool strange[NW];
    __shared__ uint64_t best;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid / 64;
    const long r = blockIdx.x;
    const char *row = a.x + r / a.n1 * a.s0 + r % a.n1 * a.s1;
    // whole vectors between the first and the last aligned one; single logits in front of and behind them
    const int head = std::min(a.V, (int)((16 - ((uintptr_t)row & 15)) & 15) / P::SIZE), vectors = (a.V - head) / P::N, tail = a.V - head - vectors * P::N;
    const char *body = row + (long)head * P::SIZE;
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
    const int lone = tid < head ? tid : tid >= NT - tail ? a.V - (NT - tid) : -1; // NT > 14
    const float single = lone >= 0 ? P::one(row, lone) : -INFINITY;
    const int64_t token = a.tokens[r];
    const float given = token >= 0 && token < a.V ? P::one(row, (int)token) : NAN;
    Sums sums = {fmaxf(single, FLOOR), 0.0f, 0.0f, fminf(fmaxf(single, FLOOR), -FLOOR) * L2E};
    bool nan = single != single;
    uint64_t bound = 0;
    float bound_value = -INFINITY;
    const auto take = [&](float x, int i) __attribute__((always_inline)) {
        const uint64_t k = key(x, i);
        if (k >= bound) {
            const int at = atomicAdd(&list->n, 1);
            if (at < CAP)
                list->keys[at] = k;
            else
                list->overrun = 1;
        }
    };
    if constexpr (WITH_TOP) {
        if (tid == 0)
            list->n = list->overrun = 0;
        // the lane's largest logit of the first step, the first of equal ones
        float most = -INFINITY;
        int at = -1;
#pragma unroll
        for (int i = 0; i < STEP; i++) {
            float x[P::N];
            P::open(now[i], x);
            const int v = i * NT + tid;
#pragma unroll
            for (int e = 0; e < P::N; e++)
                if (v < vectors && (at < 0 || x[e] > most)) {
                    most = x[e];
                    at = v * P::N + e;
                }
        }
        const uint64_t mine = at >= 0 ? key(most, head + at) : 0;
        first[tid] = lone >= 0 ? std::max(mine, key(single, lone)) : mine;
        __syncthreads();
        uint64_t group = 0;
#pragma unroll
        for (int w = 0; w < NW; w++)
            group = std::max(group, first[w * 64 + lane]);
        bound = bound_of(group, a.top);
        bound_value = bound ? number(bound) : -INFINITY;
        if (lone >= 0)
            take(single, lone);
    }
    int step = 0;
    for (int v0 = 0; v0 < vectors; v0 += STEP * NT) {
        load(v0 + STEP * NT, next);
#pragma unroll
        for (int i = 0; i < STEP; i++) {
            float x[P::N];
            P::open(now[i], x);
            const int v = v0 + i * NT + tid;
            float most = x[0];
#pragma unroll
            for (int e = 1; e < P::N; e++)
                most = fmaxf(most, x[e]);
            if (WITH_TOP && __any(most >= bound_value)) {
#pragma unroll
                for (int e = 0; e < P::N; e++)
                    if (x[e] >= bound_value && v < vectors)
                        take(x[e], head + v * P::N + e);
            }
            if (__any(most * L2E > sums.r + FAR)) {
                if (most * L2E > sums.r + FAR)
                    refer(sums, fminf(most, -FLOOR) * L2E);
            }
            // what is behind the row is minus infinity, and weighs nothing
#pragma unroll
            for (int e = 0; e < P::N; e++) {
                nan |= x[e] != x[e];
                add(sums, x[e]);
            }
        }
        step++;
        if constexpr (WITH_TOP) {
            // seldom: after four, eight, sixteen.. steps
            if (step >= 4 && (step & (step - 1)) == 0 && v0 + STEP * NT < vectors) {
                __syncthreads();
                if (wave == 0) {
                    int n = std::min(list->n, CAP);
                    const uint64_t raised = n > REFINE ? refine(*list, n, a.top, lane) : 0;
                    if (lane == 0) {
                        list->n = n;
                        list->raised = raised;
                    }
                }
                __syncthreads();
                bound = std::max(bound, list->raised);
                bound_value = bound ? number(bound) : -INFINITY;
            }
        }
#pragma unroll
        for (int i = 0; i < STEP; i++)
            now[i] = next[i];
    }
    nan = __any(nan);
    together(sums, lane);
    if (lane == 0) {
        strange[wave] = nan;
        left[wave] = sums;
    }
    __syncthreads();
    const bool odd = __any(lane < NW && strange[lane % NW]), slow = WITH_TOP && (odd || list->overrun);
    sums = lane < NW ? left[lane] : (Sums){FLOOR, 0.0f, 0.0f, FLOOR * L2E};
    together(sums, lane);
    float M = sums.big;
    const bool again = !(fabsf(M) < -0.5f * FLOOR); // else e^FLOOR is nothing beside e^M
    if (wave != 0 && !slow && !again)
        return; // the rest is the first wave's
    const float shift = __builtin_fmaf(-M, L2E, sums.r), scale = __builtin_amdgcn_exp2f(shift);
    // T is the small difference of two large ones where the reference is not the largest
    float S = scale * sums.s, T = (float)(0.69314718055994530942 * ((double)scale * ((double)shift * sums.s + sums.t)));
    if (again) {
        // logits beyond half a million, of the type's lowest value only, or of minus or plus infinity: the definition, in two passes more
        M = -INFINITY;
        for (int i = tid; i < a.V; i += NT)
            M = fmaxf(M, P::one(row, i));
        M = largest(M);
        __syncthreads();
        if (lane == 0)
            left[wave].big = M;
        __syncthreads();
        M = largest(left[lane % NW].big);
        S = T = 0.0f;
        float equal = 0.0f; // of the largest, one of which is left out
        for (int i = tid; i < a.V; i += NT) {
            const double d = (double)P::one(row, i) - M;
            const float e = d > -200.0 ? expf((float)d) : 0.0f;
            if (d == 0.0) {
                equal += 1.0f;
            } else if (e > 0.0f) {
                S += e;
                T += e * (float)d;
            }
        }
        S = sum(S);
        T = sum(T);
        equal = sum(equal);
        if (lane == 0)
            left[wave].s = S, left[wave].t = T, left[wave].r = equal;
        __syncthreads();
        S = sum(lane < NW ? left[lane].s : 0.0f) + (sum(lane < NW ? left[lane].r : 0.0f) - 1.0f);
        T = sum(lane < NW ? left[lane].t : 0.0f);
    }
    const float log1 = odd || fabsf(M) == INFINITY ? NAN : log1pf(S);
    const auto log_of = [&](float x) { return (float)((double)x - M - log1); };
    if (tid == 0) {
        a.logprobs[r] = token < 0 ? 0.0f : token < a.V ? log_of(given) : NAN;
        a.entropy[r] = (float)((double)log1 - (double)T / (1.0 + (double)S));
    }
    if constexpr (WITH_TOP) {
        const auto put = [&](int rank, uint64_t k) {
            a.top_tokens[r * a.top + rank] = (int64_t)(0xFFFFFFFFu - (uint32_t)k);
            a.top_logprobs[r * a.top + rank] = log_of(number(k));
        };
        if (!slow) {
            if (wave != 0)
                return;
            int n = list->n;
            if (n > 64)
                refine(*list, n, a.top, lane);
            for (int i = lane; i < n; i += 64) {
                const uint64_t k = list->keys[i];
                int rank = 0;
#pragma unroll 8
                for (int j = 0; j < n; j++)
                    rank += list->keys[j] > k;
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
    if (threads == 512)
        return top ? logprobs_kernel<TYPE, 512, true> : logprobs_kernel<TYPE, 512, false>;
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
    // The smallest workgroups that fill the device: few rows are over sooner with more lanes, many have less to put together with fewer.  us with 256, 512
    // and 1024 lanes: 4 rows of 32 000 logits with 8 alternatives 16.3, 10.5, 10.3; 512 of 128 000 48.4, 37.8, 34.8; 1000 of 128 000 with 20 72, 67, 74;
    // 4096 of 32 000 with 5 61, 66, 93
    const int64_t cus = cu_count();
    const int threads = rows > 6 * cus ? 256 : rows > 2 * cus ? 512 : 1024;
    const auto kernel = dtype == F32 ? kernel_of<F32>(threads, top > 0) : dtype == F16 ? kernel_of<F16>(threads, top > 0) : kernel_of<BF16>(threads, top > 0);
    hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(threads), 0, (hipStream_t)stream, a);
    return check_launch();
}
