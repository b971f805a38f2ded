// RMS norm of every head's queries and keys with its weight, and the rotary position embedding, in one pass over them; and the way back.
//   n = x * r, r = 1 / sqrt(mean(x^2) + eps)      a row x is one (sequence, token, head) vector of D values
//   y = n * w
//   z = y with the pairs (a, b) = (y[i], y[i + R/2]) of its first R values turned: a * cos[i] - b * sin[i], b * cos[i + R/2] + a * sin[i + R/2]
// and, from dz:
//   dy = dz with the pairs turned back: da * cos[i] + db * sin[i + R/2], db * cos[i + R/2] - da * sin[i]
//   dw = sum over the rows of dy * n
//   dx = r * (dy * w - n * mean(dy * w * n))
// Everything between the loads and the store is fp32; each result is rounded to the activations' type once.  n is computed again on the way back, from
// x, which is read for dw and dx anyway: nothing of the way there is kept.
//
// Memory bound: an element is read and written once on the way there, read twice and written once on the way back, some 30 operations each.  A
// row is D / 2 pairs, a lane takes V neighbouring pairs, all turned or none (eight of 16 bits, 16 bytes of either half, were slower: 53 us
// instead of 49 for the first size below); the row's 2^log lanes sum by
// exchanges.  A lane takes its pairs of HEADS heads of a token: cos, sin and the weights are loaded once for them, and all loads are in flight together.
// Four sequences of 2048 tokens, 32 + 32 heads of 128 values in fp16: 268 MB in 46 us (5.8 TB/s; a copy of 1 GiB reaches 5.1).  Two of 4096 tokens,
// 32 + 8 heads in bf16: 168 MB in 29 us there and 251 MB in 48 to 50 us back (5.8 and 5.0 to 5.2 TB/s), and 4 us for the workgroups' sums of dw.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "adkv_device.h"

#include "../../include/adkv_hip.h"

namespace adkv_rope_norm {
using adkv::check_launch;
using adkv::cu_count;
using adkv::h1;

constexpr int F32 = ADKV_DT_F32, F16 = ADKV_DT_F16, BF16 = ADKV_DT_BF16;
constexpr int NT = 256;
constexpr int V = 4; // pairs of a lane
constexpr int DIM_MAX = 512; // a row is one wave's at most
constexpr int COLUMNS = 32; // of the sums of dw

struct Strides {
    long b, h, t; // in elements; channels are contiguous
};
struct Side { // q or k
    const void *x, *w, *dz;
    void *out; // z there, dx on the way back
    Strides xs, dzs, os;
    int heads;
    int groups;  // of HEADS heads
    int first;   // workgroup
    int workers; // workgroups; none: the side is left out
};
struct Args {
    Side q, k;
    const void *cos, *sin;
    long cs_b, cs_t;
    int tokens, T, half, turned; // tokens of all sequences; D / 2; R / 2
    int lanes, log;              // of a row that have pairs; 2^log lanes are a row's
    int blocks;                  // of tokens that a workgroup takes at once
    float eps, inv_d;
    float *dw;                   // a row of D sums per workgroup
};

template <int TYPE>
struct Piece {
    static constexpr int WORDS = V * (TYPE == F32 ? 4 : 2) / 4, SIZE = TYPE == F32 ? 4 : 2;
    typedef uint32_t Raw __attribute__((ext_vector_type(WORDS)));
    static __device__ __forceinline__ Raw load(const void *p, long at)
    {
        return *(const __attribute__((address_space(1))) Raw *)((const char *)p + at * SIZE);
    }
    static __device__ __forceinline__ void store(void *p, long at, const float *f)
    {
        Raw r;
        if constexpr (TYPE == F32) {
#pragma unroll
            for (int i = 0; i < V; i++)
                r[i] = __float_as_uint(f[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; i++) {
                uint32_t w;
                if constexpr (TYPE == BF16)
                    asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(w) : "v"(f[2 * i]), "v"(f[2 * i + 1])); // to nearest even
                else
                    w = adkv::as_u32((adkv::h2){(h1)f[2 * i], (h1)f[2 * i + 1]});
                r[i] = w;
            }
        }
        *(__attribute__((address_space(1))) Raw *)((char *)p + at * SIZE) = r;
    }
    static __device__ __forceinline__ void widen(const Raw &r, float *f)
    {
#pragma unroll
        for (int i = 0; i < V; i++) {
            if constexpr (TYPE == F32)
                f[i] = __uint_as_float(r[i]);
            else if constexpr (TYPE == BF16)
                f[i] = __uint_as_float(i % 2 ? r[i / 2] & 0xFFFF0000u : r[i / 2] << 16);
            else
                f[i] = (float)adkv::as_h2(r[i / 2])[i % 2];
        }
    }
};

template <int CTRL>
__device__ __forceinline__ float beside(float v)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
// sums over the 2^log lanes of a row, in all of them
template <int N>
__device__ __forceinline__ void sum_row(float *v, int log)
{
    const auto add = [&](auto other) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < N; i++)
            v[i] += other(v[i]);
    };
    if (log > 0)
        add([](float x) { return beside<0xB1>(x); }); // lane ^ 1
    if (log > 1)
        add([](float x) { return beside<0x4E>(x); }); // lane ^ 2
    if (log > 2)
        add([](float x) { return beside<0x141>(x); }); // 7 - lane of eight
    if (log > 3)
        add([](float x) { return beside<0x140>(x); }); // 15 - lane of sixteen
    if (log > 4)
        add([](float x) { return __shfl_xor(x, 16); });
    if (log > 5)
        add([](float x) { return __shfl_xor(x, 32); });
}

// Where a lane works: its first pair, channels lo.. and hi.., and whether they are turned.
struct Lane {
    int row, lo, hi;
    bool there, turned;
    __device__ __forceinline__ explicit Lane(const Args &a)
    {
        const int j = threadIdx.x & ((1 << a.log) - 1), pair = j * V;
        row = threadIdx.x >> a.log;
        there = j < a.lanes;
        turned = there && pair < a.turned;
        lo = turned ? pair : pair + a.turned;
        hi = turned ? pair + a.turned : pair + a.half;
    }
};

__device__ __forceinline__ void turn(float *lo, float *hi, const float *cl, const float *ch, const float *sl, const float *sh)
{
#pragma unroll
    for (int e = 0; e < V; e++) {
        const float x = lo[e], y = hi[e];
        lo[e] = __builtin_fmaf(x, cl[e], -(y * sl[e]));
        hi[e] = __builtin_fmaf(y, ch[e], x * sh[e]);
    }
}
__device__ __forceinline__ void turn_back(float *lo, float *hi, const float *cl, const float *ch, const float *sl, const float *sh)
{
#pragma unroll
    for (int e = 0; e < V; e++) {
        const float x = lo[e], y = hi[e];
        lo[e] = __builtin_fmaf(x, cl[e], y * sh[e]);
        hi[e] = __builtin_fmaf(y, ch[e], -(x * sl[e]));
    }
}

template <int TYPE, int HEADS>
__global__ __launch_bounds__(NT) void forward_kernel(Args a)
{
    using P = Piece<TYPE>;
    using Raw = typename P::Raw;
    const bool is_k = (int)blockIdx.x >= a.k.first;
    const Side s = is_k ? a.k : a.q;
    const int at = (int)blockIdx.x - s.first, group = at / a.blocks, block = at - group * a.blocks;
    const Lane l(a);
    const int token = block * (NT >> a.log) + l.row;
    const bool there = l.there && token < a.tokens, turned = l.turned && token < a.tokens;
    const int b = (uint32_t)token / (uint32_t)a.T, t = token - b * a.T, h0 = group * HEADS;
    Raw lo[HEADS], hi[HEADS], cl = {}, ch = {}, sl = {}, sh = {}, wl = {}, wh = {};
#pragma unroll
    for (int j = 0; j < HEADS; j++)
        lo[j] = hi[j] = Raw{};
    if (there) {
        const long x = b * s.xs.b + t * s.xs.t;
#pragma unroll
        for (int j = 0; j < HEADS; j++) {
            const long row = x + min(h0 + j, s.heads - 1) * s.xs.h;
            lo[j] = P::load(s.x, row + l.lo);
            hi[j] = P::load(s.x, row + l.hi);
        }
        wl = P::load(s.w, l.lo);
        wh = P::load(s.w, l.hi);
    }
    if (turned) {
        const long row = b * a.cs_b + t * a.cs_t;
        cl = P::load(a.cos, row + l.lo);
        ch = P::load(a.cos, row + l.hi);
        sl = P::load(a.sin, row + l.lo);
        sh = P::load(a.sin, row + l.hi);
    }
    float x[HEADS][2 * V], sum[HEADS], w[2 * V], c[2 * V], sn[2 * V];
#pragma unroll
    for (int j = 0; j < HEADS; j++) {
        P::widen(lo[j], x[j]);
        P::widen(hi[j], x[j] + V);
        sum[j] = 0.0f;
#pragma unroll
        for (int e = 0; e < 2 * V; e++)
            sum[j] = __builtin_fmaf(x[j][e], x[j][e], sum[j]);
    }
    sum_row<HEADS>(sum, a.log);
    P::widen(wl, w);
    P::widen(wh, w + V);
    P::widen(cl, c);
    P::widen(ch, c + V);
    P::widen(sl, sn);
    P::widen(sh, sn + V);
    if (!there)
        return;
#pragma unroll
    for (int j = 0; j < HEADS; j++) {
        if (h0 + j >= s.heads)
            break;
        const float r = rsqrtf(__builtin_fmaf(sum[j], a.inv_d, a.eps));
#pragma unroll
        for (int e = 0; e < 2 * V; e++)
            x[j][e] = x[j][e] * r * w[e];
        if (turned)
            turn(x[j], x[j] + V, c, c + V, sn, sn + V);
        const long row = b * s.os.b + (h0 + j) * s.os.h + t * s.os.t;
        P::store(s.out, row + l.lo, x[j]);
        P::store(s.out, row + l.hi, x[j] + V);
    }
}

// Workgroups walk through blocks of tokens and heads with their part of dw in registers: a sum in an order that the launch alone decides.
template <int TYPE, int HEADS>
__global__ __launch_bounds__(NT) void backward_kernel(Args a)
{
    using P = Piece<TYPE>;
    using Raw = typename P::Raw;
    const bool is_k = (int)blockIdx.x >= a.k.first;
    const Side s = is_k ? a.k : a.q;
    const Lane l(a);
    __shared__ float sums[NT / 64][DIM_MAX];
    Raw wl = {}, wh = {};
    if (l.there) {
        wl = P::load(s.w, l.lo);
        wh = P::load(s.w, l.hi);
    }
    float w[2 * V], dw[2 * V];
    P::widen(wl, w);
    P::widen(wh, w + V);
#pragma unroll
    for (int e = 0; e < 2 * V; e++)
        dw[e] = 0.0f;
    const int items = s.groups * a.blocks;
    for (int at = (int)blockIdx.x - s.first; at < items; at += s.workers) {
        const int group = at / a.blocks, block = at - group * a.blocks;
        const int token = block * (NT >> a.log) + l.row;
        const bool there = l.there && token < a.tokens, turned = l.turned && token < a.tokens;
        const int b = (uint32_t)token / (uint32_t)a.T, t = token - b * a.T, h0 = group * HEADS;
        Raw xl[HEADS], xh[HEADS], gl[HEADS], gh[HEADS], cl = {}, ch = {}, sl = {}, sh = {};
#pragma unroll
        for (int j = 0; j < HEADS; j++)
            xl[j] = xh[j] = gl[j] = gh[j] = Raw{};
        if (there) {
            const long xr = b * s.xs.b + t * s.xs.t, gr = b * s.dzs.b + t * s.dzs.t;
#pragma unroll
            for (int j = 0; j < HEADS; j++) {
                if (h0 + j < s.heads) { // behind the last head zeros, which add nothing
                    xl[j] = P::load(s.x, xr + (h0 + j) * s.xs.h + l.lo);
                    xh[j] = P::load(s.x, xr + (h0 + j) * s.xs.h + l.hi);
                    gl[j] = P::load(s.dz, gr + (h0 + j) * s.dzs.h + l.lo);
                    gh[j] = P::load(s.dz, gr + (h0 + j) * s.dzs.h + l.hi);
                }
            }
        }
        if (turned) {
            const long row = b * a.cs_b + t * a.cs_t;
            cl = P::load(a.cos, row + l.lo);
            ch = P::load(a.cos, row + l.hi);
            sl = P::load(a.sin, row + l.lo);
            sh = P::load(a.sin, row + l.hi);
        }
        float c[2 * V], sn[2 * V];
        P::widen(cl, c);
        P::widen(ch, c + V);
        P::widen(sl, sn);
        P::widen(sh, sn + V);
#pragma unroll
        for (int j = 0; j < HEADS; j++) {
            float x[2 * V], g[2 * V], sum[2] = {0.0f, 0.0f};
            P::widen(xl[j], x);
            P::widen(xh[j], x + V);
            P::widen(gl[j], g);
            P::widen(gh[j], g + V);
            if (turned)
                turn_back(g, g + V, c, c + V, sn, sn + V);
#pragma unroll
            for (int e = 0; e < 2 * V; e++) {
                sum[0] = __builtin_fmaf(x[e], x[e], sum[0]);
                sum[1] = __builtin_fmaf(g[e] * w[e], x[e], sum[1]);
            }
            sum_row<2>(sum, a.log);
            if (!there || h0 + j >= s.heads)
                continue;
            const float r = rsqrtf(__builtin_fmaf(sum[0], a.inv_d, a.eps)), mean = sum[1] * r * a.inv_d;
#pragma unroll
            for (int e = 0; e < 2 * V; e++) {
                const float n = x[e] * r;
                dw[e] = __builtin_fmaf(g[e], n, dw[e]);
                x[e] = r * __builtin_fmaf(-n, mean, g[e] * w[e]);
            }
            if (s.out != nullptr) {
                const long row = b * s.os.b + (h0 + j) * s.os.h + t * s.os.t;
                P::store(s.out, row + l.lo, x);
                P::store(s.out, row + l.hi, x + V);
            }
        }
    }
    if (a.dw == nullptr)
        return;
    // the rows of a wave, then the waves
    for (int step = 1 << a.log; step < 64; step <<= 1)
#pragma unroll
        for (int e = 0; e < 2 * V; e++)
            dw[e] += __shfl_xor(dw[e], step);
    const int wave = threadIdx.x >> 6, d = a.half * 2;
    if (l.there && (threadIdx.x & 63) >> a.log == 0) {
#pragma unroll
        for (int e = 0; e < V; e++) {
            sums[wave][l.lo + e] = dw[e];
            sums[wave][l.hi + e] = dw[V + e];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < d; i += NT) {
        float v = sums[0][i];
#pragma unroll
        for (int k = 1; k < NT / 64; k++)
            v += sums[k][i];
        a.dw[(size_t)blockIdx.x * d + i] = v;
    }
}

// dw of the workgroups' rows.  A workgroup: COLUMNS channels of q or k, 32 lanes for each, which take every 32nd row.
template <int TYPE>
__global__ __launch_bounds__(1024) void weight_kernel(const float *__restrict__ rows, int q_rows, int k_rows, int D, void *dwq, void *dwk)
{
    __shared__ float sums[32][COLUMNS + 1];
    const int column = threadIdx.x % COLUMNS, part = threadIdx.x / COLUMNS, c = blockIdx.x * COLUMNS + column;
    const int n = blockIdx.y ? k_rows : q_rows;
    void *to = blockIdx.y ? dwk : dwq;
    if (to == nullptr)
        return;
    const float *from = rows + (blockIdx.y ? (size_t)q_rows * D : 0) + c;
    float v = 0.0f;
    if (c < D)
#pragma unroll 4
        for (int r = part; r < n; r += 32)
            v += from[(size_t)r * D];
    sums[part][column] = v;
    __syncthreads();
    if (part == 0 && c < D) {
        v = 0.0f;
#pragma unroll
        for (int r = 0; r < 32; r++)
            v += sums[r][column];
        if constexpr (TYPE == F32)
            ((float *)to)[c] = v;
        else if constexpr (TYPE == F16)
            ((h1 *)to)[c] = (h1)v;
        else {
            uint32_t w;
            asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(w) : "v"(v), "v"(v));
            ((uint16_t *)to)[c] = (uint16_t)w;
        }
    }
}

static int workers(int64_t items, int64_t of, int64_t all)
{
    // sixteen waves per CU for both sides together: with more, more sums of dw
    return (int)std::max<int64_t>(1, std::min<int64_t>(items, 4ll * cu_count() * of / all));
}

// sizes and the tables; also how many heads a lane takes
static int prepare(Args &a, const void *cos, const void *sin, int B, int Hq, int H, int T, int D, int R, float eps, const int64_t *table_strides,
                   int dtype, const void *const *pointers, const int64_t *const *strides, int n, int &heads)
{
    if (B <= 0 || Hq <= 0 || H <= 0 || T <= 0)
        return ADKV_E_SHAPE;
    if (D <= 0 || D > DIM_MAX || D % 8 || R <= 0 || R > D || R % 8)
        return ADKV_E_DIM;
    if (dtype != F32 && dtype != F16 && dtype != BF16)
        return ADKV_E_UNSUPPORTED;
    if ((int64_t)B * T * (Hq + H) > INT32_MAX)
        return ADKV_E_SHAPE;
    int64_t bits = (uintptr_t)cos | (uintptr_t)sin;
    for (int i = 0; i < n; i++)
        bits |= (uintptr_t)pointers[i];
    int64_t steps = table_strides[0] | table_strides[1];
    for (int i = 0; i < n; i++)
        if (strides[i] != nullptr)
            steps |= strides[i][0] | strides[i][1] | strides[i][2];
    const int size = dtype == F32 ? 4 : 2;
    bits |= steps * size;
    if (bits & (V * size - 1))
        return ADKV_E_ALIGN;
    a.cos = cos;
    a.sin = sin;
    a.cs_b = table_strides[0];
    a.cs_t = table_strides[1];
    a.tokens = B * T;
    a.T = T;
    a.half = D / 2;
    a.turned = R / 2;
    a.lanes = a.half / V;
    a.log = 0;
    while (1 << a.log < a.lanes)
        a.log++;
    const int rows = NT >> a.log;
    a.blocks = (a.tokens + rows - 1) / rows;
    a.eps = eps;
    a.inv_d = 1.0f / (float)D;
    // four heads to a lane where that leaves work for all CUs; else one, and four times the lanes
    // (the first size above 49 us with four, 59 with one; a token of 128 sequences 3.3 us with one, half a us more with four)
    heads = 4;
    if ((int64_t)a.blocks * ((Hq + 3) / 4 + (H + 3) / 4) < 4 * cu_count())
        heads = 1;
    return ADKV_OK;
}

static Side side(const void *x, const void *w, void *out, const int64_t *strides, const int64_t *out_strides, int heads, int each)
{
    Side s = {};
    s.x = x;
    s.w = w;
    s.out = out;
    s.xs = {(long)strides[0], (long)strides[1], (long)strides[2]};
    if (out_strides != nullptr)
        s.os = {(long)out_strides[0], (long)out_strides[1], (long)out_strides[2]};
    s.heads = heads;
    s.groups = (heads + each - 1) / each;
    return s;
}
} // namespace adkv_rope_norm

#define ADKV_EACH(kernel)                                            \
    (dtype == F32    ? (heads == 4 ? kernel<F32, 4> : kernel<F32, 1>) \
     : dtype == F16  ? (heads == 4 ? kernel<F16, 4> : kernel<F16, 1>) \
                     : (heads == 4 ? kernel<BF16, 4> : kernel<BF16, 1>))

extern "C" int adkv_rope_norm_qk(const void *q, const void *k, const void *cos, const void *sin, const void *q_weight, const void *k_weight,
                                 void *q_out, void *k_out, int B, int Hq, int H, int T, int D, int R, float eps, const int64_t *q_strides,
                                 const int64_t *k_strides, const int64_t *table_strides, int dtype, void *stream)
{
    using namespace adkv_rope_norm;
    if (!q || !k || !cos || !sin || !q_weight || !k_weight || !q_out || !k_out || !q_strides || !k_strides || !table_strides)
        return ADKV_E_NULL;
    Args a = {};
    int heads;
    const void *const pointers[] = {q, k, q_weight, k_weight, q_out, k_out};
    const int64_t *const strides[] = {q_strides, k_strides, nullptr, nullptr, nullptr, nullptr};
    if (int rc = prepare(a, cos, sin, B, Hq, H, T, D, R, eps, table_strides, dtype, pointers, strides, 6, heads))
        return rc;
    const int64_t qs[3] = {(int64_t)Hq * T * D, (int64_t)T * D, D}, ks[3] = {(int64_t)H * T * D, (int64_t)T * D, D};
    a.q = side(q, q_weight, q_out, q_strides, qs, Hq, heads);
    a.k = side(k, k_weight, k_out, k_strides, ks, H, heads);
    const int64_t before = (int64_t)a.q.groups * a.blocks, all = before + (int64_t)a.k.groups * a.blocks;
    if (all >= 1 << 24) // a grid is 2^32 threads at most
        return ADKV_E_SHAPE;
    a.k.first = (int)before;
    const auto kernel = ADKV_EACH(forward_kernel);
    hipLaunchKernelGGL(kernel, dim3((unsigned)all), dim3(NT), 0, (hipStream_t)stream, a);
    return check_launch();
}

extern "C" int64_t adkv_rope_norm_qk_backward_workspace_bytes(int D)
{
    if (D <= 0 || D > adkv_rope_norm::DIM_MAX)
        return ADKV_E_DIM;
    const int cus = adkv_rope_norm::cu_count();
    return cus > 0 ? (4ll * cus + 2) * D * 4 : (int64_t)ADKV_E_DEVICE;
}

extern "C" int adkv_rope_norm_qk_backward(const void *q_grad, const void *k_grad, const void *q, const void *k, const void *cos, const void *sin,
                                          const void *q_weight, const void *k_weight, void *dq, void *dk, void *dq_weight, void *dk_weight, int B,
                                          int Hq, int H, int T, int D, int R, float eps, const int64_t *q_grad_strides,
                                          const int64_t *k_grad_strides, const int64_t *q_strides, const int64_t *k_strides,
                                          const int64_t *dq_strides, const int64_t *dk_strides, const int64_t *table_strides, int dtype,
                                          void *workspace, int64_t workspace_bytes, void *stream)
{
    using namespace adkv_rope_norm;
    const bool with_q = dq || dq_weight, with_k = dk || dk_weight;
    if (!cos || !sin || !table_strides || (with_q && (!q_grad || !q || !q_weight || !q_grad_strides || !q_strides || (dq && !dq_strides))) ||
        (with_k && (!k_grad || !k || !k_weight || !k_grad_strides || !k_strides || (dk && !dk_strides))))
        return ADKV_E_NULL;
    if (!with_q && !with_k)
        return ADKV_OK;
    Args a = {};
    int heads;
    const void *pointers[8];
    const int64_t *strides[8];
    int n = 0;
    const auto put = [&](const void *p, const int64_t *s) {
        pointers[n] = p;
        strides[n++] = s;
    };
    if (with_q) {
        put(q_grad, q_grad_strides);
        put(q, q_strides);
        put(q_weight, nullptr);
        put(dq, dq ? dq_strides : nullptr);
    }
    if (with_k) {
        put(k_grad, k_grad_strides);
        put(k, k_strides);
        put(k_weight, nullptr);
        put(dk, dk ? dk_strides : nullptr);
    }
    if (int rc = prepare(a, cos, sin, B, Hq, H, T, D, R, eps, table_strides, dtype, pointers, strides, n, heads))
        return rc;
    const bool weights = dq_weight || dk_weight;
    const int64_t need = weights ? adkv_rope_norm_qk_backward_workspace_bytes(D) : 0;
    if (need < 0)
        return (int)need;
    if (weights && (!workspace || workspace_bytes < need))
        return ADKV_E_WORKSPACE;
    if ((uintptr_t)workspace & 3)
        return ADKV_E_ALIGN;
    a.dw = weights ? (float *)workspace : nullptr;
    const int64_t all = (with_q ? Hq : 0) + (with_k ? H : 0);
    if (with_q) {
        a.q = side(q, q_weight, dq, q_strides, dq ? dq_strides : nullptr, Hq, heads);
        a.q.dz = q_grad;
        a.q.dzs = {(long)q_grad_strides[0], (long)q_grad_strides[1], (long)q_grad_strides[2]};
        a.q.workers = workers((int64_t)a.q.groups * a.blocks, Hq, all);
    }
    a.k.first = a.q.workers;
    if (with_k) {
        a.k = side(k, k_weight, dk, k_strides, dk ? dk_strides : nullptr, H, heads);
        a.k.dz = k_grad;
        a.k.dzs = {(long)k_grad_strides[0], (long)k_grad_strides[1], (long)k_grad_strides[2]};
        a.k.workers = workers((int64_t)a.k.groups * a.blocks, H, all);
        a.k.first = a.q.workers;
    }
    const auto kernel = ADKV_EACH(backward_kernel);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(a.q.workers + a.k.workers)), dim3(NT), 0, (hipStream_t)stream, a);
    if (int rc = check_launch())
        return rc;
    if (weights) {
        const auto sum = dtype == F32 ? weight_kernel<F32> : dtype == F16 ? weight_kernel<F16> : weight_kernel<BF16>;
        hipLaunchKernelGGL(sum, dim3((unsigned)((D + COLUMNS - 1) / COLUMNS), 2), dim3(1024), 0, (hipStream_t)stream, a.dw, a.q.workers, a.k.workers,
                           D, dq_weight, dk_weight);
    }
    return weights ? check_launch() : ADKV_OK;
}
