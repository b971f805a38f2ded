// Attention of n new tokens per sequence over codes: a prefix whose codes all sequences share, then each sequence's own codes, the
// new tokens' among them (head dim 128, 4-bit or 2-bit codes, 1, 2, 4 or 8 query heads per KV head).
//
//   x[i, t] = scaling * q_i . K_t + mask[i, t],  t over the P prefix tokens and the own tokens up to the query's;  out_i = sum softmax(x_i)_t V_t
//
// The prefix is replayed once for the batch and multiplied with the queries of all sequences as one matrix, so that its cost does not
// grow with the batch but by matrix instructions.  The context of a KV head is cut at checkpoints into pieces, each of which leaves
// (m, l, o) = (max x, sum e^(x-m), sum e^(x-m) V) per query row; pieces are joined by M = max m, out = sum e^(m-M) o / sum e^(m-M) l.
// Scores, m, l, o are fp32; the weights e^(x-m) are rounded to fp16 for the matrix cores, relative to the largest so far.
#include <algorithm>

#include "adkv_device.h"

#include "../../include/adkv_hip.h"

#pragma clang fp contract(off)

namespace adkv_ext {
using namespace adkv;

typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef float f8v __attribute__((ext_vector_type(8)));

constexpr int D = 128;
constexpr int TILE = 64;                 // tokens
constexpr int TILE_BYTES = D * TILE * 2; // a channel's tokens are 128 consecutive bytes
constexpr int PRODUCERS = 4, CONSUMERS = 4, THREADS = 64 * (PRODUCERS + CONSUMERS);
constexpr int MAX_TOKENS = 1 << 24; // 64 bytes each: a piece's codes are addressed in 32 bits
constexpr float LOG2E = 1.44269504088896340736f;

struct Tensor { // K or V of a source
    const uint32_t *codes; // [units, n_super, D]
    const h1 *ckpt;        // [units, n_ckpt, D, 2], or null
    const h1 *zp, *sc, *al, *be, *tg;
};

// Codes and the query rows that look at them.  The prefix has a unit per KV head and the rows (sequence, token, query head of
// the group); an own source has a unit per sequence and KV head and the rows (token, query head).
struct Source {
    Tensor t[2];
    int tokens, n_super, n_ckpt;
    int interval, intervals, nseg; // a piece is a run of whole checkpoint intervals
    int units, blocks, rows;       // query blocks per unit, query rows per unit
    int items;                     // units * blocks * nseg
    int seen;                      // tokens that the first of the new tokens looks at; each later one at one more if causal
    int causal;
    int col;                       // where its tokens are in the mask
    int piece;                     // number of its first piece among all partial results
};

struct Args {
    Source s[2]; // prefix, own
    const h1 *q;
    long q_sb, q_sh, q_st;
    const void *mask;
    long m_sb, m_sh, m_st;
    int mask_dt;
    float *partial; // [pieces, rows, D]
    float2 *ml;     // [pieces, rows]: m, l
    long rows;      // B * n * Hq, in the order of the output [B, n, Hq]
    int B, H, G, n;
    int act_bf16;
    float scaling;
};

// where a channel's 16-byte pieces of a tile are: eight lanes' writes and a matrix operand's reads spread over the banks
__device__ __forceinline__ int piece_of(int c, int unit) { return c * (TILE * 2) + ((unit ^ (c >> 1 & 7)) << 4); }

template <bool MAX>
__device__ __forceinline__ float fold_quarters(float v) // over the lanes l % 16
{
    unsigned a = __builtin_bit_cast(unsigned, v), b;
    asm volatile("v_mov_b32 %0, %1" : "=v"(b) : "v"(a)); // two copies: the compiler folds a swap of a register with itself
    typedef unsigned u2v __attribute__((ext_vector_type(2)));
    u2v r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    unsigned x = r.x, y = r.y;
    asm volatile("" : "+v"(x), "+v"(y));
    v = MAX ? fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y)) : __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
    a = __builtin_bit_cast(unsigned, v);
    asm volatile("v_mov_b32 %0, %1" : "=v"(b) : "v"(a));
    r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    x = r.x;
    y = r.y;
    asm volatile("" : "+v"(x), "+v"(y));
    return MAX ? fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y)) : __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}

// ---------------------------------------------------------------------------------------------------------------- producers
// A wave replays 64 channels of K or V, one per lane, a tile at a time.
template <int BITS>
struct Producer {
    static constexpr int WPT = TILE * BITS / 32; // words of a channel per tile
    static constexpr int UPW = 32 / BITS / 8;    // units of eight tokens per word
    Lone st;
    __amdgpu_buffer_rsrc_t codes; // reads behind the last word of the piece are dropped
    int next, c, left;            // tokens that are left of the piece
    uint32_t buf[2][WPT];

    __device__ __forceinline__ void start(const Tensor &t, const Source &s, int unit, int h, int channel, int first, int t1)
    {
        c = channel;
        const int t0 = first * s.interval, pi = h * D + c;
        left = t1 - t0;
        const int words = (left + 32 / BITS - 1) / (32 / BITS);
        codes = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint32_t *>(t.codes) + ((size_t)unit * s.n_super + t0 / (32 / BITS)) * D, 0,
                                                  words * D * 4, 0x00027000);
        next = c * 4;
        h1 zp = t.zp[pi], sc = t.sc[pi];
        if (first > 0) {
            const h2 r = as_h2(*reinterpret_cast<const uint32_t *>(t.ckpt + (((size_t)unit * s.n_ckpt + first - 1) * D + c) * 2));
            zp = r.x;
            sc = r.y;
        }
        const h1 one = (h1)1.0f, be = t.be[pi], bt = be * t.tg[pi]; // omt = 1 - beta*target, both steps rounded
        st.z = as_u32((h2){zp, (h1)0.0f});
        st.r = as_u32((h2){(h1)0.0f, sc});
        st.ca = as_u32((h2){t.al[pi], one});
        st.cf = as_u32((h2){one, be});
        st.c0 = as_u32((h2){(h1)0.0f, one - bt});
        load(buf[0]);
        load(buf[1]);
    }
    __device__ __forceinline__ void load(uint32_t *b)
    {
#pragma unroll
        for (int i = 0; i < WPT; i++)
            b[i] = __builtin_amdgcn_raw_buffer_load_b32(codes, next + i * D * 4, 0, 0);
        next += WPT * D * 4;
    }
    // the next tile from the words of buffer I, which then take those of the tile after the next
    template <int I>
    __device__ __forceinline__ void tile(const uint2 *lut, uint32_t lane_copy, char *to)
    {
        uint2 e[2][4];
        lone_lookup<BITS>(e[0], lut, buf[I], 0, lane_copy);
#pragma unroll
        for (int u = 0; u < TILE / 8; u++) {
            if (u + 1 < TILE / 8)
                lone_lookup<BITS>(e[(u & 1) ^ 1], lut, buf[I], u + 1, lane_copy);
            __builtin_amdgcn_sched_barrier(0);
            uint32_t x[4];
            lone_eight(st, e[u & 1], x);
            if (left < (u + 1) * 8) { // values behind the last token are zero: their weights are, and the rest may be anything
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int n = left - u * 8 - 2 * k;
                    x[k] = n >= 2 ? x[k] : n == 1 ? x[k] & 0xFFFFu : 0u;
                }
            }
            *reinterpret_cast<uint4 *>(to + piece_of(c, u)) = make_uint4(x[0], x[1], x[2], x[3]);
            __builtin_amdgcn_sched_barrier(0);
        }
        left -= TILE;
        load(buf[I]);
    }
};

// ---------------------------------------------------------------------------------------------------------------- consumers
template <int DT>
__device__ __forceinline__ float widen(uint32_t v)
{
    return DT == ADKV_DT_F32 ? __uint_as_float(v) : DT == ADKV_DT_F16 ? (float)__builtin_bit_cast(h1, (uint16_t)v) : __uint_as_float(v << 16);
}
// a mask row at the 8 tokens from t on, of which `there` are in the source
template <int DT>
__device__ __forceinline__ f8v mask_eight(const char *row, int t, int there)
{
    constexpr int SIZE = DT == ADKV_DT_F32 ? 4 : 2;
    const char *p = row + (long)t * SIZE;
    f8v m = {};
    if (there >= 8) {
        if constexpr (SIZE == 4) {
            __builtin_memcpy(&m, p, 32);
        } else {
            uint4 u;
            __builtin_memcpy(&u, p, 16);
            m = (f8v){widen<DT>(u.x & 0xFFFFu), widen<DT>(u.x >> 16), widen<DT>(u.y & 0xFFFFu), widen<DT>(u.y >> 16),
                      widen<DT>(u.z & 0xFFFFu), widen<DT>(u.z >> 16), widen<DT>(u.w & 0xFFFFu), widen<DT>(u.w >> 16)};
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < there)
                m[e] = widen<DT>(SIZE == 4 ? reinterpret_cast<const uint32_t *>(p)[e] : reinterpret_cast<const uint16_t *>(p)[e]);
    }
    return m;
}

// NB blocks of 16 query rows.  Scores come as columns (lane l: row l % 16, tokens 8 * (l / 16) + 0..7 of every 32), which is as the
// weights are taken by the product with V; the outputs are columns too, so that a row's maximum and sum are its lanes' own.
template <int NB>
struct Consumer {
    h8v q[NB][4];
    f4v o[NB][8];
    float m[NB], l[NB];
    long out[NB];         // the row among all rows, -1: none
    int limit[NB];        // tokens of the source that it looks at
    const char *mask[NB]; // its mask at the source's first token

    __device__ __forceinline__ void start(const Args &a, const Source &s, bool prefix, int unit, int first_block, int step, int lane)
    {
        const int r16 = lane & 15, quarter = lane >> 4;
#pragma unroll
        for (int k = 0; k < NB; k++) {
            const int row = (first_block + k * step) * 16 + r16, r = min(row, s.rows - 1);
            const int g = r % a.G, token = r / a.G;
            const int b = prefix ? token / a.n : unit / a.H, i = prefix ? token % a.n : token, h = prefix ? unit : unit % a.H;
            const int hq = h * a.G + g;
            out[k] = row < s.rows ? ((long)b * a.n + i) * (a.H * a.G) + hq : -1;
            limit[k] = s.causal ? s.seen + i : s.seen;
            const h1 *src = a.q + b * a.q_sb + hq * a.q_sh + i * a.q_st + quarter * 8;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint4 u;
                __builtin_memcpy(&u, src + c * 32, 16);
                if (a.act_bf16)
                    u = make_uint4(as_u32(act2(u.x, 1)), as_u32(act2(u.y, 1)), as_u32(act2(u.z, 1)), as_u32(act2(u.w, 1)));
                q[k][c] = __builtin_bit_cast(h8v, u);
            }
            mask[k] = nullptr;
            if (a.mask != nullptr)
                mask[k] = (const char *)a.mask + (b * a.m_sb + hq * a.m_sh + i * a.m_st + s.col) * (a.mask_dt == ADKV_DT_F32 ? 4 : 2);
            m[k] = -INFINITY;
            l[k] = 0.0f;
#pragma unroll
            for (int c = 0; c < 8; c++)
                o[k][c] = (f4v){0.0f, 0.0f, 0.0f, 0.0f};
        }
    }

    // the tile of the tokens from t on
    __device__ __forceinline__ void tile(const char *keys, const char *values, int t, const Args &a, const Source &s, int lane)
    {
        typedef short s4v __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4v *Lds;
        const int r16 = lane & 15, quarter = lane >> 4;
        f4v sc[NB][2][2];
        // Block j of 16 keys out of 32: row m is token 8 * (m / 4) + 4 * j + m % 4, so that a lane gets eight consecutive ones of both
        // blocks.  A transposing read hands 16 lanes 4 channels of their tokens: lane i reads channel i / 4, the tokens of chunk i % 4.
        const auto kbase = (__attribute__((address_space(3))) const char *)keys;
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            int at[2];
#pragma unroll
            for (int i = 0; i < 2; i++)
                at[i] = piece_of(quarter * 8 + i * 4 + (r16 >> 2), kk * 4 + (r16 & 3));
#pragma unroll
            for (int j = 0; j < 2; j++) {
#pragma unroll
                for (int k = 0; k < NB; k++)
                    sc[k][kk][j] = (f4v){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const s4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(kbase + at[0] + c * 32 * TILE * 2 + j * 8));
                    const s4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(kbase + at[1] + c * 32 * TILE * 2 + j * 8));
                    const uint2 u = __builtin_bit_cast(uint2, x), v = __builtin_bit_cast(uint2, y);
                    const h8v key = __builtin_bit_cast(h8v, make_uint4(u.x, u.y, v.x, v.y));
#pragma unroll
                    for (int k = 0; k < NB; k++)
                        sc[k][kk][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, q[k][c], sc[k][kk][j], 0, 0, 0);
                }
            }
        }
        h8v w[NB][2];
#pragma unroll
        for (int k = 0; k < NB; k++) {
            float x[16];
#pragma unroll
            for (int e = 0; e < 16; e++)
                x[e] = sc[k][e >> 3][e >> 2 & 1][e & 3] * a.scaling;
            if (a.mask != nullptr) {
#pragma unroll
                for (int kk = 0; kk < 2; kk++) {
                    const int at = t + kk * 32 + quarter * 8;
                    const f8v add = a.mask_dt == ADKV_DT_F32   ? mask_eight<ADKV_DT_F32>(mask[k], at, s.tokens - at)
                                    : a.mask_dt == ADKV_DT_F16 ? mask_eight<ADKV_DT_F16>(mask[k], at, s.tokens - at)
                                                               : mask_eight<ADKV_DT_BF16>(mask[k], at, s.tokens - at);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        x[kk * 8 + e] += add[e];
                }
            }
            if (t + TILE > s.seen) {
#pragma unroll
                for (int e = 0; e < 16; e++)
                    x[e] = t + (e >> 3) * 32 + quarter * 8 + (e & 7) < limit[k] ? x[e] : -INFINITY;
            }
            float mx = x[0];
#pragma unroll
            for (int e = 1; e < 16; e++)
                mx = fmaxf(mx, x[e]);
            mx = fmaxf(m[k], fold_quarters<true>(mx));
            if (__any(mx > m[k])) {
                const float shrink = m[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m[k] - mx) * LOG2E);
                m[k] = mx;
                l[k] *= shrink;
#pragma unroll
                for (int c = 0; c < 8; c++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        o[k][c][e] *= shrink;
            }
            const float ref = mx == -INFINITY ? 0.0f : mx; // nothing but -inf so far: all weights are zero
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                x[e] = __builtin_amdgcn_exp2f((x[e] - ref) * LOG2E);
                sum += x[e];
            }
            l[k] += sum;
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                uint32_t p[4];
#pragma unroll
                for (int e = 0; e < 4; e++)
                    p[e] = as_u32((h2){(h1)x[kk * 8 + 2 * e], (h1)x[kk * 8 + 2 * e + 1]});
                w[k][kk] = __builtin_bit_cast(h8v, make_uint4(p[0], p[1], p[2], p[3]));
            }
        }
#pragma unroll
        for (int kk = 0; kk < 2; kk++)
#pragma unroll
            for (int c = 0; c < 8; c++) {
                const h8v v = *reinterpret_cast<const h8v *>(values + c * 16 * TILE * 2 + piece_of(r16, kk * 4 + quarter));
#pragma unroll
                for (int k = 0; k < NB; k++)
                    o[k][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w[k][kk], o[k][c], 0, 0, 0);
            }
    }

    __device__ __forceinline__ void finish(const Args &a, int piece, int lane)
    {
#pragma unroll
        for (int k = 0; k < NB; k++) {
            const float sum = fold_quarters<false>(l[k]);
            if (out[k] < 0)
                continue;
            const long at = piece * a.rows + out[k];
            if (lane < 16)
                a.ml[at] = make_float2(m[k], sum);
#pragma unroll
            for (int c = 0; c < 8; c++)
                *reinterpret_cast<f4v *>(a.partial + at * D + c * 16 + (lane >> 4) * 4) = o[k][c];
        }
    }
};

// Four waves replay the tile after the one that the other four multiply with: a wave of either kind per SIMD, two buffers, a
// barrier per tile.
template <int BITS, int NB>
__global__ __launch_bounds__(THREADS) void attend_kernel(Args a)
{
    // the table at LDS offset 0; two buffers of a K and a V tile
    __shared__ uint4 smem[(LUT_WORDS64 * 8 + 4 * TILE_BYTES) / 16];
    uint2 *lut = reinterpret_cast<uint2 *>(smem);
    char *tiles = reinterpret_cast<char *>(smem) + LUT_WORDS64 * 8;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const bool prefix = (int)blockIdx.x < a.s[0].items;
    const Source &s = a.s[prefix ? 0 : 1];
    int item = (int)blockIdx.x - (prefix ? 0 : a.s[0].items);
    const int block = item % s.blocks;
    item /= s.blocks;
    const int seg = item % s.nseg, unit = item / s.nseg;
    const int first = (int)((long)s.intervals * seg / s.nseg), end = (int)((long)s.intervals * (seg + 1) / s.nseg);
    const int t0 = first * s.interval, t1 = seg == s.nseg - 1 ? s.tokens : end * s.interval;
    const int ntiles = (t1 - t0 + TILE - 1) / TILE;

    if (wave < PRODUCERS) {
        Producer<BITS> p;
        p.start(s.t[wave >> 1], s, unit, prefix ? unit : unit % a.H, (wave & 1) * 64 + lane, first, t1);
        if constexpr (BITS == 4)
            lone_fill<THREADS>(lut, threadIdx.x);
        else
            lone_fill2<THREADS>(lut, threadIdx.x);
        __syncthreads();
        const uint32_t lane_copy = BITS == 4 ? (uint32_t)(lane & (LUT_COPIES - 1)) * 8u : (uint32_t)(lane & (LUT2_COPIES - 1)) * 16u;
        char *to = tiles + (wave >> 1) * TILE_BYTES;
        for (int i = 0; i <= ntiles; i += 2) { // one more than there are: the last pair of buffers is multiplied meanwhile
            if (i < ntiles)
                p.template tile<0>(lut, lane_copy, to);
            __syncthreads();
            if (i == ntiles)
                break;
            if (i + 1 < ntiles)
                p.template tile<1>(lut, lane_copy, to + 2 * TILE_BYTES);
            __syncthreads();
        }
    } else {
        const int mine = block * (NB * CONSUMERS) + wave - PRODUCERS;      // blocks of 16 rows: this one, and CONSUMERS further
        const int there = (s.rows + 15) / 16 - mine;
        const bool any = there > 0;
        Consumer<NB> c;
        if (any)
            c.start(a, s, prefix, unit, mine, CONSUMERS, lane);
        if constexpr (BITS == 4)
            lone_fill<THREADS>(lut, threadIdx.x);
        else
            lone_fill2<THREADS>(lut, threadIdx.x);
        __syncthreads();
        for (int i = 0; i < ntiles; i++) {
            __syncthreads();
            const char *from = tiles + (i & 1) * 2 * TILE_BYTES;
            if (any)
                c.tile(from, from + TILE_BYTES, t0 + i * TILE, a, s, lane);
        }
        __syncthreads();
        if (any)
            c.finish(a, s.piece + seg, lane);
    }
}

// out = sum e^(m-M) o / sum e^(m-M) l over the pieces, in their order.  Four channels per lane; bound by reading the partial outputs.
__global__ __launch_bounds__(256) void join_kernel(const float *__restrict__ partial, const float2 *__restrict__ ml, h1 *__restrict__ out,
                                                   long rows, int pieces, int act_bf16)
{
    const long row = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int c = (threadIdx.x & 31) * 4;
    if (row >= rows)
        return;
    float M = -INFINITY;
    for (int k = 0; k < pieces; k++)
        M = fmaxf(M, ml[k * rows + row].x);
    const float ref = M == -INFINITY ? 0.0f : M; // a row whose mask leaves nothing: 0 / 0
    float L = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k = 0; k < pieces; k++) {
        const float2 p = ml[k * rows + row];
        const float e = __builtin_amdgcn_exp2f((p.x - ref) * LOG2E);
        const float4 v = *reinterpret_cast<const float4 *>(partial + (k * rows + row) * D + c);
        L = __builtin_fmaf(p.y, e, L);
        o.x = __builtin_fmaf(v.x, e, o.x);
        o.y = __builtin_fmaf(v.y, e, o.y);
        o.z = __builtin_fmaf(v.z, e, o.z);
        o.w = __builtin_fmaf(v.w, e, o.w);
    }
    const float inv = 1.0f / L;
    const float r[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if (act_bf16) {
            uint32_t b[2];
#pragma unroll
            for (int k = 0; k < 2; k++) { // to nearest even, from fp32
                const uint32_t u = __float_as_uint(r[2 * i + k]);
                b[k] = (u & 0x7FFFFFFFu) > 0x7F800000u ? 0x7FC0u : (u + 0x7FFFu + (u >> 16 & 1u)) >> 16;
            }
            w[i] = b[0] | b[1] << 16;
        } else {
            w[i] = as_u32((h2){(h1)r[2 * i], (h1)r[2 * i + 1]});
        }
    }
    *reinterpret_cast<uint2 *>(out + row * D + c) = make_uint2(w[0], w[1]);
}

// The state behind token T - 1 of every channel, from the last checkpoint in front of it: at most an interval, a token at a time.
// Where token T opens an interval the state is that interval's checkpoint, which nobody may have recorded yet.
template <int BITS>
__global__ __launch_bounds__(128) void state_kernel(Source s, int H, int n_ckpt, h1 *k_state, h1 *v_state)
{
    constexpr int TPW = 32 / BITS;
    const int unit = blockIdx.x, c = threadIdx.x, pi = unit % H * D + c, T = s.tokens;
    const Tensor t = s.t[blockIdx.y];
    const h1 one = (h1)1.0f, be = t.be[pi], bt = be * t.tg[pi];
    const int first = s.interval > 0 ? min((T - 1) / s.interval, n_ckpt) : 0;
    h2 from = {t.zp[pi], t.sc[pi]};
    if (first > 0)
        from = as_h2(*reinterpret_cast<const uint32_t *>(t.ckpt + (((size_t)unit * n_ckpt + first - 1) * D + c) * 2));
    Lone st;
    st.z = as_u32((h2){from.x, (h1)0.0f});
    st.r = as_u32((h2){(h1)0.0f, from.y});
    st.ca = as_u32((h2){t.al[pi], one});
    st.cf = as_u32((h2){one, be});
    st.c0 = as_u32((h2){(h1)0.0f, one - bt});
    const uint32_t *w = t.codes + (size_t)unit * s.n_super * D + c;
    for (int at = first * s.interval; at < T; at += TPW) {
        const uint32_t word = w[(size_t)(at / TPW) * D];
#pragma unroll
        for (int i = 0; i < TPW; i++)
            if (at + i < T)
                lone_token(st, (int)(word >> (BITS * i) & Code<BITS>::FIELD) + Code<BITS>::QLO);
    }
    const uint32_t zs = as_u32((h2){lone_zp(st), lone_sc(st)});
    *reinterpret_cast<uint32_t *>((blockIdx.y ? v_state : k_state) + ((size_t)unit * D + c) * 2) = zs;
    if (s.interval > 0 && T % s.interval == 0 && T / s.interval - 1 < n_ckpt)
        *reinterpret_cast<uint32_t *>(const_cast<h1 *>(t.ckpt) + (((size_t)unit * n_ckpt + T / s.interval - 1) * D + c) * 2) = zs;
}

struct Plan {
    int nb;          // blocks of 16 rows per consumer wave
    int nseg[2];     // pieces of the prefix (0: there is none) and of an own context
    int intervals[2], blocks[2];
    long pieces() const { return nseg[0] + nseg[1]; }
};

static int usable_intervals(int tokens, int interval, int n_ckpt)
{
    return interval > 0 ? std::min((tokens + interval - 1) / interval, n_ckpt + 1) : 1;
}

// A workgroup takes a CU.  The length of a piece is chosen for the shortest launch by the model rounds of workgroups x (tiles of a
// piece + what a workgroup starts with).
static Plan plan(int B, int H, int G, int n, int P, int p_interval, int p_ckpt, int T, int interval, int n_ckpt)
{
    Plan p;
    const long rows[2] = {(long)B * n * G, (long)n * G};
    const int units[2] = {H, B * H}, tokens[2] = {P, T};
    p.nb = std::max(P > 0 ? rows[0] : 0, rows[1]) > 16 * CONSUMERS ? 2 : 1;
    p.intervals[0] = P > 0 ? usable_intervals(P, p_interval, p_ckpt) : 0;
    p.intervals[1] = usable_intervals(T, interval, n_ckpt);
    for (int i = 0; i < 2; i++)
        p.blocks[i] = (int)((rows[i] + 16 * CONSUMERS * p.nb - 1) / (16 * CONSUMERS * p.nb));
    const long cus = cu_count();
    double best = -1.0;
    p.nseg[0] = p.nseg[1] = 1;
    int chosen[2] = {p.intervals[0] ? 1 : 0, 1};
    for (int len = 4; len < (1 << 20); len += std::max(len / 4, 1)) { // tiles
        int ns[2];
        long items = 0, longest = 0;
        for (int i = 0; i < 2; i++) {
            const long tiles = (tokens[i] + TILE - 1) / TILE;
            ns[i] = (int)std::min<long>(p.intervals[i], (tiles + len - 1) / len);
            ns[i] = p.intervals[i] ? std::max(ns[i], 1) : 0;
            items += (long)units[i] * p.blocks[i] * ns[i];
            if (ns[i])
                longest = std::max(longest, (tiles + ns[i] - 1) / ns[i]);
        }
        const double cost = (double)((items + cus - 1) / cus) * (longest + 4) + 0.02 * (ns[0] + ns[1]);
        if (best < 0 || cost < best) {
            best = cost;
            chosen[0] = ns[0];
            chosen[1] = ns[1];
        }
        if (ns[0] <= 1 && ns[1] <= 1)
            break;
    }
    p.nseg[0] = chosen[0];
    p.nseg[1] = chosen[1];
    return p;
}

static int64_t pad256(int64_t n) { return (n + 255) & ~(int64_t)255; }

} // namespace adkv_ext

using namespace adkv_ext;

extern "C" {

int64_t adkv_extend_workspace_bytes(int B, int Hq, int H, int T, int n, int n_ckpt_cap, int ckpt_interval, int P, int prefix_n_ckpt_cap,
                                    int prefix_ckpt_interval)
{
    if (B <= 0 || H <= 0 || Hq <= 0 || Hq % H || T < 0 || n <= 0 || P < 0 || T > MAX_TOKENS || n > MAX_TOKENS - T || P > MAX_TOKENS)
        return 0;
    const Plan p = plan(B, H, Hq / H, n, P, prefix_n_ckpt_cap > 0 ? prefix_ckpt_interval : 0, prefix_n_ckpt_cap, T + n,
                        n_ckpt_cap > 0 ? ckpt_interval : 0, n_ckpt_cap);
    const int64_t rows = (int64_t)B * n * Hq;
    return 2 * pad256((int64_t)B * H * D * 4) + pad256(p.pieces() * rows * 8) + p.pieces() * rows * D * 4;
}

int adkv_extend(const void *q, const int64_t *q_strides, void *k_cache, void *v_cache, const void *k_new, const void *v_new,
                const int64_t *k_strides, const int64_t *v_strides, const void *const *k_params, const void *const *v_params,
                const void *mask, const int64_t *mask_strides, float scaling, void *out, int B, int Hq, int H, int T, int n, int D_,
                int n_super_cap, int bits, int act_dtype, void *k_ckpt, void *v_ckpt, int n_ckpt_cap, int ckpt_interval,
                const adkv_prefix *prefix, void *workspace, int64_t workspace_bytes, void *stream)
{
    const int mask_dt = act_dtype >> 8;
    act_dtype &= 255;
    if (!q || !k_cache || !v_cache || !k_new || !v_new || !k_params || !v_params || !out || !q_strides || (mask && !mask_strides))
        return ADKV_E_NULL;
    for (int i = 0; i < 5; i++)
        if (!k_params[i] || !v_params[i])
            return ADKV_E_NULL;
    if (B <= 0 || H <= 0 || Hq <= 0 || Hq % H || T < 0 || n <= 0 || n_super_cap <= 0 || T > MAX_TOKENS || n > MAX_TOKENS - T)
        return ADKV_E_SHAPE;
    if (D_ != D || (bits != 2 && bits != 4) || (act_dtype != ADKV_DT_F16 && act_dtype != ADKV_DT_BF16) ||
        (mask_dt != ADKV_DT_F32 && mask_dt != ADKV_DT_F16 && mask_dt != ADKV_DT_BF16))
        return ADKV_E_UNSUPPORTED;
    const int G = Hq / H, tpw = 32 / bits;
    if (G != 1 && G != 2 && G != 4 && G != 8)
        return ADKV_E_UNSUPPORTED;
    const int64_t rows = (int64_t)B * n * Hq;
    if (rows > INT32_MAX / 2 || (int64_t)B * H > INT32_MAX / 64)
        return ADKV_E_SHAPE;
    if ((T + n + tpw - 1) / tpw > n_super_cap)
        return ADKV_E_CAPACITY;
    if (((uintptr_t)k_cache & 15) || ((uintptr_t)v_cache & 15) || ((uintptr_t)q & 3) || ((uintptr_t)out & 7) || ((uintptr_t)workspace & 255))
        return ADKV_E_ALIGN;
    if ((q_strides[0] | q_strides[1] | q_strides[2]) & 1)
        return ADKV_E_ALIGN;
    if (!k_ckpt != !v_ckpt)
        return ADKV_E_NULL;
    auto bad_ckpt = [&](const void *k, const void *v, int cap, int interval) {
        return k && (cap <= 0 || interval <= 0 || interval % tpw) ? ADKV_E_SHAPE : ((uintptr_t)k & 3) || ((uintptr_t)v & 3) ? ADKV_E_ALIGN : ADKV_OK;
    };
    int rc = bad_ckpt(k_ckpt, v_ckpt, n_ckpt_cap, ckpt_interval);
    if (rc)
        return rc;
    if (!k_ckpt)
        n_ckpt_cap = ckpt_interval = 0;
    int P = 0, p_cap = 0, p_interval = 0;
    if (prefix) {
        P = prefix->tokens;
        if (!prefix->k_codes || !prefix->v_codes || !prefix->k_params || !prefix->v_params || !prefix->k_ckpt != !prefix->v_ckpt)
            return ADKV_E_NULL;
        for (int i = 0; i < 5; i++)
            if (!prefix->k_params[i] || !prefix->v_params[i])
                return ADKV_E_NULL;
        if (P < 0 || P > MAX_TOKENS || prefix->n_super <= 0)
            return ADKV_E_SHAPE;
        if ((P + tpw - 1) / tpw > prefix->n_super)
            return ADKV_E_CAPACITY;
        if (((uintptr_t)prefix->k_codes & 15) || ((uintptr_t)prefix->v_codes & 15))
            return ADKV_E_ALIGN;
        if ((rc = bad_ckpt(prefix->k_ckpt, prefix->v_ckpt, prefix->n_ckpt_cap, prefix->ckpt_interval)))
            return rc;
        if (prefix->k_ckpt) {
            p_cap = prefix->n_ckpt_cap;
            p_interval = prefix->ckpt_interval;
        }
    }
    const int64_t need = adkv_extend_workspace_bytes(B, Hq, H, T, n, n_ckpt_cap, ckpt_interval, P, p_cap, p_interval);
    if (!workspace || workspace_bytes < need)
        return ADKV_E_WORKSPACE;

    const Plan pl = plan(B, H, G, n, P, p_interval, p_cap, T + n, ckpt_interval, n_ckpt_cap);
    char *ws = (char *)workspace;
    const int64_t state_bytes = pad256((int64_t)B * H * D * 4);
    h1 *k_state = (h1 *)ws, *v_state = (h1 *)(ws + state_bytes);
    Args a;
    a.ml = (float2 *)(ws + 2 * state_bytes);
    a.partial = (float *)(ws + 2 * state_bytes + pad256(pl.pieces() * rows * 8));
    auto tensor = [](const void *codes, const void *ckpt, const void *const *p) {
        return Tensor{(const uint32_t *)codes, (const h1 *)ckpt, (const h1 *)p[0], (const h1 *)p[1], (const h1 *)p[2], (const h1 *)p[3], (const h1 *)p[4]};
    };
    Source &pre = a.s[0], &own = a.s[1];
    pre = Source{};
    if (P > 0) {
        pre.t[0] = tensor(prefix->k_codes, prefix->k_ckpt, prefix->k_params);
        pre.t[1] = tensor(prefix->v_codes, prefix->v_ckpt, prefix->v_params);
        pre.tokens = pre.seen = P;
        pre.n_super = prefix->n_super;
        pre.n_ckpt = p_cap;
        pre.interval = p_interval;
        pre.units = H;
        pre.rows = (int)((int64_t)B * n * G);
    }
    own.t[0] = tensor(k_cache, k_ckpt, k_params);
    own.t[1] = tensor(v_cache, v_ckpt, v_params);
    own.tokens = T + n;
    own.seen = T + 1;
    own.causal = 1;
    own.n_super = n_super_cap;
    own.n_ckpt = n_ckpt_cap;
    own.interval = ckpt_interval;
    own.units = B * H;
    own.rows = n * G;
    own.col = P;
    own.piece = pl.nseg[0];
    pre.causal = 0;
    pre.col = pre.piece = 0;
    int64_t items = 0;
    for (int i = 0; i < 2; i++) {
        Source &s = a.s[i];
        s.intervals = pl.intervals[i];
        s.nseg = pl.nseg[i];
        s.blocks = pl.blocks[i];
        const int64_t k = (int64_t)s.units * s.blocks * s.nseg;
        if (k > INT32_MAX)
            return ADKV_E_SHAPE;
        s.items = (int)k;
        items += k;
    }
    if (items > INT32_MAX)
        return ADKV_E_SHAPE;
    a.q = (const h1 *)q;
    a.q_sb = q_strides[0];
    a.q_sh = q_strides[1];
    a.q_st = q_strides[2];
    a.mask = mask;
    a.m_sb = a.m_sh = a.m_st = 0;
    if (mask) {
        a.m_sb = mask_strides[0];
        a.m_sh = mask_strides[1];
        a.m_st = mask_strides[2];
    }
    a.mask_dt = mask_dt;
    a.rows = rows;
    a.B = B;
    a.H = H;
    a.G = G;
    a.n = n;
    a.act_bf16 = act_dtype == ADKV_DT_BF16;
    a.scaling = scaling;

    // the new tokens' codes
    if (T > 0) {
        Source before = own;
        before.tokens = T;
        const auto kernel = bits == 4 ? state_kernel<4> : state_kernel<2>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(B * H), 2), dim3(D), 0, (hipStream_t)stream, before, H, n_ckpt_cap, k_state, v_state);
        if ((rc = check_launch()))
            return rc;
    }
    if ((rc = adkv_append_kv_pair(k_cache, v_cache, k_new, v_new, act_dtype, k_strides, v_strides, k_params, v_params, B, H, T, n, D, n_super_cap,
                                  bits, k_state, v_state, k_ckpt, v_ckpt, n_ckpt_cap, ckpt_interval, stream)))
        return rc;
    const auto kernel = bits == 4 ? (pl.nb == 2 ? attend_kernel<4, 2> : attend_kernel<4, 1>) : (pl.nb == 2 ? attend_kernel<2, 2> : attend_kernel<2, 1>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)items), dim3(THREADS), 0, (hipStream_t)stream, a);
    if ((rc = check_launch()))
        return rc;
    hipLaunchKernelGGL(join_kernel, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, (hipStream_t)stream, a.partial, a.ml, (h1 *)out, rows,
                       (int)pl.pieces(), a.act_bf16);
    return check_launch();
}

} // extern "C"
