// Causal attention over the dense rows of a prompt, grouped heads, fp16 or bf16.
//
//   x[i, t] = scaling * q_i . k_t + mask[i, t],  t up to i + (Tk - Tq);  out_i = sum_t softmax(x_i)_t v_t;  0 where a row looks at nothing
//
// One pass over the keys with the running maximum and sum of every row.  The rows of a KV head are those of all its query heads, row r being token
// r / g of head r % g, so that a block of rows spans few tokens and its keys serve g heads.
// Products are 32x32x16 matrix instructions, turned so that nothing has to change lanes between them: S^T = K Q^T leaves lane l with 16 of
// 32 scores of row l % 32, which rounded to the operands' type are as O^T = V^T P^T takes them, if V's tokens are taken in the same order (4h..4h+3,
// 4h+8.. for half h of the lanes).  V^T comes out of row-major tiles by the LDS's transposing reads.
// Weights are e^(x - m) for an m that is at most 2^8 smaller than the largest so far, so that outputs are rescaled seldom.  They are rounded to the
// operands' type for the matrix cores (fp16: after a factor of 2^7, which keeps 2^7 more of the small ones out of the subnormals); the sum that
// divides them is that of the rounded ones.  Scores, m, sums and outputs are fp32.
//
// Three forms:
//   many  a workgroup is four waves of 32 rows each over shared tiles of 64 keys and values, two tiles in the LDS, a barrier per tile
//   some  a workgroup is 64 rows, eight waves: each has 32 rows and every fourth 32 keys of them, over shared tiles of 128; joined in the LDS
//   few   a workgroup is 32 rows, its four waves walk through a quarter of the keys each in tiles of their own and are joined in the LDS; where
//         that leaves CUs without work the keys are cut into pieces for several workgroups, joined by a second kernel
// plan() says which, and what each takes.
//
// What bounds it, MI355X: long prompts the clock that the matrix cores' power allows (16384 tokens, 32 heads on 8, bf16: 1.98 ms, 1.11 PFLOP/s, matrix cores
// busy for 61 % of the time at 1.67 GHz; a library's product of 8192^3 runs at 1.40).  Batches of short ones memory and the way in and out of a workgroup
// (128 of 512 tokens, 32 heads: 539 us, 4.0 TB/s, the matrix cores 33 % busy; of 128 tokens 112 us, 4.8 TB/s; a copy runs at 5.15), and few blocks the
// chain of a single one.  A row over many keys: memory (8 x 8 heads of four, 4097 tokens: 31 us, 4.4 TB/s).
#include <math.h>

#include <algorithm>

#include "adkv_device.h"

#include "../../include/adkv_hip.h"

#pragma clang fp contract(off)

namespace adkv_prompt {
using adkv::check_launch;
using adkv::cu_count;
using adkv::load_to_lds;
using adkv::rsrc4;

typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef float f2v __attribute__((ext_vector_type(2)));

#define LDS __attribute__((address_space(3)))
#define GLOBAL __attribute__((address_space(1)))

template <typename T> __device__ __forceinline__ LDS T *shared(uint32_t at) { return (LDS T *)(uintptr_t)at; }

constexpr int WAVES = 4, NT = WAVES * 64, ROWS = 32; // rows of a wave
constexpr float LOG2E = 1.44269504088896340736f;
constexpr float SLACK = 8.0f; // how much smaller than the largest (2^) a row's reference may be
enum { F16 = ADKV_DT_F16, BF16 = ADKV_DT_BF16 };

struct Rows { // of q, k or v
    const char *p;
    long sb, sh; // bytes
    int st;
};
struct Args {
    Rows q, k, v;
    char *out;                // [B, Tq, H * g, D]
    const char *mask;
    const char *mask_end;     // behind its last element
    long m_sb, m_sh, m_st;    // elements
    const int *bounds;        // of packed sequences, n_seq + 1, or null
    float *partial;           // [pieces][rows of all][D], few rows in pieces
    f2v *ml;                  // [pieces][rows of all]
    long all;                 // rows of all
    int B, H, g, Tq, Tk, D, n_seq, mask_dt, pieces;
    int blocks, units, together; // of a unit (packed: of all sequences); units; units whose blocks are in flight together
    float scaling;
    uint32_t by_g;            // 2^32 / g rounded up
};

template <int TYPE> struct Half;
template <> struct Half<F16> {
    static constexpr float BIAS = 7.0f;
    static __device__ __forceinline__ f16v mfma(u4v a, u4v b, f16v c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2v){a, b}, h2v));
    }
    static __device__ __forceinline__ float add(uint32_t w, float sum)
    {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2v, w), (h2v){(_Float16)1.0f, (_Float16)1.0f}, sum, false);
    }
    static __device__ __forceinline__ float number(uint16_t w) { return (float)__builtin_bit_cast(_Float16, w); }
};
template <> struct Half<BF16> {
    static constexpr float BIAS = 0.0f;
    static __device__ __forceinline__ f16v mfma(u4v a, u4v b, f16v c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2v){a, b}, b2v));
    }
    static __device__ __forceinline__ float add(uint32_t w, float sum)
    {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2v, w), (b2v){(__bf16)1.0f, (__bf16)1.0f}, sum, false);
    }
    static __device__ __forceinline__ float number(uint16_t w) { return __uint_as_float((uint32_t)w << 16); }
};

__device__ __forceinline__ float other_half(float v, bool max)
{
    unsigned a = __float_as_uint(v), b = a;
    asm volatile("" : "+v"(b)); // two copies: the compiler folds a swap of a register with itself
    const u2v r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    unsigned x = r.x, y = r.y;
    asm volatile("" : "+v"(x), "+v"(y));
    return max ? fmaxf(__uint_as_float(x), __uint_as_float(y)) : __uint_as_float(x) + __uint_as_float(y);
}

// Channels that are multiplied, and that a tile's row has room for.  (80 channels, 997 tokens, 50 x 8 heads: with 96 of them 101 us, with all 128 115.)
constexpr int room(int CH) { return CH > 128 ? 256 : CH > 64 ? 128 : 64; }

// Rows of a tile are DP * 2 bytes in pieces of 16, piece c of row r at place c ^ turn(r), so that neither sixteen rows' reads of one piece
// nor a transposing read (four consecutive rows, 64 bytes of each) meet in a bank.
template <int DP> __device__ __forceinline__ constexpr int turn(int r)
{
    return DP == 64 ? (r >> 1 & 1) << 2 | (r >> 2 & 3) : (r & 3) << 2 | (r >> 2 & 3);
}

// Rows of keys or values one tile after the other, straight to the LDS, 1 KB an instruction; what is behind the last reads as zeros
template <int DP>
struct Stream {
    static constexpr int PIECES = DP / 8, EACH = 64 / PIECES; // of a row; rows per instruction
    uint64_t base;
    int left, st; // rows
    // from row `first` of `rows` on
    __device__ __forceinline__ void open(const char *p, int st_, int first, int rows)
    {
        base = (uint64_t)p + (int64_t)first * st_;
        left = rows - first;
        st = st_;
    }
    // N rows, whose first is at a multiple of 16 in its tile, to `lds`
    template <int N> __device__ __forceinline__ void ask(uint32_t lds, int lane, int D) const
    {
        const int bytes = left > 0 ? (min(left, N) - 1) * st + D * 2 : 0;
        const rsrc4 buffer = {(uint32_t)base, (uint32_t)(base >> 32), (uint32_t)bytes, 0x00027000u};
        const int r = lane / PIECES, c = lane % PIECES;
#pragma unroll
        for (int i = 0; i < N; i += EACH) {
            const int piece = c ^ turn<DP>(i + r);
            const uint32_t at = piece * 8 < D ? (uint32_t)((i + r) * st + piece * 16) : 0x7FFFFFF0u;
            load_to_lds(__builtin_amdgcn_readfirstlane(lds + (uint32_t)i * (DP * 2)), at, buffer);
        }
    }
    __device__ __forceinline__ void skip(int rows)
    {
        base += (int64_t)rows * st;
        left -= rows;
    }
};

// Where a workgroup's rows are
struct Job {
    int b, h;
    int q0, k0, n, m;  // first token of its queries and keys, how many; tokens of a sequence
    int first, rows;   // its first row and how many the sequence has
    int end;           // keys that its last row looks at
    bool nothing;      // rows that belong to no sequence: zeros
    int piece;
};

__device__ __forceinline__ int bound(const Args &a, int i) // of the sequences, and of what is in front of the first and behind the last
{
    if (i <= 0)
        return 0;
    return i > a.n_seq + 1 ? a.Tq : min(max(a.bounds[i - 1], 0), a.Tq);
}

// Of packed sequences the host knows neither how many blocks each has nor where they begin: sequence i's are from (its first row) / EACH + i on, which
// leaves room for all of them and some empty ones in between.
template <int EACH>
__device__ __forceinline__ bool find(const Args &a, int block, int lane, Job &j)
{
    int lo = 0, hi = a.n_seq + 2, x, y; // the last i whose place is not behind `block`
    while (true) {
        const int step = (hi - lo + 62) / 63, at = lo + lane * step, here = bound(a, at);
        const bool before = lane < 63 && at < hi && (int)((int64_t)here * a.g / EACH) + at <= block;
        const uint64_t which = __ballot(before);
        const int last = which ? 63 - __builtin_clzll(which) : 0;
        lo += last * step;
        hi = min(hi, lo + step);
        if (step == 1) { // the one behind it is on the next lane
            x = __builtin_amdgcn_readlane(here, last);
            y = __builtin_amdgcn_readlane(here, last + 1);
            break;
        }
    }
    j.n = j.m = max(y - x, 0);
    j.q0 = j.k0 = x;
    j.rows = j.n * a.g;
    j.first = (block - (int)((int64_t)x * a.g / EACH) - lo) * EACH;
    j.nothing = lo == 0 || lo == a.n_seq + 1;
    return j.first < j.rows;
}

__device__ __forceinline__ int token(const Args &a, int r) { return a.g == 1 ? r : (int)__umulhi((uint32_t)r, a.by_g); }

template <int EACH>
__device__ __forceinline__ bool place(const Args &a, int i, int lane, Job &j)
{
    if (a.bounds != nullptr) {
        // one after the other, all heads of a block together
        const int block = i / (a.H * a.pieces), rest = i - block * a.H * a.pieces;
        j.h = rest / a.pieces;
        j.piece = rest - j.h * a.pieces;
        j.b = 0;
        if (!find<EACH>(a, a.blocks - 1 - block, lane, j))
            return false;
    } else {
        // `together` units at a time, their longest rows first; consecutive units are on different XCDs, and a unit's blocks on one if
        // there are eight of them or a multiple of that
        j.piece = i % a.pieces;
        i /= a.pieces;
        const int batch = i / (a.together * a.blocks), here = min(a.together, a.units - batch * a.together);
        i -= batch * a.together * a.blocks;
        const int back = i / here, unit = batch * a.together + i - back * here;
        // eight sequences side by side, so that all heads of one are on an XCD, which is the only one to read their mask then (32 sequences of 700 tokens, eight
        // heads of 64 channels, bool: 35 us instead of 50; 128 of 512 without a mask: 538 instead of 550)
        const int eight = unit / (8 * a.H), of = unit - eight * 8 * a.H, beside = min(8, a.B - 8 * eight);
        j.h = of / beside;
        j.b = 8 * eight + of - j.h * beside;
        j.q0 = j.k0 = 0;
        j.n = a.Tq;
        j.m = a.Tk;
        j.rows = j.n * a.g;
        j.first = (a.blocks - 1 - back) * EACH;
        j.nothing = false;
    }
    j.end = j.nothing ? 0 : j.m - j.n + token(a, min(j.first + EACH, j.rows) - 1) + 1;
    return true;
}

// The mask of a lane's row for KB * 32 keys: SIZE bytes per key, as it is in memory.  Half h of the lanes loads keys 16 * KB * h.. of them, 16 bytes at a
// time, whatever their alignment; an exchange with the other half leaves both with the keys whose scores they have.
template <int SIZE, int KB>
struct Mask {
    static constexpr int WORDS = KB * 4 * SIZE, MORE = SIZE < 4 ? 1 : 0;
    uint32_t w[WORDS + MORE];
    uint32_t shift; // bytes in front of the lane's first
    // row: the lane's; keys k.. Nothing here waits for what is loaded.
    __device__ __forceinline__ void load(const Args &a, const char *row, int k, int lane)
    {
        typedef uint32_t u4a __attribute__((ext_vector_type(4), aligned(4)));
        const int first = k + (lane >> 5) * KB * 16;
        const char *p = row + (long)first * SIZE;
        // rows may begin between two words; loads that do so cost more than the shifts (1023 tokens, 16 bits: 97 us)
        const GLOBAL char *from = (const GLOBAL char *)((uintptr_t)p & ~(uintptr_t)3);
        if (__all((const char *)from + (WORDS + MORE) * 4 <= a.mask_end)) {
            shift = (uint32_t)(uintptr_t)p & 3;
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) {
                const u4a four = *(const GLOBAL u4a *)(from + i * 4);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    w[i + e] = four[e];
            }
            if (MORE)
                w[WORDS] = *(const GLOBAL uint32_t *)(from + WORDS * 4);
            return;
        }
        shift = 0;
        if (MORE)
            w[WORDS] = 0;
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
            w[i] = 0;
#pragma unroll
            for (int e = 0; e < 4 / SIZE; e++)
                if (first + i * 4 / SIZE + e < a.Tk) {
                    if constexpr (SIZE == 4)
                        w[i] = *(const GLOBAL uint32_t *)(p + i * 4);
                    else if constexpr (SIZE == 2)
                        w[i] |= (uint32_t)*(const GLOBAL uint16_t *)(p + i * 4 + e * 2) << e * 16;
                    else
                        w[i] |= (uint32_t)*(const GLOBAL uint8_t *)(p + i * 4 + e) << e * 8;
                }
        }
    }
    __device__ __forceinline__ void align()
    {
        if (MORE)
#pragma unroll
            for (int i = 0; i < WORDS; i++)
                w[i] = __builtin_amdgcn_alignbyte(w[i + MORE], w[i], shift);
    }
    // Of all of the wave's keys: 1 where nothing is added or hidden, -1 where all of them are hidden, 2 where the same is added to all, else 0
    __device__ __forceinline__ int alike(int dt) const
    {
        uint32_t all = ~0u, any = 0;
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
            all &= w[i];
            any |= w[i];
        }
        const uint32_t one = __builtin_amdgcn_readfirstlane(w[0]);
        if (!__all(all == one && any == one))
            return 0;
        const uint32_t none = SIZE == 1 ? 0 : SIZE == 4 ? 0xFF800000u : dt == F16 ? 0xFC00FC00u : 0xFF80FF80u, whole = SIZE == 1 ? 0x01010101u : 0;
        return one == whole ? 1 : one == none ? -1 : SIZE == 4 || (SIZE == 2 && one >> 16 == (one & 0xFFFFu)) ? 2 : 0;
    }
    __device__ __forceinline__ void exchange()
    {
#pragma unroll
        for (int i = 0; i < 2 * KB; i++)
#pragma unroll
            for (int e = 0; e < SIZE; e++) {
                const u2v r = __builtin_amdgcn_permlane32_swap(w[i * 2 * SIZE + e], w[i * 2 * SIZE + SIZE + e], false, false);
                w[i * 2 * SIZE + e] = r.x;
                w[i * 2 * SIZE + SIZE + e] = r.y;
            }
    }
    // of score e of the lane, after the exchange: what is added, or whether the key is looked at
    template <int E> __device__ __forceinline__ float of(int dt) const
    {
        constexpr int G = E >> 2, AT = G < 2 * KB ? G * 2 * SIZE : (G - 2 * KB) * 2 * SIZE + SIZE;
        if constexpr (SIZE == 1) {
            return w[AT] & 0xFFu << 8 * (E & 3) ? 1.0f : 0.0f;
        } else if constexpr (SIZE == 4) {
            return __uint_as_float(w[AT + (E & 3)]);
        } else {
            const uint32_t u = w[AT + (E >> 1 & 1)], half = E & 1 ? u >> 16 : u & 0xFFFFu;
            return dt == BF16 ? __uint_as_float(half << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)half);
        }
    }
};

constexpr float LOWEST = -3.0e38f; // of scores, in powers of two

// Score s of a key to which x is added, c being the scaling, all in powers of two.  A type's lowest value times log2(e) would be -inf, which stands for
// hidden keys only: rows of nothing but lowest values look at all of them alike.
__device__ __forceinline__ float with(float s, float x, float c)
{
    const float y = __builtin_fmaf(x, LOG2E, s * c);
    return x == -INFINITY ? -INFINITY : y < LOWEST ? LOWEST : y; // what is no number stays that
}

// A wave's 32 rows; MASK: bytes of a key's mask, 0 without one
template <int TYPE, int CH, int MASK>
struct Wave {
    using Hf = Half<TYPE>;
    static constexpr int DP = room(CH), STEPS = CH / 16, CB = CH / 32;
    u4v q[STEPS];
    f16v o[CB];
    float m, l;      // of row lane % 32: reference, in powers of two; this half's sum
    int row;         // of the sequence
    int limit;       // keys that it looks at
    int low, high;   // least and most of the wave's rows
    const char *mask;
    float c;
    int lane;
    uint32_t key_at[STEPS], value_at[STEPS]; // in a tile: of key lane % 32, and of the four tokens and channels of a transposing read

    __device__ __forceinline__ void open(const Args &a, const Job &j, int first, int lane_)
    {
        lane = lane_;
        const int r32 = lane & 31, half = lane >> 5, i16 = lane & 15;
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
            key_at[i] = r32 * (DP * 2) + ((2 * i + half) ^ turn<DP>(r32)) * 16;
            const int of = 8 * (i & 1) + 4 * half + (i16 >> 2), piece = (i >> 1) * 4 + (lane >> 4 & 1) * 2 + (i16 >> 1 & 1);
            value_at[i] = of * (DP * 2) + (piece ^ turn<DP>(of)) * 16 + (i16 & 1) * 8;
        }
        row = first + (lane & 31);
        const int r = min(row, j.rows - 1), t = token(a, r), head = j.h * a.g + r - t * a.g;
        limit = j.m - j.n + t + 1;
        low = j.m - j.n + token(a, min(first, j.rows - 1)) + 1;
        high = first < j.rows ? j.m - j.n + token(a, min(first + ROWS, j.rows) - 1) + 1 : 0;
        low = __builtin_amdgcn_readfirstlane(low);
        high = __builtin_amdgcn_readfirstlane(high);
        const char *src = a.q.p + j.b * a.q.sb + head * a.q.sh + (long)(j.q0 + t) * a.q.st;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int piece = min(2 * s + half, a.D / 8 - 1); // channels behind the last are zeros in the keys
            q[s] = *(const GLOBAL u4v *)(src + piece * 16);
        }
        if (a.scaling < 0.0f)
#pragma unroll
            for (int s = 0; s < STEPS; s++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    q[s][e] ^= 0x80008000u;
        c = fabsf(a.scaling) * LOG2E;
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int cb = 0; cb < CB; cb++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                o[cb][e] = 0.0f;
        if constexpr (MASK != 0)
            mask = a.mask + (j.b * a.m_sb + head * a.m_sh + (long)t * a.m_st) * MASK;
    }

    // q . k of KB * 32 keys in the LDS
    template <int KB> __device__ __forceinline__ void scores(uint32_t keys, f16v *sc) const
    {
#pragma unroll
        for (int kb = 0; kb < KB; kb++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                sc[kb][e] = 0.0f;
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
                sc[kb] = Hf::mfma(*shared<u4v>(key_at[s] + keys + kb * 32 * (DP * 2)), q[s], sc[kb]);
    }

    // What keys k.. are hidden behind a row's own, and the row's reference, which goes along with its sum and outputs; unit: of the scores x, more: added to them
    template <int KB> __device__ __forceinline__ void settle(float *x, int k, float unit, float more = 0.0f)
    {
        if (k + KB * 32 > low) {
            int left = limit - k - 4 * (lane >> 5);
            asm volatile("" : "+v"(left)); // a branch, not two operations more for every score of every tile
#pragma unroll
            for (int e = 0; e < KB * 16; e++)
                x[e] = (e >> 2) * 8 + (e & 3) < left ? x[e] : -INFINITY;
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < KB * 16; e++)
            top = fmaxf(top, x[e]);
        top = MASK > 1 ? __builtin_fmaf(top, unit, more) : top * unit;
        if (__any(top > m + SLACK)) {
            const float to = fmaxf(m, other_half(top, true));
            const float shrink = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= shrink;
#pragma unroll
            for (int cb = 0; cb < CB; cb++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    o[cb][e] *= shrink;
        }
    }

    template <int KB> __device__ __forceinline__ void weights(const float *x, float unit, uint32_t *w, float more = 0.0f)
    {
        const float ref = m == -INFINITY ? 0.0f : MASK > 1 ? m - Hf::BIAS - more : m - Hf::BIAS; // nothing yet: all weights are zero
#pragma unroll
        for (int e = 0; e < KB * 16; e += 2) {
            w[e >> 1] = Hf::pack(__builtin_amdgcn_exp2f(__builtin_fmaf(x[e], unit, -ref)), __builtin_amdgcn_exp2f(__builtin_fmaf(x[e + 1], unit, -ref)));
            l = Hf::add(w[e >> 1], l);
        }
    }

    template <int KB> __device__ __forceinline__ void outputs(uint32_t values, const uint32_t *w)
    {
#pragma unroll
        for (int kk = 0; kk < KB * 2; kk++) {
            const u4v p = {w[kk * 4], w[kk * 4 + 1], w[kk * 4 + 2], w[kk * 4 + 3]};
#pragma unroll
            for (int cb = 0; cb < CB; cb++) {
                u2v half[2];
#pragma unroll
                for (int d = 0; d < 2; d++)
                    half[d] = __builtin_bit_cast(u2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16(shared<s4v>(value_at[cb * 2 + d] + values + kk * 16 * (DP * 2))));
                o[cb] = Hf::mfma((u4v){half[0].x, half[0].y, half[1].x, half[1].y}, p, o[cb]);
            }
        }
    }

    // KB * 32 keys from k on, keys and values in the LDS
    template <int KB>
    __device__ __forceinline__ void tile(const Args &a, uint32_t keys, uint32_t values, int k, Mask<MASK ? MASK : 1, KB> &masked)
    {
        if (MASK != 0)
            masked.align();
        int all = MASK != 0 ? masked.alike(a.mask_dt) : 1;
        if (MASK != 0 && all < 0)
            return; // nothing to look at
        f16v sc[KB];
        scores<KB>(keys, sc);
        float x[KB * 16];
#pragma unroll
        for (int e = 0; e < KB * 16; e++)
            x[e] = sc[e >> 4][e & 15];
        float unit = c, more = 0.0f; // of x; with something added they are in powers of two
        if (MASK > 1 && all == 2) {
            // The same for all keys, a type's lowest value in front of a padded text: added to the reference, not to every score.  Where it would leave little
            // or nothing of the scores they are rounded one by one, as beside other masks, so that a row's keys are alike whatever tile they are in; where
            // with() makes the same of all of them the scores are next to nothing.
            more = masked.template of<0>(a.mask_dt) * LOG2E;
            if (more < LOWEST) {
                more = LOWEST;
                unit = 1e-30f;
            } else if (!(fabsf(more) < 131072.0f)) {
                more = 0.0f;
                all = 0;
            }
        }
        if constexpr (MASK != 0) {
            if (all == 0) {
                masked.exchange();
                if (MASK != 1)
                    unit = 1.0f;
                adkv::static_for<KB * 16>([&](auto i) {
                    constexpr int E = decltype(i)::value;
                    const float y = masked.template of<E>(a.mask_dt);
                    x[E] = MASK == 1 ? (y != 0.0f ? x[E] : -INFINITY) : with(x[E], y, c);
                });
            }
        }
        settle<KB>(x, k, unit, more);
        uint32_t w[KB * 8];
        weights<KB>(x, unit, w, more);
        outputs<KB>(values, w);
    }

    // 32 keys whose scores are there already, beside the scores of the next 32, which are put into `next`
    __device__ __forceinline__ void beside(const f16v *sc, f16v *next, uint32_t values, int k, uint32_t next_keys)
    {
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; e++)
            x[e] = sc[0][e];
        settle<1>(x, k, c);
        scores<1>(next_keys, next);
        uint32_t w[8];
        weights<1>(x, c, w);
        outputs<1>(values, w);
    }

    // whether a product's result, or the sum, is infinite or no number, or nothing is left of a row that looks at something: references of 2^30 and more are
    // rounded by what leaves no weight of the largest score
    __device__ __forceinline__ bool strange() const
    {
        const bool lost = other_half(l, false) == 0.0f && m > -INFINITY;
        float nothing[4] = {l * 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int cb = 0; cb < CB; cb++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                nothing[e & 3] = __builtin_fmaf(o[cb][e], 0.0f, nothing[e & 3]);
        return __any(lost || (nothing[0] + nothing[1]) + (nothing[2] + nothing[3]) != 0.0f);
    }

    // To the output, 16 bytes at a time: two lanes have four channels each of the same eight of a row; an exchange leaves one of them with these and
    // the other with the next eight.
    __device__ __forceinline__ void deliver(const Args &a, const Job &j)
    {
        const float sum = other_half(l, false), inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int t = token(a, row), head = j.h * a.g + row - t * a.g, half = lane >> 5;
        char *to = a.out + (((long)j.b * a.Tq + j.q0 + t) * (a.H * a.g) + head) * (a.D * 2) + half * 16;
        if (row >= j.rows)
            return;
#pragma unroll
        for (int cb = 0; cb < CB; cb++)
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
                uint32_t u[4];
#pragma unroll
                for (int i = 0; i < 4; i++)
                    u[i] = Hf::pack(o[cb][e + 2 * i] * inv, o[cb][e + 2 * i + 1] * inv);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const u2v r = __builtin_amdgcn_permlane32_swap(u[i], u[2 + i], false, false);
                    u[i] = r.x;
                    u[2 + i] = r.y;
                }
                if (cb * 32 + e * 2 + half * 8 < a.D)
                    *(GLOBAL u4v *)(to + (cb * 32 + e * 2) * 2) = (u4v){u[0], u[1], u[2], u[3]};
            }
    }

    // To the LDS: 32 rows of DP sums, in pieces of four at place piece ^ row, then the rows' m and l
    __device__ __forceinline__ void leave(uint32_t to)
    {
        const int r32 = lane & 31, h = lane >> 5;
        const float sum = other_half(l, false);
#pragma unroll
        for (int cb = 0; cb < CB; cb++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int piece = cb * 8 + (e >> 2) * 2 + h;
                *shared<f4v>(to + (r32 * (DP / 4) + (piece ^ (r32 & 15))) * 16) = (f4v){o[cb][e], o[cb][e + 1], o[cb][e + 2], o[cb][e + 3]};
            }
        if (h == 0)
            *shared<f2v>(to + ROWS * DP * 4 + r32 * 8) = (f2v){m, sum};
    }
};

constexpr int result_bytes(int DP) { return ROWS * DP * 4 + ROWS * 8; }

// The same as tile() and leave() for keys k0..k1, a row after the other and without a look at what is hidden: a hidden value that is infinite or not a
// number meets a weight of zero in a matrix product, and leaves nothing of the row.  Taken where a product's results are no numbers.
// WHOLE: all keys, straight to the output; else WIDTH keys of every STEP
template <int TYPE, int DP, int MASK, bool WHOLE, int WIDTH = 64, int STEP = 64>
__device__ __forceinline__ void carefully(const Args &a, const Job &j, int first, int k0, int k1, int lane, uint32_t to)
{
    using Hf = Half<TYPE>;
    constexpr int N = DP / 64;
    const float c = a.scaling * LOG2E;
#pragma unroll 1
    for (int i = 0; i < ROWS; i++) {
        float o[N], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int n = 0; n < N; n++)
            o[n] = 0.0f;
        const int r = min(first + i, j.rows - 1), t = token(a, r), head = j.h * a.g + r - t * a.g;
        const int end = min(k1, j.m - j.n + t + 1);
        const char *q = a.q.p + j.b * a.q.sb + head * a.q.sh + (long)(j.q0 + t) * a.q.st;
#pragma unroll 1
        for (int k = k0; k < end; k += STEP) {
            const int key = k + lane;
            float x = -INFINITY;
            if (lane < WIDTH && key < end) {
                const char *kp = a.k.p + j.b * a.k.sb + j.h * a.k.sh + (long)(j.k0 + key) * a.k.st;
                float s = 0.0f;
#pragma unroll 1
                for (int d = 0; d < a.D; d += 8) {
                    const u4v x8 = *(const GLOBAL u4v *)(q + d * 2), y8 = *(const GLOBAL u4v *)(kp + d * 2);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        s = __builtin_fmaf(Hf::number((uint16_t)(x8[e >> 1] >> (e & 1) * 16)), Hf::number((uint16_t)(y8[e >> 1] >> (e & 1) * 16)), s);
                }
                x = s * c;
                if constexpr (MASK != 0) {
                    const GLOBAL char *mp = (const GLOBAL char *)(a.mask + (j.b * a.m_sb + head * a.m_sh + (long)t * a.m_st + key) * MASK);
                    if constexpr (MASK == 1)
                        x = *mp ? x : -INFINITY;
                    else if constexpr (MASK == 4)
                        x = with(s, *(const GLOBAL float *)mp, c);
                    else
                        x = with(s, a.mask_dt == BF16 ? Half<BF16>::number(*(const GLOBAL uint16_t *)mp) : Half<F16>::number(*(const GLOBAL uint16_t *)mp), c);
                }
            }
            const uint64_t seen = __ballot(!(x == -INFINITY));
            float top = x;
            for (int d = 32; d; d >>= 1)
                top = fmaxf(top, __shfl_xor(top, d));
            const float now = fmaxf(m, top), shrink = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - now);
            m = now;
            const float ref = m == -INFINITY ? 0.0f : m - Hf::BIAS, p = x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x - ref);
            float sum = p;
            for (int d = 32; d; d >>= 1)
                sum += __shfl_xor(sum, d);
            l = l * shrink + sum;
#pragma unroll
            for (int n = 0; n < N; n++)
                o[n] *= shrink;
#pragma unroll 8
            for (int e = 0; e < WIDTH; e++) {
                const bool look = seen >> e & 1;
                const float w = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(p), e));
                const char *vp = a.v.p + j.b * a.v.sb + j.h * a.v.sh + (long)(j.k0 + min(k + e, end - 1)) * a.v.st;
#pragma unroll
                for (int n = 0; n < N; n++) {
                    const float y = Hf::number(((const GLOBAL uint16_t *)vp)[min(lane * N + n, a.D - 1)]);
                    o[n] = look ? __builtin_fmaf(w, y, o[n]) : o[n];
                }
            }
        }
        if (WHOLE) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            GLOBAL uint16_t *out = (GLOBAL uint16_t *)a.out + (((long)j.b * a.Tq + j.q0 + t) * (a.H * a.g) + head) * a.D;
#pragma unroll
            for (int n = 0; n < N; n++)
                if (first + i < j.rows && lane * N + n < a.D)
                    out[lane * N + n] = (uint16_t)Hf::pack(o[n] * inv, 0.0f);
            continue;
        }
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int d = lane * N + n;
            *shared<float>(to + (i * (DP / 4) + ((d >> 2) ^ (i & 15))) * 16 + (d & 3) * 4) = o[n];
        }
        if (lane == 0)
            *shared<f2v>(to + ROWS * DP * 4 + i * 8) = (f2v){m, l};
    }
}

// Rows first.. first + n of what is left in the LDS by `from` waves for the same rows, joined and written; lanes take four channels each
template <int TYPE, int DP, int FROM>
__device__ __forceinline__ void deliver(const Args &a, const Job &j, uint32_t at, int row0, int first, int n, int lane)
{
    using Hf = Half<TYPE>;
    constexpr int LANES = DP / 4, EACH = 64 / LANES;
    const int piece = lane % LANES;
    for (int i = first + lane / LANES; i < first + n; i += EACH) {
        if (row0 + i >= j.rows)
            break;
        float M = -INFINITY, L = 0.0f;
        f2v ml[FROM];
#pragma unroll
        for (int w = 0; w < FROM; w++) {
            ml[w] = *shared<f2v>(at + w * result_bytes(DP) + ROWS * DP * 4 + i * 8);
            M = fmaxf(M, ml[w].x);
        }
        const float ref = M == -INFINITY ? 0.0f : M;
        f4v o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < FROM; w++) {
            const f4v v = *shared<f4v>(at + w * result_bytes(DP) + (i * (DP / 4) + (piece ^ (i & 15))) * 16);
            const float e = __builtin_amdgcn_exp2f(ml[w].x - ref);
            L = __builtin_fmaf(ml[w].y, e, L);
#pragma unroll
            for (int k = 0; k < 4; k++)
                o[k] = __builtin_fmaf(v[k], e, o[k]);
        }
        if (piece * 4 >= a.D)
            continue;
        const int t = token(a, row0 + i), head = j.h * a.g + row0 + i - t * a.g;
        const long r = ((long)j.b * a.Tq + j.q0 + t) * (a.H * a.g) + head;
        if (a.pieces > 1) {
            if (piece == 0)
                *(GLOBAL f2v *)(a.ml + j.piece * a.all + r) = (f2v){M, L};
            *(GLOBAL f4v *)(a.partial + (j.piece * a.all + r) * a.D + piece * 4) = o;
            continue;
        }
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        *(GLOBAL u2v *)(a.out + (r * a.D + piece * 4) * 2) = (u2v){Hf::pack(o[0] * inv, o[1] * inv), Hf::pack(o[2] * inv, o[3] * inv)};
    }
}

// All that was asked for is there, for the compiler too: what it does not know to be there it waits for at its first use, and with it for all that
// load_to_lds() has been told since.
__device__ __forceinline__ void arrive() { __builtin_amdgcn_s_waitcnt(0x0F70); } // vmcnt(0)

template <int DP> constexpr int many_lds() { return 2 * 64 * DP * 2 * 2; }

template <int TYPE, int CH, int MASK>
__global__ __launch_bounds__(NT, CH > 128 ? 1 : 2) void many_kernel(const Args a)
{
    constexpr int DP = room(CH);
    __shared__ uint4 smem[many_lds<DP>() / 16];
    const uint32_t lds = (uint32_t)(uintptr_t)(LDS char *)(char *)smem;
    constexpr int TILE = 64, BYTES = TILE * DP * 2, EACH = TILE / WAVES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    Job j;
    if (!place<WAVES * ROWS>(a, blockIdx.x, lane, j))
        return;
    const int first = j.first + wave * ROWS;
    Wave<TYPE, CH, MASK> w;
    const char *kp = a.k.p + j.b * a.k.sb + j.h * a.k.sh + (long)j.k0 * a.k.st, *vp = a.v.p + j.b * a.v.sb + j.h * a.v.sh + (long)j.k0 * a.v.st;
    Stream<DP> keys, values;
    values.open(vp, a.v.st, wave * EACH, j.end);
    const uint32_t mine = lds + wave * EACH * DP * 2;
    if constexpr (MASK == 0) {
        // The weights of 32 keys are made beside the products of the next 32 keys' scores, so that keys are half a tile ahead of the values: tile k / 64
        // of them in the LDS begins with key k + 32.  (16384 tokens, 32 heads of 128: a tile's scores, weights and outputs one after the other take 7 % longer.)
        f16v even[1], odd[1];
        if (j.end > 0) {
            // the first 32, where the second tile of keys will be
            if (wave < 2) {
                keys.open(kp, a.k.st, wave * EACH, j.end);
                keys.template ask<EACH>(mine + BYTES, lane, a.D);
            }
            keys.open(kp, a.k.st, 32 + wave * EACH, j.end);
            keys.template ask<EACH>(mine, lane, a.D);
            values.template ask<EACH>(mine + 2 * BYTES, lane, a.D);
        }
        w.open(a, j, first, lane); // behind the loads of the tiles: all are on their way together
        arrive();
        if (j.end > 0) {
            asm volatile("s_barrier" ::: "memory");
            if (w.high > 0)
                w.template scores<1>(lds + BYTES, even);
        }
        const auto step = [&](int k, auto parity) __attribute__((always_inline)) {
            constexpr uint32_t NEXT = decltype(parity)::value * BYTES, OTHER = BYTES - NEXT, V = NEXT + 2 * BYTES, HALF = BYTES / 2;
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); // this tile is there, and nobody reads the one in front of it
            if (k + TILE < j.end) {
                keys.skip(TILE);
                values.skip(TILE);
                keys.template ask<EACH>(mine + OTHER, lane, a.D);
                values.template ask<EACH>(mine + OTHER + 2 * BYTES, lane, a.D);
            }
            if (k < w.high) { // behind the last of its keys a wave makes scores that nobody looks at
                w.beside(even, odd, lds + V, k, lds + NEXT);
                w.beside(odd, even, lds + V + HALF, k + 32, lds + NEXT + HALF);
            }
        };
        for (int k = 0; k < j.end; k += 2 * TILE) { // where the LDS is read is part of the instructions
            step(k, std::integral_constant<int, 0>{});
            if (k + TILE < j.end)
                step(k + TILE, std::integral_constant<int, 1>{});
        }
    } else {
        Mask<MASK ? MASK : 1, 2> masked, next;
        keys.open(kp, a.k.st, wave * EACH, j.end);
        if (j.end > 0) {
            keys.template ask<EACH>(mine, lane, a.D);
            values.template ask<EACH>(mine + BYTES, lane, a.D);
        }
        w.open(a, j, first, lane);
        if (0 < w.high)
            next.load(a, w.mask, 0, lane);
        int buffer = 0;
        for (int k = 0; k < j.end; k += TILE) {
            arrive();
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); // the tile is there, and nobody reads the one before it any more
            masked = next;
            if (k + TILE < w.high)
                next.load(a, w.mask, k + TILE, lane);
            if (k + TILE < j.end) {
                keys.skip(TILE);
                values.skip(TILE);
                keys.template ask<EACH>(mine + (buffer ^ 1) * 2 * BYTES, lane, a.D);
                values.template ask<EACH>(mine + (buffer ^ 1) * 2 * BYTES + BYTES, lane, a.D);
            }
            if (k < w.high)
                w.template tile<2>(a, lds + buffer * 2 * BYTES, lds + buffer * 2 * BYTES + BYTES, k, masked);
            buffer ^= 1;
        }
    }
    arrive();
    if (w.strange())
        carefully<TYPE, DP, MASK, true>(a, j, first, 0, j.end, lane, 0);
    else
        w.deliver(a, j);
}

constexpr int PARTS = 4; // of the keys
template <int DP> constexpr int some_lds() { return std::max(2 * PARTS * 32 * DP * 2 * 2, 2 * PARTS * result_bytes(DP)); }

template <int TYPE, int CH, int MASK>
__global__ __launch_bounds__(2 * NT, 1) void some_kernel(const Args a)
{
    constexpr int DP = room(CH);
    __shared__ uint4 smem[some_lds<DP>() / 16];
    const uint32_t lds = (uint32_t)(uintptr_t)(LDS char *)(char *)smem;
    constexpr int TILE = PARTS * 32, BYTES = TILE * DP * 2, EACH = 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), part = wave % PARTS, rows = wave / PARTS;
    Job j;
    if (!place<2 * ROWS>(a, blockIdx.x, lane, j))
        return;
    const int first = j.first + rows * ROWS;
    Wave<TYPE, CH, MASK> w;
    Stream<DP> keys, values;
    keys.open(a.k.p + j.b * a.k.sb + j.h * a.k.sh + (long)j.k0 * a.k.st, a.k.st, wave * EACH, j.end);
    values.open(a.v.p + j.b * a.v.sb + j.h * a.v.sh + (long)j.k0 * a.v.st, a.v.st, wave * EACH, j.end);
    const uint32_t mine = lds + wave * EACH * DP * 2;
    Mask<MASK ? MASK : 1, 1> masked, next;
    if (j.end > 0) {
        keys.template ask<EACH>(mine, lane, a.D);
        values.template ask<EACH>(mine + BYTES, lane, a.D);
    }
    w.open(a, j, first, lane);
    if (MASK != 0 && part * 32 < w.high)
        next.load(a, w.mask, part * 32, lane);
    int buffer = 0;
    for (int k = part * 32; k - part * 32 < j.end; k += TILE) {
        arrive();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); // the tile is there, and nobody reads the one before it any more
        if (MASK != 0) {
            masked = next;
            if (k + TILE < w.high)
                next.load(a, w.mask, k + TILE, lane);
        }
        if (k - part * 32 + TILE < j.end) {
            keys.skip(TILE);
            values.skip(TILE);
            keys.template ask<EACH>(mine + (buffer ^ 1) * 2 * BYTES, lane, a.D);
            values.template ask<EACH>(mine + (buffer ^ 1) * 2 * BYTES + BYTES, lane, a.D);
        }
        if (k < w.high) {
            const uint32_t at = lds + buffer * 2 * BYTES + part * 32 * DP * 2;
            w.template tile<1>(a, at, at + BYTES, k, masked);
        }
        buffer ^= 1;
    }
    arrive();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); // the tiles' place is free
    const uint32_t result = lds + wave * result_bytes(DP);
    if (w.strange())
        carefully<TYPE, DP, MASK, false, 32, TILE>(a, j, first, part * 32, j.end, lane, result);
    else
        w.leave(result);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    deliver<TYPE, DP, PARTS>(a, j, lds + rows * PARTS * result_bytes(DP), first, part * (ROWS / PARTS), ROWS / PARTS, lane);
}

template <int DP> constexpr int few_stages() { return DP > 128 ? 1 : 2; }
template <int DP> constexpr int few_lds() { return std::max(WAVES * few_stages<DP>() * 32 * DP * 2 * 2, WAVES * result_bytes(DP)); }

template <int TYPE, int CH, int MASK>
__global__ __launch_bounds__(NT, 1) void few_kernel(const Args a)
{
    constexpr int DP = room(CH);
    __shared__ uint4 smem[few_lds<DP>() / 16];
    const uint32_t lds = (uint32_t)(uintptr_t)(LDS char *)(char *)smem;
    constexpr int TILE = 32, BYTES = TILE * DP * 2, STAGES = few_stages<DP>();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    Job j;
    if (!place<ROWS>(a, blockIdx.x, lane, j))
        return;
    Wave<TYPE, CH, MASK> w;
    const int tiles = (j.end + TILE - 1) / TILE, parts = a.pieces * WAVES, part = j.piece * WAVES + wave;
    const int k0 = (int)((int64_t)tiles * part / parts) * TILE, k1 = min((int)((int64_t)tiles * (part + 1) / parts) * TILE, j.end);
    Stream<DP> keys, values;
    keys.open(a.k.p + j.b * a.k.sb + j.h * a.k.sh + (long)j.k0 * a.k.st, a.k.st, k0, j.end);
    values.open(a.v.p + j.b * a.v.sb + j.h * a.v.sh + (long)j.k0 * a.v.st, a.v.st, k0, j.end);
    const uint32_t own = lds + wave * (STAGES * 2 * BYTES);
    const auto ask = [&](uint32_t to) __attribute__((always_inline)) {
        int l = lane;
        if (DP > 128 && MASK != 0)
            asm volatile("" : "+v"(l)); // 32 addresses in a tile are made again for every tile: there is no room to keep them
        keys.template ask<TILE>(to, l, a.D);
        values.template ask<TILE>(to + BYTES, l, a.D);
        keys.skip(TILE);
        values.skip(TILE);
    };
    Mask<MASK ? MASK : 1, 1> masked, next;
    if (k0 < k1)
        ask(own);
    w.open(a, j, j.first, lane);
    if (MASK != 0 && k0 < k1)
        next.load(a, w.mask, k0, lane);
    int stage = 0;
    for (int k = k0; k < k1; k += TILE) {
        arrive();
        if (MASK != 0) {
            masked = next;
            if (k + TILE < k1)
                next.load(a, w.mask, k + TILE, lane);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // what was read of the tile that is overwritten now
        if (STAGES > 1 && k + TILE < k1)
            ask(own + (stage ^ 1) * 2 * BYTES);
        w.template tile<1>(a, own + stage * 2 * BYTES, own + stage * 2 * BYTES + BYTES, k, masked);
        if (STAGES > 1) {
            stage ^= 1;
        } else if (k + TILE < k1) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            ask(own);
        }
    }
    arrive();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const uint32_t mine = lds + wave * result_bytes(DP);
    if (w.strange())
        carefully<TYPE, DP, MASK, false>(a, j, j.first, k0, k1, lane, mine);
    else
        w.leave(mine);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    deliver<TYPE, DP, WAVES>(a, j, lds, j.first, wave * (ROWS / WAVES), ROWS / WAVES, lane);
}

// Pieces of a row to its output, four channels per lane
template <int TYPE>
__global__ __launch_bounds__(256) void join_kernel(const Args a)
{
    const int lanes = a.D / 4;
    const long i = (long)blockIdx.x * 256 + threadIdx.x, r = i / lanes;
    const int piece = (int)(i - r * lanes);
    if (r >= a.all)
        return;
    constexpr int EACH = 8; // loads on their way together
    float M = -INFINITY, L = 0.0f;
    f4v o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p0 = 0; p0 < a.pieces; p0 += EACH) {
        f2v ml[EACH];
        f4v v[EACH];
        float top = M;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const int p = min(p0 + i, a.pieces - 1);
            ml[i] = *(const GLOBAL f2v *)(a.ml + p * a.all + r);
            v[i] = *(const GLOBAL f4v *)(a.partial + (p * a.all + r) * a.D + piece * 4);
        }
#pragma unroll
        for (int i = 0; i < EACH; i++)
            top = fmaxf(top, ml[i].x);
        if (top == -INFINITY)
            continue; // nothing yet
        const float shrink = __builtin_amdgcn_exp2f(M - top);
        M = top;
        L *= shrink;
#pragma unroll
        for (int k = 0; k < 4; k++)
            o[k] *= shrink;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const float e = p0 + i < a.pieces ? __builtin_amdgcn_exp2f(ml[i].x - M) : 0.0f;
            L = __builtin_fmaf(ml[i].y, e, L);
#pragma unroll
            for (int k = 0; k < 4; k++)
                o[k] = __builtin_fmaf(v[i][k], e, o[k]);
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    *(GLOBAL u2v *)(a.out + (r * a.D + piece * 4) * 2) = (u2v){Half<TYPE>::pack(o[0] * inv, o[1] * inv), Half<TYPE>::pack(o[2] * inv, o[3] * inv)};
}

// ------------------------------------------------------------------------------------------------------------------------- host

enum { MANY_ROWS = WAVES * ROWS, SOME_ROWS = 2 * ROWS, FEW_ROWS = ROWS };
struct Plan {
    int rows; // of a workgroup: the form
    int blocks, units, together, pieces;
};

static Plan plan(int B, int Hq, int H, int Tq, int Tk, int D, int n_seq)
{
    const int g = Hq / H, cus = std::max(1, cu_count());
    const int64_t rows = (int64_t)Tq * g;
    Plan p;
    p.units = n_seq ? H : B * H;
    const auto blocks = [&](int each) { return (int)(n_seq ? rows / each + n_seq + 2 : (rows + each - 1) / each); };
    // Where 128 rows at a time leave CUs without work, or with the longest rows alone at the end, more waves share a row's keys.  Workgroups of the forms
    // for that have a CU to themselves, or share it with one more (64 channels), and two rounds of them still pay where a unit has long rows beside short
    // ones.  us of many, some, few, bf16, channels: units x tokens
    //    64: 16 x 512  10.5, 8.1, 7.3     32 x 512  10.7, 8.4, 8.1     32 x 1024  18, 14, 18     16 x 4096  60, 57, 76     64 x 1024  20, 24, 32
    //   128: 16 x 512  13.5, 11.8, 10.2    32 x 512  14.0, 12.4, 16.2   16 x 1024  22, 17, 20     16 x 2048  40, 34, 53     64 x 512   16, 20, 30
    //   256 (some do not fit): 16 x 512  27, 17      32 x 512  28, 27      16 x 1024  46, 35     64 x 256  18, 22     32 x 1024  48, 66
    const int64_t slots = D > 64 ? cus : 2ll * cus;
    const auto fits = [&](int each, int length) { // once, or twice with so many blocks of a sequence
        const int64_t all = (int64_t)p.units * blocks(each);
        return all <= slots || (all <= 2 * slots && blocks(each) >= (int64_t)length * std::max(1, n_seq));
    };
    // A tile of keys leaves nothing to share: 64 tokens of 128 channels 5.8, 8.0, 6.6 us.
    p.rows = Tk <= 64 && D <= 128 ? MANY_ROWS : fits(FEW_ROWS, D > 128 ? 16 : INT32_MAX) ? FEW_ROWS : D <= 128 && fits(SOME_ROWS, 32) ? SOME_ROWS : MANY_ROWS;
    p.blocks = blocks(p.rows);
    p.pieces = 1;
    p.together = p.units;
    if (p.rows == MANY_ROWS) {
        // Many blocks: as many units at a time as fill the device once, so that their blocks find their keys in the XCDs' caches (us with that many, twice
        // and four times as many, bf16: 128 sequences of 512 tokens, 32 heads 555, 590, 635; 64 of 300, eight heads of four queries 122, 128, 126; 101 of 278,
        // 16 heads 120, 131, 141).  Else all of them, the longest first everywhere.
        if ((int64_t)p.units * p.blocks > 8ll * cus)
            p.together = (int)std::min<int64_t>(p.units, (cus / p.blocks + 8) / 8 * 8);
    } else if (p.rows == FEW_ROWS) {
        const int64_t wide = (int64_t)p.units * p.blocks, tiles = (Tk + 31) / 32;
        // two tiles a wave at least, and none for few keys (us, 8 units of 128 channels: 512 tokens in two pieces 12.5, in one 9.8; a token behind 1000 in
        // four 9.4, in two 11.4)
        p.pieces = tiles < 24 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(cus / wide, tiles / (2 * WAVES)));
    }
    return p;
}

static int checked(int B, int Hq, int H, int Tq, int Tk, int D, int n_seq)
{
    if (B <= 0 || Hq <= 0 || H <= 0 || Tq <= 0 || Tk < Tq || n_seq < 0 || Hq % H)
        return ADKV_E_SHAPE;
    if (n_seq && (B != 1 || Tq != Tk))
        return ADKV_E_SHAPE;
    if (D <= 0 || D > 256 || D % 8)
        return ADKV_E_DIM;
    const int64_t g = Hq / H;
    // rows are counted in 31 bits and divided by g in 32; a grid is 2^32 threads at most.  The first line keeps the products below 2^63.
    if (g > 46340 || (int64_t)B * H >= 1 << 24 || (int64_t)B * Tq > INT32_MAX)
        return ADKV_E_SHAPE;
    if (Tq * g * g > INT32_MAX || Tk > INT32_MAX - 256 || (Tq * g / ROWS + n_seq + 3) * B * H > (1 << 24) - 1 || (int64_t)B * Tq * Hq > INT32_MAX)
        return ADKV_E_SHAPE;
    return ADKV_OK;
}

template <int TYPE, int CH, int MASK> static auto form_of(int rows)
{
    if constexpr (CH <= 128)
        if (rows == SOME_ROWS)
            return some_kernel<TYPE, CH, MASK>;
    return rows == MANY_ROWS ? many_kernel<TYPE, CH, MASK> : few_kernel<TYPE, CH, MASK>;
}
template <int TYPE, int MASK> static auto kernel_of(int D, int rows)
{
    return D > 128 ? form_of<TYPE, 256, MASK>(rows) : D > 96 ? form_of<TYPE, 128, MASK>(rows) : D > 64 ? form_of<TYPE, 96, MASK>(rows) : form_of<TYPE, 64, MASK>(rows);
}

} // namespace adkv_prompt

extern "C" int64_t adkv_prompt_attention_workspace_bytes(int B, int Hq, int H, int Tq, int Tk, int D, int n_seq)
{
    using namespace adkv_prompt;
    if (int rc = checked(B, Hq, H, Tq, Tk, D, n_seq))
        return rc;
    if (cu_count() <= 0)
        return ADKV_E_DEVICE;
    const Plan p = plan(B, Hq, H, Tq, Tk, D, n_seq);
    return p.pieces > 1 ? (int64_t)p.pieces * B * Tq * Hq * (D * 4 + 8) : 0;
}

extern "C" int adkv_prompt_attention(const void *q, const int64_t *q_strides, const void *k, const int64_t *k_strides, const void *v,
                                     const int64_t *v_strides, const void *mask, const int64_t *mask_strides, float scaling, const int *bounds,
                                     int n_seq, void *out, int B, int Hq, int H, int Tq, int Tk, int D, int dtype, void *workspace,
                                     int64_t workspace_bytes, void *stream)
{
    using namespace adkv_prompt;
    if (!q || !k || !v || !out || !q_strides || !k_strides || !v_strides || (mask && !mask_strides) || (n_seq > 0 && !bounds))
        return ADKV_E_NULL;
    if (int rc = checked(B, Hq, H, Tq, Tk, D, n_seq))
        return rc;
    const int type = dtype & 255, mask_dt = dtype >> 8;
    if ((type != F16 && type != BF16) || mask_dt < 0 || mask_dt > ADKV_DT_BOOL || (mask && n_seq))
        return ADKV_E_UNSUPPORTED;
    uint64_t bits = (uint64_t)q | (uint64_t)k | (uint64_t)v | (uint64_t)out;
    const int64_t *const strides[] = {q_strides, k_strides, v_strides};
    for (const int64_t *s : strides) {
        bits |= (uint64_t)(s[0] | s[1] | s[2]) * 2;
        // tiles of 64 rows are addressed in 31 bits
        if (s[0] < 0 || s[1] < 0 || s[2] < 0 || s[2] * 2 > 0x3FFFFFFF / 64)
            return ADKV_E_SHAPE;
    }
    if (bits & 15)
        return ADKV_E_ALIGN;
    const int size = mask_dt == 0 ? 4 : mask_dt == ADKV_DT_BOOL ? 1 : 2;
    if ((uint64_t)mask & (size - 1))
        return ADKV_E_ALIGN;
    if (cu_count() <= 0)
        return ADKV_E_DEVICE;
    const Plan p = plan(B, Hq, H, Tq, Tk, D, n_seq);
    const int64_t all = (int64_t)B * Tq * Hq, need = p.pieces > 1 ? p.pieces * all * (D * 4 + 8) : 0;
    if (need && (!workspace || workspace_bytes < need))
        return ADKV_E_WORKSPACE;
    if (need && (uint64_t)workspace & 15)
        return ADKV_E_ALIGN;
    Args a = {};
    const auto rows = [](const void *p, const int64_t *s) { return Rows{(const char *)p, (long)s[0] * 2, (long)s[1] * 2, (int)(s[2] * 2)}; };
    a.q = rows(q, q_strides);
    a.k = rows(k, k_strides);
    a.v = rows(v, v_strides);
    a.out = (char *)out;
    a.mask = (const char *)mask;
    if (mask) {
        a.m_sb = mask_strides[0];
        a.m_sh = mask_strides[1];
        a.m_st = mask_strides[2];
        if (a.m_sb < 0 || a.m_sh < 0 || a.m_st < 0)
            return ADKV_E_SHAPE;
        a.mask_end = a.mask + ((B - 1) * a.m_sb + (Hq - 1) * a.m_sh + (Tq - 1) * a.m_st + Tk) * size;
    }
    a.bounds = n_seq ? bounds : nullptr;
    a.partial = (float *)workspace;
    a.ml = (f2v *)((char *)workspace + (int64_t)p.pieces * all * D * 4);
    a.all = all;
    a.B = B;
    a.H = H;
    a.g = Hq / H;
    a.Tq = Tq;
    a.Tk = Tk;
    a.D = D;
    a.n_seq = n_seq;
    a.mask_dt = mask_dt;
    a.pieces = p.pieces;
    a.blocks = p.blocks;
    a.units = p.units;
    a.together = p.together;
    a.scaling = scaling;
    a.by_g = (uint32_t)(((1ull << 32) + a.g - 1) / a.g);
    const int masked = !mask ? 0 : size;
    const auto of = [&](auto type_) {
        constexpr int TYPE = decltype(type_)::value;
        return masked == 0 ? kernel_of<TYPE, 0>(D, p.rows)
            : masked == 1  ? kernel_of<TYPE, 1>(D, p.rows)
            : masked == 2  ? kernel_of<TYPE, 2>(D, p.rows)
                           : kernel_of<TYPE, 4>(D, p.rows);
    };
    const auto kernel = type == F16 ? of(std::integral_constant<int, F16>{}) : of(std::integral_constant<int, BF16>{});
    hipLaunchKernelGGL(kernel, dim3((unsigned)((int64_t)p.blocks * p.units * p.pieces)), dim3(p.rows == SOME_ROWS ? 2 * NT : NT), 0, (hipStream_t)stream, a);
    if (int rc = check_launch())
        return rc;
    if (p.pieces > 1) {
        const auto join = type == F16 ? join_kernel<F16> : join_kernel<BF16>;
        hipLaunchKernelGGL(join, dim3((unsigned)((all * (D / 4) + 255) / 256)), dim3(256), 0, (hipStream_t)stream, a);
        return check_launch();
    }
    return ADKV_OK;
}
