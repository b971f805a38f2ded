// Attention of n new tokens per sequence over codes: a prefix whose codes all sequences share, then each sequence's own codes, the
// new tokens' among them (head dim 128, 4-bit or 2-bit codes, 1, 2, 4 or 8 query heads per KV head).
//
//   x[i, t] = scaling * q_i . K_t + mask[i, t],  t over the P prefix tokens and the own tokens up to the query's;  out_i = sum softmax(x_i)_t V_t
//
// The prefix is replayed once for the batch and multiplied with the queries of all sequences as one matrix, so that its cost does not
// grow with the batch but by matrix instructions.  The context of a KV head is cut into pieces, each of which leaves
// (m, l, o) = (max x, sum e^(x-m), sum e^(x-m) V) per query row; pieces are joined by M = max m, out = sum e^(m-M) o / sum e^(m-M) l.
// Scores, m, l, o are fp32; the weights e^(x-m) are rounded to fp16 for the matrix cores, relative to the largest so far (or to one that
// is at most 2^8 times smaller: see weights()).
//
// Two ways through the codes of a source, by the query rows of a unit (a KV head of the prefix with the rows of the whole batch, or of a
// sequence with its own):
//   at most 16 (few)   attend_kernel: the waves that replay hand tiles of values to waves that multiply, through the LDS
//   more (many)        values_kernel writes the values to memory as tiles of fp16, attend_many_kernel reads them.  Replaying in the multiplying
//                      workgroup takes as many issue slots as the softmax of 256 rows, once per 256 rows, and its LDS; 8 x 512
//                      new tokens on a prefix of 4096, 32 heads, took 1000 us that way, where the two kernels take 530
#include <math.h>

#include <algorithm>

#include "adkv_device.h"

#include "../../include/adkv_hip.h"

#pragma clang fp contract(off)

namespace adkv_ext {
using namespace adkv;

typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));

constexpr int D = 128;
constexpr int PRODUCERS = 4;
// Few rows: tiles of 32 tokens, four waves that replay and four that multiply, two workgroups per CU: a wave that replays alone on its SIMD uses half
// of the issue slots.  Of 64 KB of LDS the code table (half as many copies of its entries as elsewhere) has the first half of every 256 bytes, and two
// buffers of a K and a V tile of 8 KB the second halves.
constexpr int FEW_TILE = 32, FEW_THREADS = 512, FEW_BUFFER = 32768, FEW_VALUES = 16384, FEW_FIRST = 128, FEW_LDS = 65536;
// Many rows: tiles of 64 tokens, 16 KB of keys and as many of values, two of them in the LDS; four waves of up to 32 rows.
constexpr int ALL_READS = 0x0070; // s_waitcnt's operand: all vector loads, all reads of the LDS
constexpr int TILE = 64, TILE_BYTES = 32768, TILE_VALUES = 16384, MANY_WAVES = 4, MANY_ROWS = MANY_WAVES * 32, JOINT_ROWS = 128;
constexpr int MAX_TOKENS = 1 << 24; // 64 bytes each: a piece's codes are addressed in 32 bits
constexpr float LOG2E = 1.44269504088896340736f;

struct Tensor { // K or V of a source
    const uint32_t *codes; // [units, n_super, D]
    const h1 *ckpt;        // [units, n_ckpt, D, 2], or null
    const h1 *zp, *sc, *al, *be, *tg;
};

// Codes: the prefix's, a unit per KV head, or the sequences' own ones, a unit per sequence and KV head.
struct Extent {
    int tokens, n_super, n_ckpt;
    int interval, intervals; // checkpoint intervals; the last goes on to the last token
    int seen;                // tokens that the first of the new tokens looks at; each later one at one more if causal
    int causal;
    int col;                 // where its tokens are in the mask
};
struct Source {
    Tensor t[2];
    Extent x;
};

// x / d by a multiplication with 2^64 / d, rounded up, and a shift: exact for any x and d of 31 bits, as the error is below x * d / 2^64.  (With 32
// bits x * d has to be below 2^32, which 65536 new tokens of one sequence are not.)
struct Div {
    uint32_t d, lo, hi;
};

// Query rows and the sources that they look at.  Group 0 has the rows (sequence, token, query head of the group) of a KV head and
// looks at the prefix; group 1 has the rows (token, query head) of a sequence and KV head and looks at its own codes, behind the prefix
// if `joint`.  Its items: a block of rows with one piece of the checkpoint intervals.
struct Group {
    int first_unit, blocks, nseg, rows, items;
    int from, to;          // sources
    int per_piece, longer; // intervals of a piece; the first `longer` ones have one more
    int piece, split;      // number of its first partial result; partial results per piece
    Div by_unit, by_block;
};

struct Args {
    Source s[2]; // prefix, own; many rows: the codes are tiles of values, of units from the group's first on, and intervals are tiles
    Group g[2];
    const h1 *q;
    long q_sb, q_sh, q_st;
    const void *mask;
    long m_sb, m_sh, m_st;
    int mask_dt;
    float *partial; // [partial results, rows, D]
    float2 *ml;     // [partial results, rows]: m, l
    h1 *out;        // not null: a row has one partial result, and goes here
    long rows;      // B * n * Hq, in the order of the output [B, n, Hq]
    int H, log_g;
    Div by_head, by_token;
    int n;
    int act_bf16;
    float scaling; // not negative: the queries' signs are changed instead
    int negate;
    // one new token: quantised by the waves that replay the own tokens in front of it, its row here
    int append;
    const uint16_t *x[2];
    long x_sb[2], x_sh[2];
};

// The arguments are read where the launch has put them: indexed by what a wave is at, a copy would live in scratch memory.
#define ADKV_KERNARG const __attribute__((address_space(4)))
typedef ADKV_KERNARG Args KArgs;
__device__ __forceinline__ int quotient(uint32_t x, uint32_t d, uint32_t lo, uint32_t hi)
{
    return d == 1 ? (int)x : (int)(((uint64_t)x * hi + __umulhi(x, lo)) >> 32);
}
__device__ __forceinline__ int divide(int x, const Div &by) { return quotient(x, by.d, by.lo, by.hi); }
__device__ __forceinline__ int divide(int x, ADKV_KERNARG Div &by) { return quotient(x, by.d, by.lo, by.hi); }
// all of a structure at once: field by field, between branches, every read is a wait
template <typename T>
__device__ __forceinline__ T all_of(ADKV_KERNARG T &from)
{
    struct Words {
        uint32_t w[sizeof(T) / 4];
    } x;
    const auto p = (ADKV_KERNARG uint32_t *)&from;
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 4; i++)
        x.w[i] = p[i];
    return __builtin_bit_cast(T, x);
}
// a pointer from there is one to global memory, which the compiler cannot know
template <typename T>
__device__ __forceinline__ __attribute__((address_space(1))) T *global(T *p) { return (__attribute__((address_space(1))) T *)p; }

// The tiles of a workgroup, one after the other: those of an item's piece in one source, then in the other, then the next item's.  What
// the arguments have of an item or a span is read when it is opened: a read per tile is a wait per tile.
template <int TOKENS>
struct Walk {
    int i, group, b, h, block, seg, end; // item; end: interval behind its piece, counted over its sources
    int rows, prefix;                    // of the group; intervals of the prefix if the piece may begin there
    int src, first, t0, t1, k, n;        // span: a run of tokens of a source, in tiles; the tile
    int items;
    bool ends;                           // the span is its item's last
    __device__ __forceinline__ Walk(KArgs &a, int items_, int item) : i(item), items(items_) { open(a); }
    __device__ __forceinline__ void open(KArgs &a)
    {
        group = i < a.g[0].items ? 0 : 1;
        const Group g = all_of(a.g[group]);
        int at = i - (group ? a.g[0].items : 0);
        const int of_launch = divide(at, g.by_unit), unit = of_launch + g.first_unit;
        at -= of_launch * (g.blocks * g.nseg);
        seg = divide(at, g.by_block);
        block = at - seg * g.blocks;
        b = group ? divide(unit, a.by_head) : 0;
        h = unit - b * a.H;
        rows = g.rows;
        prefix = g.from == 0 ? a.s[0].x.intervals : 0;
        const int begin = seg * g.per_piece + min(seg, g.longer);
        end = begin + g.per_piece + (seg < g.longer ? 1 : 0);
        span(a, begin < prefix ? begin : begin - prefix, begin < prefix ? 0 : 1);
    }
    __device__ __forceinline__ void span(KArgs &a, int first_, int src_)
    {
        src = src_;
        first = first_;
        const Extent s = all_of(a.s[src].x);
        const int e = src ? end - prefix : end;
        t0 = first * s.interval;
        t1 = e >= s.intervals ? s.tokens : e * s.interval;
        k = 0;
        n = (t1 - t0 + TOKENS - 1) / TOKENS;
        ends = src == 1 || end <= prefix;
    }
    __device__ __forceinline__ bool last_of_item() const { return k + 1 == n && ends; }
    __device__ __forceinline__ bool more() const { return i + (int)gridDim.x < items; }
    __device__ __forceinline__ bool last() const { return last_of_item() && !more(); }
    // to the next tile, which is there
    __device__ __forceinline__ void go(KArgs &a)
    {
        if (++k < n)
            return;
        if (!ends) {
            span(a, 0, 1);
        } else {
            i += gridDim.x;
            open(a);
        }
    }
    __device__ __forceinline__ int code_unit(KArgs &a) const { return src ? b * a.H + h : h; }
};

// Where a tile's values are, in pieces of 16 bytes whose order changes with the channel so that what is accessed in one clock lies in different
// banks.  32 channels are 4096 bytes, 16 are 2048, in either kind of tile.
// Many rows: a channel's 64 tokens are a row of 128 bytes.  Keys: piece u is tokens 8u..; the transposing reads of 16 lanes take 32 bytes of four
// consecutive channels.  Values: piece 4 * kk + r is tokens 32 * kk + 4 * r.. and 32 * kk + 16 + 4 * r.., the ones whose weights a lane of
// quarter r has; reads take 16 bytes of sixteen channels.
// Few rows: two channels' 32 tokens are 128 bytes, piece u of either is tokens 8u..
__device__ __forceinline__ int few_piece(int c, int u) { return (c >> 1) * 256 + ((((c & 1) << 2 | u) ^ (c & 2) ^ (c >> 2 & 1)) << 4); }
__device__ __forceinline__ int many_key_piece(int c, int u) { return c * 128 + ((u ^ (c & 3) << 1 ^ (c >> 2 & 1)) << 4); }
__device__ __forceinline__ int many_value_piece(int c, int u) { return c * 128 + ((u ^ (c >> 1 & 7)) << 4); }
template <bool FEW> __device__ __forceinline__ int key_piece(int c, int u) { return FEW ? few_piece(c, u) : many_key_piece(c, u); }
template <bool FEW> __device__ __forceinline__ int value_piece(int c, int u) { return FEW ? few_piece(c, u) : many_value_piece(c, u); }

template <bool MAX>
__device__ __forceinline__ float fold_quarters(float v) // over the lanes l % 16
{
    unsigned a = __builtin_bit_cast(unsigned, v), b = a;
    // Two copies: the compiler folds a swap of a register with itself.  The copy is its own: behind one in a block of assembly it would
    // not keep the two wait states that the swap needs.
    asm volatile("" : "+v"(b));
    u2v r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    unsigned x = r.x, y = r.y;
    asm volatile("" : "+v"(x), "+v"(y));
    v = MAX ? fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y)) : __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
    b = a = __builtin_bit_cast(unsigned, v);
    asm volatile("" : "+v"(b));
    r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    x = r.x;
    y = r.y;
    asm volatile("" : "+v"(x), "+v"(y));
    return MAX ? fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y)) : __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}

__device__ __forceinline__ void store_four(h1 *to, f4v v, int act_bf16)
{
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if (act_bf16) {
            uint32_t b[2];
#pragma unroll
            for (int k = 0; k < 2; k++) { // to nearest even, from fp32
                const uint32_t u = __float_as_uint(v[2 * i + k]);
                b[k] = (u & 0x7FFFFFFFu) > 0x7F800000u ? 0x7FC0u : (u + 0x7FFFu + (u >> 16 & 1u)) >> 16;
            }
            w[i] = b[0] | b[1] << 16;
        } else {
            w[i] = as_u32((h2){(h1)v[2 * i], (h1)v[2 * i + 1]});
        }
    }
    *(__attribute__((address_space(1))) u2v *)to = (u2v){w[0], w[1]};
}

// ---------------------------------------------------------------------------------------------------------------- producers
// A wave replays 64 channels of K or V, one per lane, a tile at a time.

__device__ __forceinline__ Lone state_of(h2 zp_sc, h1 al, h1 be, h1 tg)
{
    const h1 one = (h1)1.0f, bt = be * tg; // omt = 1 - beta*target, both steps rounded
    Lone st;
    st.z = as_u32((h2){zp_sc.x, (h1)0.0f});
    st.r = as_u32((h2){(h1)0.0f, zp_sc.y});
    st.ca = as_u32((h2){al, one});
    st.cf = as_u32((h2){one, be});
    st.c0 = as_u32((h2){(h1)0.0f, one - bt});
    return st;
}

// Where a span's loads are
struct Feed {
    const uint32_t *codes, *ck;
    const h1 *zp, *sc, *al, *be, *tg;
    const uint16_t *x;
    int bytes;
    template <int BITS> __device__ __forceinline__ void open(KArgs &a, const Walk<FEW_TILE> &at, int kind)
    {
        const Extent s = all_of(a.s[at.src].x);
        const Tensor t = all_of(a.s[at.src].t[kind]);
        const int unit = at.code_unit(a);
        constexpr int TPW = 32 / BITS;
        codes = t.codes + ((size_t)unit * s.n_super + at.t0 / TPW) * D;
        bytes = (at.t1 - at.t0 + TPW - 1) / TPW * (D * 4);
        // the first span has no checkpoint: any word will do
        ck = at.first > 0 ? reinterpret_cast<const uint32_t *>(t.ckpt) + ((size_t)unit * s.n_ckpt + at.first - 1) * D : codes;
        zp = t.zp + at.h * D;
        sc = t.sc + at.h * D;
        al = t.al + at.h * D;
        be = t.be + at.h * D;
        tg = t.tg + at.h * D;
        x = a.x[kind] + at.b * a.x_sb[kind] + at.h * a.x_sh[kind];
    }
};

// What a tile needs from memory, loaded two tiles ahead.  There is no condition around the loads of the words: the compiler would wait for every load
// in flight behind one.  (With words loaded behind each whole tile, and none behind the last one of an item, a tile of 64 tokens took 2.4 us, the
// memory's latency.)
template <int BITS>
struct Loads {
    static constexpr int WPT = FEW_TILE * BITS / 32; // words of a channel per tile
    uint32_t w[WPT], ck;
    h1 zp, sc, al, be, tg;
    uint16_t fresh;

    __device__ __forceinline__ void start(const Feed &f, int k, int c)
    {
        // reads behind the last word of the span are dropped
        const auto codes = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint32_t *>(f.codes), 0, f.bytes, 0x00027000);
        const int next = (k * WPT * D + c) * 4;
#pragma unroll
        for (int i = 0; i < WPT; i++)
            w[i] = __builtin_amdgcn_raw_buffer_load_b32(codes, next + i * D * 4, 0, 0);
        if (k > 0)
            return;
        ck = global(f.ck)[c];
        zp = global(f.zp)[c];
        sc = global(f.sc)[c];
        al = global(f.al)[c];
        be = global(f.be)[c];
        tg = global(f.tg)[c];
        fresh = global(f.x)[c];
    }
    __device__ __forceinline__ Lone state(bool from_ckpt) const { return state_of(from_ckpt ? as_h2(ck) : (h2){zp, sc}, al, be, tg); }
};

__device__ __forceinline__ void put_unit(char *to, int c, int u, const uint32_t *x)
{
    *reinterpret_cast<uint4 *>(to + few_piece(c, u)) = make_uint4(x[0], x[1], x[2], x[3]);
}

// a whole tile from the words w
template <int BITS>
__device__ __forceinline__ void whole_tile(Lone &st, const uint32_t *w, const uint2 *lut, uint32_t lane_copy, char *to, int c)
{
    uint2 e[2][4];
    lone_lookup<BITS>(e[0], lut, w, 0, lane_copy);
#pragma unroll
    for (int u = 0; u < FEW_TILE / 8; u++) {
        if (u + 1 < FEW_TILE / 8)
            lone_lookup<BITS>(e[(u & 1) ^ 1], lut, w, u + 1, lane_copy);
        __builtin_amdgcn_sched_barrier(0);
        uint32_t x[4];
        lone_eight(st, e[u & 1], x);
        put_unit(to, c, u, x);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// The last tile of a span: fewer tokens than a tile has, or as many with the appended one among them.  What is behind them is zero: its weights
// are, and the rest of a buffer may be anything.  append: the n-th token is new, the last of its stream.
template <int BITS, bool KEYS>
__device__ __forceinline__ void part_tile(Lone &st, const uint32_t *w, char *to, int c, int n, bool append, uint16_t fresh, KArgs &a,
                                          const Walk<FEW_TILE> &at)
{
    constexpr int TPW = 32 / BITS;
    for (int u = 0; u < FEW_TILE / 8; u++) {
        uint32_t x[4] = {};
        if (u * 8 < n) {
            uint32_t word = 0;
#pragma unroll
            for (int k = 0; k < FEW_TILE / TPW; k++)
                word = u * 8 / TPW == k ? w[k] : word;
            word >>= u * 8 % TPW * BITS;
            const int there = min(n - u * 8 - (append ? 1 : 0), 8); // old ones
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < there)
                    x[i >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, lone_token(st, (int)(word >> BITS * i & Code<BITS>::FIELD) + Code<BITS>::QLO))
                                 << (i & 1) * 16;
            if (append && there >= 0 && there < 8 && u * 8 + there == n - 1) {
                const Extent s = all_of(a.s[1].x);
                const Tensor t = all_of(a.s[1].t[KEYS ? 0 : 1]);
                const int unit = at.code_unit(a), T = at.t1 - 1;
                const auto ck = global(reinterpret_cast<uint32_t *>(const_cast<h1 *>(t.ckpt))) + (size_t)unit * s.n_ckpt * D + c;
                // the state in front of token T, and behind it, where an interval ends there
                const int j = s.interval > 0 ? T / s.interval : 0, rest = s.interval > 0 ? T - j * s.interval : 1;
                if (rest == 0 && j > 0 && j <= s.n_ckpt)
                    ck[(size_t)(j - 1) * D] = as_u32((h2){lone_zp(st), lone_sc(st)});
                const int q = quantize<BITS>(act2(fresh, a.act_bf16).x, lone_zp(st), lone_sc(st));
                const auto home = global(const_cast<uint32_t *>(t.codes)) + ((size_t)unit * s.n_super + T / TPW) * D + c;
                const int sh = T % TPW * BITS;
                uint32_t whole = 0;
#pragma unroll
                for (int k = 0; k < FEW_TILE / TPW; k++)
                    whole = u * 8 / TPW == k ? w[k] : whole;
                *home = (whole & ~(Code<BITS>::FIELD << sh)) | (uint32_t)(q - Code<BITS>::QLO) << sh;
                const uint32_t v = (uint32_t)__builtin_bit_cast(uint16_t, lone_token(st, q)) << (there & 1) * 16;
#pragma unroll
                for (int k = 0; k < 4; k++)
                    x[k] |= there >> 1 == k ? v : 0u;
                if (rest + 1 == s.interval && j < s.n_ckpt)
                    ck[(size_t)j * D] = as_u32((h2){lone_zp(st), lone_sc(st)});
            }
        }
        put_unit(to, c, u, x);
    }
}

template <int BITS, bool KEYS>
__device__ __forceinline__ void produce(KArgs &a, int items, const uint2 *lut, char *tiles, int c, int lane)
{
    constexpr int KIND = KEYS ? 0 : 1, COPIES = (BITS == 4 ? LUT_COPIES : LUT2_COPIES) / 2;
    const uint32_t lane_copy = (uint32_t)(lane & (COPIES - 1)) * (BITS == 4 ? 8u : 16u);
    const int append_end = a.append ? a.s[1].x.tokens : -1;
    Loads<BITS> ahead[2];
    uint16_t fresh = 0;
    Walk<FEW_TILE> at(a, items, blockIdx.x), then = at, next = at; // the tile, the one after it, the one whose loads go out next
    Feed feed;
    feed.open<BITS>(a, next, KIND);
    auto step = [&]() __attribute__((always_inline)) {
        if (next.last())
            return; // the same again, never used
        next.go(a);
        if (next.k == 0)
            feed.open<BITS>(a, next, KIND);
    };
    ahead[0].start(feed, next.k, c);
    step();
    then = next;
    ahead[1].start(feed, next.k, c);
    __syncthreads(); // the table
    Lone st = {};
    // returns whether that was the last
    auto tile = [&](auto ic) __attribute__((always_inline)) {
        constexpr int I = decltype(ic)::value;
        const Loads<BITS> cur = ahead[I];
        step();
        ahead[I].start(feed, next.k, c);
        if (at.k == 0) {
            st = cur.state(at.first > 0);
            fresh = cur.fresh;
        }
        char *to = tiles + I * FEW_BUFFER + (KEYS ? 0 : FEW_VALUES);
        const int left = at.t1 - at.t0 - at.k * FEW_TILE;
        const bool append = at.src && at.t1 == append_end;
        if (left > FEW_TILE || (left == FEW_TILE && !append))
            whole_tile<BITS>(st, cur.w, lut, lane_copy, to, c);
        else
            part_tile<BITS, KEYS>(st, cur.w, to, c, left, append, fresh, a, at);
        __syncthreads();
        if (at.last())
            return true;
        at = then;
        then = next;
        return false;
    };
    while (!tile(std::integral_constant<int, 0>{}) && !tile(std::integral_constant<int, 1>{}))
        ;
}

// ---------------------------------------------------------------------------------------------------------------- consumers
// The mask of a lane's 4 * J tokens of a step, as it is in memory; rows are as aligned as their elements.
template <int J, int MASK>
struct MaskRaw {
    static constexpr int WORDS = 2 * J * MASK; // MASK: 1 of 16 bits, 2 fp32
    typedef uint32_t u2a __attribute__((ext_vector_type(2), aligned(2)));
    typedef uint32_t u4a __attribute__((ext_vector_type(4), aligned(4)));
    uint32_t w[WORDS];
    // tokens t + 16 * i.. for i < J, of which `there` are in the source
    __device__ __forceinline__ void load(const char *row, int t, int there)
    {
        const auto p = global(row + (long)t * (2 * MASK));
        if (__all(there >= 16 * (J - 1) + 4)) {
#pragma unroll
            for (int i = 0; i < J; i++) {
                if constexpr (MASK == 1) {
                    const u2a u = *(const __attribute__((address_space(1))) u2a *)(p + i * 32);
                    w[2 * i] = u.x;
                    w[2 * i + 1] = u.y;
                } else {
                    const u4a u = *(const __attribute__((address_space(1))) u4a *)(p + i * 64);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        w[4 * i + e] = u[e];
                }
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < WORDS; e++)
            w[e] = 0;
#pragma unroll
        for (int e = 0; e < 4 * J; e++) {
            const int at = (e >> 2) * 16 + (e & 3);
            if (at < there) {
                if constexpr (MASK == 1)
                    w[e >> 1] |= (uint32_t)((const __attribute__((address_space(1))) uint16_t *)p)[at] << (e & 1) * 16;
                else
                    w[e] = ((const __attribute__((address_space(1))) uint32_t *)p)[at];
            }
        }
    }
    __device__ __forceinline__ bool anything() const
    {
        uint32_t any = 0;
#pragma unroll
        for (int e = 0; e < WORDS; e++)
            any |= w[e];
        return any != 0;
    }
    // x = x * scaling + mask
    __device__ __forceinline__ void add(float *x, float scaling, int dt) const
    {
        if constexpr (MASK == 2) {
#pragma unroll
            for (int e = 0; e < 4 * J; e++)
                x[e] = __builtin_fmaf(x[e], scaling, __uint_as_float(w[e]));
        } else if (dt == ADKV_DT_F16) {
#pragma unroll
            for (int e = 0; e < 2 * J; e++) {
                x[2 * e] = __builtin_fmaf(x[2 * e], scaling, (float)as_h2(w[e]).x);
                x[2 * e + 1] = __builtin_fmaf(x[2 * e + 1], scaling, (float)as_h2(w[e]).y);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 2 * J; e++) {
                x[2 * e] = __builtin_fmaf(x[2 * e], scaling, __uint_as_float(w[e] << 16));
                x[2 * e + 1] = __builtin_fmaf(x[2 * e + 1], scaling, __uint_as_float(w[e] & 0xFFFF0000u));
            }
        }
    }
};
template <int J> struct MaskRaw<J, 0> {
};

// NB blocks of 16 query rows, J times 16 tokens a step.  Scores come as columns (lane l: row l % 16, of every 16 tokens 4 * (l / 16) + 0..3),
// which is as the weights are taken by the product with V; the outputs are columns too, so that a row's maximum and sum are its lanes' own.
// Without a mask scores are kept as q.K and the scaling is the exponent's: e^(scaling * (s - m)) is one multiply-add and an exp2.
// MASK: 0 none, 1 of 16 bits, 2 fp32; m is then the largest of scaling * s + mask.
template <int NB, int J, int MASK>
struct Consumer {
    static constexpr bool FEW = J == 1;
    using W = Walk<FEW ? FEW_TILE : TILE>;
    static constexpr int NC = FEW ? 4 : 8; // blocks of 16 channels of the outputs
    h8v q[NB][4];
    f4v o[NB][NC];
    float m[NB], l[NB];
    int row[NB];          // of the unit
    int limit[NB];        // tokens of the source that it looks at, and that the span has
    const char *mask[NB]; // its mask at the source's first token
    int seen, tokens;     // of the source: what every row looks at (of the span), all
    MaskRaw<J, MASK> masks[NB];

    // of row r of a unit: sequence, token, query head
    __device__ __forceinline__ static void place(KArgs &a, const W &at, int r, int &b, int &i, int &hq)
    {
        const int token = r >> a.log_g;
        b = at.group ? at.b : divide(token, a.by_token);
        i = at.group ? token : token - b * a.n;
        hq = (at.h << a.log_g) + (r & ((1 << a.log_g) - 1));
    }
    // the queries' loads, of blocks `block`, block + stride..; ready() makes them what is multiplied
    __device__ __forceinline__ static void load(KArgs &a, const W &at, int block, int stride, int lane, h8v (*to)[4])
    {
        const int rows = at.rows;
#pragma unroll
        for (int k = 0; k < NB; k++) {
            int b, i, hq;
            place(a, at, min((block + k * stride) * 16 + (lane & 15), rows - 1), b, i, hq);
            const h1 *src = a.q + b * a.q_sb + hq * a.q_sh + i * a.q_st + (lane >> 4) * 8;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                // rows are 4-byte aligned
                typedef uint32_t u4a __attribute__((ext_vector_type(4), aligned(4)));
                to[k][c] = __builtin_bit_cast(h8v, (u4v)*(const __attribute__((address_space(1))) u4a *)(src + c * 32));
            }
        }
    }
    __device__ __forceinline__ void ready(KArgs &a, const h8v (*from)[4])
    {
        const uint32_t sign = a.negate ? 0x80008000u : 0u;
#pragma unroll
        for (int k = 0; k < NB; k++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint4 u = __builtin_bit_cast(uint4, from[k][c]);
                if (a.act_bf16)
                    u = make_uint4(as_u32(act2(u.x, 1)), as_u32(act2(u.y, 1)), as_u32(act2(u.z, 1)), as_u32(act2(u.w, 1)));
                q[k][c] = __builtin_bit_cast(h8v, make_uint4(u.x ^ sign, u.y ^ sign, u.z ^ sign, u.w ^ sign));
            }
    }
    __device__ __forceinline__ void clear(KArgs &a, const W &at, int block, int stride, int lane)
    {
#pragma unroll
        for (int k = 0; k < NB; k++) {
            row[k] = (block + k * stride) * 16 + (lane & 15);
            m[k] = -INFINITY;
            l[k] = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; c++)
                o[k][c] = (f4v){0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    // What a row looks at of a span's source, up to the span's end: of few rows a span may end inside a tile, and the tile's rest, which is
    // zero there, is the next span's.
    __device__ __forceinline__ void look(KArgs &a, const W &at)
    {
        const Extent s = all_of(a.s[at.src].x);
        seen = min(s.seen, at.t1);
        tokens = s.tokens;
#pragma unroll
        for (int k = 0; k < NB; k++) {
            int b, i, hq;
            place(a, at, min(row[k], at.rows - 1), b, i, hq);
            limit[k] = min(s.causal ? s.seen + i : s.seen, at.t1);
            if constexpr (MASK != 0)
                mask[k] = (const char *)a.mask + (b * a.m_sb + hq * a.m_sh + i * a.m_st + s.col) * (MASK == 2 ? 4 : 2);
        }
    }

    // the mask of the tokens from t on
    template <int NA> __device__ __forceinline__ void look_at(int t, int lane, MaskRaw<J, MASK> *to)
    {
        if constexpr (MASK != 0) {
            t += (lane >> 4) * 4;
#pragma unroll
            for (int k = 0; k < NA; k++)
                to[k].load(mask[k], t, tokens - t);
        }
    }
    // the scores of the step-th step of a tile, as q.K
    template <int NA> __device__ __forceinline__ void scores(const char *keys, int step, int lane, f4v (*sc)[J])
    {
        typedef short s4v __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4v *Lds;
        const int r16 = lane & 15, quarter = lane >> 4;
        // A transposing read hands 16 lanes four channels of 16 tokens: lane i reads channel i / 4, tokens 4 * (i % 4)..
        const auto kbase = (__attribute__((address_space(3))) const char *)keys;
#pragma unroll
        for (int j = 0; j < J; j++) {
            int at[2];
#pragma unroll
            for (int i = 0; i < 2; i++)
                at[i] = key_piece<FEW>(quarter * 8 + i * 4 + (r16 >> 2), (step * J + j) * 2 + (r16 >> 1 & 1)) + (r16 & 1) * 8;
#pragma unroll
            for (int k = 0; k < NA; k++)
                sc[k][j] = (f4v){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const s4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(kbase + at[0] + c * 4096));
                const s4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(kbase + at[1] + c * 4096));
                const uint2 u = __builtin_bit_cast(uint2, x), v = __builtin_bit_cast(uint2, y);
                const h8v key = __builtin_bit_cast(h8v, make_uint4(u.x, u.y, v.x, v.y));
#pragma unroll
                for (int k = 0; k < NA; k++)
                    sc[k][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, q[k][c], sc[k][j], 0, 0, 0);
            }
        }
        // Beside a mask a branch may follow, and the compiler then counts one wait state too few between a product and what reads it.
        if constexpr (MASK != 0)
#pragma unroll
            for (int k = 0; k < NA; k++)
                asm volatile("s_nop 7" : "+v"(sc[k][J - 1]));
    }

    // scores of the tokens from t on to weights of fp16; the row's maximum, sum and outputs go along
    template <int NA> __device__ __forceinline__ void weights(KArgs &a, int t, int lane, const f4v (*sc)[J], uint32_t (*w)[2 * J])
    {
        const int quarter = lane >> 4;
#pragma unroll
        for (int k = 0; k < NA; k++) {
            float x[4 * J];
#pragma unroll
            for (int e = 0; e < 4 * J; e++)
                x[e] = sc[k][e >> 2][e & 3];
            bool plain = true; // x are products yet, and nothing is added to them
            if constexpr (MASK != 0) {
                plain = !__any(masks[k].anything());
                if (!plain)
                    masks[k].add(x, a.scaling, a.mask_dt);
            }
            if (t + 16 * J > seen) {
#pragma unroll
                for (int e = 0; e < 4 * J; e++)
                    x[e] = t + (e >> 2) * 16 + quarter * 4 + (e & 3) < limit[k] ? x[e] : -INFINITY;
            }
            float mx = x[0];
#pragma unroll
            for (int e = 1; e < 4 * J; e++)
                mx = fmaxf(mx, x[e]);
            // The largest so far is looked for again only where a weight would be more than 2^8: weights relative to one that is smaller than the
            // largest by up to that are as exact.
            const float c = MASK != 0 ? LOG2E : a.scaling * LOG2E; // of m; with masks scores, else products
            if (MASK != 0 && plain)
                mx *= a.scaling;
            if (__any((mx - m[k]) * c > 8.0f || m[k] == -INFINITY)) {
                mx = fmaxf(m[k], fold_quarters<true>(mx));
                const float shrink = m[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m[k] - mx) * c);
                m[k] = mx;
                l[k] *= shrink;
#pragma unroll
                for (int cc = 0; cc < NC; cc++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        o[k][cc][e] *= shrink;
            }
            const float ref = m[k] == -INFINITY ? 0.0f : m[k]; // nothing but -inf so far: all weights are zero
            float sum = 0.0f;
            if (MASK != 0 && __any(fabsf(ref) > 1024.0f)) {
                // The difference first: beside a mask the largest may be as large as its type's lowest value, also for rows of a plain tile,
                // of which later tokens are all that they could look at (-inf, which has to stay that).
                const float unit = plain ? a.scaling : 1.0f;
#pragma unroll
                for (int e = 0; e < 4 * J; e++)
                    x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], unit, -ref) * c);
            } else {
                const float unit = MASK != 0 && plain ? a.scaling * LOG2E : c;
#pragma unroll
                for (int e = 0; e < 4 * J; e++)
                    x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], unit, -ref * c));
            }
#pragma unroll
            for (int e = 0; e < 4 * J; e++)
                sum += x[e];
            l[k] += sum;
#pragma unroll
            for (int e = 0; e < 2 * J; e++)
                w[k][e] = as_u32((h2){(h1)x[2 * e], (h1)x[2 * e + 1]});
        }
    }
    // Half of a product's 32 tokens where a step has 16: the other half is zero on both sides.
    template <int NA> __device__ __forceinline__ void outputs(const char *values, int step, int lane, const uint32_t (*w)[2 * J])
    {
#pragma unroll
        for (int kk = 0; kk < (J + 1) / 2; kk++)
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const int quarter = lane >> 4, piece = FEW ? step * 2 + (quarter >> 1) : (step * (J / 2) + kk) * 4 + quarter;
                const char *p = values + c * 2048 + value_piece<FEW>(lane & 15, piece);
                uint4 v;
                if constexpr (FEW) {
                    const uint2 half = *reinterpret_cast<const uint2 *>(p + (quarter & 1) * 8);
                    v = make_uint4(half.x, half.y, 0, 0);
                } else {
                    v = *reinterpret_cast<const uint4 *>(p);
                }
#pragma unroll
                for (int k = 0; k < NA; k++) {
                    const uint4 p4 = FEW ? make_uint4(w[k][0], w[k][1], 0, 0) : make_uint4(w[k][kk * 4], w[k][kk * 4 + 1], w[k][kk * 4 + 2], w[k][kk * 4 + 3]);
                    o[k][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, v), __builtin_bit_cast(h8v, p4), o[k][c], 0, 0, 0);
                }
            }
    }

    // part: of a piece's partial results; c0: the first block of channels
    __device__ __forceinline__ void finish(KArgs &a, const W &at, int part, int c0, int lane)
    {
        const Group g = all_of(a.g[at.group]);
#pragma unroll
        for (int k = 0; k < NB; k++) {
            const float sum = fold_quarters<false>(l[k]);
            if (row[k] >= at.rows)
                continue;
            int b, i, hq;
            place(a, at, row[k], b, i, hq);
            const long r = ((long)b * a.n + i) * (a.H << a.log_g) + hq;
            if (a.out != nullptr) {
                const float inv = 1.0f / sum;
#pragma unroll
                for (int c = 0; c < NC; c++)
                    store_four(a.out + r * D + (c0 + c) * 16 + (lane >> 4) * 4, o[k][c] * inv, a.act_bf16);
                continue;
            }
            const long to = (g.piece + at.seg * g.split + part) * a.rows + r;
            if (lane < 16 && c0 == 0)
                *(__attribute__((address_space(1))) f2v *)global(a.ml + to) = (f2v){MASK != 0 || m[k] == -INFINITY ? m[k] : m[k] * a.scaling, sum};
#pragma unroll
            for (int c = 0; c < NC; c++)
                *(__attribute__((address_space(1))) f4v *)global(a.partial + to * D + (c0 + c) * 16 + (lane >> 4) * 4) = o[k][c];
        }
    }
};

// Few rows: two pairs of waves multiply half of a tile's tokens each, with partial results of their own, a wave for half of the channels of the
// outputs; both make the weights.
template <int MASK>
__device__ __forceinline__ void consume(KArgs &a, int items, const char *tiles, int wave, int lane)
{
    using C = Consumer<1, 1, MASK>;
    const int step = wave & 1, c0 = (wave >> 1) * 4;
    C c;
    h8v ahead[1][4]; // the next item's queries, from this one's start on
    typename C::W at(a, items, blockIdx.x), next = at; // next: the next item's first tile
    C::load(a, at, 0, 0, lane, ahead);
    c.ready(a, ahead);
    __syncthreads(); // the table
    bool opened = true; // at the item's first tile
    auto tile = [&](auto ic) __attribute__((always_inline)) {
        const char *from = tiles + decltype(ic)::value * FEW_BUFFER;
        const bool ends = at.last_of_item(), more = at.more();
        const int t = at.t0 + at.k * FEW_TILE + step * 16;
        if (opened) {
            c.clear(a, at, 0, 0, lane);
            if (more) {
                next = typename C::W(a, items, at.i + gridDim.x);
                C::load(a, next, 0, 0, lane, ahead);
            }
        }
        if (at.k == 0)
            c.look(a, at);
        opened = ends;
        c.template look_at<1>(t, lane, c.masks);
        __syncthreads();
        if (t < at.t1) { // of a span's last tile half may be empty
            f4v sc[1][1];
            uint32_t w[1][2];
            c.template scores<1>(from, step, lane, sc);
            c.template weights<1>(a, t, lane, sc, w);
            c.template outputs<1>(from + FEW_VALUES + c0 * 2048, step, lane, w);
        }
        if (!ends) {
            at.go(a);
            return false;
        }
        if (more)
            c.ready(a, ahead); // in front of the stores, which it would wait for
        c.finish(a, at, step, c0, lane);
        at = next;
        return !more;
    };
    while (!tile(std::integral_constant<int, 0>{}) && !tile(std::integral_constant<int, 1>{}))
        ;
}

// The code table with its copies in the first half of every 256 bytes (see Shape, lone_fill, lone_fill2)
template <int BITS, int NT>
__device__ __forceinline__ void fill_half(char *lds, int tid)
{
    for (int i = tid; i < LUT_ENTRIES * 8; i += NT) {
        const int b = i >> 3;
        const auto entry = [](int code) { return as_u32(splat((h1)(code - (BITS == 4 ? 8 : 2)))) & 0x7FFFFFFFu; };
        uint4 v;
        if constexpr (BITS == 4) {
            const uint32_t x = entry(b & 15), y = entry(b >> 4);
            v = make_uint4(x, y, x, y);
        } else {
            v = make_uint4(entry(b & 3), entry(b >> 2 & 3), entry(b >> 4 & 3), entry(b >> 6));
        }
        *reinterpret_cast<uint4 *>(lds + b * 256 + (i & 7) * 16) = v;
    }
}

// Four waves replay the tile after the one that the others multiply with, one per SIMD, through two buffers and a barrier per tile.
// A workgroup goes on to its next item without a gap.  Replay, hand-over through the LDS and products of a tile are some 2000 cycles of every
// SIMD whether its rows are one or sixteen, which bounds it; a limit of the replay it is not (a step's own kernels, without the hand-over,
// replay 2.7 times as many tokens in a time).  128 sequences of 32 heads with 65 tokens each: 43 us (codes of 34 MB are 7); a
// prefix of 8192 tokens and 4 sequences of 1001, 32 heads: 36 us.
template <int BITS, int MASK>
__global__ __launch_bounds__(FEW_THREADS) void attend_kernel(Args)
{
    KArgs &a = *(KArgs *)__builtin_amdgcn_kernarg_segment_ptr();
    __shared__ uint4 smem[FEW_LDS / 16]; // the table at LDS offset 0
    const uint2 *lut = reinterpret_cast<const uint2 *>(smem);
    char *tiles = reinterpret_cast<char *>(smem) + FEW_FIRST;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int items = a.g[0].items + a.g[1].items;
    fill_half<BITS, FEW_THREADS>(reinterpret_cast<char *>(smem), threadIdx.x);
    if (wave < 2)
        produce<BITS, true>(a, items, lut, tiles, wave * 64 + lane, lane);
    else if (wave < PRODUCERS)
        produce<BITS, false>(a, items, lut, tiles, (wave - 2) * 64 + lane, lane);
    else
        consume<MASK>(a, items, tiles, wave - PRODUCERS, lane);
}

// ---------------------------------------------------------------------------------------------------------------- many rows
struct Images {
    Source s[2]; // the sources' codes
    char *to[2]; // their tiles, of the units from `first` on
    int first[2], runs[2], items[2]; // runs of checkpoint intervals per unit
    int H;
    Div by_run[2];
};

// The values of a run of tokens of K and V as tiles in memory, as the LDS has them: a wave for 64 channels of either, two workgroups to a CU.  Bound by its
// stores: 4096 tokens of 32 heads are 67 MB of values, 17 us (3.9 TB/s).  Workgroups of four runs, four waves to a SIMD with one table, are done later
// (the call with 5 new tokens of 16 sequences behind 2048, 8 heads, 67 us instead of 57).
template <int BITS>
__global__ __launch_bounds__(256) void values_kernel(Images im)
{
    constexpr int TPW = 32 / BITS, WPC = TILE / TPW; // words of a channel per chunk of 64 tokens
    __shared__ uint4 smem[LUT_WORDS64 / 2 + 4 * 256];
    uint2 *lut = reinterpret_cast<uint2 *>(smem);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    int item = (int)blockIdx.x;
    const bool own = item >= im.items[0];
    const int kind = wave >> 1, c = (wave & 1) * 64 + lane;
    item -= own ? im.items[0] : 0;
    const Extent &x = own ? im.s[1].x : im.s[0].x;
    const Tensor &t = own ? (kind ? im.s[1].t[1] : im.s[1].t[0]) : (kind ? im.s[0].t[1] : im.s[0].t[0]);
    const int runs = own ? im.runs[1] : im.runs[0], of_launch = divide(item, own ? im.by_run[1] : im.by_run[0]);
    const int unit = of_launch + (own ? im.first[1] : im.first[0]), run = item - of_launch * runs;
    const int per = x.intervals / runs, longer = x.intervals % runs, first = run * per + min(run, longer), end = first + per + (run < longer ? 1 : 0);
    const int t0 = first * x.interval, t1 = end >= x.intervals ? x.tokens : end * x.interval;
    const int h = own ? unit % im.H : unit, pi = h * D + c;

    const int words = (t1 - t0 + TPW - 1) / TPW;
    // reads behind the last word are dropped
    const auto codes = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint32_t *>(t.codes) + ((size_t)unit * x.n_super + t0 / TPW) * D, 0, words * D * 4,
                                                         0x00027000);
    int next = c * 4;
    uint32_t w[2][WPC];
    auto load = [&](uint32_t *to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < WPC; i++)
            to[i] = __builtin_amdgcn_raw_buffer_load_b32(codes, next + i * D * 4, 0, 0);
        next += WPC * D * 4;
    };
    load(w[0]);
    load(w[1]);
    h2 from = {t.zp[pi], t.sc[pi]};
    if (first > 0)
        from = as_h2(*reinterpret_cast<const uint32_t *>(t.ckpt + (((size_t)unit * x.n_ckpt + first - 1) * D + c) * 2));
    Lone st = state_of(from, t.al[pi], t.be[pi], t.tg[pi]);
    if constexpr (BITS == 4)
        lone_fill<256>(lut, threadIdx.x);
    else
        lone_fill2<256>(lut, threadIdx.x);
    __syncthreads();
    const uint32_t lane_copy = BITS == 4 ? (uint32_t)(lane & (LUT_COPIES - 1)) * 8u : (uint32_t)(lane & (LUT2_COPIES - 1)) * 16u;
    const int tiles = (x.tokens + TILE - 1) / TILE;
    const auto image = global((own ? im.to[1] : im.to[0]) + (size_t)of_launch * tiles * TILE_BYTES + kind * TILE_VALUES);
    // unit n of eight tokens of the source
    auto put = [&](int n, const uint32_t *v) __attribute__((always_inline)) {
        const auto to = image + (size_t)(n >> 3) * TILE_BYTES;
        const int u = n & 7;
        if (kind == 0) {
            *(__attribute__((address_space(1))) u4v *)(to + many_key_piece(c, u)) = (u4v){v[0], v[1], v[2], v[3]};
        } else {
            const int piece = (u & 4) + (u & 1) * 2, half = (u & 2) * 4;
            *(__attribute__((address_space(1))) u2v *)(to + many_value_piece(c, piece) + half) = (u2v){v[0], v[1]};
            *(__attribute__((address_space(1))) u2v *)(to + many_value_piece(c, piece + 1) + half) = (u2v){v[2], v[3]};
        }
    };
    // A whole tile by way of the LDS, 32 channels at a time, which makes a store of the wave 1 KB in a row instead of 16 bytes of 64 rows.
    u4v *stage = reinterpret_cast<u4v *>(smem + LUT_WORDS64 / 2) + wave * 256;
    auto put_tile = [&](int n, const uint32_t (*v)[4]) __attribute__((always_inline)) {
        const auto to = image + (size_t)(n >> 3) * TILE_BYTES + (wave & 1) * 8192 + lane * 16;
#pragma unroll
        for (int part = 0; part < 2; part++) {
            if (lane >> 5 == part) {
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    const int k = (u & 4) + u % 4 / 2, j = u % 2 * 2;
                    if (kind == 0)
                        stage[many_key_piece(lane & 31, u) >> 4] = (u4v){v[u][0], v[u][1], v[u][2], v[u][3]};
                    else
                        stage[many_value_piece(lane & 31, u) >> 4] = (u4v){v[k][j], v[k][j + 1], v[k + 2][j], v[k + 2][j + 1]};
                }
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < 4; i++)
                *(__attribute__((address_space(1))) u4v *)(to + part * 4096 + i * 1024) = stage[i * 64 + lane];
            __builtin_amdgcn_wave_barrier();
        }
    };
    int n = t0 >> 3, left = t1 - t0;
    const bool whole = (n & 7) == 0;
    auto chunk = [&](uint32_t *from) __attribute__((always_inline)) {
        uint32_t cur[WPC], v[8][4];
#pragma unroll
        for (int i = 0; i < WPC; i++)
            cur[i] = from[i];
        load(from);
        uint2 e[2][4];
        lone_lookup<BITS>(e[0], lut, cur, 0, lane_copy);
#pragma unroll
        for (int u = 0; u < 8; u++) {
            if (u < 7)
                lone_lookup<BITS>(e[(u & 1) ^ 1], lut, cur, u + 1, lane_copy);
            __builtin_amdgcn_sched_barrier(0);
            lone_eight(st, e[u & 1], v[u]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (whole) {
            put_tile(n, v);
        } else {
#pragma unroll
            for (int u = 0; u < 8; u++)
                put(n + u, v[u]);
        }
        n += 8;
        left -= TILE;
    };
    for (;;) {
        if (left < TILE)
            break;
        chunk(w[0]);
        if (left < TILE) {
#pragma unroll
            for (int i = 0; i < WPC; i++)
                w[0][i] = w[1][i];
            break;
        }
        chunk(w[1]);
    }
    // the rest, and zeros up to the end of the source's last tile: their weights are zero, and what is there may be anything
    const int stop = t1 == x.tokens ? tiles * 8 : n + (left + 7) / 8;
    for (int u = 0; n < stop; u++, n++) {
        uint32_t v[4] = {};
        if (u * 8 < left) {
            uint32_t word = 0;
#pragma unroll
            for (int k = 0; k < WPC; k++)
                word = u * 8 / TPW == k ? w[0][k] : word;
            word >>= u * 8 % TPW * BITS;
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (u * 8 + i < left)
                    v[i >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, lone_token(st, (int)(word >> BITS * i & Code<BITS>::FIELD) + Code<BITS>::QLO))
                                 << (i & 1) * 16;
        }
        put(n, v);
    }
}

// A tile in 32 loads of 1 KB straight to the LDS, eight by each of four waves.
struct Fetch {
    static constexpr uint32_t PART = TILE_BYTES / MANY_WAVES;
    uint32_t from, to;
    __device__ __forceinline__ Fetch(int wave, int lane) : from((uint32_t)wave * PART + (uint32_t)lane * 16u), to((uint32_t)wave * PART) {}
    __device__ __forceinline__ void tile(const char *image, uint32_t lds) const
    {
        const uint64_t base = (uint64_t)image;
        const rsrc4 buffer = {(uint32_t)base, (uint32_t)(base >> 32) & 0xFFFFu, (uint32_t)TILE_BYTES, 0x00027000u};
#pragma unroll
        for (uint32_t i = 0; i < PART; i += 1024)
            load_to_lds(lds + to + i, from + i, buffer);
    }
};

// Two tiles in the LDS, one being multiplied with and one on its way, a barrier per tile; two workgroups to a CU, which wait at different times (one
// of eight waves and three tiles: 512 masked tokens of 8 sequences 690 us instead of 530).  Workgroups of one XCD take neighbouring items,
// which read the same tiles.  A wave's tile with 32 rows is 1024 cycles of matrix instructions and some 1500 of others, half of them the softmax;
// with two waves to a SIMD it takes 2900, 3500 with a mask: neither pipe is full (matrix cores 29 to 35 % busy), the wave that waits for its reads or
// results is not covered by one other.  512 tokens of 8 sequences, 32 heads, over 4096 tokens, masked: 430 to 510 us by the clock that the card
// holds, 570 to 670 TFLOP/s; without fetching its tiles 11 % less, without exponentials 7 % less.  A wave of the SIMD a tile behind, a
// raised priority for the softmax or for one of two workgroups and reads of the LDS issued a group ahead changed nothing; a raised priority for the
// products made it 810.  Tiles that hold later tokens only are walked through like others: a call that is mostly its own new tokens takes up to twice what it
// needs (2048 tokens of 32 heads with nothing in front of them 169 us, 235 behind 2048 others).
template <int MASK>
__global__ __launch_bounds__(MANY_WAVES * 64, 2) void attend_many_kernel(Args)
{
    using C = Consumer<2, 4, MASK>;
    KArgs &a = *(KArgs *)__builtin_amdgcn_kernarg_segment_ptr();
    __shared__ uint4 smem[2 * TILE_BYTES / 16];
    char *tiles = reinterpret_cast<char *>(smem);
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)tiles;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int items = a.g[0].items + a.g[1].items;
    const int here = gridDim.x % 8 == 0 ? blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8 : blockIdx.x;
    const Fetch fetch(wave, lane);
    C c;
    Walk<TILE> at(a, items, here), next = at; // the tile, the one that is fetched next
    const char *image = nullptr;              // of the latter
    auto open = [&]() __attribute__((always_inline)) {
        const size_t unit = next.code_unit(a) - (next.src ? a.g[1].first_unit : 0);
        image = (const char *)a.s[next.src].t[0].codes + (unit * a.s[next.src].x.intervals + next.first) * TILE_BYTES;
    };
    auto step = [&]() __attribute__((always_inline)) {
        if (next.last())
            return; // the same again, never used
        image += TILE_BYTES;
        next.go(a);
        if (next.k == 0)
            open();
    };
    auto block = [&](const Walk<TILE> &w) __attribute__((always_inline)) { return w.block * (2 * MANY_WAVES) + wave; };
    open();
    fetch.tile(image, lds);
    C::load(a, at, block(at), MANY_WAVES, lane, c.q);
    bool opened = true, looked = false; // the tile's mask is there
    MaskRaw<4, MASK> coming[2];
    int buffer = 0;
    for (;;) {
        if (opened) {
            c.ready(a, c.q);
            c.clear(a, at, block(at), MANY_WAVES, lane);
        }
        if (at.k == 0)
            c.look(a, at);
        const int t = at.t0 + at.k * TILE, mine = (at.rows + 15) / 16 - block(at); // blocks from this wave's first on
        const bool ends = at.last_of_item(), done = at.last();
        opened = ends;
        step();
        __builtin_amdgcn_s_waitcnt(ALL_READS); // this wave's part of the tile is there, what it read of the last one, and loads that the compiler would wait for later
        __builtin_amdgcn_s_barrier();          // and everyone's; and nobody reads the tile before it any more
        asm volatile("" ::: "memory");
        // Loads end in order, and a wait for a mask would be one for a tile that is fetched in front of it or behind it: the next tile's
        // mask is loaded with the tile.  (fp32 masks have no registers for that.)
        if constexpr (MASK == 1) {
            if (looked) {
#pragma unroll
                for (int k = 0; k < 2; k++)
                    c.masks[k] = coming[k];
            } else if (mine > 0) {
                c.template look_at<2>(t, lane, c.masks);
            }
            looked = mine > 0 && at.k + 1 < at.n;
            if (looked)
                c.template look_at<2>(t + TILE, lane, coming);
        }
        if constexpr (MASK == 2)
            if (mine > 0)
                c.template look_at<2>(t, lane, c.masks);
        fetch.tile(image, lds + (buffer ^ 1) * TILE_BYTES);
        const char *from = tiles + buffer * TILE_BYTES;
        Walk<TILE> then = at;
        auto multiply = [&](auto na) __attribute__((always_inline)) {
            constexpr int NA = decltype(na)::value;
            f4v sc[2][4];
            uint32_t w[2][8];
            c.template scores<NA>(from, 0, lane, sc);
            c.template weights<NA>(a, t, lane, sc, w);
            c.template outputs<NA>(from + TILE_VALUES, 0, lane, w);
        };
        if (mine > MANY_WAVES)
            multiply(std::integral_constant<int, 2>{});
        else if (mine > 0)
            multiply(std::integral_constant<int, 1>{});
        if (!done) {
            if (ends) {
                then = Walk<TILE>(a, items, at.i + gridDim.x);
                C::load(a, then, block(then), MANY_WAVES, lane, c.q);
            } else {
                then.go(a);
            }
        }
        if (ends && mine > 0)
            c.finish(a, at, 0, 0, lane);
        if (done)
            break;
        at = then;
        buffer ^= 1;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // nothing is written to the LDS any more
}

// out = sum e^(m-M) o / sum e^(m-M) l over the pieces.  Four channels per lane, 32 lanes per row, WAYS of them for a share of the
// pieces each, in a fixed order: where rows are few the pieces are many and a lane that walks through all of them waits for each
// (128 rows of 100 pieces 25 us, with WAYS = 8 five).  Whole calls with WAYS = 8 and 1, us: 128 rows 44 and 64, 1024 rows 42 and 43 or 59 and 62, 4096
// rows 93.5 and 95.0, 8192 rows 103 and 102, 16384 rows 122 and 119, 32768 rows 127 and 118; 5120 rows of few pieces 57 and 56.
template <int WAYS>
__global__ __launch_bounds__(256) void join_kernel(const float *__restrict__ partial, const float2 *__restrict__ ml, h1 *__restrict__ out,
                                                   long rows, int pieces, int act_bf16)
{
    constexpr int ROWS = 8 / WAYS;
    __shared__ f4v part[WAYS > 1 ? 256 : 1];
    __shared__ f2v stat[WAYS > 1 ? 8 : 1];
    const int group = threadIdx.x >> 5, way = group % WAYS, c = (threadIdx.x & 31) * 4;
    const long row = min((long)blockIdx.x * ROWS + group / WAYS, rows - 1);
    float M = -INFINITY;
    for (int k = way; k < pieces; k += WAYS)
        M = fmaxf(M, ml[k * rows + row].x);
    if constexpr (WAYS > 1) {
        if (c == 0)
            stat[group].x = M;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAYS; i++)
            M = fmaxf(M, stat[group / WAYS * WAYS + i].x);
    }
    const float ref = M == -INFINITY ? 0.0f : M; // a row whose mask leaves nothing: 0 / 0
    float L = 0.0f;
    f4v o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int k = way; k < pieces; k += WAYS) {
        const float2 p = ml[k * rows + row];
        const float e = __builtin_amdgcn_exp2f((p.x - ref) * LOG2E);
        const f4v v = *reinterpret_cast<const f4v *>(partial + (k * rows + row) * D + c);
        L = __builtin_fmaf(p.y, e, L);
#pragma unroll
        for (int i = 0; i < 4; i++)
            o[i] = __builtin_fmaf(v[i], e, o[i]);
    }
    if constexpr (WAYS > 1) {
        part[threadIdx.x] = o;
        if (c == 0)
            stat[group].y = L;
        __syncthreads();
        if (way > 0)
            return;
#pragma unroll
        for (int i = 1; i < WAYS; i++) {
            L += stat[group + i].y;
            o += part[threadIdx.x + i * 32];
        }
    }
    if ((long)blockIdx.x * ROWS + group / WAYS < rows)
        store_four(out + row * D + c, o * (1.0f / L), act_bf16);
}

// The state behind token T - 1 of every channel, from the last checkpoint in front of it: at most an interval, a token at a time, three dependent
// operations each (200 tokens: 7 us, 13 with codes taken apart one by one).
// Where token T opens an interval the state is that interval's checkpoint, which nobody may have recorded yet.
template <int BITS>
__global__ __launch_bounds__(128) void state_kernel(Source s, int H, int n_ckpt, h1 *k_state, h1 *v_state)
{
    constexpr int TPW = 32 / BITS;
    const int unit = blockIdx.x, c = threadIdx.x, pi = unit % H * D + c, T = s.x.tokens;
    const Tensor t = s.t[blockIdx.y];
    const h1 one = (h1)1.0f, be = t.be[pi], bt = be * t.tg[pi];
    const int first = s.x.interval > 0 ? min((T - 1) / s.x.interval, n_ckpt) : 0;
    h2 from = {t.zp[pi], t.sc[pi]};
    if (first > 0)
        from = as_h2(*reinterpret_cast<const uint32_t *>(t.ckpt + (((size_t)unit * n_ckpt + first - 1) * D + c) * 2));
    const h1 al = t.al[pi], omt = one - bt;
    h1 zp = from.x, sc = from.y;
    // token k of a word, whose code and factor of the scale wait for nothing
    auto token = [&](h1 q, h1 f) __attribute__((always_inline)) {
        zp = __builtin_fmaf16(al, q * sc, zp);
        sc = sc * f;
    };
    auto pair = [&](uint32_t w, int k, h2 &q, h2 &f) __attribute__((always_inline)) {
        constexpr uint32_t FIELD = Code<BITS>::FIELD;
        const int at = 2 * BITS * k;
        const uint32_t lo = w >> at & FIELD, hi = w >> (at + BITS) & FIELD;
        q = as_h2(0x64006400u | hi << 16 | lo) - splat((h1)(1024 - Code<BITS>::QLO)); // 1024 + code, then exact
        f = __builtin_elementwise_fma(splat(be), as_h2(as_u32(q) & 0x7FFF7FFFu), splat(omt));
    };
    const uint32_t *w = t.codes + (size_t)unit * s.x.n_super * D + c;
    constexpr int AHEAD = 8;
    uint32_t buf[2][AHEAD];
    const int at0 = first * s.x.interval / TPW, words = (T + TPW - 1) / TPW, whole = T / TPW;
    auto load = [&](int at, uint32_t *b) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            b[i] = w[(size_t)min(at + i, words - 1) * D];
    };
    load(at0, buf[0]);
    for (int at = at0; at < words; at += AHEAD) {
        load(at + AHEAD, buf[1]);
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (at + i < whole) {
#pragma unroll
                for (int k = 0; k < TPW / 2; k++) {
                    h2 q, f;
                    pair(buf[0][i], k, q, f);
                    token(q.x, f.x);
                    token(q.y, f.y);
                }
            } else {
#pragma unroll
                for (int k = 0; k < TPW / 2; k++) {
                    h2 q, f;
                    pair(buf[0][i], k, q, f);
                    if ((at + i) * TPW + 2 * k < T)
                        token(q.x, f.x);
                    if ((at + i) * TPW + 2 * k + 1 < T)
                        token(q.y, f.y);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            buf[0][i] = buf[1][i];
    }
    const uint32_t zs = as_u32((h2){zp, sc});
    *reinterpret_cast<uint32_t *>((blockIdx.y ? v_state : k_state) + ((size_t)unit * D + c) * 2) = zs;
    if (s.x.interval > 0 && T % s.x.interval == 0 && T / s.x.interval - 1 < n_ckpt)
        *reinterpret_cast<uint32_t *>(const_cast<h1 *>(t.ckpt) + (((size_t)unit * n_ckpt + T / s.x.interval - 1) * D + c) * 2) = zs;
}

struct Plan {
    bool joint;                     // the prefix is walked with the rows of each sequence by themselves
    bool there[2], few[2];          // of a group
    int nseg[2], blocks[2], split[2];
    int intervals[2], tiles[2];     // of a source
    bool image[2];                  // whether the source is written out as tiles of values
    int batch;                      // units of the own source whose tiles are there at a time
    long pieces() const { return (long)nseg[0] * split[0] + (long)nseg[1] * split[1]; }
    int64_t image_bytes(int i, int H) const { return image[i] ? (int64_t)(i ? batch : H) * tiles[i] * TILE_BYTES : 0; }
};

static int usable_intervals(int tokens, int interval, int n_ckpt)
{
    return interval > 0 ? std::max(std::min((tokens + interval - 1) / interval, n_ckpt + 1), 1) : 1;
}

constexpr int64_t IMAGE_MAX = 1ll << 30; // bytes of own tiles at a time, unless one unit's are more

// Rows of a sequence that fill a workgroup walk through the prefix by themselves, and their outputs need no joining (512 tokens of 8 sequences 520 us,
// 680 with the prefix apart; at 40 rows 60 us instead of 58).  Workgroups
// walk through items, two per CU.  The length of a piece is chosen for the shortest call by the model (us): a workgroup's items x
// (64 tokens of a piece x 1.3 or, of many rows, 2.3, + 1), and 4 TB/s for the partial results, written and read.  With 0.8 and 1.4, these, 2.2 and 3.8,
// us: 257 new tokens of 4 sequences behind 3001, 8 heads of 4 queries, 157, 145, 146; 33 of one behind 6000 48.4, 45.5, 46.1; a token of 4 sequences
// over 8192 + 1000 45.7, 43.7, 43.9; of 128 over 4096 + 64 92.5, 93.5, 95.0; of 48 over 7777 + 301, 4 queries, 62.5, 61.0, 60.5; seven other sizes within 2 %.
// T: the own tokens in front of the new ones.
static Plan plan(int B, int H, int G, int n, int P, int p_interval, int p_ckpt, int T, int interval, int n_ckpt)
{
    Plan p = {};
    const long rows[2] = {(long)B * n * G, (long)n * G}, units[2] = {H, (long)B * H}, total = (long)B * n * G * H;
    p.joint = P > 0 && rows[1] >= JOINT_ROWS;
    p.there[0] = P > 0 && !p.joint;
    p.there[1] = true;
    p.intervals[0] = P > 0 ? usable_intervals(P, p_interval, p_ckpt) : 0;
    // the state in front of a single new token may not be recorded yet
    p.intervals[1] = usable_intervals(n == 1 ? T : T + n, interval, n_ckpt);
    p.tiles[0] = (P + TILE - 1) / TILE;
    p.tiles[1] = (T + n + TILE - 1) / TILE;
    for (int i = 0; i < 2; i++)
        p.few[i] = rows[i] <= 16;
    p.image[0] = p.joint || (p.there[0] && !p.few[0]);
    p.image[1] = !p.few[1];
    p.batch = (int)std::max<int64_t>(1, std::min<int64_t>((long)B * H, IMAGE_MAX / ((int64_t)p.tiles[1] * TILE_BYTES)));
    // groups of one kind share a launch
    for (int k = 0; k < 2; k++) {
        const bool f = k == 0;
        const long slots = cu_count() * 2L;
        const bool in[2] = {p.there[0] && p.few[0] == f, p.few[1] == f};
        if (!in[0] && !in[1])
            continue;
        const double tile = f ? 1.3 : 2.3;
        double best = -1.0;
        for (int len = 1; len < (1 << 20); len += std::max(len / 4, 1)) { // of 64 tokens
            int ns[2] = {0, 0};
            long items = 0, longest = 0, pieces = 0;
            bool shortest = true;
            for (int i = 0; i < 2; i++) {
                if (!in[i])
                    continue;
                const long tiles = p.tiles[i] + (i && p.joint ? p.tiles[0] : 0), most = f ? p.intervals[i] : tiles;
                p.blocks[i] = f ? 1 : (int)((rows[i] + MANY_ROWS - 1) / MANY_ROWS);
                p.split[i] = f ? 2 : 1;
                ns[i] = (int)std::max<long>(std::min<long>(most, (tiles + len - 1) / len), 1);
                items += units[i] * p.blocks[i] * ns[i];
                longest = std::max(longest, (tiles + ns[i] - 1) / ns[i]);
                pieces += (long)ns[i] * p.split[i];
                shortest = shortest && ns[i] == 1;
            }
            const bool direct = pieces == 1 && !(p.there[0] && !in[0]);
            const double cost = (double)((items + slots - 1) / slots) * (longest * tile + 1.0) + (direct ? 0.0 : 4.0 + pieces * total * 1024 / 4e6);
            if (best < 0 || cost < best) {
                best = cost;
                for (int i = 0; i < 2; i++)
                    if (in[i])
                        p.nseg[i] = ns[i];
            }
            if (shortest)
                break;
        }
    }
    return p;
}

static int64_t pad256(int64_t n) { return (n + 255) & ~(int64_t)255; }

static int64_t workspace_bytes_of(const Plan &p, int B, int H, int64_t rows)
{
    return 2 * pad256((int64_t)B * H * D * 4) + pad256(p.pieces() * rows * 8) + pad256(p.pieces() * rows * D * 4) + p.image_bytes(0, H) + p.image_bytes(1, H);
}

// rows of the joining launch: a grid is 2^32 threads at most, 32 for a row
constexpr int64_t JOIN_MAX = (1ll << 27) - 8;

} // namespace adkv_ext

using namespace adkv_ext;

extern "C" {

int64_t adkv_extend_workspace_bytes(int B, int Hq, int H, int T, int n, int n_ckpt_cap, int ckpt_interval, int P, int prefix_n_ckpt_cap,
                                    int prefix_ckpt_interval)
{
    if (B <= 0 || H <= 0 || Hq <= 0 || Hq % H || T < 0 || n <= 0 || P < 0 || T > MAX_TOKENS || n > MAX_TOKENS - T || P > MAX_TOKENS)
        return 0;
    const Plan p = plan(B, H, Hq / H, n, P, prefix_n_ckpt_cap > 0 ? prefix_ckpt_interval : 0, prefix_n_ckpt_cap, T,
                        n_ckpt_cap > 0 ? ckpt_interval : 0, n_ckpt_cap);
    return workspace_bytes_of(p, B, H, (int64_t)B * n * Hq);
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
    // everything is refused here, in front of the launches: a call that fails has changed nothing
    if (n > 1)
        for (int i = 0; i < 2; i++) { // rows that the encoder reads, as aligned words
            const int64_t *st = i ? v_strides : k_strides;
            if ((uintptr_t)(i ? v_new : k_new) & 3)
                return ADKV_E_ALIGN;
            if (st && (st[0] < 0 || st[1] < 0 || st[2] < D || ((st[0] | st[1] | st[2]) & 1)))
                return ADKV_E_SHAPE;
        }
    const Plan pl = plan(B, H, G, n, P, p_interval, p_cap, T, ckpt_interval, n_ckpt_cap);
    if (pl.pieces() > 1 && rows > JOIN_MAX)
        return ADKV_E_SHAPE;
    for (int i = 0; i < 2; i++) // items are counted in 32 bits, and beyond the last by a launch's workgroups
        if (pl.there[i] && (i ? (int64_t)B * H : H) * pl.blocks[i] * pl.nseg[i] > INT32_MAX / 4)
            return ADKV_E_SHAPE;
    if (!workspace || workspace_bytes < workspace_bytes_of(pl, B, H, rows))
        return ADKV_E_WORKSPACE;

    char *ws = (char *)workspace;
    const int64_t state_bytes = pad256((int64_t)B * H * D * 4);
    h1 *k_state = (h1 *)ws, *v_state = (h1 *)(ws + state_bytes);
    Args a;
    a.ml = (float2 *)(ws + 2 * state_bytes);
    a.partial = (float *)(ws + 2 * state_bytes + pad256(pl.pieces() * rows * 8));
    char *images[2];
    images[0] = (char *)a.partial + pad256(pl.pieces() * rows * D * 4);
    images[1] = images[0] + pl.image_bytes(0, H);
    auto tensor = [](const void *codes, const void *ckpt, const void *const *p) {
        return Tensor{(const uint32_t *)codes, (const h1 *)ckpt, (const h1 *)p[0], (const h1 *)p[1], (const h1 *)p[2], (const h1 *)p[3], (const h1 *)p[4]};
    };
    auto div = [](int64_t d) {
        const uint64_t mul = ~0ull / (uint64_t)d + 1; // of 1 it is 2^64, and not used
        return Div{(uint32_t)d, (uint32_t)mul, (uint32_t)(mul >> 32)};
    };
    Source &pre = a.s[0], &own = a.s[1];
    pre = Source{};
    if (P > 0) {
        pre.t[0] = tensor(prefix->k_codes, prefix->k_ckpt, prefix->k_params);
        pre.t[1] = tensor(prefix->v_codes, prefix->v_ckpt, prefix->v_params);
        pre.x.tokens = pre.x.seen = P;
        pre.x.n_super = prefix->n_super;
        pre.x.n_ckpt = p_cap;
        pre.x.interval = p_interval;
        pre.x.intervals = pl.intervals[0];
    }
    own = Source{};
    own.t[0] = tensor(k_cache, k_ckpt, k_params);
    own.t[1] = tensor(v_cache, v_ckpt, v_params);
    own.x.tokens = T + n;
    own.x.seen = T + 1;
    own.x.causal = 1;
    own.x.n_super = n_super_cap;
    own.x.n_ckpt = n_ckpt_cap;
    own.x.interval = ckpt_interval;
    own.x.intervals = pl.intervals[1];
    own.x.col = P;
    a.by_head = div(H);
    a.by_token = div(n);
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
    a.H = H;
    a.log_g = G == 1 ? 0 : G == 2 ? 1 : G == 4 ? 2 : 3;
    a.n = n;
    a.act_bf16 = act_dtype == ADKV_DT_BF16;
    // hidden tokens are -inf times it, which has to stay -inf: a scaling of zero is a small one
    a.scaling = scaling == 0.0f ? 1e-30f : fabsf(scaling);
    a.negate = scaling < 0.0f;
    a.append = n == 1;

    const int64_t *strides[2] = {k_strides, v_strides}; // as adkv_append_kv_pair has them
    for (int i = 0; i < 2; i++) {
        a.x[i] = (const uint16_t *)(i ? v_new : k_new);
        a.x_sb[i] = strides[i] ? strides[i][0] : (int64_t)H * n * D;
        a.x_sh[i] = strides[i] ? strides[i][1] : (int64_t)n * D;
    }
    if (n > 1) {
        if (T > 0) {
            Source before = own;
            before.x.tokens = T;
            const auto kernel = bits == 4 ? state_kernel<4> : state_kernel<2>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)(B * H), 2), dim3(D), 0, (hipStream_t)stream, before, H, n_ckpt_cap, k_state, v_state);
            if ((rc = check_launch()))
                return rc;
        }
        if ((rc = adkv_append_kv_pair(k_cache, v_cache, k_new, v_new, act_dtype, k_strides, v_strides, k_params, v_params, B, H, T, n, D,
                                      n_super_cap, bits, k_state, v_state, k_ckpt, v_ckpt, n_ckpt_cap, ckpt_interval, stream)))
            return rc;
    }
    const bool direct = pl.pieces() == 1;
    a.out = direct ? (h1 *)out : nullptr;
    const int kind = !mask ? 0 : mask_dt == ADKV_DT_F32 ? 2 : 1;
    const Source sources[2] = {pre, own};
    // units [u0, u1) of a group
    auto group = [&](int i, int u0, int u1) {
        Group g = {};
        g.first_unit = u0;
        g.blocks = pl.blocks[i];
        g.nseg = pl.nseg[i];
        g.rows = (int)(i ? (int64_t)n * G : (int64_t)B * n * G);
        g.from = i == 0 || pl.joint ? 0 : 1;
        g.to = i;
        const int intervals = pl.few[i] ? pl.intervals[i] : pl.tiles[i] + (i && pl.joint ? pl.tiles[0] : 0);
        g.per_piece = intervals / g.nseg;
        g.longer = intervals % g.nseg;
        g.piece = i ? pl.nseg[0] * pl.split[0] : 0;
        g.split = pl.split[i];
        g.by_unit = div((int64_t)g.blocks * g.nseg);
        g.by_block = div(g.blocks);
        g.items = (int)((int64_t)(u1 - u0) * g.blocks * g.nseg);
        return g;
    };
    typedef void (*Kernel)(Args);
    if ((pl.there[0] && pl.few[0]) || pl.few[1]) {
        static const Kernel kernels[2][3] = {{attend_kernel<4, 0>, attend_kernel<4, 1>, attend_kernel<4, 2>},
                                             {attend_kernel<2, 0>, attend_kernel<2, 1>, attend_kernel<2, 2>}};
        a.g[0] = pl.there[0] && pl.few[0] ? group(0, 0, H) : Group{};
        a.g[1] = pl.few[1] ? group(1, 0, B * H) : Group{};
        const int64_t items = (int64_t)a.g[0].items + a.g[1].items;
        hipLaunchKernelGGL(kernels[bits == 2][kind], dim3((unsigned)std::min<int64_t>(items, 2 * cu_count())), dim3(FEW_THREADS), 0,
                           (hipStream_t)stream, a);
        if ((rc = check_launch()))
            return rc;
    }
    if (pl.image[0] || pl.image[1]) {
        static const Kernel kernels[3] = {attend_many_kernel<0>, attend_many_kernel<1>, attend_many_kernel<2>};
        for (int i = 0; i < 2; i++)
            if (pl.image[i]) {
                a.s[i].t[0].codes = (const uint32_t *)images[i];
                a.s[i].x.interval = TILE;
                a.s[i].x.intervals = pl.tiles[i];
            }
        for (int u0 = 0; u0 < B * H; u0 += pl.batch) {
            const int u1 = std::min(B * H, u0 + pl.batch);
            Images im = {};
            im.H = H;
            for (int i = 0; i < 2; i++) {
                im.s[i] = sources[i];
                im.to[i] = images[i];
                im.first[i] = i ? u0 : 0;
                const int units = !pl.image[i] || (i == 0 && u0 > 0) ? 0 : i ? u1 - u0 : H;
                // a run per wave slot: four waves a run, sixteen a CU
                im.runs[i] = std::max(1, std::min(pl.intervals[i], 4 * cu_count() / std::max(units, 1)));
                im.items[i] = units * im.runs[i];
                im.by_run[i] = div(im.runs[i]);
            }
            const int items = im.items[0] + im.items[1];
            if (items > 0) {
                hipLaunchKernelGGL(bits == 4 ? values_kernel<4> : values_kernel<2>, dim3((unsigned)items), dim3(256), 0, (hipStream_t)stream, im);
                if ((rc = check_launch()))
                    return rc;
            }
            a.g[0] = pl.there[0] && !pl.few[0] && u0 == 0 ? group(0, 0, H) : Group{};
            a.g[1] = pl.image[1] ? group(1, u0, u1) : Group{};
            const int64_t work = (int64_t)a.g[0].items + a.g[1].items;
            if (work > 0) {
                hipLaunchKernelGGL(kernels[kind], dim3((unsigned)std::min<int64_t>(work, 2 * cu_count())), dim3(MANY_WAVES * 64), 0, (hipStream_t)stream, a);
                if ((rc = check_launch()))
                    return rc;
            }
            if (!pl.image[1])
                break;
        }
    }
    if (direct)
        return ADKV_OK;
    const auto join = rows <= 8192 && pl.pieces() >= 4 ? join_kernel<8> : join_kernel<1>;
    const int64_t per = rows <= 8192 && pl.pieces() >= 4 ? 1 : 8;
    hipLaunchKernelGGL(join, dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, (hipStream_t)stream, a.partial, a.ml, (h1 *)out, rows,
                       (int)pl.pieces(), a.act_bf16);
    return check_launch();
}

} // extern "C"
