// Sequences of a cache copied over one another: row r of every tensor becomes what row index[r] was, all layers' tensors in a launch or two.
//
// Nothing but memory: a row that moves is read and written once, one that stays is not touched.  In place any map is taken, whatever the order in
// which rows overwrite each other: a wave takes a column of the tensors (1 KB or less, of all rows), and has read what it needs of it before it
// writes.  Columns are independent, so that there is nothing to wait for between waves.  A wave has 8 or 16 loads of up to 1 KB in flight: the moved rows of
// as many columns as that gives, or, with more rows, of a narrower column.  All waves are resident, each with an equal share of the columns; stores go past
// the caches.
// MI355X, one layer's worth after another's so that nothing is in a cache: one of four beams of 603 tokens, 32 layers of 32 heads (166 MB read and written)
// 38 us, 4.4 TB/s; 12 of 64 sequences of 4096 tokens (416 MB) 88, 4.7 TB/s; sixteen of one of 8001 (368 MB) 75, 4.9 TB/s; a large copy runs at 5.15.
#include <algorithm>
#include <memory>
#include <new>

#include "adkv_device.h"

#include "../../include/adkv_hip.h"

namespace adkv_sequences {
using adkv::check_launch;
using adkv::cu_count;

typedef uint32_t u4v __attribute__((ext_vector_type(4)));
#define GLOBAL __attribute__((address_space(1)))

constexpr int WAVES = 4, BLOCK = 1024; // bytes of a column
// Rows up to which a wave has 8 slots, and five fit a SIMD by their registers; with more rows it has 16, and three fit.  us with 8 and 16: 4 rows 38, 51;
// 48 rows, 12 of them moved, 88, 105; 50 21, 21; 78 42, 31; 122 104, 78.  (4 slots, six waves: 42, 88; 29; 165; 387.)
constexpr int FEW = 64;
constexpr int waves_per_cu(int SLOTS) { return SLOTS == 8 ? 20 : 12; }
constexpr int TENSORS = 96;                         // of a launch
constexpr int MOST = 1024;                          // rows: with all of them moved 16 slots have columns of 16 bytes

struct Tensor {
    const char *from;
    char *to;
    int segments;        // of a row (heads)
    int pitch, to_pitch; // of a segment, bytes
    int used, width;     // columns up to `used` are copied, from there to `width` they are zeros
    int first;           // column of all
};
struct Args {
    const int64_t *index;
    int rows, batch, n, units, waves;
    Tensor t[TENSORS];
};
static_assert(sizeof(Args) <= 4096, "kernel arguments");

// A row may be another one's source: what is read of a column is there before any of it is written.
__device__ __forceinline__ void all_read() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <bool INTO, int SLOTS>
__global__ __launch_bounds__(WAVES * 64) void take_kernel(const Args a)
{
    __shared__ int2 list[MOST];
    __shared__ int count;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (threadIdx.x == 0)
        count = 0;
    __syncthreads();
    // the rows that move, in any order
    for (int r = threadIdx.x; r < a.rows; r += WAVES * 64) {
        const int64_t from = a.index[r];
        const bool there = from >= 0 && from < a.batch;
        if (INTO || (there && from != r))
            list[atomicAdd(&count, 1)] = make_int2(r, there ? (int)from : -1);
    }
    __syncthreads();
    const int m = __builtin_amdgcn_readfirstlane(count), me = (int)blockIdx.x * WAVES + wave;
    if (m == 0 || me >= a.waves)
        return;
    // this wave's share of the columns, which may be of several tensors
    int unit = (int)((int64_t)a.units * me / a.waves);
    const int last = (int)((int64_t)a.units * (me + 1) / a.waves);
    int which = 0;
    for (int i = 0; i < a.n; i += 64)
        which += __popcll(__ballot(i + lane < a.n && a.t[min(i + lane, TENSORS - 1)].first <= unit));
    which--;
    int log = 0; // up to SLOTS rows: 2^log slots are a column's; more: 2^log rows are a slot's
    while ((m <= SLOTS ? 1 : SLOTS) << log < m)
        log++;
    const int2 mine = list[min(lane, m - 1)];
    u4v x[SLOTS];
    for (; unit < last; which++) {
        const Tensor t = a.t[which];
        const int blocks = (t.width + BLOCK - 1) / BLOCK; // columns of a segment
        const long from_row = (long)t.segments * t.pitch, to_row = (long)t.segments * t.to_pitch;
        const int end = min(last, t.first + t.segments * blocks);
        if (m <= SLOTS) {
            for (; unit < end; unit = min(unit + (SLOTS >> log), end)) {
                const int seg0 = (unit - t.first) / blocks, block0 = unit - t.first - seg0 * blocks;
                auto each = [&](auto &&f) __attribute__((always_inline)) {
                    int seg = seg0, block = block0;
#pragma unroll
                    for (int i = 0; i < SLOTS; i++) {
                        const int row = i & ((1 << log) - 1);
                        if (i > 0 && row == 0 && ++block == blocks) {
                            block = 0;
                            seg++;
                        }
                        if (row < m && unit + (i >> log) < end)
                            f(i, __builtin_amdgcn_readlane(mine.x, row), __builtin_amdgcn_readlane(mine.y, row), seg, block * BLOCK + lane * 16);
                    }
                };
                each([&](int i, int, int from, int seg, int at) __attribute__((always_inline)) {
                    x[i] = (u4v){0, 0, 0, 0};
                    if ((!INTO || from >= 0) && at < t.used)
                        x[i] = *(const GLOBAL u4v *)(t.from + from * from_row + (long)seg * t.pitch + at);
                });
                all_read();
                each([&](int i, int to, int, int seg, int at) __attribute__((always_inline)) {
                    if (at < t.width)
                        __builtin_nontemporal_store(x[i], (GLOBAL u4v *)(t.to + to * to_row + (long)seg * t.to_pitch + at));
                });
            }
            continue;
        }
        const int wide = BLOCK >> log, sub = lane >> (6 - log), in = (lane & ((64 >> log) - 1)) * 16;
        for (; unit < end; unit++) {
            const int seg = (unit - t.first) / blocks, block = unit - t.first - seg * blocks;
            for (int part = 0; part < 1 << log; part++) {
                const int at = block * BLOCK + part * wide + in;
#pragma unroll
                for (int i = 0; i < SLOTS; i++) {
                    const int p = (i << log) + sub;
                    x[i] = (u4v){0, 0, 0, 0};
                    if (p < m && at < t.used) {
                        const int from = list[p].y;
                        if (!INTO || from >= 0)
                            x[i] = *(const GLOBAL u4v *)(t.from + from * from_row + (long)seg * t.pitch + at);
                    }
                }
                all_read();
#pragma unroll
                for (int i = 0; i < SLOTS; i++) {
                    const int p = (i << log) + sub;
                    if (p < m && at < t.width)
                        __builtin_nontemporal_store(x[i], (GLOBAL u4v *)(t.to + list[p].x * to_row + (long)seg * t.to_pitch + at));
                }
            }
        }
    }
}

struct Extent {
    uint64_t begin, end;
    bool written;
};

// whether any that is written shares memory with another one
static bool overlapping(Extent *first, Extent *last)
{
    std::sort(first, last, [](const Extent &a, const Extent &b) { return a.begin < b.begin; });
    uint64_t any = 0, written = 0; // ends of what is in front
    for (; first != last; first++) {
        const Extent &e = *first;
        if (e.begin < written || (e.written && e.begin < any))
            return true;
        any = std::max(any, e.end);
        if (e.written)
            written = std::max(written, e.end);
    }
    return false;
}

} // namespace adkv_sequences

extern "C" int adkv_take_sequences(const adkv_rows *tensors, int n, const int64_t *index, int rows, int batch, void *stream)
{
    using namespace adkv_sequences;
    if (n < 0 || rows < 0 || batch <= 0 || rows > MOST)
        return ADKV_E_SHAPE;
    if ((n > 0 && !tensors) || (rows > 0 && !index))
        return ADKV_E_NULL;
    bool into = false;
    for (int i = 0; i < n; i++) {
        const adkv_rows &t = tensors[i];
        if (!t.data)
            return ADKV_E_NULL;
        if (i == 0)
            into = t.into != nullptr;
        if (into != (t.into != nullptr))
            return ADKV_E_UNSUPPORTED;
        if (t.segments < 0 || t.used < 0 || t.pitch < t.used || (into && t.into_pitch < t.used) || (!into && rows > batch) || t.pitch > INT32_MAX - BLOCK ||
            t.into_pitch > INT32_MAX - BLOCK)
            return ADKV_E_SHAPE;
        // no memory is that large, and products of what is taken stay below 2^63
        if (t.segments > INT32_MAX || t.segments * std::max(t.pitch, into ? t.into_pitch : 0) > INT64_MAX / std::max(batch, MOST))
            return ADKV_E_SHAPE;
        if (((uint64_t)t.data | (uint64_t)t.into | (uint64_t)t.pitch | (uint64_t)(into ? t.into_pitch : 0) | (uint64_t)t.used) & 15)
            return ADKV_E_ALIGN;
    }
    // rows that are written while another tensor's are read
    const std::unique_ptr<Extent[]> all(new (std::nothrow) Extent[2 * (size_t)n]);
    if (!all)
        return ADKV_E_WORKSPACE;
    size_t extents = 0;
    for (int i = 0; i < n && rows > 0; i++) {
        const adkv_rows &t = tensors[i];
        if (t.segments * t.used > 0)
            all[extents++] = {(uint64_t)t.data, (uint64_t)t.data + (uint64_t)batch * t.segments * t.pitch, !into};
        if (into && t.segments * t.into_pitch > 0)
            all[extents++] = {(uint64_t)t.into, (uint64_t)t.into + (uint64_t)rows * t.segments * t.into_pitch, true};
    }
    if (overlapping(all.get(), all.get() + extents))
        return ADKV_E_UNSUPPORTED;
    for (int at = 0; at < n && rows > 0;) {
        Args a = {};
        a.index = index;
        a.rows = rows;
        a.batch = batch;
        int64_t units = 0;
        for (; at < n && a.n < TENSORS; at++) {
            const adkv_rows &r = tensors[at];
            Tensor t = {};
            t.from = (const char *)r.data;
            t.to = into ? (char *)r.into : (char *)r.data;
            t.pitch = (int)r.pitch;
            t.to_pitch = into ? (int)r.into_pitch : t.pitch;
            int64_t used = r.used, width = into ? t.to_pitch : used, segments = r.segments;
            if (used == t.pitch && used == t.to_pitch && segments * used <= INT32_MAX - BLOCK) { // one piece
                width = used *= segments;
                t.pitch = t.to_pitch = (int)used;
                segments = 1;
            }
            t.segments = (int)segments;
            t.used = (int)used;
            t.width = (int)width;
            const int64_t blocks = (width + BLOCK - 1) / BLOCK;
            if (segments * blocks == 0)
                continue;
            if (units + segments * blocks > INT32_MAX / 2) {
                if (units == 0)
                    return ADKV_E_SHAPE;
                break;
            }
            t.first = (int)units;
            a.t[a.n++] = t;
            units += segments * blocks;
        }
        if (a.n == 0)
            continue;
        a.units = (int)units;
        const bool few = rows <= FEW;
        a.waves = (int)std::min<int64_t>(units, (int64_t)waves_per_cu(few ? 8 : 16) * cu_count());
        const auto kernel = into ? (few ? take_kernel<true, 8> : take_kernel<true, 16>) : few ? take_kernel<false, 8> : take_kernel<false, 16>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.waves + WAVES - 1) / WAVES)), dim3(WAVES * 64), 0, (hipStream_t)stream, a);
        if (int rc = check_launch())
            return rc;
    }
    return ADKV_OK;
}
