// Block tables and slot maps from request lengths, on the GPU: what a serving loop does between two steps of a paged
// cache, without the lengths leaving the device.
//
// extend: sequence b holds ceil(len / P) blocks and grows by n tokens. With fits = (len + n <= S * P, and the tokens up to
// and including b's are at most max_tokens), ask = fits ? blocks missing : 0 and upto its inclusive sum over the batch,
// b is granted if fits and (ask == 0 or upto <= free_count): blocks go out in batch order and stop at the first sequence
// that the free stack cannot serve. The k-th block asked for is free[free_count - 1 - k].
// trim: the blocks behind ceil(keep / P) go back, in batch order, to free[free_count], free[free_count + 1], ...
//
// A few hundred bytes to a megabyte move; what counts is latency. One launch each: every CTA works out the prefix sums
// of the whole batch for itself in shared memory (up to BT_MAX_BATCH sequences: consecutive ones per thread, one block-wide
// scan of two sums; a scan per BT_THREADS sequences took 2048 of them 6.6 us), which spares a second launch or a barrier
// across the grid, and then takes its share of the outputs, counted in table entries and slots: whose they are is found by
// binary search in the sums. One after the other in a graph: extend 256 sequences by a token each 4.9 us, 64 sequences by
// 263 k tokens 6.1 us; trim 256 sequences 2.9 us, 2048 sequences 4.7 us: dependent loads, a scan and a search one behind
// the other.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ftk {

constexpr int BT_THREADS = 256;
constexpr int BT_MAX_BATCH = 8192;

struct BlockTableParams {
    int* table;               // [B, width]; extend writes the new entries, trim reads
    const int* lens;          // [B] tokens held
    const int* change;        // [B] extend: tokens to add; trim: tokens to keep
    int* free_blocks;         // [capacity] stack; extend reads its top, trim writes behind it
    const int* free_count;    // [1]
    int* slots;               // [max_tokens] (extend)
    int* starts;              // [B + 1] (extend)
    int* lens_out;            // [B]
    int* count_out;           // [1]
    int B, width, page, capacity, max_tokens;
};

// The next launch may begin once this one no longer waits for the one before it: with the permission given first, every
// launch of a queue lets its own successor in while it waits itself, and 2048 sequences trimmed 400 times in a row take
// 8.7 us a launch instead of 4.6 (100 times: 6.9).
__device__ __forceinline__ void bt_begin() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

struct Sums {
    long long a, b;
};
// Inclusive sums over the block of two values per thread; `total` gets the sums of all.
__device__ __forceinline__ Sums bt_scan(Sums v, Sums* red, Sums& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long a = __shfl_up_sync(0xffffffffu, v.a, o), b = __shfl_up_sync(0xffffffffu, v.b, o);
        if (lane >= o) { v.a += a; v.b += b; }
    }
    __syncthreads();                                   // red is free again
    if (lane == 31) red[warp] = v;
    __syncthreads();
    total = Sums{0, 0};
#pragma unroll
    for (int w = 0; w < BT_THREADS / 32; ++w) {
        const Sums t = red[w];
        if (w < warp) { v.a += t.a; v.b += t.b; }
        total.a += t.a;
        total.b += t.b;
    }
    return v;
}
// Division by the page size: a shift where it is a power of two (every sequence takes four of them per launch). The
// dividends are below 2^32: lengths and page sizes are below 2^31.
struct Pages {
    unsigned int page;
    int shift;                                         // -1: not a power of two
    __device__ __forceinline__ explicit Pages(int p) {
        page = (unsigned int)p;
        shift = (p & (p - 1)) ? -1 : 31 - __clz(p);
    }
    __device__ __forceinline__ int whole(unsigned int rows) const { return (int)(shift >= 0 ? rows >> shift : rows / page); }
    __device__ __forceinline__ int blocks(long long tokens) const { return whole((unsigned int)(tokens + page - 1)); }
};
// last index in [0, n) whose sum is at most x (the sums do not decrease, s[0] <= x); the top bit of an entry is a flag
__device__ __forceinline__ int bt_find(const int* s, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((s[mid] & 0x7fffffff) <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}
constexpr int BT_REFUSED = (int)0x80000000;

__global__ void __launch_bounds__(BT_THREADS) block_table_extend_kernel(const BlockTableParams p) {
    extern __shared__ int bt_smem[];
    int* s_start = bt_smem;                            // [B + 1] tokens before b's (2^31 - 1 at most)
    int* s_off = bt_smem + p.B + 1;                    // [B] blocks asked for before b's; BT_REFUSED: none for b
    __shared__ Sums red[BT_THREADS / 32];
    __shared__ int s_taken;
    bt_begin();
    const int tid = threadIdx.x;
    const long long room = (long long)p.width * p.page;
    const Pages pages(p.page);
    const int count = min(max(__ldg(p.free_count), 0), p.capacity);
    if (tid == 0) { s_taken = 0; s_start[0] = 0; }
    // this thread's sequences [b0, b1), one after the other: f(b, tokens held, tokens to add)
    const int each = (p.B + BT_THREADS - 1) / BT_THREADS;
    const int b0 = min(tid * each, p.B), b1 = min(b0 + each, p.B);
    auto sequences = [&](auto f) {
#pragma unroll 4
        for (int b = b0; b < b1; ++b) f(b, (long long)max(__ldg(p.lens + b), 0), (long long)max(__ldg(p.change + b), 0));
    };
    auto missing = [&](long long len, long long add) { return pages.blocks(len + add) - pages.blocks(len); };
    Sums mine{0, 0}, all;
    sequences([&](int, long long len, long long add) {
        mine.a += add;
        if (len + add <= room) mine.b += missing(len, add);
    });
    Sums before = bt_scan(mine, red, all);
    before.a -= mine.a;
    if (all.a > p.max_tokens) {
        // some sequences have tokens behind the slot map's end and ask for nothing: the second sum again
        long long end = before.a;
        mine.b = 0;
        sequences([&](int, long long len, long long add) {
            end += add;
            if (len + add <= room && end <= p.max_tokens) mine.b += missing(len, add);
        });
        before.b = bt_scan(Sums{0, mine.b}, red, all).b;
    }
    before.b -= mine.b;
    sequences([&](int b, long long len, long long add) {
        before.a += add;
        const bool fits = len + add <= room && before.a <= p.max_tokens;
        const int ask = fits ? missing(len, add) : 0;
        const long long upto = before.b + ask;
        const bool granted = fits && (ask == 0 || upto <= count);
        if (granted && ask) atomicMax(&s_taken, (int)upto);            // (who is granted blocks comes before who is not)
        s_start[b + 1] = (int)min(before.a, 0x7fffffffll);
        s_off[b] = (int)min(before.b, 0x7fffffffll) | (granted ? 0 : BT_REFUSED);
        before.b = upto;
        if (blockIdx.x == 0) {
            p.starts[b + 1] = s_start[b + 1];
            p.lens_out[b] = (int)(granted ? len + add : len);
        }
    });
    __syncthreads();
    const int taken = s_taken;
    if (blockIdx.x == 0 && tid == 0) {
        p.starts[0] = 0;
        *p.count_out = count - taken;
    }
    // ---- the new entries of the table
    const int gtid = (int)blockIdx.x * BT_THREADS + tid, threads = (int)gridDim.x * BT_THREADS;
    for (int e = gtid; e < taken; e += threads) {
        const int b = bt_find(s_off, p.B, e);
        const int held = pages.blocks(max(__ldg(p.lens + b), 0));
        p.table[(size_t)b * p.width + held + (e - s_off[b])] = __ldg(p.free_blocks + (count - 1 - e));
    }
    // ---- the slot map, 4 tokens per thread
    const int last = p.B ? s_start[p.B] : 0;
    const bool wide = (reinterpret_cast<uintptr_t>(p.slots) & 15u) == 0;
    for (long long t0 = (long long)gtid * 4; t0 < p.max_tokens; t0 += (long long)threads * 4) {
        int out[4] = {-1, -1, -1, -1};
        int b = -1, end = 0, len = 0, first = 0, off = -1, held = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (t0 + k >= p.max_tokens || t0 + k >= last) break;
            const int t = (int)(t0 + k);
            if (b < 0 || t >= end) {
                // the sequence with start <= t < end: the next one that has tokens, most often the next one
                b = b >= 0 && s_start[b + 2] > t ? b + 1 : bt_find(s_start, p.B + 1, t);
                first = s_start[b];
                end = s_start[b + 1];
                off = s_off[b];
                len = max(__ldg(p.lens + b), 0);
                held = pages.blocks(len);
            }
            if (off < 0) continue;
            const int pos = len + (t - first);         // < width * page
            const int pg = pages.whole((unsigned)pos);
            // entries that this launch writes are taken from where they come from
            const int blk = pg < held ? __ldg(p.table + (size_t)b * p.width + pg)
                                      : __ldg(p.free_blocks + (count - 1 - off - (pg - held)));
            out[k] = blk * p.page + (pos - pg * p.page);
        }
        if (wide && t0 + 4 <= p.max_tokens) {
            *reinterpret_cast<int4*>(p.slots + t0) = make_int4(out[0], out[1], out[2], out[3]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (t0 + k < p.max_tokens) p.slots[t0 + k] = out[k];
        }
    }
}

__global__ void __launch_bounds__(BT_THREADS) block_table_trim_kernel(const BlockTableParams p) {
    extern __shared__ int bt_smem[];
    int* s_off = bt_smem;                              // [B] blocks given back before b's
    __shared__ Sums red[BT_THREADS / 32];
    bt_begin();
    const int tid = threadIdx.x;
    const long long room = (long long)p.width * p.page;
    const Pages pages(p.page);
    const int count = min(max(__ldg(p.free_count), 0), p.capacity);
    const int each = (p.B + BT_THREADS - 1) / BT_THREADS;
    const int b0 = min(tid * each, p.B), b1 = min(b0 + each, p.B);
    auto sequences = [&](auto f) {                     // f(b, tokens kept, blocks given back)
#pragma unroll 4
        for (int b = b0; b < b1; ++b) {
            const int len = (int)min((long long)max(__ldg(p.lens + b), 0), room);
            const int keep = min(max(__ldg(p.change + b), 0), len);
            f(b, keep, pages.blocks(len) - pages.blocks(keep));
        }
    };
    Sums mine{0, 0}, all;
    sequences([&](int, int, int back) { mine.a += back; });
    long long before = bt_scan(mine, red, all).a - mine.a;
    const long long gone = all.a;
    sequences([&](int b, int keep, int back) {
        s_off[b] = (int)min(before, 0x7fffffffll);
        before += back;
        if (blockIdx.x == 0) p.lens_out[b] = keep;
    });
    const int pushed = (int)min(gone, (long long)(p.capacity - count));      // (a stack that is full takes no more)
    if (blockIdx.x == 0 && tid == 0) *p.count_out = count + pushed;
    __syncthreads();
    for (int e = (int)blockIdx.x * BT_THREADS + tid; e < pushed; e += (int)gridDim.x * BT_THREADS) {
        const int b = bt_find(s_off, p.B, e);
        const int len = (int)min((long long)max(__ldg(p.lens + b), 0), room);
        const int keep = min(max(__ldg(p.change + b), 0), len);
        p.free_blocks[count + e] = __ldg(p.table + (size_t)b * p.width + pages.blocks(keep) + (e - s_off[b]));
    }
}

}  // namespace ftk
