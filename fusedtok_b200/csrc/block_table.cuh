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
// of the whole batch for itself in shared memory (up to BT_MAX_BATCH sequences, two block-wide scans per BT_THREADS
// sequences), which spares a second launch or a barrier across the grid, and then takes its share of the outputs: a warp
// per sequence for table entries, a thread per 4 tokens for slots, the token's sequence found by binary search.
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

// Inclusive sum over the block of one value per thread; `total` gets the sum of all.
__device__ __forceinline__ long long bt_scan(long long v, long long* red, long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    __syncthreads();                                   // red is free again
    if (lane == 31) red[warp] = v;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < BT_THREADS / 32; ++w) {
        if (w < warp) v += red[w];
        total += red[w];
    }
    return v;
}
__device__ __forceinline__ int bt_blocks(long long tokens, int page) { return (int)((tokens + page - 1) / page); }

__global__ void __launch_bounds__(BT_THREADS) block_table_extend_kernel(const BlockTableParams p) {
    extern __shared__ int bt_smem[];
    int* s_end = bt_smem;                              // [B] tokens up to and including b's (INT_MAX at most)
    int* s_off = bt_smem + p.B;                        // [B] blocks asked for before b's; -1: refused
    __shared__ long long red[BT_THREADS / 32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x;
    const long long room = (long long)p.width * p.page;
    const int count = min(max(__ldg(p.free_count), 0), p.capacity);
    long long tokens = 0, asked = 0, taken = 0;
    for (int base = 0; base < p.B; base += BT_THREADS) {
        const int b = base + tid;
        const long long len = b < p.B ? max(__ldg(p.lens + b), 0) : 0;
        const long long add = b < p.B ? max(__ldg(p.change + b), 0) : 0;
        long long all, all_asked;
        const long long end = tokens + bt_scan(add, red, all);
        const bool fits = len + add <= room && end <= p.max_tokens;
        const int ask = fits ? bt_blocks(len + add, p.page) - bt_blocks(len, p.page) : 0;
        const long long upto = asked + bt_scan(ask, red, all_asked);
        const bool granted = fits && (ask == 0 || upto <= count);
        long long got;
        bt_scan(granted ? ask : 0, red, got);
        if (b < p.B) {
            s_end[b] = (int)min(end, 0x7fffffffll);
            s_off[b] = granted ? (int)(upto - ask) : -1;
            if (blockIdx.x == 0) {
                p.starts[b + 1] = s_end[b];
                p.lens_out[b] = (int)(granted ? len + add : len);
            }
        }
        tokens += all;
        asked += all_asked;
        taken += got;
    }
    if (blockIdx.x == 0 && tid == 0) {
        p.starts[0] = 0;
        *p.count_out = count - (int)taken;
    }
    __syncthreads();
    // ---- the new entries of the table, a warp per sequence
    const int lane = tid & 31;
    const int warps = (int)gridDim.x * (BT_THREADS / 32);
    for (int b = (int)blockIdx.x * (BT_THREADS / 32) + (tid >> 5); b < p.B; b += warps) {
        const int off = s_off[b];
        if (off < 0) continue;
        const long long len = max(__ldg(p.lens + b), 0);
        const int add = s_end[b] - (b ? s_end[b - 1] : 0);
        const int held = bt_blocks(len, p.page), ask = bt_blocks(len + add, p.page) - held;
        for (int j = lane; j < ask; j += 32) p.table[(size_t)b * p.width + held + j] = __ldg(p.free_blocks + (count - 1 - off - j));
    }
    // ---- the slot map, 4 tokens per thread
    const int last = p.B ? s_end[p.B - 1] : 0;
    const long long stride = (long long)gridDim.x * BT_THREADS * 4;
    for (long long t0 = ((long long)blockIdx.x * BT_THREADS + tid) * 4; t0 < p.max_tokens; t0 += stride) {
        int out[4] = {-1, -1, -1, -1};
        int b = -1, end = 0, len = 0, first = 0, off = -1, held = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int t = (int)(t0 + k);
            if (t0 + k >= p.max_tokens || t >= last) break;
            if (b < 0 || t >= end) {                   // first sequence whose tokens reach past t
                int lo = b < 0 ? 0 : b + 1, hi = p.B - 1;
                if (b >= 0 && s_end[lo] > t) hi = lo;
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (s_end[mid] > t) hi = mid;
                    else lo = mid + 1;
                }
                b = lo;
                end = s_end[b];
                first = b ? s_end[b - 1] : 0;
                off = s_off[b];
                len = max(__ldg(p.lens + b), 0);
                held = bt_blocks(len, p.page);
            }
            if (off < 0) continue;
            const int pos = len + (t - first);         // < width * page
            const int pg = pos / p.page;
            // entries that this launch writes are taken from where they come from
            const int blk = pg < held ? __ldg(p.table + (size_t)b * p.width + pg)
                                      : __ldg(p.free_blocks + (count - 1 - off - (pg - held)));
            out[k] = blk * p.page + (pos - pg * p.page);
        }
        if (t0 + 4 <= p.max_tokens && (reinterpret_cast<uintptr_t>(p.slots) & 15u) == 0) {
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
    __shared__ long long red[BT_THREADS / 32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x;
    const long long room = (long long)p.width * p.page;
    const int count = min(max(__ldg(p.free_count), 0), p.capacity);
    auto bounds = [&](int b, int& keep, int& left, int& held) {
        const int len = (int)min((long long)max(__ldg(p.lens + b), 0), room);
        keep = min(max(__ldg(p.change + b), 0), len);
        left = bt_blocks(keep, p.page);
        held = bt_blocks(len, p.page);
    };
    long long gone = 0;
    for (int base = 0; base < p.B; base += BT_THREADS) {
        const int b = base + tid;
        int keep = 0, left = 0, held = 0;
        if (b < p.B) bounds(b, keep, left, held);
        long long all;
        const long long upto = gone + bt_scan(held - left, red, all);
        if (b < p.B) {
            s_off[b] = (int)min(upto - (held - left), 0x7fffffffll);
            if (blockIdx.x == 0) p.lens_out[b] = keep;
        }
        gone += all;
    }
    if (blockIdx.x == 0 && tid == 0) *p.count_out = (int)min(count + gone, (long long)p.capacity);
    __syncthreads();
    const int lane = tid & 31;
    const int warps = (int)gridDim.x * (BT_THREADS / 32);
    for (int b = (int)blockIdx.x * (BT_THREADS / 32) + (tid >> 5); b < p.B; b += warps) {
        int keep, left, held;
        bounds(b, keep, left, held);
        const long long at = (long long)count + s_off[b];
        for (int j = left + lane; j < held; j += 32)
            if (at + (j - left) < p.capacity) p.free_blocks[at + (j - left)] = __ldg(p.table + (size_t)b * p.width + j);
    }
}

}  // namespace ftk
