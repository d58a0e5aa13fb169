// Append to a paged cache held in 8 bits: the tokens of a call, given with a slot each (block * page + offset), are
// rounded to the code type under one scale per (block, kv head) for K and one for V.
//
// Tokens with consecutive slots inside one block form a RUN. For a run with first offset o, per kv head and for K and V
// each (M = 127 for int8, 448 for e4m3):
//     old = o > 0 ? scale : 0;   new = max(old, max|x| / M);   codes of rows < o: round(code * old / new);
//     codes of the run's rows: round(x / new);   rows behind the run: untouched.
// round() is to the nearest code of the EXACT quotient, ties to even. The fast quotient x * (1 / new) may be off by two
// units in its last place, which matters next to a border between two codes: both x * r_lo and x * r_hi, r_lo and r_hi
// being 1 / new less and plus 2^-21 of it, are rounded, and where they give different codes the sign of
// fma(-border, new, x) decides, exactly. (Borders are not rare: two bfloat16 values have a quotient of two 8-bit numbers,
// and about 1 in 5000 of 448 m / M lies on one.) Rounding the rows before the run again is a map from 256 codes to 256
// codes, worked out once per run in float64 and applied bytewise; it runs only when the new tokens raise the scale. A
// block whose tokens are not all finite gets the scale NaN, and reads as NaN.
//
// Bound by HBM for prompts (2 bytes read and 1 written per 16-bit element: about 17 instructions an element may cost),
// by latency for a decode step. A CTA of 4 warps takes a window of tokens, finds its runs once, and appends them for 4
// (kv head, K or V) pairs. A warp copies rows with cp.async into a ring of two 4 KB slots of its own (a 16-row block of
// 128 half-precision elements fills one): the next run is on its way while one is looked through for its maximum and then
// rounded, both out of shared memory, and no register holds data in flight. Runs of up to two slots are a warp's own, a
// warp per pair and no barrier; longer ones the four warps share, pair by pair (up to 8 slots, a 128-row block of the same
// rows; a run beyond that is copied twice, the second time from L2).
// 266 k tokens of 8 x 128 half-precision values to int8 (1.64 GB): 257 us in a graph of four calls, 6390 GB/s, and 275 - 290 us
// when calls follow each other for long (copies alone, without the rounding, took 277 us then). (A CTA per run: 1476 us; a
// warp per run with its rows in registers: 546 us, 412 us with the runs of a window found at once.) 256 tokens of one step:
// 7.2 us, 32 tokens 3.5 us: a chain of dependent loads for the first token of a warp, 2 us of instructions for each further one.
#pragma once

#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "common.cuh"

namespace ftk {

struct AppendQ8Params {
    const void* x_new[2];     // k_new, v_new [N, Hkv, D]
    uint8_t* pool[2];         // K and V codes [blocks, Hkv, page, D]
    float* scales;            // [blocks, Hkv, 2]
    const int* slots;         // [N]; a slot outside [0, blocks * page) is passed over
    int N, Hkv, D, page;
    long long rows;           // blocks * page
    int window;               // tokens per CTA, at most AQ_THREADS
    int groups;               // CTAs per window: 4 of the 2 * Hkv (kv head, K or V) pairs each
};

constexpr int AQ_THREADS = 128, AQ_WARPS = AQ_THREADS / 32;
constexpr int AQ_BATCH = 256;                         // vectors per ring slot, 8 per lane
constexpr int AQ_SLOT_BYTES = AQ_BATCH * 16;
// Slots of a warp's ring. With four of them three CTAs fit an SM instead of five (266 k tokens: 422 us instead of 313); with
// one a warp waits for every run it begins (345 us).
constexpr int AQ_RING = 2;

template <typename T, int V> struct Vec;
template <> struct Vec<float, 4> {
    float4 d;
    __device__ __forceinline__ void load(const float* p) { d = *reinterpret_cast<const float4*>(p); }
    __device__ __forceinline__ void get(float (&x)[4]) const { x[0] = d.x; x[1] = d.y; x[2] = d.z; x[3] = d.w; }
};
template <typename T> __device__ __forceinline__ float2 widen2(uint32_t u);
template <> __device__ __forceinline__ float2 widen2<__nv_bfloat16>(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 widen2<__half>(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <typename T> struct Vec<T, 8> {
    uint4 d;
    __device__ __forceinline__ void load(const T* p) { d = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const float2 a = widen2<T>(d.x), b = widen2<T>(d.y), c = widen2<T>(d.z), e = widen2<T>(d.w);
        x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = c.x; x[5] = c.y; x[6] = e.x; x[7] = e.y;
    }
};
template <typename T> struct Vec<T, 4> {
    uint2 d;
    __device__ __forceinline__ void load(const T* p) { d = *reinterpret_cast<const uint2*>(p); }
    __device__ __forceinline__ void get(float (&x)[4]) const {
        const float2 a = widen2<T>(d.x), b = widen2<T>(d.y);
        x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
    }
};

// Largest magnitude so far and of a vector, two halves at a time; a NaN stays.
template <typename T> struct Top;
template <> struct Top<float> {
    uint32_t m = 0;                                   // as bits: their order is that of the values, infinities and NaN on top
    __device__ __forceinline__ void add(const Vec<float, 4>& v) {
        m = max(max(max(m, __float_as_uint(v.d.x) & 0x7fffffffu), max(__float_as_uint(v.d.y) & 0x7fffffffu, __float_as_uint(v.d.z) & 0x7fffffffu)),
                __float_as_uint(v.d.w) & 0x7fffffffu);
    }
    __device__ __forceinline__ uint32_t bits() const { return m; }
};
template <typename T> struct Top {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    uint32_t m = 0;
    __device__ __forceinline__ void two(uint32_t u) {
        const T2 r = __hmax2_nan(*reinterpret_cast<T2*>(&m), __habs2(*reinterpret_cast<T2*>(&u)));
        m = *reinterpret_cast<const uint32_t*>(&r);
    }
    __device__ __forceinline__ void add(const Vec<T, 8>& v) { two(v.d.x); two(v.d.y); two(v.d.z); two(v.d.w); }
    __device__ __forceinline__ void add(const Vec<T, 4>& v) { two(v.d.x); two(v.d.y); }
    __device__ __forceinline__ uint32_t bits() const {       // as float32 bits
        const float2 x = widen2<T>(m & 0x7fff7fffu);
        return max(__float_as_uint(x.x), __float_as_uint(x.y));
    }
};
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d)
        : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)), "l"(*reinterpret_cast<unsigned long long*>(&c)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d)
        : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
    return *reinterpret_cast<float2*>(&d);
}

// Rounding to codes. four(): four products x * r as packed codes; fast(): those for r_lo, described above, and whether the
// ones for r_hi differ (not 0). of_quotient(): a float64 quotient.
template <typename KV> struct Rounder;
template <> struct Rounder<int8_t> {
    static constexpr float M = 127.0f;
    // 1.5 * 2^23 + q: the sum's last bits are q rounded to a whole number, ties to even
    static __device__ __forceinline__ float2 sum2(const float* x, float r) {
        return fma2(make_float2(x[0], x[1]), make_float2(r, r), make_float2(12582912.0f, 12582912.0f));
    }
    static __device__ __forceinline__ uint32_t pack(float2 a, float2 b) {
        return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040),
                           __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
    }
    static __device__ __forceinline__ uint32_t four(const float* x, float r) { return pack(sum2(x, r), sum2(x + 2, r)); }
    static __device__ __forceinline__ uint32_t fast(const float* x, float r_lo, float r_hi, uint32_t& codes) {
        const float2 a = sum2(x, r_lo), b = sum2(x + 2, r_lo), c = sum2(x, r_hi), d = sum2(x + 2, r_hi);
        codes = pack(a, b);
        uint32_t differ = __float_as_uint(a.x) ^ __float_as_uint(c.x);
        differ |= __float_as_uint(a.y) ^ __float_as_uint(c.y);
        differ |= __float_as_uint(b.x) ^ __float_as_uint(d.x);
        differ |= __float_as_uint(b.y) ^ __float_as_uint(d.y);
        return differ;
    }
    static __device__ __forceinline__ float number(uint32_t c) { return (float)(int8_t)c; }
    static __device__ __forceinline__ double value(uint32_t c) { return (double)(int8_t)c; }
    static __device__ __forceinline__ uint32_t of_quotient(double q) {
        return (uint32_t)(int)fmin(fmax(rint(q), -127.0), 127.0) & 255u;
    }
};
template <> struct Rounder<__nv_fp8_e4m3> {
    static constexpr float M = 448.0f;
    static __device__ __forceinline__ uint32_t four(const float* x, float r) {
        const float2 a = mul2(make_float2(x[0], x[1]), make_float2(r, r)), b = mul2(make_float2(x[2], x[3]), make_float2(r, r));
        uint32_t codes;
        asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\tmov.b32 %0, {l, h};\n\t}"
            : "=r"(codes) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
        return codes;
    }
    static __device__ __forceinline__ uint32_t fast(const float* x, float r_lo, float r_hi, uint32_t& codes) {
        codes = four(x, r_lo);
        return codes ^ four(x, r_hi);
    }
    static __device__ __forceinline__ float number(uint32_t c) {
        return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
    }
    static __device__ __forceinline__ double value(uint32_t c) {
        return (double)__half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
    }
    // truncated to float32 with the last bit set when anything was cut off: a value that rounds to 4 significant bits
    // like the quotient itself
    static __device__ __forceinline__ uint32_t of_quotient(double q) {
        float f = __double2float_rz(q);
        if ((double)f != q) f = __uint_as_float(__float_as_uint(f) | 1u);
        return (uint32_t)__nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3);
    }
};
// Four values of which some round differently at r_lo and at r_hi (which gives the code of the larger magnitude): the
// border between the two codes has few bits, so the sign of x - border * s is exact in one fused multiply-add.
template <typename KV>
__device__ __noinline__ uint32_t four_settled(float x0, float x1, float x2, float x3, float s, float r_lo, float r_hi) {
    const float x[4] = {x0, x1, x2, x3};
    const uint32_t lo = Rounder<KV>::four(x, r_lo), hi = Rounder<KV>::four(x, r_hi);
    uint32_t w = lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t a = lo >> (8 * e) & 255u, b = hi >> (8 * e) & 255u;
        const float d = fmaf(-0.5f * (Rounder<KV>::number(a) + Rounder<KV>::number(b)), s, x[e]);
        const float beyond = x[e] < 0.0f ? -d : d;
        if (a != b && (beyond > 0.0f || (beyond == 0.0f && (a & 1u)))) w = (w & ~(255u << (8 * e))) | (b << (8 * e));
    }
    return w;
}
// Four quotients the long way, for scales that have no normal reciprocal.
template <typename KV>
__device__ __noinline__ uint32_t four_exact(float a, float b, float c, float d, float s) {
    return Rounder<KV>::of_quotient((double)a / (double)s) | (Rounder<KV>::of_quotient((double)b / (double)s) << 8) |
           (Rounder<KV>::of_quotient((double)c / (double)s) << 16) | (Rounder<KV>::of_quotient((double)d / (double)s) << 24);
}

struct Run {
    int first, n;             // its tokens
    int blk, off;             // and where they go
};

__device__ __forceinline__ void aq_wait(int pending) {           // all but the last `pending` groups of this thread's copies
    static_assert(AQ_RING == 2, "");
    if (pending <= 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
    else asm volatile("cp.async.wait_group 1;" ::: "memory");
}

// T: type of the new rows, KV: code type, V: elements per vector (16 bytes where D and the alignment allow, else 4). LONG: a
// run may have more batches than a warp's ring has slots (it costs registers and a division per batch).
template <typename T, typename KV, int V, bool LONG>
__global__ void __launch_bounds__(AQ_THREADS, 5) kv_append_q8_kernel(const AppendQ8Params p) {
    __shared__ __align__(16) uint8_t s_ring[AQ_WARPS][AQ_RING][AQ_SLOT_BYTES];
    __shared__ Run s_run[AQ_THREADS];
    __shared__ uint32_t s_goes_on[AQ_WARPS], s_begins[AQ_WARPS];
    __shared__ int s_beyond;
    __shared__ uint8_t s_map[AQ_WARPS][256];
    __shared__ uint32_t s_top[2][AQ_WARPS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int win = (int)(blockIdx.x / (unsigned)p.groups), group = (int)(blockIdx.x - (unsigned)win * p.groups);
    const long long w0 = (long long)win * p.window;
    const int here = (int)min((long long)p.window, p.N - w0);                 // tokens of this window

    // ---- the runs that begin in the window. A token goes on with the run before it if its slot is the next one of the
    // same block
    int slot = -1, before = -1;
    if (tid < here) {
        slot = __ldg(p.slots + w0 + tid);
        if (w0 + tid > 0) before = __ldg(p.slots + w0 + tid - 1);
    }
    const bool in_pool = slot >= 0 && slot < p.rows;
    const bool goes_on = in_pool && before >= 0 && before == slot - 1 && slot % p.page != 0;
    const uint32_t on = __ballot_sync(0xffffffffu, goes_on), begins = __ballot_sync(0xffffffffu, in_pool && !goes_on);
    if (lane == 0) { s_goes_on[warp] = on; s_begins[warp] = begins; }
    // how far the last token's run reaches beyond the window (warp 0; one step for blocks of up to 32 rows)
    if (warp == 0) {
        const int last = __ldg(p.slots + w0 + here - 1);
        int beyond = 0;
        if (last >= 0 && last < p.rows) {
            const int room = (int)min((long long)(p.page - 1 - last % p.page), p.N - (w0 + here));
            while (beyond < room) {
                const int j = beyond + lane;
                const bool ok = j < room && __ldg(p.slots + w0 + here + j) == last + 1 + j;
                const uint32_t m = __ballot_sync(0xffffffffu, ok);
                beyond += m == 0xffffffffu ? 32 : __ffs(~m) - 1;
                if (m != 0xffffffffu) break;
            }
        }
        if (lane == 0) s_beyond = beyond;
    }
    __syncthreads();
    int runs = 0, rank = 0;
#pragma unroll
    for (int k = 0; k < AQ_WARPS; ++k) {
        if (k < warp) rank += __popc(s_begins[k]);
        runs += __popc(s_begins[k]);
    }
    if (in_pool && !goes_on) {
        int n = 1;                                    // up to the first token behind that does not go on
        while (tid + n < here && (s_goes_on[(tid + n) >> 5] >> ((tid + n) & 31) & 1u)) ++n;
        if (tid + n == here) n += s_beyond;
        const int blk = slot / p.page;
        s_run[rank + __popc(begins & ((1u << lane) - 1u))] = Run{(int)(w0 + tid), n, blk, slot - blk * p.page};
    }
    __syncthreads();
    auto copy = [](uint32_t dst, const T* from) {
        if constexpr (V * sizeof(T) == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(from) : "memory");
        else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(from) : "memory");
    };
    // ---- the warp's copies, a batch of 256 vectors at a time. A run of up to AQ_RING batches is a warp's own, for the
    // pair group * 4 + warp. A longer one is the CTA's, for the four pairs in turn, and the warps share its batches; if a
    // warp's share is more than its ring holds it copies it twice, for the maximum and for the rounding. A run's rows are
    // one stretch of its block: vector v goes to byte V * v behind the first.
    const int pairs = min(4, 2 * p.Hkv - group * 4);
    uint8_t* my = s_ring[warp][0] + lane * (V * sizeof(T));
    constexpr int PER = AQ_BATCH / 32;                // vectors per lane and batch, 32 apart
    const int vpr = p.D / V;                          // vectors per row
    const int jump = 32 / vpr, rest = 32 - jump * vpr;
    const size_t stride = (size_t)p.Hkv * p.D;
    struct Share {
        int nb, first, every, count, times;           // batches; this warp's: first, first + every, ..., `count`, copied `times`
        bool own;                                     // the run is the warp's own
    };
    auto share = [&](const Run& r) {
        Share s;
        s.nb = (r.n * vpr + AQ_BATCH - 1) / AQ_BATCH;
        s.own = !LONG || s.nb <= AQ_RING;
        s.first = s.own ? 0 : warp;
        s.every = s.own ? 1 : AQ_WARPS;
        s.count = s.own ? s.nb : (s.nb - warp + AQ_WARPS - 1) / AQ_WARPS;
        s.times = s.own || s.nb <= AQ_RING * AQ_WARPS ? 1 : 2;
        if (LONG && s.own && warp >= pairs) s.count = 0;
        return s;
    };
    if (!LONG && warp >= pairs) return;
    const int lane_row = lane / vpr, lane_col = lane - lane_row * vpr;
    const int batch_rows = AQ_BATCH / vpr, batch_cols = AQ_BATCH - batch_rows * vpr;
    int at_run = 0, at_pair = 0, at_batch = 0, issued = 0;      // what is to be requested next
    auto request = [&]() {                            // one batch into the next slot (at the end: an empty group)
        while (at_run < runs) {
            const Run r = s_run[at_run];
            const Share sh = share(r);
            if (LONG && at_batch >= sh.count * sh.times) {      // the next pair, or the next run
                at_batch = 0;
                if (sh.own || ++at_pair == pairs) { at_pair = 0; ++at_run; }
                continue;
            }
            const int pair = group * 4 + (sh.own ? warp : at_pair);
            const int which = pair >= p.Hkv, head = pair - which * p.Hkv;
            int row, col;                             // this lane's first vector
            if constexpr (LONG) {
                const int v = (sh.first + (at_batch < sh.count ? at_batch : at_batch - sh.count) * sh.every) * AQ_BATCH + lane;
                row = v / vpr;
                col = v - row * vpr;
            } else {
                row = lane_row + at_batch * batch_rows;
                col = lane_col + at_batch * batch_cols;
                if (col >= vpr) { col -= vpr; ++row; }
            }
            const uint32_t dst = (uint32_t)__cvta_generic_to_shared(my + (issued & (AQ_RING - 1)) * AQ_SLOT_BYTES);
            const T* from = static_cast<const T*>(which ? p.x_new[1] : p.x_new[0]) + (size_t)(r.first + row) * stride + (size_t)head * p.D + col * V;
            if (rest == 0) {                          // a lane stays in its column
                const size_t step = (size_t)jump * stride;
#pragma unroll
                for (int h = 0; h < PER; ++h) {
                    if (row + h * jump < r.n) copy(dst + h * 32 * (V * (int)sizeof(T)), from);
                    from += step;
                }
            } else {
#pragma unroll
                for (int h = 0; h < PER; ++h) {
                    if (row < r.n) copy(dst + h * 32 * (V * (int)sizeof(T)), from);
                    row += jump;
                    col += rest;
                    from += (size_t)jump * stride + rest * V;
                    if (col >= vpr) { col -= vpr; ++row; from += stride - p.D; }
                }
            }
            ++at_batch;
            if (!LONG && at_batch == sh.count) { at_batch = 0; ++at_run; }
            break;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        ++issued;
    };
    for (int i = 0; i < AQ_RING; ++i) request();
    int used = 0, turn = 0;                           // batches done with (`issued` is always used + AQ_RING); CTA runs so far
    for (int k = 0; k < runs; ++k) {
        const Run run = s_run[k];
        const Share sh = share(run);
        const int off = run.off, total = run.n * vpr;
        const bool resident = sh.times == 1;
        for (int q = 0; q < (sh.own ? 1 : pairs); ++q) {
            if (LONG && sh.own && warp >= pairs) break;
            const int pair = group * 4 + (sh.own ? warp : q);
            const int which = pair >= p.Hkv, head = pair - which * p.Hkv;
            const size_t bh = (size_t)run.blk * p.Hkv + head;
            uint8_t* dst = (which ? p.pool[1] : p.pool[0]) + bh * p.page * p.D;
            float* scale = p.scales + bh * 2 + which;
            const float old = off > 0 ? __ldcg(scale) : 0.0f;
            // f(h) for this lane's vectors of batch i, whole batches without a test
            auto each = [&](int i, auto f) {
                if ((i + 1) * AQ_BATCH <= total) {
#pragma unroll
                    for (int h = 0; h < PER; ++h) f(h);
                } else {
#pragma unroll
                    for (int h = 0; h < PER; ++h) {
                        if (i * AQ_BATCH + h * 32 >= total) break;
                        if (i * AQ_BATCH + h * 32 + lane < total) f(h);
                    }
                }
            };
            auto slot_of = [&](int j) { return my + ((used + (resident ? j : 0)) & (AQ_RING - 1)) * AQ_SLOT_BYTES; };
            auto vector = [](const uint8_t* at, int h) {
                Vec<T, V> v;
                v.load(reinterpret_cast<const T*>(at + h * 32 * (V * (int)sizeof(T))));
                return v;
            };

            // ---- the largest magnitude
            Top<T> most;
            if (resident) aq_wait(AQ_RING - sh.count);
            for (int j = 0; j < sh.count; ++j) {
                if (!resident) aq_wait(AQ_RING - 1);
                const uint8_t* at = slot_of(j);
                each(sh.first + j * sh.every, [&](int h) { most.add(vector(at, h)); });
                if (!resident) { ++used; request(); }
            }
            uint32_t top = __reduce_max_sync(0xffffffffu, most.bits());
            if (!sh.own) {
                if (lane == 0) s_top[turn & 1][warp] = top;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < AQ_WARPS; ++w) top = max(top, s_top[turn & 1][w]);
                ++turn;
            }
            float now = fmaxf(old, __fdiv_rn(__uint_as_float(top), Rounder<KV>::M));
            if (top >= 0x7f800000u || old != old) now = __uint_as_float(0x7fc00000u);
            const bool fine = now > 0.0f && now < INFINITY;

            // ---- rows before the run, when the scale rose
            if (off > 0 && fine && now != old) {
                uint8_t* map = s_map[sh.own ? warp : 0];
                const int t = sh.own ? lane : tid, every = sh.own ? 32 : AQ_THREADS;
                if (!sh.own) __syncthreads();         // (warp 0 may be at its own run's map)
                for (int c = t; c < 256; c += every)
                    map[c] = (uint8_t)Rounder<KV>::of_quotient(Rounder<KV>::value((uint32_t)c) * (double)old / (double)now);
                if (sh.own) __syncwarp();
                else __syncthreads();
                auto again = [&](uint32_t u) {
                    return (uint32_t)map[u & 255u] | ((uint32_t)map[(u >> 8) & 255u] << 8) | ((uint32_t)map[(u >> 16) & 255u] << 16) |
                           ((uint32_t)map[u >> 24] << 24);
                };
                if (((reinterpret_cast<uintptr_t>(dst) | (uintptr_t)p.D) & 15u) == 0) {
                    uint4* quads = reinterpret_cast<uint4*>(dst);
                    const int count = off * (p.D >> 4);
#pragma unroll 4
                    for (int c = t; c < count; c += every) {
                        const uint4 u = quads[c];
                        quads[c] = make_uint4(again(u.x), again(u.y), again(u.z), again(u.w));
                    }
                } else {
                    uint32_t* words = reinterpret_cast<uint32_t*>(dst);
                    const int count = off * (p.D >> 2);
#pragma unroll 4
                    for (int c = t; c < count; c += every) words[c] = again(words[c]);
                }
                if (sh.own) __syncwarp();             // the map is free for the next run
                else __syncthreads();
            }
            // (every load of the scale precedes this store: the reduction above is in between)
            if ((sh.own ? lane : tid) == 0) *scale = now;

            // ---- the run's rows. Where 1 / new would not be a normal number, or new itself has few bits, all go the exact way
            const uint32_t unusual = now > 1e-30f && now < 1e30f ? 0u : 1u;
            const float r = 1.0f / now;
            const float r_lo = r - r * 4.76837158e-7f, r_hi = r + r * 4.76837158e-7f;          // 2^-21
            uint8_t* out = dst + (size_t)off * p.D + lane * V;
            for (int j = 0; j < sh.count; ++j) {
                if (!resident) aq_wait(AQ_RING - 1);
                const int i = sh.first + j * sh.every;
                const uint8_t* at = slot_of(j);
                uint8_t* to = out + (size_t)i * (AQ_BATCH * V);
                each(i, [&](int h) {
                    float x[V];
                    vector(at, h).get(x);
                    uint32_t w[V / 4], differ = unusual;
#pragma unroll
                    for (int e = 0; e < V / 4; ++e) differ |= Rounder<KV>::fast(x + 4 * e, r_lo, r_hi, w[e]);
                    if (differ) {
#pragma unroll
                        for (int e = 0; e < V / 4; ++e) {
                            if (!unusual) w[e] = four_settled<KV>(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3], now, r_lo, r_hi);
                            else w[e] = fine ? four_exact<KV>(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3], now) : 0u;
                        }
                    }
                    if constexpr (V == 8) *reinterpret_cast<uint2*>(to + h * (32 * V)) = make_uint2(w[0], w[1]);
                    else *reinterpret_cast<uint32_t*>(to + h * (32 * V)) = w[0];
                });
                if (!resident) { ++used; request(); }
            }
            if (resident)
                for (int j = 0; j < sh.count; ++j) { ++used; request(); }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

}  // namespace ftk
