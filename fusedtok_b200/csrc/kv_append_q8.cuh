// Append to a paged cache held in 8 bits: the tokens of a call, given with a slot each (block * page + offset), are
// rounded to the code type under one scale per (block, kv head) for K and one for V.
//
// Tokens with consecutive slots inside one block form a RUN. For a run with first offset o, per kv head and for K and V
// each (M = 127 for int8, 448 for e4m3):
//     old = o > 0 ? scale : 0;   new = max(old, max|x| / M);   codes of rows < o: round(code * old / new);
//     codes of the run's rows: round(x / new);   rows behind the run: untouched.
// round() is to the nearest code of the EXACT quotient, ties to even. The fast quotient x * (1 / new) may be off by two
// units in its last place, which matters next to a border between two codes, so the border is decided exactly: for
// int8 by the sign of fma(-(k + 1/2), new, x), for e4m3 by a float64 quotient in the few cases (about 1 in 10^5) whose
// fast one lies within 4 units of a border or below the smallest normal code. Rounding the rows before the run again
// is a map from 256 codes to 256 codes, worked out once per run in float64 and applied bytewise; it runs only when the
// new tokens raise the scale. A block whose tokens are not all finite gets the scale NaN, and reads as NaN.
//
// Bound by HBM for prompts (2 bytes read and 1 written per 16-bit element), by latency for a decode step. One CTA per
// (run, kv head, K or V): the run's rows are read once, 16 bytes per thread with up to 8 loads in flight, and kept in
// registers between the maximum and the rounding (a 64-row block of 128 half-precision elements fits exactly; what does
// not fit is read again, from L2). With many tokens a CTA looks after a window of tokens and its runs in turn.
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
};

constexpr int AQ_THREADS = 128;
constexpr int AQ_HELD = 8;    // vectors a thread keeps

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

// Rounding of x / s to a code; r is 1 / s. (s > 0 and finite, |x / s| at most about M)
template <typename KV> struct Rounder;
template <> struct Rounder<int8_t> {
    static constexpr float M = 127.0f;
    static __device__ __forceinline__ uint32_t code(float x, float s, float r) {
        // h is the border nearest to the quotient; which side of it x / s lies on is the sign of x - h s, exactly
        const float h = floorf(x * r) + 0.5f;
        const float d = fmaf(-h, s, x);
        float t = h + copysignf(0.5f, d);
        if (d == 0.0f) t = rintf(h);
        t = fminf(fmaxf(t, -127.0f), 127.0f);
        return (uint32_t)(int)t & 255u;
    }
    static __device__ __forceinline__ uint32_t pair(float a, float b, float s, float r) {
        return code(a, s, r) | (code(b, s, r) << 8);
    }
    static __device__ __forceinline__ double value(uint32_t c) { return (double)(int8_t)c; }
    static __device__ __forceinline__ uint32_t of_quotient(double q) {
        return (uint32_t)(int)fmin(fmax(rint(q), -127.0), 127.0) & 255u;
    }
};
template <> struct Rounder<__nv_fp8_e4m3> {
    static constexpr float M = 448.0f;
    // nearest code of a float64 quotient: truncated to float32 with the last bit set when anything was cut off, a value
    // that rounds to 4 significant bits like the quotient itself
    static __device__ __noinline__ uint32_t of_quotient(double q) {
        float f = __double2float_rz(q);
        if ((double)f != q) f = __uint_as_float(__float_as_uint(f) | 1u);
        return (uint32_t)__nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3);
    }
    static __device__ __forceinline__ double value(uint32_t c) {
        return (double)__half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
    }
    static __device__ __forceinline__ bool near_border(float y) {
        const uint32_t u = __float_as_uint(y) & 0x7fffffffu;
        // borders of normal codes: bit 19 set, the 19 bits below it clear. Below 2^-6 the codes are evenly spaced.
        const uint32_t low = (u + 4u) & 0xfffffu;
        return (low - 0x80000u) <= 8u || (u < 0x3c800000u && u != 0u);
    }
    static __device__ __forceinline__ uint32_t pair(float a, float b, float s, float r) {
        const float ya = a * r, yb = b * r;
        uint32_t c = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(ya, yb), __NV_SATFINITE, __NV_E4M3);
        if (near_border(ya)) c = (c & 0xff00u) | of_quotient((double)a / (double)s);
        if (near_border(yb)) c = (c & 0x00ffu) | (of_quotient((double)b / (double)s) << 8);
        return c;
    }
};

// T: type of the new rows, KV: code type, V: elements per vector (16 bytes where D and the alignment allow, else 4 elements).
template <typename T, typename KV, int V>
__global__ void __launch_bounds__(AQ_THREADS) kv_append_q8_kernel(const AppendQ8Params p) {
    __shared__ int s_run[AQ_THREADS];
    __shared__ int s_runs, s_n;
    __shared__ uint32_t s_top[AQ_THREADS / 32];
    __shared__ uint8_t s_map[256];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int head = blockIdx.y, which = blockIdx.z;
    const T* x_new = static_cast<const T*>(p.x_new[which]);
    const int vpr = p.D / V;                          // vectors per row
    const int jump = AQ_THREADS / vpr, rest = AQ_THREADS - jump * vpr;
    const size_t stride = (size_t)p.Hkv * p.D;

    // ---- first tokens of the runs in this CTA's window
    if (tid == 0) s_runs = 0;
    __syncthreads();
    const long long i0 = (long long)blockIdx.x * p.window + tid;
    if (tid < p.window && i0 < p.N) {
        const int slot = __ldg(p.slots + i0);
        if (slot >= 0 && slot < p.rows) {
            const int before = i0 ? __ldg(p.slots + i0 - 1) : -1;
            if (!(before >= 0 && before == slot - 1 && slot % p.page != 0)) s_run[atomicAdd(&s_runs, 1)] = (int)i0;
        }
    }
    __syncthreads();
    const int runs = s_runs;
    for (int k = 0; k < runs; ++k) {
        const int i = s_run[k];
        const int slot = __ldg(p.slots + i);
        const int blk = slot / p.page, off = slot - blk * p.page;
        const int most = min(p.page - off, p.N - i);
        if (tid == 0) s_n = most;
        __syncthreads();
        for (int j = 1 + tid; j < most; j += AQ_THREADS)
            if (__ldg(p.slots + i + j) != slot + j) {
                atomicMin(&s_n, j);
                break;
            }
        __syncthreads();
        const int n = s_n;
        const T* src = x_new + (size_t)i * stride + (size_t)head * p.D;
        const size_t bh = (size_t)blk * p.Hkv + head;
        uint8_t* dst = p.pool[which] + bh * p.page * p.D;
        float* scale = p.scales + bh * 2 + which;
        const float old = off > 0 ? *scale : 0.0f;

        // ---- the largest magnitude, as bits (their order is that of the values, infinities and NaN on top)
        Vec<T, V> held[AQ_HELD];
        uint32_t top = 0;
        int row = tid / vpr, col = tid - row * vpr;
        const int row0 = row, col0 = col;
        auto step = [&](int& r, int& c) {
            r += jump;
            c += rest;
            if (c >= vpr) { c -= vpr; ++r; }
        };
#pragma unroll
        for (int h = 0; h < AQ_HELD; ++h) {
            if (row < n) held[h].load(src + (size_t)row * stride + col * V);
            step(row, col);
        }
        {
            int r = row0, c = col0;
#pragma unroll
            for (int h = 0; h < AQ_HELD; ++h) {
                if (r < n) {
                    float x[V];
                    held[h].get(x);
#pragma unroll
                    for (int e = 0; e < V; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
                }
                step(r, c);
            }
        }
        while (row < n) {
            Vec<T, V> more;
            more.load(src + (size_t)row * stride + col * V);
            float x[V];
            more.get(x);
#pragma unroll
            for (int e = 0; e < V; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
            step(row, col);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) s_top[warp] = top;
        __syncthreads();
#pragma unroll
        for (int wv = 0; wv < AQ_THREADS / 32; ++wv) top = max(top, s_top[wv]);
        float now = fmaxf(old, __fdiv_rn(__uint_as_float(top), Rounder<KV>::M));
        if (top >= 0x7f800000u || old != old) now = __uint_as_float(0x7fc00000u);
        const bool fine = now > 0.0f && now < INFINITY;

        // ---- rows before the run, when the scale rose
        if (off > 0 && fine && now != old) {
            for (int c = tid; c < 256; c += AQ_THREADS)
                s_map[c] = (uint8_t)Rounder<KV>::of_quotient(Rounder<KV>::value((uint32_t)c) * (double)old / (double)now);
            __syncthreads();
            uint32_t* words = reinterpret_cast<uint32_t*>(dst);
            const int count = off * (p.D >> 2);
#pragma unroll 4
            for (int c = tid; c < count; c += AQ_THREADS) {
                const uint32_t u = words[c];
                words[c] = (uint32_t)s_map[u & 255u] | ((uint32_t)s_map[(u >> 8) & 255u] << 8) |
                           ((uint32_t)s_map[(u >> 16) & 255u] << 16) | ((uint32_t)s_map[u >> 24] << 24);
            }
        }
        if (tid == 0) *scale = now;

        // ---- the run's rows. Scales below 2^-100 are moved up first (the border test must not underflow)
        const float up = now < 7.9e-31f ? 1152921504606846976.0f : 1.0f;       // 2^60
        const float s = now * up, r1 = fine ? 1.0f / s : 0.0f;
        auto put = [&](const Vec<T, V>& v, int r, int c) {
            float x[V];
            v.get(x);
            uint32_t w[V / 4];
#pragma unroll
            for (int e = 0; e < V / 4; ++e) {
                w[e] = 0;
                if (fine)
                    w[e] = Rounder<KV>::pair(x[4 * e] * up, x[4 * e + 1] * up, s, r1) |
                           (Rounder<KV>::pair(x[4 * e + 2] * up, x[4 * e + 3] * up, s, r1) << 16);
            }
            uint8_t* to = dst + (size_t)(off + r) * p.D + c * V;
            if constexpr (V == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint32_t*>(to) = w[0];
        };
        row = row0;
        col = col0;
#pragma unroll
        for (int h = 0; h < AQ_HELD; ++h) {
            if (row < n) put(held[h], row, col);
            step(row, col);
        }
        while (row < n) {
            Vec<T, V> more;
            more.load(src + (size_t)row * stride + col * V);
            put(more, row, col);
            step(row, col);
        }
        __syncthreads();                              // s_n, s_top and s_map are free for the next run
    }
}

}  // namespace ftk
