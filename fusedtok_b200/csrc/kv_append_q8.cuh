// Append to a paged cache held in 8 bits: the tokens of a call, given with a slot each (block * page + offset), are
// rounded to the code type under one scale per (block, kv head) for K and one for V.
//
// Tokens with consecutive slots inside one block form a RUN. For a run with first offset o, per kv head and for K and V
// each (M = 127 for int8, 448 for e4m3):
//     old = o > 0 ? scale : 0;   new = max(old, max|x| / M);   codes of rows < o: round(code * old / new);
//     codes of the run's rows: round(x / new);   rows behind the run: untouched.
// round() is to the nearest code of the EXACT quotient, ties to even. The fast quotient x * (1 / new) may be off by two
// units in its last place, which matters next to a border between two codes: both x * r_lo and x * r_hi, r_lo and r_hi
// being 1 / new less and plus 2^-21 of it, are rounded, and where they give different codes (about 1 value in 10^5) the
// quotient is worked out in float64. Rounding the rows before the run again is a map from 256 codes to 256 codes, worked
// out once per run in float64 and applied bytewise; it runs only when the new tokens raise the scale. A block whose
// tokens are not all finite gets the scale NaN, and reads as NaN.
//
// Bound by HBM for prompts (2 bytes read and 1 written per 16-bit element: about 17 instructions an element may cost),
// by latency for a decode step. A team of TEAM threads takes a (run, kv head, K or V): the run's rows are read once,
// 16 bytes per thread with up to 8 loads in flight, and kept in registers between the maximum and the rounding. A warp
// holds 4 KB, a 16-row block of 128 half-precision elements, and needs no barrier; larger blocks take a CTA of 4 warps (a
// 64-row block of the same rows); what does not fit is read again, from L2. With many tokens a team looks after a window
// of tokens and its runs in turn.
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
    int window, windows;      // tokens per team, at most TEAM, and teams along the tokens
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

// Largest magnitude of a vector as bits (their order is that of the values, infinities and NaN on top): of halves as
// halves, two at a time.
template <typename T, int V> __device__ __forceinline__ uint32_t top_bits(const Vec<T, V>& v) {
    if constexpr (std::is_same<T, float>::value) {
        return max(max(__float_as_uint(v.d.x) & 0x7fffffffu, __float_as_uint(v.d.y) & 0x7fffffffu),
                   max(__float_as_uint(v.d.z) & 0x7fffffffu, __float_as_uint(v.d.w) & 0x7fffffffu));
    } else if constexpr (V == 8) {
        return __vmaxu2(__vmaxu2(v.d.x & 0x7fff7fffu, v.d.y & 0x7fff7fffu), __vmaxu2(v.d.z & 0x7fff7fffu, v.d.w & 0x7fff7fffu));
    } else {
        return __vmaxu2(v.d.x & 0x7fff7fffu, v.d.y & 0x7fff7fffu);
    }
}
template <typename T> __device__ __forceinline__ uint32_t max_bits(uint32_t a, uint32_t b) {
    if constexpr (std::is_same<T, float>::value) return max(a, b);
    else return __vmaxu2(a, b);
}
// ... and as float32 bits
template <typename T> __device__ __forceinline__ uint32_t wide_bits(uint32_t a) {
    if constexpr (std::is_same<T, float>::value) return a;
    else {
        const float2 x = widen2<T>(a);
        return max(__float_as_uint(x.x), __float_as_uint(x.y));
    }
}

// Rounding to codes. fast(): four quotients x / s as packed codes, r_lo and r_hi as described above; false where they
// straddle a border. of_quotient(): a float64 quotient.
template <typename KV> struct Rounder;
template <> struct Rounder<int8_t> {
    static constexpr float M = 127.0f;
    static __device__ __forceinline__ bool fast(const float* x, float r_lo, float r_hi, uint32_t& codes) {
        // 1.5 * 2^23 + q: the sum's last bits are q rounded to a whole number, ties to even
        uint32_t c[4], differ = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            c[e] = __float_as_uint(fmaf(x[e], r_lo, 12582912.0f));
            differ |= c[e] ^ __float_as_uint(fmaf(x[e], r_hi, 12582912.0f));
        }
        codes = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
        return differ == 0;
    }
    static __device__ __forceinline__ double value(uint32_t c) { return (double)(int8_t)c; }
    static __device__ __forceinline__ uint32_t of_quotient(double q) {
        return (uint32_t)(int)fmin(fmax(rint(q), -127.0), 127.0) & 255u;
    }
};
template <> struct Rounder<__nv_fp8_e4m3> {
    static constexpr float M = 448.0f;
    static __device__ __forceinline__ uint32_t four(const float* x, float r) {
        return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[0] * r, x[1] * r), __NV_SATFINITE, __NV_E4M3) |
               ((uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[2] * r, x[3] * r), __NV_SATFINITE, __NV_E4M3) << 16);
    }
    static __device__ __forceinline__ bool fast(const float* x, float r_lo, float r_hi, uint32_t& codes) {
        codes = four(x, r_lo);
        return codes == four(x, r_hi);
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
template <typename KV>
__device__ __noinline__ uint32_t four_exact(float a, float b, float c, float d, float s) {
    return Rounder<KV>::of_quotient((double)a / (double)s) | (Rounder<KV>::of_quotient((double)b / (double)s) << 8) |
           (Rounder<KV>::of_quotient((double)c / (double)s) << 16) | (Rounder<KV>::of_quotient((double)d / (double)s) << 24);
}

// T: type of the new rows, KV: code type, V: elements per vector (16 bytes where D and the alignment allow, else 4
// elements), TEAM: threads per (run, kv head, K or V), a warp or the CTA.
template <typename T, typename KV, int V, int TEAM>
__global__ void __launch_bounds__(AQ_THREADS) kv_append_q8_kernel(const AppendQ8Params p) {
    constexpr int TEAMS = AQ_THREADS / TEAM, WARPS = TEAM / 32;
    __shared__ int s_run[TEAMS][TEAM];
    __shared__ int s_runs[TEAMS], s_n[TEAMS];
    __shared__ uint32_t s_top[AQ_THREADS / 32];
    __shared__ uint8_t s_map[TEAMS][256];
    auto sync = [] {
        if constexpr (TEAM == 32) __syncwarp();
        else __syncthreads();
    };
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int team = threadIdx.x / TEAM, tid = threadIdx.x % TEAM, lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * TEAMS + team;
    if (item >= (long long)p.windows * 2 * p.Hkv) return;                // (whole teams leave)
    const int head = (int)(item % p.Hkv), which = (int)(item / p.Hkv & 1);
    const T* x_new = static_cast<const T*>(which ? p.x_new[1] : p.x_new[0]);
    uint8_t* pool = which ? p.pool[1] : p.pool[0];
    const int vpr = p.D / V;                          // vectors per row
    const int jump = TEAM / vpr, rest = TEAM - jump * vpr;
    const size_t stride = (size_t)p.Hkv * p.D;

    // ---- first tokens of the runs in this team's window
    if (tid == 0) s_runs[team] = 0;
    sync();
    const long long i0 = item / (2 * p.Hkv) * p.window + tid;
    if (tid < p.window && i0 < p.N) {
        const int slot = __ldg(p.slots + i0);
        const int before = i0 ? __ldg(p.slots + i0 - 1) : -1;
        if (slot >= 0 && slot < p.rows && !(before >= 0 && before == slot - 1 && slot % p.page != 0))
            s_run[team][atomicAdd(&s_runs[team], 1)] = (int)i0;
    }
    sync();
    const int runs = s_runs[team];
    for (int k = 0; k < runs; ++k) {
        const int i = s_run[team][k];
        const int slot = __ldg(p.slots + i);
        const int blk = slot / p.page, off = slot - blk * p.page;
        const int most = min(p.page - off, p.N - i);
        const size_t bh = (size_t)blk * p.Hkv + head;
        uint8_t* dst = pool + bh * p.page * p.D;
        float* scale = p.scales + bh * 2 + which;
        const float old = off > 0 ? *scale : 0.0f;
        int n = most;
        if (most > 1) {
            if (tid == 0) s_n[team] = most;
            sync();
            for (int j = 1 + tid; j < most; j += TEAM)
                if (__ldg(p.slots + i + j) != slot + j) {
                    atomicMin(&s_n[team], j);
                    break;
                }
            sync();
            n = s_n[team];
        }
        const T* src = x_new + (size_t)i * stride + (size_t)head * p.D;

        // ---- the largest magnitude
        Vec<T, V> held[AQ_HELD];
        uint32_t top = 0;
        const int row0 = tid / vpr, col0 = tid - row0 * vpr;
        int row = row0, col = col0;
        auto step = [&](int& r, int& c) {
            r += jump;
            c += rest;
            if (c >= vpr) { c -= vpr; ++r; }
        };
#pragma unroll
        for (int h = 0; h < AQ_HELD; ++h) {
            held[h] = Vec<T, V>{};
            if (row < n) held[h].load(src + (size_t)row * stride + col * V);
            step(row, col);
        }
#pragma unroll
        for (int h = 0; h < AQ_HELD; ++h) top = max_bits<T>(top, top_bits<T, V>(held[h]));
        while (row < n) {
            Vec<T, V> more;
            more.load(src + (size_t)row * stride + col * V);
            top = max_bits<T>(top, top_bits<T, V>(more));
            step(row, col);
        }
        top = __reduce_max_sync(0xffffffffu, wide_bits<T>(top));
        if constexpr (WARPS > 1) {
            if (lane == 0) s_top[threadIdx.x >> 5] = top;
            sync();
#pragma unroll
            for (int wv = 0; wv < WARPS; ++wv) top = max(top, s_top[wv]);
        }
        float now = fmaxf(old, __fdiv_rn(__uint_as_float(top), Rounder<KV>::M));
        if (top >= 0x7f800000u || old != old) now = __uint_as_float(0x7fc00000u);
        const bool fine = now > 0.0f && now < INFINITY;

        // ---- rows before the run, when the scale rose
        if (off > 0 && fine && now != old) {
            for (int c = tid; c < 256; c += TEAM)
                s_map[team][c] = (uint8_t)Rounder<KV>::of_quotient(Rounder<KV>::value((uint32_t)c) * (double)old / (double)now);
            sync();
            const uint8_t* map = s_map[team];
            uint32_t* words = reinterpret_cast<uint32_t*>(dst);
            const int count = off * (p.D >> 2);
#pragma unroll 4
            for (int c = tid; c < count; c += TEAM) {
                const uint32_t u = words[c];
                words[c] = (uint32_t)map[u & 255u] | ((uint32_t)map[(u >> 8) & 255u] << 8) |
                           ((uint32_t)map[(u >> 16) & 255u] << 16) | ((uint32_t)map[u >> 24] << 24);
            }
        }
        // (in a warp team the loads of `scale` by the other lanes precede this store: the reduction above is in between)
        if (tid == 0) *scale = now;

        // ---- the run's rows. Where 1 / new would not be a normal number, or new itself has few bits, all go the exact way
        const bool plain = now > 1e-30f && now < 1e30f;
        const float r = 1.0f / now;
        const float r_lo = r - r * 4.76837158e-7f, r_hi = r + r * 4.76837158e-7f;          // 2^-21
        auto put = [&](const Vec<T, V>& v, int rr, int c) {
            float x[V];
            v.get(x);
            uint32_t w[V / 4];
#pragma unroll
            for (int e = 0; e < V / 4; ++e) {
                const float* y = x + 4 * e;
                if (!(Rounder<KV>::fast(y, r_lo, r_hi, w[e]) && plain)) w[e] = fine ? four_exact<KV>(y[0], y[1], y[2], y[3], now) : 0u;
            }
            uint8_t* to = dst + (size_t)(off + rr) * p.D + c * V;
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
        sync();                                       // s_n, s_top and s_map are free for the next run
    }
}

}  // namespace ftk
