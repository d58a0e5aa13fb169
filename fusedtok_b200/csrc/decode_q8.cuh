// Decode attention over a paged cache held in 8 bits (int8 or e4m3 codes) with one scale per (block, kv head)
// for K and one for V: out = softmax_t(ks[t] * q . k8_t / sqrt(D)) . (vs[t] * v8_t).
//
// What bounds it: HBM. A cache row is 2 * D bytes for 4 * G * D flops (G query heads per kv head). Half the bytes of a
// 16-bit cache for the same arithmetic, so the conversions count: every code becomes a half exactly once, in
// registers, on its way from shared memory to the tensor cores. Both code types are exact in half precision, and
// the scales never touch the codes: ks multiplies the finished score, vs is folded into the softmax weight.
//
// Structure (see decode_tc.cuh for the parts both share): one persistent CTA per SM; all tiles of all units cut at equal
// cost into one range per CTA, worked out on the device from lens. Four kinds of warps, every one walking the range for
// itself:
//  * 4 producer warps stream 64-row tiles with TMA into a ring in shared memory, every fourth tile each;
//  * 8 consumer warps, in groups of two that take tiles in turn, keep an online softmax over their rows in registers.
//    Nothing makes them meet: at the end of a segment (the range's part of a unit) a warp leaves its state (m, l, O) in a
//    buffer and goes on;
//  * 2 helper warps prepare the query fragments of the next segments, 2 fold the 8 states of the last ones. With both done
//    by the consumers, and barriers between them, every segment cost a CTA about 4 us (12 tiles' worth), and 64 ragged
//    sequences took 130 us instead of 90.
// Measured (B200, back to back in a graph; called one behind the other for long 4 to 6 % more, the third 4 to 13 %, by what
// the power cap leaves of the clock): 32 sequences x 4096 rows, 32 / 8 heads of 128, bf16 and int8: 49.7 us, 5.4 TB/s; 64 ragged ones of
// 128 - 8192 rows, fp16 and e4m3: 90 us, 6.1 TB/s; 4 x 131072 rows, 64 / 8 heads, bf16 and e4m3: 165 us, 6.5 TB/s, the copy
// rate. What is left of the first is its ends: 3.3 us from the release of the launch to the first copy (lengths read, ranges
// located, table entries read), 1.5 us from a CTA's last tile to its exit, 2.7 us for the merge behind. With 16 heads per kv
// head (83 us) the consumers are the limit: the issue slots are 42 % busy, the tensor pipe 29 %, and two consumer warps a
// scheduler are too few to cover what each waits for. With 16-row blocks of 64-wide heads it is the rate of 1 KB copies (61 us;
// 54 us with 64-row blocks).
//  * Stage layout: a block's (page x D) bytes are contiguous in the pool, so the pool is described to TMA as 128-byte
//    lines with the 128-byte swizzle, whatever D is; row r, 16-byte chunk c of a tile sits at line-linear address
//    r * D + 16 c, swizzled. One copy per block and tile for K, one for V; the two scales of the block follow with an
//    8-byte cp.async that signals the same mbarrier.
//  * K and V are the A operand of mma.m16n8k16 (rows / head dim on M, query heads on N). ldmatrix moves 16-bit units,
//    i.e. pairs of codes: for K the pair is two neighbouring d, the order of d inside a 16-step is permuted and the
//    query fragments are loaded in that same order; for V^T (transposing load) the pair is two neighbouring d of one
//    row, the byte permutation that widens the codes also splits them, and a 16-row block of O^T holds the even d in
//    its upper half and the odd d in its lower half.
//  * Weights: with |vs| = c * 2^e, 1 <= c < 2, the running maximum R is that of s + e (log2 units) and the weight
//    w = 2^(s + e - R) lies in [0, 1]: the MMA gets w * c, rounded to half relative to the largest CONTRIBUTION so far, and
//    l += w * 2^-e, the sum of 2^(s - R), stays in fp32. w * c goes in as 2^14 times itself, the most a half has room for: a
//    weight keeps its 22 bits down to 2^-17 of the largest contribution and loses at most 2^-39 of that below. (Without the
//    factor half precision ends at 2^-25, and thousands of rows 17 natural log units below one row, whose sum is
//    what there is to see when that row's V is small, were lost altogether.) e is counted from a warp's first block that is not zero, so that
//    both stay in range as long as the V scales of a sequence differ by less than 2^60 (those that are zero aside, which set no
//    exponent). A block more than 2^60 above that one moves e's zero up; blocks more than 2^60 below the largest keep their
//    part in l, and in O what is left of it.
//  * A weight goes to the tensor cores in two halves, its value rounded to half and the remainder: 22 bits, whatever the type of
//    q. Rounded once (2^-12 of the weight at most) it added as much error to a float16 result as the result's own rounding.
//    SPLIT: with at most 4 query heads per unit (8 with two column blocks) each head takes two of the 8 MMA columns for the two
//    parts of q and of the weights, at no cost in MMAs. float32 calls always run this way (q needs 22 bits too), 16-bit calls
//    when their heads fit. Without SPLIT q, 16 bits as it is, goes in one half, and the remainders of the weights take an MMA
//    of their own into the same accumulators: with 8 heads per kv head 53.7 us instead of 52.8 (32 x 4096 rows, captured; 4 x
//    131072 rows called for long, under the power cap, 172 - 187 us instead of 167 - 177), with 16 79.4 instead of 72.8.
//  * A unit that lies in one range is finished in place. Otherwise the CTAs leave (m, l, acc) partials, at most two per
//    range, in a workspace that belongs to the call, and q8_merge_kernel, launched behind with programmatic stream
//    serialization, folds them in range order. No counters, no state between calls: calls on different streams, and
//    captured graphs, cannot meet in it.
// Every mbarrier wait is bounded (2 s); on expiry the kernel records a status code and runs to completion.
#pragma once

#include <cuda_fp8.h>

#include "decode_tc.cuh"

namespace ftk {

constexpr int Q8_NP = 4;                        // producer warps
constexpr int Q8_QWARPS = 2, Q8_FWARPS = 2;     // helper warps: query fragments, folds
constexpr int Q8_HELPERS = Q8_QWARPS + Q8_FWARPS;
constexpr int Q8_THREADS = (NCW + Q8_HELPERS + Q8_NP) * 32;
static_assert(Q8_THREADS == 512, "the register split below counts 16 warps");
constexpr float Q8_ROOM = 16384.0f;             // the largest weight goes to the tensor cores as a half between this and twice it
constexpr int Q8_MAX_SPLIT = 32;                // generic kernel: most ranges a unit is cut into

struct Q8Params : DecodeParams {
    const float2* scales;      // [blocks][Hkv] (K, V)
    long long blocks;          // blocks of the pool
    int4* desc;                // [ncta] unit whose merge starts in this range: (b, unit of b, partials, -)
    int out_dt;                // type of q and out: 0 float32, 1 bfloat16, 2 float16
    int nsplit;                // generic kernel: ranges per unit
    int full;                  // the tensor-core kernel's grid takes every SM
    int device;                // index of the device (host side)
};

// q and out carry their type at run time: only the first and last step of a unit look at it.
struct AnyOut {};
__device__ __forceinline__ float4 load4_any(const void* base, size_t at, int dt) {
    if (dt == 0) return Store<float>::ld4(static_cast<const float*>(base) + at);
    if (dt == 1) return Store<__nv_bfloat16>::ld4(static_cast<const __nv_bfloat16*>(base) + at);
    return Store<__half>::ld4(static_cast<const __half*>(base) + at);
}
__device__ __forceinline__ void store4_any(void* base, size_t at, int dt, float4 v) {
    if (dt == 0) Store<float>::st4(static_cast<float*>(base) + at, v);
    else if (dt == 1) Store<__nv_bfloat16>::st4(static_cast<__nv_bfloat16*>(base) + at, v);
    else Store<__half>::st4(static_cast<__half*>(base) + at, v);
}
__device__ __forceinline__ void store2_any(void* base, size_t at, int dt, float a, float b) {
    if (dt == 0) Store<float>::st2(static_cast<float*>(base) + at, a, b);
    else if (dt == 1) Store<__nv_bfloat16>::st2(static_cast<__nv_bfloat16*>(base) + at, a, b);
    else Store<__half>::st2(static_cast<__half*>(base) + at, a, b);
}
template <> __device__ inline void zero_rows<AnyOut>(const DecodeParams& p, int b, unsigned int) {
    const int dt = static_cast<const Q8Params&>(p).out_dt;
    const int n = p.Hq * p.D;
    for (int i = 0; i < n; i += 4) store4_any(p.out, (size_t)b * n + i, dt, make_float4(0.f, 0.f, 0.f, 0.f));
}

// ---- 8-bit codes to half pairs -------------------------------------------------
// `pairs`: bytes (0, 1) and (2, 3) of a word; `crossed`: bytes (0, 2) and (1, 3).
template <typename KV> struct Codes;
template <> struct Codes<int8_t> {
    // byte u = code + 128 as the low mantissa bits of 1024 (0x6400 | u is the half 1024 + u), less 1152: exact
    static __device__ __forceinline__ uint32_t off(uint32_t x) {
        const __half2 v = __hsub2(*reinterpret_cast<__half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    static __device__ __forceinline__ void pairs(uint32_t r, uint32_t& a, uint32_t& b) {
        const uint32_t u = r ^ 0x80808080u;
        a = off(__byte_perm(u, 0x64646464u, 0x4140));
        b = off(__byte_perm(u, 0x64646464u, 0x4342));
    }
    static __device__ __forceinline__ void crossed(uint32_t r, uint32_t& a, uint32_t& b) {
        const uint32_t u = r ^ 0x80808080u;
        a = off(__byte_perm(u, 0x64646464u, 0x4240));
        b = off(__byte_perm(u, 0x64646464u, 0x4341));
    }
    static __device__ __forceinline__ float4 floats(uint32_t r) {
        return make_float4((float)(int8_t)(r & 255u), (float)(int8_t)((r >> 8) & 255u), (float)(int8_t)((r >> 16) & 255u),
                           (float)(int8_t)(r >> 24));
    }
};
template <> struct Codes<__nv_fp8_e4m3> {
    static __device__ __forceinline__ void pairs(uint32_t r, uint32_t& a, uint32_t& b) {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(a), "=r"(b) : "r"(r));
    }
    static __device__ __forceinline__ void crossed(uint32_t r, uint32_t& a, uint32_t& b) {
        pairs(__byte_perm(r, r, 0x3120), a, b);
    }
    static __device__ __forceinline__ float4 floats(uint32_t r) {
        uint32_t a, b;
        pairs(r, a, b);
        const float2 lo = __half22float2(*reinterpret_cast<__half2*>(&a)), hi = __half22float2(*reinterpret_cast<__half2*>(&b));
        return make_float4(lo.x, lo.y, hi.x, hi.y);
    }
};

template <int D, int NBK, bool SPLIT, int WPT> struct Q8Cfg {
    static_assert(D % 16 == 0 && D >= 64 && D <= 256, "head dim: a multiple of 16 from 64 to 256");
    static constexpr int KV_BYTES = TILE * D;          // a multiple of 1024: the swizzle phase of every stage is the same
    static constexpr int STAGE_BYTES = 2 * KV_BYTES;
    // 128 KB of tiles in flight per SM, as in the 16-bit kernel; a multiple of the number of groups, so that a stage is
    // always consumed by the same group, which then sees every phase of its barrier in order
    static constexpr int NG = NCW / WPT;               // groups of consumer warps, taking tiles in turn
    static constexpr int RB = 4 / WPT;                 // 16-row blocks of a tile per warp
    static constexpr int NS = (131072 / STAGE_BYTES) / NG * NG;
    static_assert(NS >= NG && NS % Q8_NP == 0, "ring shorter than the groups");
    static constexpr int HEADS = NBK * (SPLIT ? 4 : 8);
    static constexpr int ACC_STRIDE = D + 4;
    static constexpr int STATE_BYTES = NCW * HEADS * ACC_STRIDE * 4;             // the warps' O of one segment
    // segments whose states may wait to be folded: as many as fit beside the ring (sequences of a tile or two keep several
    // segments in flight; 256 of 60 - 200 rows: 44 us with two)
    static constexpr int NF = STATE_BYTES <= 17408 ? 4 : STATE_BYTES <= 34816 ? 2 : 1;
    static constexpr int NQ = NF == 4 ? 4 : 2;         // segments whose query fragments may be ready
    static constexpr int Q_BYTES = NBK * (D / 16) * 32 * 8;                      // query fragments of a segment
    // The CTA is launched with 128 registers per thread; the 2 consumer warpgroups take more, the 2 others give up as many.
    static constexpr int REGS_CONSUMER = NBK * D <= 128 ? 152 : 168, REGS_OTHER = 256 - REGS_CONSUMER;
    static constexpr int OFF_STATE = NS * STAGE_BYTES;
    static constexpr int OFF_ML = OFF_STATE + NF * STATE_BYTES;                  // [NF][NCW][HEADS] (m, l)
    static constexpr int OFF_Q = OFF_ML + NF * NCW * HEADS * 8;                  // [NQ] fragments
    static constexpr int OFF_KF = OFF_Q + NQ * Q_BYTES;                          // [NQ][16] score factors
    static constexpr int OFF_SCALE = OFF_KF + NQ * 16 * 4;                       // [NS][4] (K, V) scales of the stage's blocks
    static constexpr int OFF_BAR = OFF_SCALE + NS * 4 * 8;                       // full[NS], empty[NS], q full / empty [NQ], state full / empty [4]
    static constexpr int OFF_SCHED = OFF_BAR + (2 * NS + 2 * NQ + 8) * 8;
    static constexpr int OFF_ABORT = OFF_SCHED + (int)sizeof(SchedShared);
    static constexpr int OFF_PREFIX = (OFF_ABORT + 16 + 15) & ~15;
    static constexpr int OFF_ZPRE = OFF_PREFIX + (SCHED_MAX_B + 1) * 4;
    static constexpr int SMEM_BYTES = OFF_ZPRE + (SCHED_MAX_B + 1) * 4 + 8;
    static_assert(SMEM_BYTES <= 232448, "exceeds the 227 KB of shared memory a CTA can have");
};

__device__ __forceinline__ void tma_load_lines(uint32_t dst, const CUtensorMap* map, int line, uint32_t bar, uint64_t pol) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%2, %3}], [%4], %5;"
        ::"r"(dst), "l"(map), "r"(0), "r"(line), "r"(bar), "l"(pol)
        : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
// this thread's arrival on `bar`, made when its cp.async copies so far have landed
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// Powers of two f, g with f * g = 1 and |x| * f in [2^14, 2^15) for a row's largest magnitude x (NaN for a row that is not
// finite; f is 2^127 for x below 2^-112): as large as a half can hold, so that small elements of the row keep most bits.
__device__ __forceinline__ void row_exponent(float x, float& f, float& g) {
    const int e = (int)(__float_as_uint(x) >> 23 & 255u), to = min(268 - e, 254);
    f = __uint_as_float((uint32_t)to << 23);
    g = to == 254 ? __uint_as_float(0x00400000u) : __uint_as_float((uint32_t)(254 - to) << 23);
    if (e == 255) f = __uint_as_float(0x7fc00000u);
}

// ---- the kernel ----------------------------------------------------------------
// KV: code type. NBK: 8-column blocks of the MMA. SPLIT: two columns per query head (see above).
template <typename KV, int D, int NBK, bool SPLIT, int WPT>
__global__ void __launch_bounds__(Q8_THREADS, 1)
decode_q8_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Q8Params p) {
    using Cfg = Q8Cfg<D, NBK, SPLIT, WPT>;
    extern __shared__ __align__(1024) uint8_t smem[];
    SchedShared* sh = reinterpret_cast<SchedShared*>(smem + Cfg::OFF_SCHED);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Cfg::OFF_ABORT);
    const uint32_t smem_base = smem_u32(smem);
    const uint32_t bar_full = smem_base + Cfg::OFF_BAR;
    const uint32_t bar_empty = bar_full + Cfg::NS * 8;
    const uint32_t bar_q_full = bar_empty + Cfg::NS * 8, bar_q_empty = bar_q_full + Cfg::NQ * 8;
    const uint32_t bar_state_full = bar_q_empty + Cfg::NQ * 8, bar_state_empty = bar_state_full + 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = (int)blockIdx.x;

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        if (smem_base & 1023u) {
            *abort_flag = 1;
            atomicCAS(p.status, ST_OK, ST_SMEM_MISALIGNED);
        }
        for (int s = 0; s < Cfg::NS; ++s) {
            mbar_init(bar_full + s * 8, 33);           // the announced bytes, and each producer lane's scales
            mbar_init(bar_empty + s * 8, WPT);
        }
        for (int s = 0; s < Cfg::NQ; ++s) {
            mbar_init(bar_q_full + s * 8, Q8_QWARPS);
            mbar_init(bar_q_empty + s * 8, NCW);
        }
        for (int s = 0; s < Cfg::NF; ++s) {
            mbar_init(bar_state_full + s * 8, NCW);
            mbar_init(bar_state_empty + s * 8, Q8_FWARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_v) : "memory");
    }
    __syncthreads();
    // The merge may come and wait early where this grid takes every SM. Where it leaves some free, the merge would let the next
    // launches of a queue in as well, all of them waiting there (1 x 512 rows, 8 CTAs: 8.2 us a call instead of 7.3;
    // with the permission late on a full grid: 32 x 4096 rows 0.3 us more).
    if (p.full) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int upb = p.Hkv * p.NCH;
    const unsigned int* prefix = nullptr;
    const unsigned int* zprefix = nullptr;
    long long total;
    Plan pl;
    if (!p.lens) {
        total = (long long)p.B * tiles_of(p.T) * upb;
        pl = make_plan(total, p.ncta, 0, 0);
        if (total > 0) plan_enable_cost(pl, (long long)p.B * tiles_of(p.T), p.B, upb, nullptr, nullptr, tiles_of(p.T), 1, 3);
        asm volatile("griddepcontrol.wait;" ::: "memory");
    } else {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        unsigned int* table = reinterpret_cast<unsigned int*>(smem + Cfg::OFF_PREFIX);
        unsigned int* ztable = reinterpret_cast<unsigned int*>(smem + Cfg::OFF_ZPRE);
        total = sched_prefix<AnyOut>(p, sh, table, ztable, 0);
        prefix = table;
        zprefix = ztable;
        pl = make_plan(total, p.ncta, 0, 0);
        if (total > 0) plan_enable_cost(pl, prefix[p.B], zprefix[p.B], upb, prefix, zprefix, 0, 1, 3);
    }
    if (!p.full) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (*abort_flag) {
        if (threadIdx.x == 0) p.desc[cta] = make_int4(0, 0, 0, 0);
        return;
    }
    // every warp locates the CTA's range for itself
    Walker w = {};
    if (total > 0) {
        if (pl.ctot) w = walker_locate_cost_range(p, pl, cta);
        else if (!range_empty(pl, cta)) w = walker_locate(p, prefix, range_start(pl, cta), range_start(pl, cta + 1));
    }

    constexpr int KSTEPS = D / 16;
    constexpr int HB = SPLIT ? 4 : 8;              // query heads per column block
    constexpr int HEADS = Cfg::HEADS, RB = Cfg::RB;

    if (warp >= NCW + Q8_HELPERS) {
        // ===================== producer warps =====================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::REGS_OTHER));
        // Every Q8_NP-th tile of the range. A single producer would have to issue a 16 KB tile of 2 KB blocks every 350 ns,
        // and falls behind (measured: 94 us for 32 x 4096 rows instead of 57). A tile's table entries are fetched while the
        // tile before it goes out.
        const int pw = warp - NCW - Q8_HELPERS;
        const uint64_t pol = policy_evict_first();
        const int page_shift = __ffs(p.page) - 1;
        int issued = 0, s = pw;
        uint32_t ph = 0;
        bool gave_up = false;
        auto blocks_of = [&](const Walker& t) {                             // blocks (or parts of one) tile t has rows in
            return p.page <= TILE ? (min(TILE, t.len - t.ti * TILE) + p.page - 1) >> p.box_shift : 1;
        };
        auto entry = [&](const Walker& t) {                                 // lane j: the j-th of them
            return lane < blocks_of(t) ? __ldg(p.table + (size_t)t.b * p.tbl_width + ((t.ti * TILE + (lane << p.box_shift)) >> page_shift)) : 0;
        };
        for (int i = 0; i < pw && w.g < w.end; ++i) walker_advance(p, w);
        int blk = w.g < w.end ? entry(w) : 0;
        while (w.g < w.end) {
            Walker next = w;
            if (w.ti + Q8_NP < w.nt) {
                next.g += Q8_NP;
                next.ti += Q8_NP;
            } else {
                for (int i = 0; i < Q8_NP && next.g < next.end; ++i) walker_advance(p, next);
            }
            const int next_blk = next.g < next.end ? entry(next) : 0;
            const int kv = w.ub / p.NCH;
            const int npg = blocks_of(w);
            // (device table values are trusted; an entry outside the pool only has to stay an address, and is reported by the
            // self-checking build)
            if (!FTK_ROW_OK(p, ((long long)blk * p.Hkv + kv) * p.page) || !(blk >= 0 && blk < p.blocks)) blk = 0;
            const long long unit_row = ((long long)blk * p.Hkv + kv) * p.page + (p.page <= TILE ? 0 : (w.ti * TILE) & (p.page - 1));
            const int line = (int)(unit_row * D >> 7);
            const uint32_t bytes = (uint32_t)(npg << p.box_shift) * (uint32_t)(2 * D);
            if (!mbar_wait(bar_empty + s * 8, ph ^ 1u, abort_flag, p.status, ST_WAIT_EMPTY_TIMEOUT)) {
                gave_up = true;
                break;
            }
            const uint32_t fb = bar_full + s * 8;
            if (lane == 0) mbar_expect_tx(fb, bytes);
            __syncwarp();                                                   // expect_tx before any complete_tx
            if (lane < npg) {
                const uint32_t dst = smem_base + s * Cfg::STAGE_BYTES + (uint32_t)(lane << p.box_shift) * (uint32_t)D;
                tma_load_lines(dst, &tm_k, line, fb, pol);
                tma_load_lines(dst + Cfg::KV_BYTES, &tm_v, line, fb, pol);
                cp_async8(smem_base + Cfg::OFF_SCALE + (s * 4 + lane) * 8, p.scales + (size_t)blk * p.Hkv + kv);
            }
            cp_async_arrive(fb);
            ++issued;
            w = next;
            blk = next_blk;
            s += Q8_NP;
            if (s >= Cfg::NS) { s -= Cfg::NS; ph ^= 1u; }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (gave_up || *abort_flag) {
            // do not leave the CTA while its own copies may still be landing: wait (bounded) for the last phase of every
            // stage this warp issued
            constexpr int OWN = Cfg::NS / Q8_NP;
            const int first = issued > OWN ? issued - OWN : 0;
            for (int i = first; i < issued; ++i) {
                const unsigned long long b0 = global_ns();
                while (!mbar_try_wait(bar_full + (pw + (i % OWN) * Q8_NP) * 8, (uint32_t)((i / OWN) & 1))) {
                    if (global_ns() - b0 > WAIT_LIMIT_NS) {
                        atomicCAS(p.status, ST_OK, ST_DRAIN_TIMEOUT);
                        break;
                    }
                }
            }
        }
        return;
    }

    if (warp >= NCW) {
        // ===================== helper warps =====================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::REGS_OTHER));
        // tiles of the segment that begins at t, and the step to the next segment
        auto seg_tiles = [](const Walker& t) { return (int)min(t.end - t.g, (long long)(t.nt - t.ti)); };
        auto to_next = [&](Walker& t) {
            const int n = seg_tiles(t);
            t.g += n - 1;
            t.ti += n - 1;
            walker_advance(p, t);
        };
        if (warp < NCW + Q8_QWARPS) {
            // ---- The query rows of each segment's unit as B fragments, each row scaled by a power of two into the range of
            // a half. A warp takes every other head; a lane the 4 elements that make a fragment register pair. The rows
            // are requested one segment before they are worked on.
            const int hw = warp - NCW;
            constexpr int PER = (HEADS + Q8_QWARPS - 1) / Q8_QWARPS, LR = (D / 4 + 31) / 32;
            float4 x[PER][LR];
            auto request = [&]() {
                const int kv = w.ub / p.NCH, ch = w.ub - kv * p.NCH;
                const int gvalid = min(p.GC, p.G - ch * p.GC);
                const size_t row0 = ((size_t)w.b * p.Hq + kv * p.G + ch * p.GC) * D;
#pragma unroll
                for (int i = 0; i < PER; ++i)
#pragma unroll
                    for (int r = 0; r < LR; ++r) {
                        const int g = hw + i * Q8_QWARPS, c = lane + 32 * r;
                        x[i][r] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (g < gvalid && c < D / 4) x[i][r] = load4_any(p.q, row0 + (size_t)g * D + c * 4, p.out_dt);
                    }
            };
            if (w.g < w.end) request();
            for (int k = 0; w.g < w.end; ++k) {
                const int buf = k % Cfg::NQ;
                mbar_wait(bar_q_empty + buf * 8, (uint32_t)((k / Cfg::NQ) & 1) ^ 1u, abort_flag, p.status, ST_WAIT_RANGE_TIMEOUT);
                uint2* frag = reinterpret_cast<uint2*>(smem + Cfg::OFF_Q + buf * Cfg::Q_BYTES);
                float* kf = reinterpret_cast<float*>(smem + Cfg::OFF_KF) + buf * 16;
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const int g = hw + i * Q8_QWARPS;
                    uint32_t top = 0;                       // as bits: NaN and infinity are the largest
#pragma unroll
                    for (int r = 0; r < LR; ++r)
                        top = max(max(top, max(__float_as_uint(x[i][r].x) & 0x7fffffffu, __float_as_uint(x[i][r].y) & 0x7fffffffu)),
                                  max(__float_as_uint(x[i][r].z) & 0x7fffffffu, __float_as_uint(x[i][r].w) & 0x7fffffffu));
                    top = __reduce_max_sync(0xffffffffu, top);
                    float fx, gx;
                    row_exponent(__uint_as_float(top), fx, gx);
#pragma unroll
                    for (int r = 0; r < LR; ++r) {
                        const int c = lane + 32 * r;
                        if (c < D / 4) {
                            const float e[4] = {x[i][r].x * fx, x[i][r].y * fx, x[i][r].z * fx, x[i][r].w * fx};
                            const uint2 hi = make_uint2(pack2<__half>(e[0], e[1]), pack2<__half>(e[2], e[3]));
                            const int nbk = g / HB, col = SPLIT ? 2 * (g % HB) : g % HB;
                            uint2* to = frag + ((size_t)nbk * KSTEPS + (c >> 2)) * 32 + col * 4 + (c & 3);
                            to[0] = hi;
                            if constexpr (SPLIT) {
                                const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&hi.x));
                                const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi.y));
                                to[4] = make_uint2(pack2<__half>(e[0] - a.x, e[1] - a.y), pack2<__half>(e[2] - b.x, e[3] - b.y));
                            }
                        }
                    }
                    if (lane == 0) kf[g] = gx * p.scale * LOG2E;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_q_full + buf * 8);
                to_next(w);
                if (w.g < w.end) request();
            }
            return;
        }
        // ---- The consumers' states of each segment, folded into the output or into a partial.
        const int tid = threadIdx.x - (NCW + Q8_QWARPS) * 32;
        int4 merge = make_int4(0, 0, 0, 0);           // the unit that begins in this range and ends in a later one
        if (w.g >= w.end) {
            // nothing here: an empty partial, which a merge that spans this range passes over
            for (int i = tid; i < p.GC; i += Q8_FWARPS * 32)
                *reinterpret_cast<float2*>(p.ws_ml + ((size_t)2 * cta * p.GC + i) * 2) = make_float2(-INFINITY, 0.0f);
        }
        for (int k = 0; w.g < w.end; ++k) {
            const int n = seg_tiles(w);
            const bool begins = w.ti == 0, ends = w.ti + n == w.nt, whole = begins && ends;
            const int kv = w.ub / p.NCH, ch = w.ub - kv * p.NCH;
            const int gvalid = min(p.GC, p.G - ch * p.GC);
            const size_t out0 = ((size_t)w.b * p.Hq + kv * p.G + ch * p.GC) * D;
            const size_t slot = (size_t)2 * cta + (begins ? 1 : 0);
            if (begins && !ends) {
                int last;
                if (pl.ctot) last = cost_owner(pl, cost_of_unit(pl, w.b, w.ub, w.nt) + (long long)pl.ka * (w.nt - 1));
                else last = range_of(pl, w.g + w.nt - 1);              // w stands on the unit's first tile
                merge = make_int4(w.b, w.ub, last - cta + 1, 0);
            }
            to_next(w);
            const int buf = k % Cfg::NF;
            const float* s_acc = reinterpret_cast<const float*>(smem + Cfg::OFF_STATE + buf * Cfg::STATE_BYTES);
            const float2* s_ml = reinterpret_cast<const float2*>(smem + Cfg::OFF_ML) + buf * NCW * HEADS;
            mbar_wait(bar_state_full + buf * 8, (uint32_t)((k / Cfg::NF) & 1), abort_flag, p.status, ST_WAIT_FULL_TIMEOUT);
            for (int it = tid; it < gvalid * (D / 4); it += Q8_FWARPS * 32) {
                const int g = it / (D / 4), d = (it % (D / 4)) * 4;
                // Every thread works the weights of its head out for itself: 8 exponentials, and no barrier. A warp that had
                // no tile of this segment (l == 0) left no O: what is read in its place is not used.
                float2 ml[NCW];
                float4 v[NCW];
                float m = -INFINITY, l = 0.0f;
#pragma unroll
                for (int ww = 0; ww < NCW; ++ww) {
                    ml[ww] = s_ml[ww * HEADS + g];
                    v[ww] = *reinterpret_cast<const float4*>(s_acc + ((size_t)ww * HEADS + g) * Cfg::ACC_STRIDE + d);
                    m = fmaxf(m, ml[ww].x);
                }
                const float safe = m == -INFINITY ? 0.0f : m;
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int ww = 0; ww < NCW; ++ww) {
                    const bool some = ml[ww].y != 0.0f;
                    const float f = ex2(ml[ww].x - safe);
                    l = fmaf(ml[ww].y, f, l);
                    a.x = fmaf(some ? v[ww].x : 0.0f, f, a.x);
                    a.y = fmaf(some ? v[ww].y : 0.0f, f, a.y);
                    a.z = fmaf(some ? v[ww].z : 0.0f, f, a.z);
                    a.w = fmaf(some ? v[ww].w : 0.0f, f, a.w);
                }
                if (whole) {
                    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
                    store4_any(p.out, out0 + (size_t)g * D + d, p.out_dt, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
                } else if (FTK_SLOT_OK(p, slot, 0)) {
                    *reinterpret_cast<float4*>(p.ws_acc + (slot * p.GC + g) * D + d) = a;
                    if (d == 0) *reinterpret_cast<float2*>(p.ws_ml + (slot * p.GC + g) * 2) = make_float2(m, l);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_state_empty + buf * 8);
        }
        if (tid == 0) p.desc[cta] = merge;
        return;
    }

    // ======================= consumer warps =======================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::REGS_CONSUMER));
    const int cg = warp / WPT, wr = warp % WPT;
    const int quad = lane >> 2, qi = lane & 3;
    const float neg_inf = -INFINITY;

    constexpr int NLD = (KSTEPS + 1) / 2;          // ldmatrix.x4 per 16 rows: two 16-byte chunks of 16 rows
    constexpr int HPT = SPLIT ? 1 : 2;             // heads per column block that this thread holds the scores of
    uint32_t qb[NBK][KSTEPS][2];
    float acc[NBK][KSTEPS][4];                     // O^T block mt: d = 16 mt + 2 quad ([0], [1]) and + 1 ([2], [3])
    float kf[NBK][HPT];                            // score factor of the head: its row's exponent / sqrt(D) * log2(e)
    float m_run[NBK][HPT], l_run[NBK][HPT];        // R of the head; this thread's share of l
    // biased exponent that this warp counts V scales from (-127: only blocks of zeros so far, -126: no rows), and the largest
    // exponent so far, counted from there
    int e0 = -126, top = 0;

    // Byte offset of chunk 2 i + csel of row r inside a tile, swizzled. `csel` and the row are the lane's.
    const int lrow = ((lane >> 3) & 1) * 8 + (lane & 7), csel = lane >> 4;
    auto chunk_off = [&](int j, int i) -> uint32_t {
        const uint32_t lin = (uint32_t)((wr * RB + j) * 16 + lrow) * (uint32_t)D + (uint32_t)(2 * i + csel) * 16u;
        return lin ^ (((lin >> 7) & 7u) << 4);
    };

    int i0 = 0, own = cg, s = cg;
    uint32_t ph = 0;

    auto process = [&](auto ragged_tag, int rows_valid) {
        constexpr bool RAGGED = decltype(ragged_tag)::value;
        const uint32_t st_k = smem_base + s * Cfg::STAGE_BYTES;
        const uint32_t st_v = st_k + Cfg::KV_BYTES;
        const float2* sc = reinterpret_cast<const float2*>(smem + Cfg::OFF_SCALE) + s * 4;
        float2 ks[RB];
#pragma unroll
        for (int j = 0; j < RB; ++j) {
            const int r0 = (wr * RB + j) * 16;
            ks[j] = sc[r0 >> p.box_shift];
            // a block of the tile that holds no valid row was not copied, nor were its scales
            if (RAGGED && r0 >= rows_valid) ks[j] = make_float2(0.0f, 0.0f);
        }
        constexpr int PF = 2;
        constexpr int N = RB * NLD;
        uint32_t f[PF][4];
        // ---- S^T = K Q^T
        float sa[NBK][RB][4];
#pragma unroll
        for (int nbk = 0; nbk < NBK; ++nbk)
#pragma unroll
            for (int j = 0; j < RB; ++j) sa[nbk][j][0] = sa[nbk][j][1] = sa[nbk][j][2] = sa[nbk][j][3] = 0.0f;
#pragma unroll
        for (int n = 0; n < PF; ++n) ldsm_x4(st_k + chunk_off(n / NLD, n % NLD), f[n][0], f[n][1], f[n][2], f[n][3]);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int j = n / NLD, i = n % NLD;
            uint32_t (&r)[4] = f[n % PF];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int kk = 2 * i + half;
                if (kk < KSTEPS) {
                    uint32_t a0, a1, a2, a3;
                    Codes<KV>::pairs(r[2 * half], a0, a2);
                    Codes<KV>::pairs(r[2 * half + 1], a1, a3);
#pragma unroll
                    for (int nbk = 0; nbk < NBK; ++nbk)
                        mma16816<__half>(sa[nbk][j], a0, a1, a2, a3, qb[nbk][kk][0], qb[nbk][kk][1]);
                }
            }
            if (n + PF < N) ldsm_x4(st_k + chunk_off((n + PF) / NLD, (n + PF) % NLD), r[0], r[1], r[2], r[3]);
        }
#pragma unroll
        for (int n = 0; n < PF; ++n) ldsm_x4_t(st_v + chunk_off(n / NLD, n % NLD), f[n][0], f[n][1], f[n][2], f[n][3]);
        // ---- online softmax, in units of log2
        // Exponents of the blocks' vs less e0: at most 60. Otherwise (and always while e0 is negative) there is something to settle
        int d[RB], hi = -255;
#pragma unroll
        for (int j = 0; j < RB; ++j) {
            d[j] = (int)(__float_as_uint(ks[j].y) >> 23 & 255u) - e0;
            hi = max(hi, d[j]);
        }
        if (hi > 60) {
            if (e0 < 0) {                // a block of zeros says nothing about the others: the first that is not one sets e0
                top = 0;
                e0 = -127;
#pragma unroll
                for (int j = RB - 1; j >= 0; --j)
                    if (ks[j].y != 0.0f) e0 = min(max((int)(__float_as_uint(ks[j].y) >> 23 & 255u), 61), 194);
            }
            hi = -255;
#pragma unroll
            for (int j = 0; j < RB; ++j) {
                d[j] = min((int)(__float_as_uint(ks[j].y) >> 23 & 255u), 254) - abs(e0);
                hi = max(hi, d[j]);
            }
            if (hi > 60) {               // e0 moves up, and R with it
                const int by = hi - 60;
                const float f = __uint_as_float((uint32_t)(127 + by / 2) << 23), g = __uint_as_float((uint32_t)(127 + by - by / 2) << 23);
                e0 += by;
                top -= by;
                hi = 60;
#pragma unroll
                for (int j = 0; j < RB; ++j) d[j] -= by;
#pragma unroll
                for (int nbk = 0; nbk < NBK; ++nbk)
#pragma unroll
                    for (int e = 0; e < HPT; ++e) {
                        m_run[nbk][e] -= (float)by;
                        l_run[nbk][e] = l_run[nbk][e] * f * g;
                    }
            }
        }
        // Per block: that exponent, 2^-it, and what is left of vs (e0 + d covers 1 .. 254, every finite scale). Rows 60 and more below
        // the largest, those of a block of zeros among them, add to l and only have to keep R in range of their s
        top = max(top, hi);
        float de[RB], ge[RB], ce[RB];
#pragma unroll
        for (int j = 0; j < RB; ++j) {
            d[j] = max(d[j], top - 60);
            de[j] = (float)d[j];
            ge[j] = __uint_as_float((uint32_t)(127 - d[j]) << 23);
            ce[j] = ks[j].y * __uint_as_float(max((uint32_t)(254 - abs(e0) - d[j]) << 23, 0x00400000u)) * Q8_ROOM;
        }
        uint32_t pb[NBK][RB][2];
        [[maybe_unused]] uint32_t pr[SPLIT ? 1 : NBK][RB][2];      // what the rounding to half left of the weights
#pragma unroll
        for (int nbk = 0; nbk < NBK; ++nbk) {
            float pw[HPT][RB][2];
#pragma unroll
            for (int e = 0; e < HPT; ++e) {
                float v[RB][2];
                float mx = neg_inf;
#pragma unroll
                for (int j = 0; j < RB; ++j) {
                    const float fac = kf[nbk][e] * ks[j].x;
                    const int r_lo = (wr * RB + j) * 16 + quad;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        v[j][h] = fmaf(SPLIT ? sa[nbk][j][2 * h] + sa[nbk][j][2 * h + 1] : sa[nbk][j][2 * h + e], fac, de[j]);
                        if (RAGGED && r_lo + 8 * h >= rows_valid) v[j][h] = neg_inf;
                        mx = fmaxf(mx, v[j][h]);
                    }
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float m_old = m_run[nbk][e];
                const float m_new = fmaxf(m_old, mx);
                const float m_safe = m_new == neg_inf ? 0.0f : m_new;
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < RB; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float w8 = ex2(v[j][h] - m_safe);
                        sum = fmaf(w8, ge[j], sum);
                        pw[e][j][h] = w8 * ce[j];
                    }
                if (m_new != m_old) {
                    // in two steps for l, which may be 2^60 and more: what is left of it counts where 2^(m_old - m_new) is 0 in
                    // float32
                    const float half = ex2(0.5f * (m_old - m_safe)), alpha = half * half;
                    m_run[nbk][e] = m_new;
                    l_run[nbk][e] = l_run[nbk][e] * half * half;
#pragma unroll
                    for (int mt = 0; mt < KSTEPS; ++mt) {
                        if constexpr (SPLIT) {
                            acc[nbk][mt][0] *= alpha; acc[nbk][mt][1] *= alpha;
                            acc[nbk][mt][2] *= alpha; acc[nbk][mt][3] *= alpha;
                        } else {
                            acc[nbk][mt][e] *= alpha;
                            acc[nbk][mt][2 + e] *= alpha;
                        }
                    }
                }
                l_run[nbk][e] += sum;
            }
#pragma unroll
            for (int j = 0; j < RB; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if constexpr (SPLIT) {
                        const float hi = __half2float(__float2half_rn(pw[0][j][h]));
                        pb[nbk][j][h] = movmatrix_trans(pack2<__half>(hi, pw[0][j][h] - hi));
                    } else {
                        const uint32_t hi = pack2<__half>(pw[0][j][h], pw[HPT - 1][j][h]);
                        const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                        pb[nbk][j][h] = movmatrix_trans(hi);
                        pr[nbk][j][h] = movmatrix_trans(pack2<__half>(pw[0][j][h] - r.x, pw[HPT - 1][j][h] - r.y));
                    }
                }
        }
        // ---- O^T += V^T P^T
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int j = n / NLD, i = n % NLD;
            uint32_t (&r)[4] = f[n % PF];
            if constexpr (RAGGED) {
                // rows at and past the end may hold anything, NaN codes included: a zero weight times them has to be zero
                const int t = (wr * RB + j) * 16 + qi * 2;
                const uint32_t lo = (t < rows_valid ? 0x0000ffffu : 0u) | (t + 1 < rows_valid ? 0xffff0000u : 0u);
                const uint32_t hi = (t + 8 < rows_valid ? 0x0000ffffu : 0u) | (t + 9 < rows_valid ? 0xffff0000u : 0u);
                r[0] &= lo; r[1] &= hi; r[2] &= lo; r[3] &= hi;
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int mt = 2 * i + half;
                if (mt < KSTEPS) {
                    uint32_t a0, a1, a2, a3;
                    Codes<KV>::crossed(r[2 * half], a0, a1);
                    Codes<KV>::crossed(r[2 * half + 1], a2, a3);
#pragma unroll
                    for (int nbk = 0; nbk < NBK; ++nbk) {
                        mma16816<__half>(acc[nbk][mt], a0, a1, a2, a3, pb[nbk][j][0], pb[nbk][j][1]);
                        if constexpr (!SPLIT) mma16816<__half>(acc[nbk][mt], a0, a1, a2, a3, pr[nbk][j][0], pr[nbk][j][1]);
                    }
                }
            }
            if (n + PF < N) ldsm_x4_t(st_v + chunk_off((n + PF) / NLD, (n + PF) % NLD), r[0], r[1], r[2], r[3]);
        }
    };

    for (int k = 0; w.g < w.end; ++k) {
        const long long left = w.end - w.g;
        const int n = (int)(left < (long long)(w.nt - w.ti) ? left : (long long)(w.nt - w.ti));
        const bool mine = own < i0 + n;            // this group has a tile of the segment
        // ---- the segment's query fragments
        e0 = -126;
        {
            const int buf = k % Cfg::NQ;
            mbar_wait(bar_q_full + buf * 8, (uint32_t)((k / Cfg::NQ) & 1), abort_flag, p.status, ST_WAIT_RANGE_TIMEOUT);
            if (mine) {
                const uint2* frag = reinterpret_cast<const uint2*>(smem + Cfg::OFF_Q + buf * Cfg::Q_BYTES) + lane;
                const float* s_kf = reinterpret_cast<const float*>(smem + Cfg::OFF_KF) + buf * 16;
#pragma unroll
                for (int nbk = 0; nbk < NBK; ++nbk) {
#pragma unroll
                    for (int kk = 0; kk < KSTEPS; ++kk) {
                        const uint2 f = frag[(nbk * KSTEPS + kk) * 32];
                        qb[nbk][kk][0] = f.x;
                        qb[nbk][kk][1] = f.y;
                    }
#pragma unroll
                    for (int e = 0; e < HPT; ++e) kf[nbk][e] = s_kf[nbk * HB + (SPLIT ? qi : 2 * qi + e)];
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_q_empty + buf * 8);
        }
#pragma unroll
        for (int nbk = 0; nbk < NBK; ++nbk) {
#pragma unroll
            for (int e = 0; e < HPT; ++e) {
                m_run[nbk][e] = neg_inf;
                l_run[nbk][e] = 0.0f;
            }
#pragma unroll
            for (int mt = 0; mt < KSTEPS; ++mt) acc[nbk][mt][0] = acc[nbk][mt][1] = acc[nbk][mt][2] = acc[nbk][mt][3] = 0.0f;
        }
        // ---- this group's tiles of the segment
        for (; own < i0 + n; own += Cfg::NG) {
            const bool ok = mbar_wait(bar_full + s * 8, ph, abort_flag, p.status, ST_WAIT_FULL_TIMEOUT);
            const int rows_valid = w.len - (w.ti + (own - i0)) * TILE;      // >= 1
            if (ok) {
                if (rows_valid >= TILE) process(std::false_type{}, TILE);
                else if (wr * (RB * 16) < rows_valid) process(std::true_type{}, rows_valid);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_empty + s * 8);
            s += Cfg::NG;
            if (s >= Cfg::NS) { s -= Cfg::NS; ph ^= 1u; }
        }
        i0 += n;
        // ---- leave the warp's state for the helpers
        {
            const int buf = k % Cfg::NF;
            float* s_acc = reinterpret_cast<float*>(smem + Cfg::OFF_STATE + buf * Cfg::STATE_BYTES);
            float2* s_ml = reinterpret_cast<float2*>(smem + Cfg::OFF_ML) + buf * NCW * HEADS;
            // 2^e0 without the room: sums of vs * v8 again
            const float unit = e0 < 0 ? 1.0f : __uint_as_float((uint32_t)e0 << 23) * (1.0f / Q8_ROOM);
            mbar_wait(bar_state_empty + buf * 8, (uint32_t)((k / Cfg::NF) & 1) ^ 1u, abort_flag, p.status, ST_WAIT_EMPTY_TIMEOUT);
#pragma unroll
            for (int nbk = 0; nbk < NBK; ++nbk) {
#pragma unroll
                for (int e = 0; e < HPT; ++e) {
                    float l = l_run[nbk][e];
                    l += __shfl_xor_sync(0xffffffffu, l, 4);
                    l += __shfl_xor_sync(0xffffffffu, l, 8);
                    l += __shfl_xor_sync(0xffffffffu, l, 16);
                    const int g = nbk * HB + (SPLIT ? qi : qi * 2 + e);
                    // Warps count V scales from different exponents. Where that has left l far from 1 (2^-60 to 2^60), its
                    // exponent goes back into m, so that the folds, which compare m alone, lose nothing
                    const int le = (int)(__float_as_uint(l) >> 23) - 127, k = le > 32 ? le - 32 : le < -32 ? le + 32 : 0;
                    const float back = __uint_as_float((uint32_t)(127 - k) << 23);
                    if (quad == 0) s_ml[warp * HEADS + g] = make_float2(m_run[nbk][e] + (float)k, l * back);
                    if (e0 != -126) {
                        float* my = s_acc + ((size_t)warp * HEADS + g) * Cfg::ACC_STRIDE + quad * 2;
#pragma unroll
                        for (int mt = 0; mt < KSTEPS; ++mt) {
                            float2 o;
                            if constexpr (SPLIT) o = make_float2(acc[nbk][mt][0] + acc[nbk][mt][1], acc[nbk][mt][2] + acc[nbk][mt][3]);
                            else o = make_float2(acc[nbk][mt][e], acc[nbk][mt][2 + e]);
                            *reinterpret_cast<float2*>(my + mt * 16) = make_float2(o.x * unit * back, o.y * unit * back);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_state_full + buf * 8);
        }
        w.g += n - 1;
        w.ti += n - 1;
        walker_advance(p, w);
    }
}

// ---- generic kernel ---------------------------------------------------------------
// Every other shape (head dims outside the list above or up to 512, blocks of other than a power of two >= 16 rows,
// unaligned operands, more sequences than the schedule's table holds): CUDA cores, float32 throughout. One CTA per (unit of
// up to 4 heads, range): a unit's rows are cut into nsplit equal ranges, a warp takes every eighth group of 4 rows, a lane
// every 32nd word of 4 codes. Bound by instruction issue (the 5-step reductions of the scores), not by bandwidth.
constexpr int Q8G_HEADS = 4;
template <typename KV, int LC>
__global__ void __launch_bounds__(256)
decode_q8_generic_kernel(const Q8Params p) {
    __shared__ float s_acc[8][LC * 128];
    __shared__ float2 s_ml[8][Q8G_HEADS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int upb = p.Hkv * p.NCH;
    const long long unit = blockIdx.x / (unsigned)p.nsplit;
    const int part = (int)(blockIdx.x - unit * p.nsplit);
    const int b = (int)(unit / upb), ub = (int)(unit - (long long)b * upb);
    const int kv = ub / p.NCH, ch = ub % p.NCH;
    const int gvalid = min(Q8G_HEADS, p.G - ch * Q8G_HEADS);
    const int h0 = kv * p.G + ch * Q8G_HEADS;
    const int len = seq_len(p, b);
    const int per = (len + p.nsplit - 1) / p.nsplit;
    const int begin = min(len, part * per), end = min(len, begin + per);
    const int words = p.D >> 2;
    float4 q[Q8G_HEADS][LC], acc[Q8G_HEADS][LC];
    float m[Q8G_HEADS], l[Q8G_HEADS];
#pragma unroll
    for (int g = 0; g < Q8G_HEADS; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.0f;
#pragma unroll
        for (int c = 0; c < LC; ++c) {
            q[g][c] = acc[g][c] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (g < gvalid && lane + 32 * c < words)
                q[g][c] = load4_any(p.q, ((size_t)b * p.Hq + h0 + g) * p.D + (size_t)(lane + 32 * c) * 4, p.out_dt);
        }
    }
    const float to2 = p.scale * LOG2E;
    constexpr int R = 4;
    for (int t0 = begin + warp * R; t0 < end; t0 += 8 * R) {
        uint32_t kw[R][LC], vw[R][LC];
        float2 sc[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int t = min(t0 + r, end - 1);
            int blk = __ldg(p.table + (size_t)b * p.tbl_width + t / p.page);
            if (!FTK_ROW_OK(p, ((long long)blk * p.Hkv + kv) * p.page) || !(blk >= 0 && blk < p.blocks)) blk = 0;
            sc[r] = __ldg(p.scales + (size_t)blk * p.Hkv + kv);
            const size_t row = ((size_t)blk * p.Hkv + kv) * p.page + t % p.page;
#pragma unroll
            for (int c = 0; c < LC; ++c) {
                kw[r][c] = vw[r][c] = 0;
                if (lane + 32 * c < words) {
                    kw[r][c] = __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(p.k) + row * p.D) + lane + 32 * c);
                    vw[r][c] = __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(p.v) + row * p.D) + lane + 32 * c);
                }
            }
        }
        float s[R][Q8G_HEADS];
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int g = 0; g < Q8G_HEADS; ++g) s[r][g] = 0.0f;
#pragma unroll
            for (int c = 0; c < LC; ++c) {
                const float4 k = Codes<KV>::floats(kw[r][c]);
#pragma unroll
                for (int g = 0; g < Q8G_HEADS; ++g)
                    s[r][g] = fmaf(q[g][c].w, k.w, fmaf(q[g][c].z, k.z, fmaf(q[g][c].y, k.y, fmaf(q[g][c].x, k.x, s[r][g]))));
            }
#pragma unroll
            for (int g = 0; g < Q8G_HEADS; ++g) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) s[r][g] += __shfl_xor_sync(0xffffffffu, s[r][g], o);
                s[r][g] = t0 + r < end ? s[r][g] * (sc[r].x * to2) : -INFINITY;
            }
        }
#pragma unroll
        for (int g = 0; g < Q8G_HEADS; ++g) {
            float mx = m[g];
#pragma unroll
            for (int r = 0; r < R; ++r) mx = fmaxf(mx, s[r][g]);
            const float safe = mx == -INFINITY ? 0.0f : mx;
            const float alpha = ex2(m[g] - safe);
            m[g] = mx;
            l[g] *= alpha;
#pragma unroll
            for (int c = 0; c < LC; ++c) { acc[g][c].x *= alpha; acc[g][c].y *= alpha; acc[g][c].z *= alpha; acc[g][c].w *= alpha; }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float w8 = ex2(s[r][g] - safe);
                l[g] += w8;
                s[r][g] = t0 + r < end ? w8 * sc[r].y : 0.0f;
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (t0 + r >= end) break;
#pragma unroll
            for (int c = 0; c < LC; ++c) {
                const float4 v = Codes<KV>::floats(vw[r][c]);
#pragma unroll
                for (int g = 0; g < Q8G_HEADS; ++g) {
                    acc[g][c].x = fmaf(s[r][g], v.x, acc[g][c].x);
                    acc[g][c].y = fmaf(s[r][g], v.y, acc[g][c].y);
                    acc[g][c].z = fmaf(s[r][g], v.z, acc[g][c].z);
                    acc[g][c].w = fmaf(s[r][g], v.w, acc[g][c].w);
                }
            }
        }
    }
    if (lane == 0)
#pragma unroll
        for (int g = 0; g < Q8G_HEADS; ++g) s_ml[warp][g] = make_float2(m[g], l[g]);
#pragma unroll
    for (int g = 0; g < Q8G_HEADS; ++g) {
        __syncthreads();
#pragma unroll
        for (int c = 0; c < LC; ++c) *reinterpret_cast<float4*>(&s_acc[warp][(lane + 32 * c) * 4]) = acc[g][c];
        __syncthreads();
        if (g >= gvalid) continue;
        for (int d = threadIdx.x * 2; d < p.D; d += 512) {
            float mg = -INFINITY;
#pragma unroll
            for (int w = 0; w < 8; ++w) mg = fmaxf(mg, s_ml[w][g].x);
            const float safe = mg == -INFINITY ? 0.0f : mg;
            float a0 = 0.0f, a1 = 0.0f, lg = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                const float f = ex2(s_ml[w][g].x - safe);
                a0 += s_acc[w][d] * f;
                a1 += s_acc[w][d + 1] * f;
                lg += s_ml[w][g].y * f;
            }
            if (p.nsplit == 1) {
                const float inv = lg != 0.0f ? 1.0f / lg : 0.0f;
                store2_any(p.out, ((size_t)b * p.Hq + h0 + g) * p.D + d, p.out_dt, a0 * inv, a1 * inv);
            } else {
                const size_t pr = (size_t)blockIdx.x * Q8G_HEADS + g;
                *reinterpret_cast<float2*>(p.ws_acc + pr * p.D + d) = make_float2(a0, a1);
                if (d == 0) *reinterpret_cast<float2*>(p.ws_ml + pr * 2) = make_float2(mg, lg);
            }
        }
    }
}

// ---- merge -------------------------------------------------------------------------
// Folds the partials of the units that were cut. TC: block c looks at the unit that begins in range c of the tensor-core
// kernel and ends in a later one, if any: its first partial is slot 2 c + 1, the next ones the even slots behind.
// Otherwise block u folds the nsplit slots of unit u of the generic kernel. All latency: the (m, l) of up to 32 partials and
// the first sums of each thread's are requested together; 4 teams of threads take every fourth partial, and their sums
// are added in order (one team: 1.5 us more with 19 partials; 2 or 8: 0.6 us more). gridDim.y blocks share a unit's sums,
// 128 float4 at a time.
constexpr int Q8M_TEAMS = 4, Q8M_TEAM = 128, Q8M_THREADS = Q8M_TEAMS * Q8M_TEAM;
template <bool TC>
__global__ void __launch_bounds__(Q8M_THREADS) q8_merge_kernel(const Q8Params p) {
    __shared__ float s_w[16][32];                   // weights of a round of 32 partials; -1: empty, its sums unwritten
    __shared__ float s_top[16], s_l[16], s_scale[16];
    __shared__ float4 s_sum[Q8M_TEAMS - 1][Q8M_TEAM];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int c = (int)blockIdx.x, tid = threadIdx.x;
    const int upb = p.Hkv * p.NCH;
    int b, ub, parts;
    if (TC) {
        const int4 d = __ldcg(p.desc + c);
        if (d.z < 2) return;
        b = d.x; ub = d.y; parts = d.z;
    } else {
        b = c / upb; ub = c - b * upb; parts = p.nsplit;
    }
    auto slot = [&](int j) -> size_t { return TC ? (j ? (size_t)2 * (c + j) : (size_t)2 * c + 1) : (size_t)c * parts + j; };
    const int kv = ub / p.NCH, ch = ub % p.NCH;
    const int gv = min(p.GC, p.G - ch * p.GC);
    const int h0 = kv * p.G + ch * p.GC;
    const int warp = tid >> 5, lane = tid & 31;
    const int team = tid / Q8M_TEAM, at = tid % Q8M_TEAM;
    const int quads = p.D >> 2, items = gv * quads;
    if (tid < 16) { s_top[tid] = -INFINITY; s_l[tid] = 0.0f; }
    const int i_first = (int)blockIdx.y * Q8M_TEAM;
    for (int i0 = i_first; i0 < items; i0 += (int)gridDim.y * Q8M_TEAM) {
        const int it = i0 + at;
        const int g = it < items ? it / quads : 0, d = it < items ? (it - g * quads) * 4 : 0;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int j0 = 0; j0 < parts; j0 += 32) {
            const int n = min(32, parts - j0);
            __syncthreads();
            // every fourth partial of the round, requested before anything is known about the weights (an empty one's slot
            // is allocated, its contents are not used)
            float4 v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int j = team + Q8M_TEAMS * q;
                v[q] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (it < items && j < n) v[q] = __ldcg(reinterpret_cast<const float4*>(p.ws_acc + (slot(j0 + j) * p.GC + g) * p.D + d));
            }
            if (i0 == i_first || parts > 32) {
                for (int gg = warp; gg < gv; gg += Q8M_THREADS / 32) {
                    float2 ml = make_float2(-INFINITY, 0.0f);
                    if (lane < n) ml = __ldcg(reinterpret_cast<const float2*>(p.ws_ml + (slot(j0 + lane) * p.GC + gg) * 2));
                    const float before = j0 ? s_top[gg] : -INFINITY;
                    float now = ml.y != 0.0f ? ml.x : -INFINITY;
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, o));
                    now = fmaxf(now, before);
                    const float safe = now == -INFINITY ? 0.0f : now;
                    const float f = ex2(ml.x - safe);
                    s_w[gg][lane] = ml.y != 0.0f ? f : -1.0f;
                    float sum = ml.y != 0.0f ? ml.y * f : 0.0f;
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if (lane == 0) {
                        s_scale[gg] = ex2(before - safe);
                        s_l[gg] = (j0 ? s_l[gg] * s_scale[gg] : 0.0f) + sum;
                        s_top[gg] = now;
                    }
                    __syncwarp();
                }
            }
            __syncthreads();
            if (j0) {
                const float r = s_scale[g];
                a.x *= r; a.y *= r; a.z *= r; a.w *= r;
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int j = team + Q8M_TEAMS * q;
                if (j >= n) break;
                const float f = s_w[g][j];
                if (f == -1.0f) continue;
                a.x = fmaf(v[q].x, f, a.x); a.y = fmaf(v[q].y, f, a.y); a.z = fmaf(v[q].z, f, a.z); a.w = fmaf(v[q].w, f, a.w);
            }
        }
        if (team) s_sum[team - 1][at] = a;
        __syncthreads();
        if (!team && it < items) {
#pragma unroll
            for (int t = 0; t < Q8M_TEAMS - 1; ++t) {
                const float4 v = s_sum[t][at];
                a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
            }
            const float l = s_l[g];
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;
            store4_any(p.out, ((size_t)b * p.Hq + h0 + g) * p.D + d, p.out_dt, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
        }
    }
}

}  // namespace ftk
