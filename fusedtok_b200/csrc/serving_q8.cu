// Host side of the 8-bit paged cache: argument checks, kernel selection and launch of the entry points
// fusedtok_attention_decode_paged_q8_*, fusedtok_kv_append_paged_q8_launch and fusedtok_block_table_*_launch
// (include/fusedtok_b200.h). No counterpart in the reference, which keeps its caches in the type of its queries and its
// block tables on the host (python/fusedtok/__init__.py:849-940 takes the table as given).

#include "../../include/fusedtok_b200.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>

#include "block_table.cuh"
#include "decode_q8.cuh"
#include "host.h"
#include "kv_append_q8.cuh"

namespace ftk {
cudaError_t q8_launch_int8_pow2(const CUtensorMap&, const CUtensorMap&, const Q8Params&, int nbk, bool split, cudaStream_t);
cudaError_t q8_launch_int8_other(const CUtensorMap&, const CUtensorMap&, const Q8Params&, int nbk, bool split, cudaStream_t);
cudaError_t q8_launch_e4m3_pow2(const CUtensorMap&, const CUtensorMap&, const Q8Params&, int nbk, bool split, cudaStream_t);
cudaError_t q8_launch_e4m3_other(const CUtensorMap&, const CUtensorMap&, const Q8Params&, int nbk, bool split, cudaStream_t);
}  // namespace ftk

namespace {

using namespace ftk;
using host::fail;

// bounded waits that expired in a decode launch; the one word is all the kernels keep between launches
__device__ int g_q8_status[64];

int runtime_fail(const char* what, cudaError_t e) {
    return fail(FUSEDTOK_RUNTIME_ERROR, std::string(what) + ": " + cudaGetErrorString(e));
}

// The current device and its status word (whose address is looked up once per device).
int status_word(int* device, int** word) {
    static std::atomic<int*> known[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return runtime_fail("cudaGetDevice", e);
    if (dev < 0 || dev >= 64) return fail(FUSEDTOK_RUNTIME_ERROR, "device index out of range");
    int* at = known[dev].load(std::memory_order_relaxed);
    if (!at) {
        void* base = nullptr;
        if ((e = cudaGetSymbolAddress(&base, g_q8_status)) != cudaSuccess) return runtime_fail("status word", e);
        at = static_cast<int*>(base) + dev;
        known[dev].store(at, std::memory_order_relaxed);
    }
    *device = dev;
    *word = at;
    return FUSEDTOK_OK;
}

// A launch whose kernel begins with griddepcontrol.wait, so that it may be set up while the one before it ends.
template <typename K, typename P>
int launch_pdl(K kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t cs, const P& p, const char* what) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = cs;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return runtime_fail(what, e);
    }
    return host::launched(what);
}

inline size_t up256(size_t x) { return (x + 255) / 256 * 256; }
inline bool power_of_two(int x) { return x > 0 && (x & (x - 1)) == 0; }

// How a decode call runs, from its shape and (`aligned`) its operands' alignment.
struct Q8Plan {
    bool tc = false, split = false;
    int GC = 1, NCH = 1, nbk = 1, ncta = 1, nsplit = 1, box_shift = 6;
    long long units = 0;
    size_t ml_b = 0, acc_b = 0, desc_b = 0;
    size_t bytes() const { return ml_b + acc_b + desc_b; }
};

Q8Plan plan_q8(int dtype, int batch, int hq, int hkv, int page, int width, int dim, int sms, bool aligned) {
    Q8Plan pl;
    const int G = hq / hkv;
    const long long rows = (long long)width * page;
    const long long tiles = (rows + TILE - 1) / TILE;
    const bool dims = dim == 64 || dim == 80 || dim == 96 || dim == 128 || dim == 192 || dim == 256;
    pl.tc = aligned && dims && power_of_two(page) && page >= 16 && batch <= SCHED_MAX_B && (long long)batch * tiles < (1ll << 31);
    if (pl.tc) {
        // two MMA columns per head where the heads then still fit one 8-column block: free, and float32's only way
        const int blocks = dim <= 128 ? 2 : 1;                  // column blocks whose accumulators fit the registers
        pl.split = dtype == 0 || G <= 4;
        const int per = pl.split ? 4 : 8;
        pl.nbk = std::min(blocks, (G + per - 1) / per);
        pl.GC = std::min(G, pl.nbk * per);
        pl.NCH = (G + pl.GC - 1) / pl.GC;
        pl.units = (long long)batch * hkv * pl.NCH;
        // As many CTAs as units where those have at most 8 tiles and are no more than the SMs: with equal lengths every unit is
        // then one CTA's, which works through 8 tiles in less time than partials and their fold take (8 heads of 64 x 512 rows:
        // 7.2 us on 8 CTAs, 9.2 on 64). Unequal lengths are cut at equal cost all the same, into fewer parts. With 16 tiles heads
        // of 64 would still gain (9.0 and 9.8); larger heads and groups, whose tiles take longer, were not measured there.
        pl.ncta = (int)(tiles <= 8 && pl.units <= sms ? pl.units : std::max<long long>(1, std::min<long long>(sms, pl.units * tiles)));
        for (pl.box_shift = 4; (1 << pl.box_shift) < std::min(page, TILE);) ++pl.box_shift;
        const size_t slots = (size_t)2 * pl.ncta;
        pl.ml_b = up256(slots * pl.GC * 8);
        pl.acc_b = up256(slots * pl.GC * dim * 4);
        pl.desc_b = up256((size_t)pl.ncta * sizeof(int4));
    } else {
        pl.GC = Q8G_HEADS;
        pl.NCH = (G + Q8G_HEADS - 1) / Q8G_HEADS;
        pl.units = (long long)batch * hkv * pl.NCH;
        // about two CTAs per SM, and no range below 64 rows
        const long long want = (2ll * sms + pl.units - 1) / std::max<long long>(1, pl.units);
        pl.nsplit = (int)std::max<long long>(1, std::min<long long>({want, (rows + 63) / 64, (long long)Q8_MAX_SPLIT}));
        if (pl.nsplit > 1) {
            const size_t slots = (size_t)pl.units * pl.nsplit;
            pl.ml_b = up256(slots * pl.GC * 8);
            pl.acc_b = up256(slots * pl.GC * dim * 4);
        }
    }
    return pl;
}

int decode_q8_check(int batch, int hq, int hkv, int page, int width, int dim) {
    if (batch < 0 || hq < 1 || hkv < 1 || dim < 1)
        return fail(FUSEDTOK_INVALID_ARGUMENT, "attention shapes must satisfy batch>=0, heads>=1, rows>=0, dim>=1");
    if (hq % hkv != 0)
        return fail(FUSEDTOK_INVALID_ARGUMENT, "q heads must be a multiple of kv heads (contiguous GQA groups)");
    if (dim % 4 != 0 || dim > 512) return fail(FUSEDTOK_INVALID_ARGUMENT, "dim must be a multiple of 4 and at most 512");
    if (page < 1) return fail(FUSEDTOK_INVALID_ARGUMENT, "page size must be >= 1");
    if (width < 0) return fail(FUSEDTOK_INVALID_ARGUMENT, "table width must be >= 0");
    if ((long long)width * page > (1LL << 30)) return fail(FUSEDTOK_INVALID_ARGUMENT, "table capacity too large");
    return FUSEDTOK_OK;
}

// A pool as 128-byte lines: its blocks are contiguous, so a box of lines is a run of rows whatever the head dim.
int encode_lines(host::EncodeTiledFn encode, CUtensorMap* map, const void* base, unsigned long long bytes, int box_lines) {
    const cuuint64_t gdim[2] = {128u, (cuuint64_t)(bytes >> 7)};
    const cuuint64_t gstride[1] = {128u};
    const cuuint32_t box[2] = {128u, (cuuint32_t)box_lines};
    const cuuint32_t estr[2] = {1u, 1u};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), gdim, gstride, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(FUSEDTOK_RUNTIME_ERROR, "cuTensorMapEncodeTiled failed (code " + std::to_string((int)r) + ")");
    return FUSEDTOK_OK;
}

int block_table_check(const BlockTableParams& p) {
    if (p.B < 0 || p.width < 0 || p.page < 1 || p.capacity < 0 || p.max_tokens < 0)
        return fail(FUSEDTOK_INVALID_ARGUMENT, "block table shapes must satisfy batch>=0, width>=0, page>=1, capacity>=0, tokens>=0");
    if (p.B > BT_MAX_BATCH)
        return fail(FUSEDTOK_INVALID_ARGUMENT, "block table operators take at most " + std::to_string(BT_MAX_BATCH) + " sequences");
    if ((long long)p.width * p.page > (1LL << 30)) return fail(FUSEDTOK_INVALID_ARGUMENT, "table capacity too large");
    return FUSEDTOK_OK;
}

}  // namespace

namespace ftk {
namespace host {
int q8_status(int* status) {
    int dev = 0, word = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return runtime_fail("cudaGetDevice", e);
    *status = 0;
    if (dev < 0 || dev >= 64) return FUSEDTOK_OK;
    const size_t at = (size_t)dev * sizeof(int);
    if ((e = cudaMemcpyFromSymbol(&word, g_q8_status, sizeof(int), at)) != cudaSuccess) return runtime_fail("status read failed", e);
    if (word != 0) {
        const int zero = 0;
        if ((e = cudaMemcpyToSymbol(g_q8_status, &zero, sizeof(int), at)) != cudaSuccess) return runtime_fail("status clear failed", e);
        *status = word;
    }
    return FUSEDTOK_OK;
}
}  // namespace host
}  // namespace ftk

extern "C" {

long long fusedtok_attention_decode_paged_q8_workspace(int dtype, int batch, int q_heads, int kv_heads, int page, int tbl_width, int dim) {
    if (dtype < 0 || dtype > 2) return -(long long)fail(FUSEDTOK_INVALID_ARGUMENT, "dtype must be 0 (f32), 1 (bf16) or 2 (fp16)");
    int rc = decode_q8_check(batch, q_heads, kv_heads, page, tbl_width, dim);
    if (rc) return -(long long)rc;
    if (batch == 0 || tbl_width == 0) return 0;
    int sms = 0;
    if ((rc = host::current_sm_count(&sms))) return -(long long)rc;
    // whichever kernel the operands' alignment selects
    return (long long)std::max(plan_q8(dtype, batch, q_heads, kv_heads, page, tbl_width, dim, sms, true).bytes(),
                               plan_q8(dtype, batch, q_heads, kv_heads, page, tbl_width, dim, sms, false).bytes());
}

int fusedtok_attention_decode_paged_q8_launch(int dtype, int store, const void* q, const void* k_pool, const void* v_pool,
                                              const float* kv_scales, const int* table, const int* lens, void* out,
                                              void* workspace, long long workspace_bytes, int batch, int q_heads, int kv_heads,
                                              int page, int tbl_width, long long num_blocks, int dim, uintptr_t stream) {
    if (dtype < 0 || dtype > 2) return fail(FUSEDTOK_INVALID_ARGUMENT, "dtype must be 0 (f32), 1 (bf16) or 2 (fp16)");
    if (store < 0 || store > 1) return fail(FUSEDTOK_INVALID_ARGUMENT, "store must be 0 (int8) or 1 (e4m3)");
    int rc = decode_q8_check(batch, q_heads, kv_heads, page, tbl_width, dim);
    if (rc) return rc;
    if (batch == 0) return FUSEDTOK_OK;
    if (num_blocks < 0) return fail(FUSEDTOK_INVALID_ARGUMENT, "the pool must have at least 0 blocks");
    if (!q || !out) return fail(FUSEDTOK_INVALID_ARGUMENT, "null attention operand");
    const size_t es = dtype == 0 ? 4 : 2;
    cudaStream_t cs = (cudaStream_t)stream;
    if (tbl_width == 0 || num_blocks == 0) {                 // no cache rows at all: zero rows, like the other decode operators
        const cudaError_t e = cudaMemsetAsync(out, 0, (size_t)batch * q_heads * dim * es, cs);
        return e == cudaSuccess ? FUSEDTOK_OK : runtime_fail("attention zero fill failed", e);
    }
    if (!k_pool || !v_pool || !kv_scales || !table) return fail(FUSEDTOK_INVALID_ARGUMENT, "null attention operand");
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & (4 * es - 1))
        return fail(FUSEDTOK_INVALID_ARGUMENT, "attention operands must be aligned to 4 elements");
    const uintptr_t pools = reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool);
    if ((pools & 3u) || (reinterpret_cast<uintptr_t>(kv_scales) & 7u))
        return fail(FUSEDTOK_INVALID_ARGUMENT, "pools must be aligned to 4 bytes and scales to 8");
    int sms = 0;
    if ((rc = host::current_sm_count(&sms))) return rc;
    const unsigned long long pool_bytes = (unsigned long long)num_blocks * kv_heads * page * dim;
    const bool aligned = (pools & 15u) == 0 && (pool_bytes >> 7) < (1ull << 31);
    const Q8Plan pl = plan_q8(dtype, batch, q_heads, kv_heads, page, tbl_width, dim, sms, aligned);
    if (pl.units * pl.nsplit > 0x7fffffffll) return fail(FUSEDTOK_INVALID_ARGUMENT, "attention shape too large for one launch");
    if (pl.bytes() && (!workspace || workspace_bytes < (long long)pl.bytes() || (reinterpret_cast<uintptr_t>(workspace) & 15u)))
        return fail(FUSEDTOK_INVALID_ARGUMENT, "the decode workspace must be 16-byte aligned device memory of at least " +
                                                   std::to_string(pl.bytes()) + " bytes");
    Q8Params p;
    memset(&p, 0, sizeof(p));
    p.q = q; p.k = k_pool; p.v = v_pool; p.out = out; p.lens = lens; p.table = table;
    p.B = batch; p.Hq = q_heads; p.Hkv = kv_heads; p.G = q_heads / kv_heads; p.T = tbl_width * page; p.D = dim;
    p.page = page; p.tbl_width = tbl_width;
    p.scale = 1.0f / sqrtf((float)dim);
    p.GC = pl.GC; p.NCH = pl.NCH; p.ncta = pl.ncta;
    p.full = pl.ncta >= sms;
    p.box_shift = pl.box_shift; p.box_rows = 1 << pl.box_shift;
    p.scales = reinterpret_cast<const float2*>(kv_scales);
    p.blocks = num_blocks;
    p.out_dt = dtype;
    p.nsplit = pl.nsplit;
    char* ws = static_cast<char*>(workspace);
    p.ws_ml = reinterpret_cast<float*>(ws);
    p.ws_acc = reinterpret_cast<float*>(ws + pl.ml_b);
    p.desc = reinterpret_cast<int4*>(ws + pl.ml_b + pl.acc_b);
    p.bound_slots = 2u * (unsigned)pl.ncta;
    p.bound_rows = (unsigned long long)num_blocks * kv_heads * page;
    if ((rc = status_word(&p.device, &p.status))) return rc;
    cudaError_t e = cudaSuccess;
    // Blocks per unit of the merge: one for every 128 sums where that makes no more of them than SMs (4 sequences of 571 - 2061
    // rows, 4 kv heads: with 16 heads each 20.3 us instead of 22.8, with 8 14.1 instead of 14.8), else one (32 x 4096 rows, 8 kv heads
    // of 16: 82.2 us, and 85.3 with four: blocks without a unit to merge hold the next launch up)
    const long long per_unit = (pl.GC * (dim / 4) + Q8M_TEAM - 1) / Q8M_TEAM;
    const unsigned slices = pl.units * per_unit <= sms ? (unsigned)per_unit : 1u;
    if (pl.tc) {
        host::EncodeTiledFn encode = nullptr;
        if ((rc = host::encoder(&encode))) return rc;
        CUtensorMap mk, mv;
        const int lines = p.box_rows * dim / 128;
        if ((rc = encode_lines(encode, &mk, k_pool, pool_bytes, lines))) return rc;
        if ((rc = encode_lines(encode, &mv, v_pool, pool_bytes, lines))) return rc;
        const bool pow2 = power_of_two(dim);
        if (store == 0) e = pow2 ? q8_launch_int8_pow2(mk, mv, p, pl.nbk, pl.split, cs) : q8_launch_int8_other(mk, mv, p, pl.nbk, pl.split, cs);
        else e = pow2 ? q8_launch_e4m3_pow2(mk, mv, p, pl.nbk, pl.split, cs) : q8_launch_e4m3_other(mk, mv, p, pl.nbk, pl.split, cs);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return runtime_fail("8-bit decode kernel launch", e);
        }
        if ((rc = host::launched("8-bit decode kernel launch"))) return rc;
        return launch_pdl(q8_merge_kernel<true>, dim3((unsigned)pl.ncta, slices), dim3(Q8M_THREADS), 0, cs, p, "8-bit decode merge launch");
    }
    const dim3 grid((unsigned)(pl.units * pl.nsplit));
    const int lc = dim <= 128 ? 1 : dim <= 256 ? 2 : 4;
#define FTK_GO(KV, LC) rc = launch_pdl(decode_q8_generic_kernel<KV, LC>, grid, dim3(256), 0, cs, p, "8-bit decode generic kernel launch")
    if (store == 0) { if (lc == 1) FTK_GO(int8_t, 1); else if (lc == 2) FTK_GO(int8_t, 2); else FTK_GO(int8_t, 4); }
    else { if (lc == 1) FTK_GO(__nv_fp8_e4m3, 1); else if (lc == 2) FTK_GO(__nv_fp8_e4m3, 2); else FTK_GO(__nv_fp8_e4m3, 4); }
#undef FTK_GO
    if (rc || pl.nsplit == 1) return rc;
    return launch_pdl(q8_merge_kernel<false>, dim3((unsigned)pl.units, slices), dim3(Q8M_THREADS), 0, cs, p, "8-bit decode merge launch");
}

int fusedtok_kv_append_paged_q8_launch(int dtype, int store, const void* k_new, const void* v_new, const int* slots, void* k_pool,
                                       void* v_pool, float* kv_scales, int tokens, int kv_heads, int dim, int page,
                                       long long num_blocks, uintptr_t stream) {
    if (dtype < 0 || dtype > 2) return fail(FUSEDTOK_INVALID_ARGUMENT, "dtype must be 0 (f32), 1 (bf16) or 2 (fp16)");
    if (store < 0 || store > 1) return fail(FUSEDTOK_INVALID_ARGUMENT, "store must be 0 (int8) or 1 (e4m3)");
    if (tokens < 0 || kv_heads < 1 || kv_heads > 65535 || dim < 1 || num_blocks < 0)
        return fail(FUSEDTOK_INVALID_ARGUMENT, "kv append shapes must satisfy tokens>=0, 65535>=heads>=1, dim>=1, blocks>=0");
    if (dim % 4 != 0 || dim > 512) return fail(FUSEDTOK_INVALID_ARGUMENT, "dim must be a multiple of 4 and at most 512");
    if (page < 1) return fail(FUSEDTOK_INVALID_ARGUMENT, "page size must be >= 1");
    if (num_blocks * page > 0x7fffffffll) return fail(FUSEDTOK_INVALID_ARGUMENT, "the pool has more rows than a slot can name");
    if ((long long)page * dim > 0x7fffffffll) return fail(FUSEDTOK_INVALID_ARGUMENT, "a block's rows of one head must be below 2^31 bytes");
    if (tokens == 0 || num_blocks == 0) return FUSEDTOK_OK;
    if (!k_new || !v_new || !slots || !k_pool || !v_pool || !kv_scales) return fail(FUSEDTOK_INVALID_ARGUMENT, "null kv append operand");
    const size_t es = dtype == 0 ? 4 : 2;
    const uintptr_t news = reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new);
    const uintptr_t pools = reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool);
    if ((news & (4 * es - 1)) || (pools & 3u) || (reinterpret_cast<uintptr_t>(kv_scales) & 3u))
        return fail(FUSEDTOK_INVALID_ARGUMENT, "new rows must be aligned to 4 elements, pools and scales to 4 bytes");
    const uintptr_t ka = reinterpret_cast<uintptr_t>(k_pool), va = reinterpret_cast<uintptr_t>(v_pool);
    if ((ka < va ? va - ka : ka - va) < (unsigned long long)num_blocks * kv_heads * page * dim)
        return fail(FUSEDTOK_INVALID_ARGUMENT, "the K and V pools must not overlap");
    int sms = 0;
    const int rc = host::current_sm_count(&sms);
    if (rc) return rc;
    AppendQ8Params p;
    p.x_new[0] = k_new; p.x_new[1] = v_new;
    p.pool[0] = static_cast<uint8_t*>(k_pool); p.pool[1] = static_cast<uint8_t*>(v_pool);
    p.scales = kv_scales; p.slots = slots;
    p.N = tokens; p.Hkv = kv_heads; p.D = dim; p.page = page;
    p.rows = num_blocks * page;
    const bool wide = es == 2 && dim % 8 == 0 && (news & 15u) == 0 && (pools & 7u) == 0;
    p.groups = (2 * kv_heads + 3) / 4;
    // as few tokens per CTA as leave all CTAs resident at once (5 per SM), up to 128
    const long long work = (long long)tokens * p.groups, room = 5ll * sms;
    p.window = (int)std::min<long long>((work + room - 1) / room, (long long)AQ_THREADS);
    const long long ctas = ((tokens + p.window - 1) / p.window) * (long long)p.groups;
    if (ctas > 0x7fffffffll) return fail(FUSEDTOK_INVALID_ARGUMENT, "too many tokens and heads for one launch");
    const dim3 grid((unsigned)ctas);
    cudaStream_t cs = (cudaStream_t)stream;
    const char* what = "8-bit kv append kernel launch";
    // no run is longer than a block
    const bool lng = (long long)page * dim > (long long)AQ_RING * AQ_BATCH * (wide ? 8 : 4);
#define FTK_LAUNCH(T, KV, V)                                                                                            \
    return lng ? launch_pdl(kv_append_q8_kernel<T, KV, V, true>, grid, dim3(AQ_THREADS), 0, cs, p, what)                \
               : launch_pdl(kv_append_q8_kernel<T, KV, V, false>, grid, dim3(AQ_THREADS), 0, cs, p, what)
#define FTK_GO(T, V)                                        \
    do {                                                    \
        if (store == 0) FTK_LAUNCH(T, int8_t, V);           \
        FTK_LAUNCH(T, __nv_fp8_e4m3, V);                    \
    } while (0)
    if (dtype == 0) FTK_GO(float, 4);
    if (dtype == 1) { if (wide) FTK_GO(__nv_bfloat16, 8); FTK_GO(__nv_bfloat16, 4); }
    if (wide) FTK_GO(__half, 8);
    FTK_GO(__half, 4);
#undef FTK_GO
#undef FTK_LAUNCH
}

int fusedtok_block_table_extend_launch(int* table, const int* lens, const int* new_lens, const int* free_blocks,
                                       const int* free_count, int* slots, int* starts, int* lens_out, int* free_count_out,
                                       int batch, int tbl_width, int page, int free_capacity, int max_tokens, uintptr_t stream) {
    BlockTableParams p{table, lens, new_lens, const_cast<int*>(free_blocks), free_count, slots, starts, lens_out, free_count_out,
                       batch, tbl_width, page, free_capacity, max_tokens};
    int rc = block_table_check(p);
    if (rc) return rc;
    if ((batch && (!lens || !new_lens || !lens_out)) || (batch && tbl_width && !table) || (free_capacity && !free_blocks) ||
        !free_count || !free_count_out || !starts || (max_tokens && !slots))
        return fail(FUSEDTOK_INVALID_ARGUMENT, "null block table operand");
    int sms = 0;
    if ((rc = host::current_sm_count(&sms))) return rc;
    // 4 slots per thread; every CTA repeats the prefix sums, so no more of them than that and a few for the table
    const long long want = std::max<long long>(((long long)max_tokens + BT_THREADS * 4 - 1) / (BT_THREADS * 4), (batch + 255) / 256);
    const dim3 grid((unsigned)std::max<long long>(1, std::min<long long>(want, sms)));
    const size_t smem = (size_t)batch * 8 + 4;
    if (smem > 40000) {
        const cudaError_t e = cudaFuncSetAttribute(block_table_extend_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BT_MAX_BATCH * 8 + 4);
        if (e != cudaSuccess) return runtime_fail("cudaFuncSetAttribute", e);
    }
    return launch_pdl(block_table_extend_kernel, grid, dim3(BT_THREADS), smem, (cudaStream_t)stream, p, "block table extend launch");
}

int fusedtok_block_table_trim_launch(const int* table, const int* lens, const int* keep_lens, int* free_blocks, const int* free_count,
                                     int* lens_out, int* free_count_out, int batch, int tbl_width, int page, int free_capacity,
                                     uintptr_t stream) {
    BlockTableParams p{const_cast<int*>(table), lens, keep_lens, free_blocks, free_count, nullptr, nullptr, lens_out, free_count_out,
                       batch, tbl_width, page, free_capacity, 0};
    int rc = block_table_check(p);
    if (rc) return rc;
    if ((batch && (!lens || !keep_lens || !lens_out)) || (batch && tbl_width && !table) || (free_capacity && !free_blocks) ||
        !free_count || !free_count_out)
        return fail(FUSEDTOK_INVALID_ARGUMENT, "null block table operand");
    int sms = 0;
    if ((rc = host::current_sm_count(&sms))) return rc;
    // an entry per thread if a quarter of all that the table has go back
    const long long want = ((long long)batch * tbl_width + 4 * BT_THREADS - 1) / (4 * BT_THREADS);
    const dim3 grid((unsigned)std::max<long long>(1, std::min<long long>(want, sms)));
    return launch_pdl(block_table_trim_kernel, grid, dim3(BT_THREADS), (size_t)batch * 4, (cudaStream_t)stream, p, "block table trim launch");
}

}  // extern "C"
