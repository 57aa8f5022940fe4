// paged.cu — host side of the operators over the paged cache (include/fiber_paged.h).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <atomic>

#include "fiber_cuda.h"
#include "fiber_paged.h"
#include "launch.cuh"
#include "paged_append.cuh"
#include "paged_rows.cuh"
#include "paged_tile.cuh"

using namespace fiber;

void fiber_set_error_message(const char *msg);  // fiber_cuda.cu

namespace {

int fail(int code, const char *fmt, ...) {
    char msg[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof(msg), fmt, ap);
    va_end(ap);
    fiber_set_error_message(msg);
    return code;
}

int sm_count() {
    static int cache[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if (!cache[dev]) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        cache[dev] = n;
    }
    return cache[dev];
}

std::atomic<int> drill{0};

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// A stride in elements that TMA and 16-byte accesses can use.
bool stride_ok(int64_t s, int64_t least) { return s >= least && s % 8 == 0 && s < (1ll << 38); }

int check_view(const char *fn, const fiber_kv_view_t *kv) {
    if (!kv || !kv->k_pool || !kv->v_pool || !kv->page_table) return fail(FIBER_EARG, "%s: null cache", fn);
    if (kv->type != FIBER_TYPE_F16 && kv->type != FIBER_TYPE_BF16)
        return fail(FIBER_EARG, "%s: cache type %d is not F16 or BF16", fn, kv->type);
    if (kv->head_dim != 64 && kv->head_dim != 128)
        return fail(FIBER_EARG, "%s: head_dim %d is not 64 or 128", fn, kv->head_dim);
    const int P = kv->page_size;
    if (P < 16 || P > 256 || (P & (P - 1)))
        return fail(FIBER_EARG, "%s: page_size %d is not 16, 32, 64, 128 or 256", fn, P);
    if (kv->n_kv_heads <= 0 || kv->n_pages <= 0 || kv->n_slots <= 0 || kv->max_pages <= 0)
        return fail(FIBER_EARG, "%s: bad cache shape (kv_heads=%d pages=%d slots=%d max_pages=%d)", fn, kv->n_kv_heads,
                    kv->n_pages, kv->n_slots, kv->max_pages);
    // positions are rounded up to whole tiles and pages in 32 bits
    if ((int64_t)kv->max_pages * P > 0x7fffff00) return fail(FIBER_EARG, "%s: a slot holds more than 2^31 - 256 positions", fn);
    if (!aligned16(kv->k_pool) || !aligned16(kv->v_pool)) return fail(FIBER_EARG, "%s: pools must be 16-byte aligned", fn);
    if (!stride_ok(kv->pos_stride, kv->head_dim) || !stride_ok(kv->head_stride, kv->head_dim) ||
        !stride_ok(kv->page_stride, kv->head_dim))
        return fail(FIBER_EARG, "%s: strides must be multiples of 8 elements, at least head_dim", fn);
    return FIBER_OK;
}

int check_batch(const char *fn, const fiber_ragged_t *b) {
    if (!b || b->n_seqs < 0 || b->n_tokens < 0) return fail(FIBER_EARG, "%s: bad batch", fn);
    if (b->n_seqs && b->n_tokens && (!b->q_start || !b->kv_len))
        return fail(FIBER_EARG, "%s: null q_start or kv_len", fn);
    return FIBER_OK;
}

// Token rows of `width` values in elements of `size` bytes.
int check_rows(const char *fn, const char *what, const void *p, int64_t ld, int64_t width, int size) {
    if (!p) return fail(FIBER_EARG, "%s: null %s", fn, what);
    if (ld < width || (ld * size) % 16 || ld >= (1ll << 38) || !aligned16(p))
        return fail(FIBER_EARG, "%s: %s rows must be 16-byte aligned and hold %lld values (ld=%lld)", fn, what,
                    (long long)width, (long long)ld);
    return FIBER_OK;
}

PagedView dev_view(const fiber_kv_view_t *kv) {
    PagedView v;
    v.k = (uint16_t *)kv->k_pool;
    v.v = (uint16_t *)kv->v_pool;
    v.table = kv->page_table;
    v.n_kv = kv->n_kv_heads;
    v.page_shift = 0;
    while ((1 << v.page_shift) < kv->page_size) v.page_shift++;
    v.n_pages = kv->n_pages;
    v.n_slots = kv->n_slots;
    v.max_pages = kv->max_pages;
    v.page_stride = kv->page_stride;
    v.head_stride = kv->head_stride;
    v.pos_stride = kv->pos_stride;
    return v;
}

RaggedDev dev_batch(const fiber_ragged_t *b) {
    RaggedDev r;
    r.n_seqs = b->n_seqs;
    r.n_tokens = b->n_tokens;
    r.slot0 = 0;
    r.q_start = b->q_start;
    r.kv_len = b->kv_len;
    r.slot = b->slot;
    return r;
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return (PFN_cuTensorMapEncodeTiled_v12000)fn;
    }();
    return encode;
}

// Map of a pool: (head_dim, page_size, n_kv, n_pages), box of 64 dims x `rows` positions of
// one page, 128-byte swizzle; what lies outside reads as zeros.
bool pool_map(CUtensorMap *map, const void *pool, const fiber_kv_view_t *kv, int rows) {
    auto enc = encoder();
    if (!enc) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)kv->head_dim, (cuuint64_t)kv->page_size, (cuuint64_t)kv->n_kv_heads,
                                (cuuint64_t)kv->n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)kv->pos_stride * 2, (cuuint64_t)kv->head_stride * 2,
                                   (cuuint64_t)kv->page_stride * 2};
    const cuuint32_t box[4] = {64u, (cuuint32_t)std::min(rows, kv->page_size), 1u, 1u}, one[4] = {1, 1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void *>(pool), dims, strides, box, one,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Map of the query rows: (head_dim, n_heads, n_tokens), box of 64 dims x the group's heads x
// a tile's tokens.
bool query_map(CUtensorMap *map, const void *q, int hd, int n_heads, int group, long long ldq, int n_tokens) {
    auto enc = encoder();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)n_heads, (cuuint64_t)n_tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)ldq * 2};
    const cuuint32_t box[3] = {64u, (cuuint32_t)group, (cuuint32_t)(PT_ROWS / group)}, one[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void *>(q), dims, strides, box, one,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class TI, bool BF>
cudaError_t launch_append(const AppendParams &p, int hd, cudaStream_t st) {
    const long long warps = (long long)p.b.n_tokens * append_warps_per_token(p.n_heads + 2 * p.kv.n_kv, hd);
    const long long grid = (warps + APPEND_THREADS / 32 - 1) / (APPEND_THREADS / 32);
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    return launch_pdl(hd == 64 ? kv_append_kernel<TI, BF, 64> : kv_append_kernel<TI, BF, 128>, dim3((unsigned)grid),
                      dim3(APPEND_THREADS), 0, st, p);
}

// Workspace: status, tickets, then the split units' softmax states.
constexpr size_t WS_TICKETS = 256, WS_PARTS = WS_TICKETS + 4096;
constexpr int WS_MAX_CTAS = 1024;

// {unit, half, full, snap, share, root}
constexpr AttnCost PR_COST = {3, 1, 1, 8, 1, 0.8f}, PT_COST = {4, 3, 4, 4, 4, 1.0f};

struct AttnShape {
    bool tile;        // tile kernel, else row kernel
    int n_cta, rows;  // CTAs of a launch, rows of a unit's state
};

// Up to 16 rows per KV head the row kernel reads K and V once; above, once per 16 rows. 24
// sequences over 6,000 positions, 8 KV heads, fp16, us (events around a call), row / tile kernel:
//     rows         16           20           32           64          128
//     dim 64    74 / 102    111 / 102    113 / 102    209 / 102    303 / 107
//     dim 128  126 / 123    206 / 124    207 / 124    379 / 126    691 / 131
// In calls that leave SMs idle the row kernel is ahead to 32 rows (8 sequences over 1,500, dim 64: 24 / 27).
bool tile_kernel(const fiber_kv_view_t *kv, const fiber_ragged_t *b, int n_heads) {
    return b->max_q * (long long)(n_heads / kv->n_kv_heads) > PR_ROWS;
}

AttnShape attn_shape(const fiber_kv_view_t *kv, const fiber_ragged_t *b, int n_heads) {
    if (tile_kernel(kv, b, n_heads))
        return {true, std::min(sm_count(), WS_MAX_CTAS), 2 * PT_ROWS};
    return {false, std::min(sm_count() * PR_CTAS_PER_SM, WS_MAX_CTAS), PR_ROWS};
}

size_t ws_bytes_of(const AttnShape &s, int hd) { return WS_PARTS + (size_t)2 * s.n_cta * s.rows * (hd + 2) * 4; }

// Raise a kernel's shared-memory limit, once per device.
template <class K>
cudaError_t allow_smem(K kernel, int bytes, bool (&ready)[64]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && ready[dev])) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) ready[dev] = true;
    return e;
}

template <int HD, bool BF>
cudaError_t launch_attn(const AttnPagedParams &p, const AttnShape &s, cudaStream_t st) {
    static bool ready_tile[64], ready_rows[64];
    if (s.tile) {
        cudaError_t e = allow_smem(attn_tile_kernel<HD, BF>, pt_smem<HD>(), ready_tile);
        return e ? e : launch_pdl(attn_tile_kernel<HD, BF>, dim3(s.n_cta), dim3(PT_THREADS), pt_smem<HD>(), st, p);
    }
    cudaError_t e = allow_smem(attn_rows_kernel<HD, BF>, pr_smem<HD>(), ready_rows);
    return e ? e : launch_pdl(attn_rows_kernel<HD, BF>, dim3(s.n_cta), dim3(PR_THREADS), pr_smem<HD>(), st, p);
}

int check_attn(const char *fn, const fiber_kv_view_t *kv, const fiber_ragged_t *b, int n_heads) {
    int rc = check_view(fn, kv);
    if (rc == FIBER_OK) rc = check_batch(fn, b);
    if (rc) return rc;
    if (b->n_tokens && b->max_q < 1) return fail(FIBER_EARG, "%s: max_q %d", fn, b->max_q);
    if (n_heads <= 0 || n_heads % kv->n_kv_heads || n_heads / kv->n_kv_heads > 128)
        return fail(FIBER_EARG, "%s: %d query heads over %d KV heads", fn, n_heads, kv->n_kv_heads);
    // Rows of a sequence, and the cost of a launch (attn_plan_build), are counted in 32 bits: at
    // most this many units, none of more steps than the table has room for.
    const int group = n_heads / kv->n_kv_heads;
    const bool tile = tile_kernel(kv, b, n_heads);
    const double rows = (double)b->n_tokens * group, ru = tile ? 2 * pt_tile_rows(group) : PR_ROWS;
    const double units = (rows / ru + std::min(b->n_seqs, PG_MAX_SEQS)) * kv->n_kv_heads;
    const AttnCost cost = tile ? PT_COST : PR_COST;
    const double steps = (double)kv->max_pages * kv->page_size / (tile ? PT_BK : PR_BK) + 1;
    if (rows > 2147483647. - 2 * PT_ROWS || units * (cost.unit + cost.full * steps) > 4294967295.)
        return fail(FIBER_EARG, "%s: batch too large (%d tokens over %d positions)", fn, b->n_tokens,
                    kv->max_pages * kv->page_size);
    return FIBER_OK;
}

}  // namespace

extern "C" int fiber_kv_view(const kv_cache_t *kv, int layer, fiber_kv_view_t *out) {
    if (!kv || !out || layer < 0 || layer >= kv->n_layers) return fail(FIBER_EARG, "fiber_kv_view: bad argument (layer %d)", layer);
    memset(out, 0, sizeof(*out));
    const int64_t head = (int64_t)kv->page_size * kv->head_dim;
    out->type = FIBER_TYPE_F16;
    out->head_dim = kv->head_dim;
    out->n_kv_heads = kv->n_kv_heads;
    out->page_size = kv->page_size;
    out->n_pages = kv->n_pages;
    out->n_slots = kv->max_batch;
    out->max_pages = kv->max_pages_per_seq;
    out->pos_stride = kv->head_dim;
    out->head_stride = head;
    out->page_stride = head * kv->n_kv_heads * kv->n_layers;
    out->k_pool = kv->k_pool + (size_t)layer * kv->n_kv_heads * head;
    out->v_pool = kv->v_pool + (size_t)layer * kv->n_kv_heads * head;
    out->page_table = kv->page_table;
    return FIBER_OK;
}

extern "C" int fiber_kv_append(const fiber_kv_view_t *kv, const fiber_ragged_t *batch, int in_type, const void *d_q,
                               int64_t ldq, const void *d_k, int64_t ldk, const void *d_v, int64_t ldv, int n_heads,
                               const fiber_rope_t *rope, void *d_q_out, int64_t ldo, void *stream) {
    const char *fn = "fiber_kv_append";
    int rc = check_view(fn, kv);
    if (rc == FIBER_OK) rc = check_batch(fn, batch);
    if (rc) return rc;
    if (in_type != FIBER_TYPE_F32 && in_type != kv->type)
        return fail(FIBER_EARG, "%s: input type %d is neither F32 nor the cache's type %d", fn, in_type, kv->type);
    if (batch->n_seqs == 0 || batch->n_tokens == 0) return FIBER_OK;
    const int size = in_type == FIBER_TYPE_F32 ? 4 : 2, hd = kv->head_dim;
    if (!d_q != !d_q_out) return fail(FIBER_EARG, "%s: d_q and d_q_out go together", fn);
    if (d_q) {
        if (n_heads <= 0) return fail(FIBER_EARG, "%s: n_heads %d", fn, n_heads);
        if ((rc = check_rows(fn, "q", d_q, ldq, (int64_t)n_heads * hd, size))) return rc;
        if ((rc = check_rows(fn, "q_out", d_q_out, ldo, (int64_t)n_heads * hd, 2))) return rc;
    }
    if ((rc = check_rows(fn, "k", d_k, ldk, (int64_t)kv->n_kv_heads * hd, size))) return rc;
    if ((rc = check_rows(fn, "v", d_v, ldv, (int64_t)kv->n_kv_heads * hd, size))) return rc;
    if (rope && (!rope->table || !aligned16(rope->table) || rope->max_pos <= 0 || rope->dim <= 0 || rope->dim % 16 ||
                 rope->dim > hd))
        return fail(FIBER_EARG, "%s: bad rope (dim %d, a multiple of 16 up to head_dim; table 16-byte aligned)", fn, rope->dim);
    if (d_q && d_q == d_q_out && (in_type == FIBER_TYPE_F32 || ldq != ldo))
        return fail(FIBER_EARG, "%s: in place, q and q_out have one type and one row stride", fn);
    AppendParams p;
    memset(&p, 0, sizeof(p));
    p.kv = dev_view(kv);
    p.b = dev_batch(batch);
    p.q = d_q;
    p.k = d_k;
    p.v = d_v;
    p.ldq = ldq;
    p.ldk = ldk;
    p.ldv = ldv;
    p.ldo = ldo;
    p.n_heads = d_q ? n_heads : 0;
    if (rope) {
        p.rope = (const float2 *)rope->table;
        p.max_pos = rope->max_pos;
        p.rot = rope->dim;
        p.adjacent = rope->adjacent != 0;
    }
    p.q_out = (uint16_t *)d_q_out;
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (kv->type == FIBER_TYPE_F16)
        e = in_type == FIBER_TYPE_F32 ? launch_append<float, false>(p, hd, st) : launch_append<__half, false>(p, hd, st);
    else
        e = in_type == FIBER_TYPE_F32 ? launch_append<float, true>(p, hd, st) : launch_append<__nv_bfloat16, true>(p, hd, st);
    return e == cudaSuccess ? FIBER_OK : fail(FIBER_ECUDA, "%s: %s", fn, cudaGetErrorString(e));
}

extern "C" size_t fiber_attn_paged_workspace(const fiber_kv_view_t *kv, const fiber_ragged_t *batch, int n_heads) {
    if (check_attn("fiber_attn_paged_workspace", kv, batch, n_heads)) return 0;
    return ws_bytes_of(attn_shape(kv, batch, n_heads), kv->head_dim);
}

extern "C" int fiber_attn_paged(const fiber_kv_view_t *kv, const fiber_ragged_t *batch, const void *d_q, int64_t ldq,
                                void *d_out, int64_t ldo, int n_heads, float scale, int window, void *d_ws,
                                size_t ws_bytes, void *stream) {
    const char *fn = "fiber_attn_paged";
    int rc = check_attn(fn, kv, batch, n_heads);
    if (rc) return rc;
    if (!(scale > 0.f) || !isfinite(scale)) return fail(FIBER_EARG, "%s: scale must be positive and finite", fn);
    if (window < 0) return fail(FIBER_EARG, "%s: window %d", fn, window);
    if (batch->n_seqs == 0 || batch->n_tokens == 0) return FIBER_OK;
    const int hd = kv->head_dim;
    if ((rc = check_rows(fn, "q", d_q, ldq, (int64_t)n_heads * hd, 2))) return rc;
    if ((rc = check_rows(fn, "out", d_out, ldo, (int64_t)n_heads * hd, 2))) return rc;
    const AttnShape shape = attn_shape(kv, batch, n_heads);
    if (!d_ws || !aligned16(d_ws) || ws_bytes < ws_bytes_of(shape, hd))
        return fail(FIBER_EARG, "%s: workspace of %zu bytes, 16-byte aligned, needed (%zu given)", fn,
                    ws_bytes_of(shape, hd), ws_bytes);
    if (d_q == d_out)  // a row that is computed again reads its query after its first result is stored
        return fail(FIBER_EARG, "%s: d_q and d_out are the same buffer", fn);
    AttnPagedParams p;
    memset(&p, 0, sizeof(p));
    p.kv = dev_view(kv);
    p.b = dev_batch(batch);
    p.q = (const uint16_t *)d_q;
    p.out = (uint16_t *)d_out;
    p.ldq = ldq;
    p.ldo = ldo;
    p.n_heads = n_heads;
    p.group = n_heads / kv->n_kv_heads;
    p.by_group = make_div((uint32_t)p.group);
    p.by_ru = make_div(shape.tile ? 2u * pt_tile_rows(p.group) : (unsigned)PR_ROWS);
    p.window = window >= kv->max_pages * kv->page_size ? 0 : window;  // wider than a slot: no window
    p.cost = shape.tile ? PT_COST : PR_COST;
    p.scale = scale;
    p.scale_log2 = (float)((double)scale * 1.4426950408889634);
    p.drill = drill.load();
    p.wait_limit = p.drill ? PG_DRILL_CYCLES : PG_WAIT_CYCLES;
    uint8_t *ws = (uint8_t *)d_ws;
    p.status = (int *)ws;
    p.tickets = (unsigned int *)(ws + WS_TICKETS);
    p.part_ml = (float *)(ws + WS_PARTS);
    p.part_o = p.part_ml + (size_t)2 * shape.n_cta * shape.rows * 2;
    const int bk = shape.tile ? PT_BK : PR_BK;
    if (!pool_map(&p.kmap, kv->k_pool, kv, bk) || !pool_map(&p.vmap, kv->v_pool, kv, bk) ||
        (shape.tile && !query_map(&p.qmap, d_q, hd, n_heads, p.group, ldq, batch->n_tokens)))
        return fail(FIBER_ECUDA, "%s: cannot build the tensor maps", fn);
    cudaStream_t st = (cudaStream_t)stream;
    for (int s0 = 0; s0 < batch->n_seqs; s0 += PG_MAX_SEQS) {
        p.b.n_seqs = std::min(PG_MAX_SEQS, batch->n_seqs - s0);
        p.b.q_start = batch->q_start + s0;
        p.b.kv_len = batch->kv_len + s0;
        p.b.slot = batch->slot ? batch->slot + s0 : nullptr;
        p.b.slot0 = s0;
        cudaError_t e;
        if (kv->type == FIBER_TYPE_F16)
            e = hd == 64 ? launch_attn<64, false>(p, shape, st) : launch_attn<128, false>(p, shape, st);
        else
            e = hd == 64 ? launch_attn<64, true>(p, shape, st) : launch_attn<128, true>(p, shape, st);
        if (e != cudaSuccess) return fail(FIBER_ECUDA, "%s: %s", fn, cudaGetErrorString(e));
    }
    return FIBER_OK;
}

extern "C" int fiber_attn_paged_drill(int on) {
    drill.store(on != 0);
    return FIBER_OK;
}

extern "C" int fiber_attn_paged_status(const void *d_ws, void *stream) {
    if (!d_ws) return fail(FIBER_EARG, "fiber_attn_paged_status: null workspace");
    int status = 0;
    cudaError_t e = cudaMemcpyAsync(&status, d_ws, sizeof(int), cudaMemcpyDeviceToHost, (cudaStream_t)stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize((cudaStream_t)stream);
    if (e != cudaSuccess) return fail(FIBER_ECUDA, "fiber_attn_paged_status: %s", cudaGetErrorString(e));
    if (status == PG_BAD_BATCH) return fail(FIBER_EARG, "fiber_attn_paged: q_start decreases");
    if (status == PG_BAD_SM) return fail(FIBER_ECUDA, "fiber_attn_paged: shared or tensor memory is not where the kernel needs it");
    return status == 0 ? FIBER_OK : fail(FIBER_ETIMEOUT, "fiber_attn_paged: a wait inside the kernel gave up");
}
