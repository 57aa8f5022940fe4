// paged_rows.cuh — attention over the paged cache for few rows per KV head (single
// tokens, a few drafted tokens): units of 16 (token, head) rows.
//
// Bound by the cache's bytes: each K and V row is read once per 16 rows and costs them
// 4 * 16 * head_dim operations, far below the tensor cores' rate, so the kernel is a stream
// of 64-key tiles through a shared-memory ring (TMA, one producer warp) and the four
// consumer warps must only keep up. Each takes 16 of a tile's keys with a softmax state of
// its own (m, l, o), so no barrier is needed per tile; the four states are joined at the
// end of a unit. mma.sync m16n8k16 serves here because a 16-row operand fills it, where a
// 128-row tcgen05 tile would be seven eighths empty: the tile kernel streams such rows at
// 4.4 to 4.8 TB/s, this one at 5.7 to 6.2 (two tokens over 242,802 positions, 995 MB: 161 us, 94% of
// a plain copy's rate; 64 tokens over 211,722 positions in pages of 16: 144 us, 92%). A short
// call is latency: one token over 384 positions takes 7.0 us on the device, of which 4.9 remain
// at 101 positions.
#pragma once
#include "paged.cuh"

namespace fiber {

constexpr int PR_ROWS = 16;
constexpr int PR_BK_SHIFT = 6, PR_BK = 1 << PR_BK_SHIFT;
constexpr int PR_WARPS = 4;
constexpr int PR_THREADS = 32 * (PR_WARPS + 1);
constexpr int PR_CTAS_PER_SM = 2;

// Weights are 2^(score - maximum + pr_shift), the largest 2^15 in fp16: without the shift those
// below 2^-25 of the largest rounded to zero in the product with V but not in the sum: 100,000
// such keys can be 0.3 % of an output. Maximum, sum and output share the factor, so nothing
// else changes, and it costs no time.
template <bool BF>
HDCE float pr_shift() { return BF ? 0.f : 15.f; }

template <int HD>
HDCE int pr_stage_bytes() { return 2 * PR_BK * HD * 2; }
template <int HD>
HDCE int pr_stages() { return HD == 128 ? 3 : 6; }

struct PrShared {
    AttnPlan plan;
    uint64_t full[8], empty[8];
    float ml[PR_WARPS][PR_ROWS][2];
    int bad;        // some row's result is not finite
    int joined[2];  // this CTA has joined the cut unit at the start / at the end of its share
    int last;
    int fail;
};
template <int HD>
HDCE int pr_smem() { return pr_stages<HD>() * pr_stage_bytes<HD>() + (int)sizeof(PrShared) + 1024; }

FDEV void pr_bar() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
FDEV void pr_ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
FDEV void pr_ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
template <bool BF>
FDEV void pr_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Byte offset of 16-byte piece `c` of row `r` in a tile of [head_dim / 64][64 rows][128 B],
// 128-byte swizzle.
FDEV uint32_t pr_off(int r, int c) { return (uint32_t)((c >> 3) * (PR_BK * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

// Index of float4 `c4` of row r in a warp's [16][HD / 4] output block: rotated by the row
// so that the fragments' rows fall on different banks.
template <int HD>
FDEV int pr_oidx(int r, int c4) { return r * (HD / 4) + (c4 ^ (r & 7)); }

template <int HD, bool BF>
__global__ void __launch_bounds__(PR_THREADS, PR_CTAS_PER_SM) attn_rows_kernel(const __grid_constant__ AttnPagedParams p) {
    constexpr int NST = pr_stages<HD>(), SB = pr_stage_bytes<HD>(), C4 = HD / 4;
    extern __shared__ uint8_t pr_raw[];
    uint8_t *ring = pr_raw + ((1024u - (pg_saddr(pr_raw) & 1023u)) & 1023u);
    PrShared &sh = *reinterpret_cast<PrShared *>(ring + NST * SB);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < NST; s++) {
            pg_init(&sh.full[s], 1);
            pg_init(&sh.empty[s], PR_WARPS + p.drill);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sh.fail = 0;
        sh.bad = 0;
        sh.joined[0] = sh.joined[1] = 0;
    }
    if (tid == 32 * PR_WARPS) {
        pg_prefetch_map(&p.kmap);
        pg_prefetch_map(&p.vmap);
    }
    __syncthreads();
    pdl_trigger();
    pdl_wait();
    uint32_t longest;
    const uint32_t total = attn_plan_build<PR_THREADS>(sh.plan, p, PR_ROWS, PR_BK_SHIFT, longest);
    const int n_cta = attn_ctas(p, total, longest), cta = blockIdx.x;
    if (cta >= n_cta) return;
    const uint32_t x0 = attn_share(total, n_cta, cta), x1 = attn_share(total, n_cta, cta + 1);
    AttnUnit u;
    attn_unit_find(u, sh.plan, p, PR_ROWS, PR_BK_SHIFT, x0);

    if (warp == PR_WARPS) {
        // ---- producer: lane b issues box b of a tile (rows of one page x 64 head dims)
        const int box_rows = min(1 << p.kv.page_shift, PR_BK), nrb = PR_BK / box_rows;
        constexpr int HALVES = HD / 64;
        const int n_box = 2 * HALVES * nrb;  // K boxes, then V boxes; at most 16
        const bool is_v = lane >= HALVES * nrb;
        const int half = (lane / nrb) % HALVES, rb = lane % nrb;
        const uint32_t dst0 = (is_v ? SB / 2 : 0) + half * (PR_BK * 128) + rb * box_rows * 128;
        uint32_t it = 0;
        bool ok = true;
        for (;;) {
            const int b = u.u0 < x0 ? attn_step_at(u, p, x0) : 0, e = u.u0 + u.cost > x1 ? attn_step_at(u, p, x1) : u.steps;
            if (u.hi > u.lo) {
                const int32_t *tab = p.kv.table + (long long)u.slot * p.kv.max_pages;
                const int used = (u.hi + (1 << p.kv.page_shift) - 1) >> p.kv.page_shift;
                for (int k = b; k < e; k++, it++) {
                    const int key = (((u.lo >> PR_BK_SHIFT) + k) << PR_BK_SHIFT) + rb * box_rows;
                    const int lp = key >> p.kv.page_shift;
                    int page = p.kv.n_pages;  // outside the tensor: reads as zeros
                    if (lane < n_box && lp < used) page = tab[lp];
                    const int st = it % NST;
                    if (it >= NST) ok = pg_wait(&sh.empty[st], (it / NST - 1) & 1, &sh.fail, p.wait_limit);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (lane == 0) pg_expect_tx(&sh.full[st], SB);
                    __syncwarp();
                    if (lane < n_box)
                        pg_tma4(pg_saddr(ring + st * SB) + dst0, is_v ? &p.vmap : &p.kmap, half * 64,
                                key & ((1 << p.kv.page_shift) - 1), u.g, page, &sh.full[st]);
                }
            }
            if (!ok || u.u0 + u.cost >= x1) break;
            attn_unit_next(u, sh.plan, p, PR_ROWS, PR_BK_SHIFT);
        }
        // every copy has landed before the CTA exits
        if (lane == 0)
            for (uint32_t s = 0; s < NST && s < it; s++)
                pg_drain(&sh.full[s], (s + (it - 1 - s) / NST * NST) / NST & 1);
        if (lane == 0 && sh.fail) *p.status = PG_GAVE_UP;
        return;
    }

    // ---- consumers: warp w takes keys 16 w .. 16 w + 15 of each tile
    const int g8 = lane >> 2, t4 = lane & 3;
    uint32_t it = 0;
    for (;;) {
        const int b = u.u0 < x0 ? attn_step_at(u, p, x0) : 0, e = u.u0 + u.cost > x1 ? attn_step_at(u, p, x1) : u.steps;
        const bool whole = b == 0 && e == u.steps, any = u.hi > u.lo;
        const int p0 = u.kv - u.nq;
        // query fragments, and the positions that rows g8 and g8 + 8 see
        uint32_t qa[HD / 16][4];
        int rlo[2], rhi[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int r = g8 + 8 * h, t = fdiv(u.row0 + r, p.by_group), head = u.g * p.group + u.row0 + r - t * p.group;
            const bool in = r < u.rows;
            rhi[h] = in ? p0 + t + 1 : 0;
            rlo[h] = p.window > 0 ? max(0, p0 + t - p.window + 1) : 0;
            const uint16_t *src = p.q + (long long)(u.q0 + t) * p.ldq + (long long)head * HD + 2 * t4;
#pragma unroll
            for (int k = 0; k < HD / 16; k++) {
                qa[k][h] = in && any ? *reinterpret_cast<const uint32_t *>(src + 16 * k) : 0u;
                qa[k][h + 2] = in && any ? *reinterpret_cast<const uint32_t *>(src + 16 * k + 8) : 0u;
            }
        }
        float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int n = 0; n < HD / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
        // every row of the unit sees the keys in [all_lo, all_hi): no mask needed there
        const int all_hi = max(0, p0 + fdiv(u.row0, p.by_group) + 1);
        const int all_lo = p.window > 0 ? max(0, p0 + fdiv(u.row0 + u.rows - 1, p.by_group) - p.window + 1) : 0;
        int st = 0;
        if (any && b < e) {
            for (int k = b; k < e; k++, it++) {
                st = it % NST;
                // after a timeout: runs through, status says so
                pg_wait_warp(&sh.full[st], (it / NST) & 1, &sh.fail, p.wait_limit);
                uint8_t *kt = ring + st * SB, *vt = kt + SB / 2;
                const int key0 = (((u.lo >> PR_BK_SHIFT) + k) << PR_BK_SHIFT) + 16 * warp;
                const bool edge = key0 < all_lo || key0 + 16 > all_hi;
                if (edge && (key0 < u.lo || key0 + 16 > u.hi)) {
                    // values no row sees may hold anything: weight 0 must meet 0 there
                    const int r = lane >> 1, c0 = (lane & 1) * (HD / 16);
                    if (key0 + r < u.lo || key0 + r >= u.hi)
#pragma unroll
                        for (int c = 0; c < HD / 16; c++)
                            *reinterpret_cast<uint4 *>(vt + pr_off(16 * warp + r, c0 + c)) = make_uint4(0, 0, 0, 0);
                    pg_proxy_fence();  // the ring's next copy into these rows comes after
                    __syncwarp();
                }
                float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
                const uint32_t kb = pg_saddr(kt), vb = pg_saddr(vt);
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int kk = 0; kk < HD / 32; kk++) {
                        uint32_t r[4];
                        pr_ldsm4(r, kb + pr_off(16 * warp + 8 * n + (lane & 7), 4 * kk + (lane >> 3)));
                        pr_mma<BF>(s[n], qa[2 * kk], r[0], r[1]);
                        pr_mma<BF>(s[n], qa[2 * kk + 1], r[2], r[3]);
                    }
                if (edge)
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            const int key = key0 + 8 * n + 2 * t4 + (c & 1);
                            if (key < rlo[c >> 1] || key >= rhi[c >> 1]) s[n][c] = -INFINITY;
                        }
                uint32_t pa[4];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float mx = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float mn = fmaxf(m[h], mx * p.scale_log2);
                    const float base = mn == -INFINITY ? 0.f : mn;
                    if (mn != m[h]) {
                        const float f = exp2f(m[h] - base);
                        m[h] = mn;
                        l[h] *= f;
#pragma unroll
                        for (int n = 0; n < HD / 8; n++) {
                            o[n][2 * h] *= f;
                            o[n][2 * h + 1] *= f;
                        }
                    }
                    const float nb = pr_shift<BF>() - base;
                    float e[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) e[c] = exp2f(fmaf(s[c >> 1][2 * h + (c & 1)], p.scale_log2, nb));
                    l[h] += (e[0] + e[1]) + (e[2] + e[3]);
                    pa[h] = pack2<BF>(e[0], e[1]);
                    pa[2 + h] = pack2<BF>(e[2], e[3]);
                }
#pragma unroll
                for (int n = 0; n < HD / 16; n++) {
                    uint32_t r[4];
                    pr_ldsm4t(r, vb + pr_off(16 * warp + (lane & 15), 2 * n + (lane >> 4)));
                    pr_mma<BF>(o[2 * n], pa, r[0], r[1]);
                    pr_mma<BF>(o[2 * n + 1], pa, r[2], r[3]);
                }
                __syncwarp();
                if (k + 1 < e && lane == 0) pg_arrive(&sh.empty[st]);
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                if (t4 == 0) {
                    sh.ml[warp][g8 + 8 * h][0] = m[h];
                    sh.ml[warp][g8 + 8 * h][1] = l[h];
                }
            }
            // the unit's last stage, consumed, holds the warps' outputs until they are joined
            pr_bar();
            float *buf = reinterpret_cast<float *>(ring + st * SB);
            float *mine = buf + warp * PR_ROWS * HD;
#pragma unroll
            for (int n = 0; n < HD / 8; n++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    *reinterpret_cast<float2 *>(mine + 4 * pr_oidx<HD>(g8 + 8 * h, 2 * n + (t4 >> 1)) + 2 * (t4 & 1)) =
                        make_float2(o[n][2 * h], o[n][2 * h + 1]);
            pr_bar();
            const int pslot = 2 * cta + (b > 0 ? 0 : 1);
            for (int i = tid; i < u.rows * C4; i += 32 * PR_WARPS) {
                const int r = i / C4, c4 = i % C4;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < PR_WARPS; w++) M = fmaxf(M, sh.ml[w][r][0]);
                const float base = M == -INFINITY ? 0.f : M;
                float L = 0.f;
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < PR_WARPS; w++) {
                    const float f = exp2f(sh.ml[w][r][0] - base);
                    const float4 v = reinterpret_cast<const float4 *>(buf + w * PR_ROWS * HD)[pr_oidx<HD>(r, c4)];
                    L = fmaf(f, sh.ml[w][r][1], L);
                    a.x = fmaf(f, v.x, a.x);
                    a.y = fmaf(f, v.y, a.y);
                    a.z = fmaf(f, v.z, a.z);
                    a.w = fmaf(f, v.w, a.w);
                }
                if (whole) {
                    const float inv = 1.f / L;
                    const int t = fdiv(u.row0 + r, p.by_group), head = u.g * p.group + u.row0 + r - t * p.group;
                    const bool sees = p0 + t >= 0;
                    a = sees ? make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f);
                    if (attn_spoiled<BF>(a.x) || attn_spoiled<BF>(a.y) || attn_spoiled<BF>(a.z) || attn_spoiled<BF>(a.w)) sh.bad = 1;
                    *reinterpret_cast<uint2 *>(p.out + (long long)(u.q0 + t) * p.ldo + (long long)head * HD + 4 * c4) =
                        make_uint2(pack2<BF>(a.x, a.y), pack2<BF>(a.z, a.w));
                } else {
                    reinterpret_cast<float4 *>(p.part_o)[((long long)pslot * PR_ROWS + r) * C4 + c4] = a;
                    if (c4 == 0) {
                        p.part_ml[(pslot * PR_ROWS + r) * 2] = M;
                        p.part_ml[(pslot * PR_ROWS + r) * 2 + 1] = L;
                    }
                }
            }
            pg_proxy_fence();
            pr_bar();
            if (lane == 0) pg_arrive(&sh.empty[st]);
            if (!whole) {
                // ---- join the CTAs' states of this unit
                const int ca = attn_owner(total, n_cta, attn_place(u, p, 0)), cb = attn_owner(total, n_cta, attn_place(u, p, u.steps - 1));
                if (tid == 0) {
                    sh.last = pg_ticket(&p.tickets[ca]) == (unsigned)(cb - ca);
                    if (sh.last) {
                        p.tickets[ca] = 0u;
                        sh.joined[b > 0 ? 0 : 1] = 1;
                    }
                }
                pr_bar();
                if (sh.last) {
                    for (int i = tid; i < u.rows * C4; i += 32 * PR_WARPS) {
                        // eight states at a time, their loads all in flight together
                        constexpr int W = 8;
                        const int r = i / C4, c4 = i % C4;
                        const float2 *ml = reinterpret_cast<const float2 *>(p.part_ml) + r;
                        const float4 *po = reinterpret_cast<const float4 *>(p.part_o) + r * C4 + c4;
                        float M = -INFINITY, L = 0.f;
                        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
                        for (int c = ca; c <= cb; c += W) {
                            float2 s[W];
                            float4 v[W];
#pragma unroll
                            for (int k = 0; k < W; k++) {
                                const int sl = 2 * min(c + k, cb) + (min(c + k, cb) == ca ? 1 : 0);
                                s[k] = __ldcg(ml + sl * PR_ROWS);
                                v[k] = __ldcg(po + (long long)sl * (PR_ROWS * C4));
                            }
                            float mn = M;
#pragma unroll
                            for (int k = 0; k < W; k++) mn = fmaxf(mn, s[k].x);
                            const float base = mn == -INFINITY ? 0.f : mn, f0 = exp2f(M - base);
                            M = mn;
                            L *= f0;
                            a = make_float4(a.x * f0, a.y * f0, a.z * f0, a.w * f0);
#pragma unroll
                            for (int k = 0; k < W; k++) {
                                if (c + k > cb) break;
                                const float f = exp2f(s[k].x - base);
                                L = fmaf(f, s[k].y, L);
                                a.x = fmaf(f, v[k].x, a.x);
                                a.y = fmaf(f, v[k].y, a.y);
                                a.z = fmaf(f, v[k].z, a.z);
                                a.w = fmaf(f, v[k].w, a.w);
                            }
                        }
                        const float inv = 1.f / L;
                        const int t = fdiv(u.row0 + r, p.by_group), head = u.g * p.group + u.row0 + r - t * p.group;
                        const bool sees = p0 + t >= 0;
                        a = sees ? make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f);
                        if (attn_spoiled<BF>(a.x) || attn_spoiled<BF>(a.y) || attn_spoiled<BF>(a.z) || attn_spoiled<BF>(a.w)) sh.bad = 1;
                        *reinterpret_cast<uint2 *>(p.out + (long long)(u.q0 + t) * p.ldo + (long long)head * HD + 4 * c4) =
                            make_uint2(pack2<BF>(a.x, a.y), pack2<BF>(a.z, a.w));
                    }
                    pr_bar();
                }
            }
            pr_bar();  // sh.ml is reused by the next unit
        } else if (b < e) {  // no row of the unit sees a key
            for (int i = tid; i < u.rows * C4; i += 32 * PR_WARPS) {
                const int r = i / C4, c4 = i % C4;
                const int t = fdiv(u.row0 + r, p.by_group), head = u.g * p.group + u.row0 + r - t * p.group;
                *reinterpret_cast<uint2 *>(p.out + (long long)(u.q0 + t) * p.ldo + (long long)head * HD + 4 * c4) =
                    make_uint2(0u, 0u);
            }
        }
        if (u.u0 + u.cost >= x1) break;
        attn_unit_next(u, sh.plan, p, PR_ROWS, PR_BK_SHIFT);
    }
    if (lane == 0 && sh.fail) *p.status = PG_GAVE_UP;
    pr_bar();
    if (sh.bad && !sh.fail) attn_exact_rows<HD, BF>(p, sh.plan, n_cta, sh.joined, PR_ROWS, PR_BK_SHIFT, PR_WARPS);
}

}  // namespace fiber
