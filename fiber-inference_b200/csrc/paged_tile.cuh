// paged_tile.cuh — attention over the paged cache for chunks of tokens on the
// 5th-generation tensor cores.
//
// A unit is two tiles (A, B) of up to 128 rows (token, head of the group) of one sequence
// and KV head, and walks the 128-key tiles that its rows see. One CTA per SM:
//   warps 0-3   softmax of tile A, one row per thread: scores from tensor memory, running
//               maximum and sum, probabilities back to tensor memory in 16 bits
//   warps 4-7   the same for tile B
//   warps 8, 11 issue the MMAs of tile A and of tile B: S = Q K^T (operands in shared
//               memory), then O += P V with P read from tensor memory (with one warp for
//               both a step took 4,590 cycles: every wait of one tile also held up the other)
//   warp 9      producer: Q, K and V tiles by TMA (K / V boxes go page by page)
//   warp 10     scheduler: works out the CTA's units ahead of the others
// Tensor memory: S_A, S_B (128 columns each), O_A, O_B (head_dim columns each). A key tile
// is worked through in two halves of 64 keys, each with its own 64 columns of S, whose
// front half its probabilities overwrite: while the softmax of one half runs, the tensor
// core multiplies the other half's probabilities with V and computes its next scores, so
// a softmax warp finds its next scores ready.
//
// Bound by the softmax warps, then by power. A step of both tiles (128 keys, head_dim 128)
// takes 3,760 cycles; its products alone are 2,560 (S of 64 keys is bound by reading Q and K
// from shared memory: 48 cycles per MMA where the arithmetic is 32), 2,920 with the hand-overs.
// One S of 128 keys per step needs 2,048 but puts products and softmax in a row: 3,880. 2,048
// tokens after 14,005 positions take 439 us from a cool start (1,150 TFLOP/s) and 509 at
// 1,000 W, where the clock falls to 1.5 GHz.
//
// The output accumulators are rescaled only when a row's maximum has grown by more than
// 2^9 (fp16) or 2^40 (bf16) since the last time: a rescale waits for the product before
// it and costs its 32 rows about 3,000 cycles.
#pragma once
#include "paged.cuh"

namespace fiber {

constexpr int PT_ROWS = 128;                          // rows of a tile
constexpr int PT_BK_SHIFT = 7, PT_BK = 1 << PT_BK_SHIFT;  // keys of a tile
constexpr int PT_THREADS = 384;
// Powers of two a row's maximum may grow before O is rescaled, and the power of two that a weight
// at the maximum has. A larger probability is no less exact, so only the range of the 16-bit type
// and of the fp32 sums limits their sum: 2^15 for fp16 (below 65,504); 2^40 for bf16 leaves 2^87
// to the sums. In fp16 a weight below 2^-25 rounds to zero in the product with V but not in the
// sum, so a part of the range lies below the maximum: what is lost is at most 2^-31 of it a key. (A
// growth of 2^9 costs no time against 2^15, 2^7 costs 4 %: 257 us instead of 247 for two chunks
// beside 40 single tokens, with random heads.)
template <bool BF>
HDCE float pt_growth() { return BF ? 40.f : 9.f; }
template <bool BF>
HDCE float pt_shift() { return BF ? 0.f : 6.f; }

// Tokens and rows of a tile: whole tokens (all heads of the group).
HDCE int pt_tile_rows(int group) { return PT_ROWS / group * group; }

template <int HD>
HDCE int pt_tile_bytes() { return 128 * HD * 2; }  // a Q, K or V tile: [HD / 64][128 rows][128 B], 128-byte swizzle
template <int HD>
HDCE int pt_stages() { return HD == 128 ? 5 : 8; }

// A unit (or this CTA's piece of it) as the scheduler hands it to the other warps.
struct PtWork {
    int q0, slot, g;       // first token row of the sequence, cache slot, KV head
    int p0;                // position of the sequence's first token
    int row0, rows[2];     // first row of tile A, rows of tiles A and B
    int lo, hi;            // positions any row of the unit sees
    int kt0, b, e;         // key tile of step 0; this piece's steps
    int ab[2], ae[2];      // half steps (64 keys) [ab, ae) in which the tile has work
    int mode;              // PT_WHOLE, PT_PIECE or PT_END
    int slot_of, ca, cb;   // piece: its state's place, first and last CTA of the unit
};
enum : int { PT_WHOLE = 0, PT_PIECE = 1, PT_END = 2 };
constexpr int PT_CONSUMERS = 11;  // warps that read the work records

struct PtShared {
    AttnPlan plan;
    uint64_t kvfull[8], kvfree[8];
    uint64_t qfull, qfree;
    uint64_t sfull[2][2], pready[2][2];  // [tile][half]
    uint64_t pvdone[2], odone[2];        // a product with V has finished; a unit's last one has
    uint64_t wfull[2], wfree[2];
    uint64_t join, mdone;
    PtWork work[2];
    uint32_t tmem;
    int n_cta;      // CTAs that have work
    int bad;        // some row's result is not finite
    int joined[2];  // this CTA has joined the cut unit at the start / at the end of its share
    int last;
    int fail;
};
template <int HD>
HDCE int pt_smem() { return (2 + pt_stages<HD>()) * pt_tile_bytes<HD>() + (int)sizeof(PtShared); }
static_assert(pt_smem<128>() <= 227 * 1024 && pt_smem<64>() <= 227 * 1024, "shared memory of one CTA");

FDEV uint64_t pt_desc(uint32_t saddr, uint32_t lbo) {
    // 128-byte swizzle (2 << 61), version 1, 8-row groups 1024 B apart; lbo: for the operand
    // whose rows are K (V), the next 64 columns
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// kind::f16: D fp32, A and B both fp16 or both bf16, M 128; b_rows_k: B is [K][N] in memory
template <bool BF>
HDCE uint32_t pt_idesc(int n, bool b_rows_k) {
    return (1u << 4) | ((BF ? 1u : 0u) << 7) | ((BF ? 1u : 0u) << 10) | ((b_rows_k ? 1u : 0u) << 16) |
           ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// The issuing warp runs converged and every MMA and commit is predicated on its elected
// lane: descriptors then stay in uniform registers. Issued from a divergent branch
// (lane 0 alone) each operand is moved there one by one, about 130 cycles per MMA of 64.
FDEV uint32_t pt_elect() {
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r;
}
FDEV void pt_mma_ss(uint32_t me, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(me)
        : "memory");
}
FDEV void pt_mma_ts(uint32_t me, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(me)
        : "memory");
}
FDEV void pt_commit(uint32_t me, uint64_t *bar) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(pg_saddr(bar)),
        "r"(me)
        : "memory");
}
FDEV void pt_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
FDEV void pt_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
FDEV void pt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of this warp's 32 lanes (one row per thread)
FDEV void pt_ld32(float *v, uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
          "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(addr)
        : "memory");
}
FDEV void pt_ld16(float *v, uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(addr)
        : "memory");
}
FDEV void pt_st16(uint32_t addr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
FDEV float pt_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two fp32 values in one 64-bit register
FDEV uint64_t pt_two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
FDEV float2 pt_both(uint64_t r) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(r));
    return f;
}
FDEV uint64_t pt_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
FDEV uint64_t pt_add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
FDEV uint64_t pt_mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
FDEV float pt_max(float a, float b) {  // NaN if either is (fmaxf returns the other)
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// 2^x of two values on the FMA pipe: x = n + f with n the nearest integer (added and
// subtracted 1.5 * 2^23), 2^f by a minimax polynomial of degree 4 on [-1/2, 1/2] (Remez
// exchange on the relative error, 2.7e-6 in fp32), times 2^n, whose bits are n + 127 in the
// exponent. x is clamped to -127, whose 2^n is all zero bits: a masked key's weight has to
// be exactly 0 (bf16 holds 2^-126, and values up to 2^127 would meet it).
// A score that is NaN stays NaN, so that its row is seen to need the exact pass.
FDEV float2 pt_exp2_poly(float x0, float x1) {
    const uint64_t magic = pt_two(12582912.f, 12582912.f), minus = pt_two(-12582912.f, -12582912.f);
    const uint64_t x = pt_two(pt_max(x0, -127.f), pt_max(x1, -127.f));
    const uint64_t t = pt_add2(x, magic);
    const uint64_t n = pt_add2(t, minus);
    const uint64_t f = pt_fma2(n, pt_two(-1.f, -1.f), x);
    uint64_t y = pt_fma2(pt_two(0.009570102207362652f, 0.009570102207362652f), f, pt_two(0.05591785907745361f, 0.05591785907745361f));
    y = pt_fma2(y, f, pt_two(0.240247443318367f, 0.240247443318367f));
    y = pt_fma2(y, f, pt_two(0.6931217908859253f, 0.6931217908859253f));
    y = pt_fma2(y, f, pt_two(0.9999992847442627f, 0.9999992847442627f));
    const float2 e = pt_both(t);
    return pt_both(pt_mul2(y, pt_two(__uint_as_float((__float_as_uint(e.x) << 23) + 0x3f800000u),
                                     __uint_as_float((__float_as_uint(e.y) << 23) + 0x3f800000u))));
}
// Completion of tensor-memory loads, tied to the registers they fill
FDEV void pt_wait_ld(float *v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
                 :
                 : "memory");
}
FDEV void pt_tie16(float *v) {
    asm volatile("" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                      "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]));
}
// The lowest n bits (none below 0, all from 32)
FDEV uint32_t pt_below(int n) { return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1u); }

// Pairs of every 4 whose exponentials run on the FMA pipe instead of the special-function
// unit, which alone would need 2 x 1,024 cycles per step (2,048 tokens after 14,005
// positions: none 470 us, one in four 439, two 454).
constexpr int PT_POLY = 1;

template <int HD, bool BF>
__global__ void __launch_bounds__(PT_THREADS, 1) attn_tile_kernel(const __grid_constant__ AttnPagedParams p) {
    constexpr int NST = pt_stages<HD>(), TB = pt_tile_bytes<HD>(), HALVES = HD / 64;
    extern __shared__ __align__(1024) uint8_t pt_raw[];
    uint8_t *qbuf = pt_raw, *ring = pt_raw + 2 * TB;
    PtShared &sh = *reinterpret_cast<PtShared *>(ring + NST * TB);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (pg_saddr(pt_raw) & 1023u) {  // never: the operand tiles must start on 1024 bytes
        if (tid == 0) *p.status = PG_BAD_SM;
        return;
    }
    if (tid == 0) {
        for (int s = 0; s < NST; s++) {
            pg_init(&sh.kvfull[s], 1);
            pg_init(&sh.kvfree[s], 2 + p.drill);
        }
        pg_init(&sh.qfull, 1);
        pg_init(&sh.qfree, 2);
        for (int t = 0; t < 2; t++) {
            for (int h = 0; h < 2; h++) {
                pg_init(&sh.sfull[t][h], 1);
                pg_init(&sh.pready[t][h], 4);
            }
            pg_init(&sh.pvdone[t], 1);
            pg_init(&sh.odone[t], 1);
            pg_init(&sh.wfull[t], 1);
            pg_init(&sh.wfree[t], PT_CONSUMERS);
        }
        pg_init(&sh.join, 8);
        pg_init(&sh.mdone, 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sh.fail = 0;
        sh.bad = 0;
        sh.joined[0] = sh.joined[1] = 0;
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(pg_saddr(&sh.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 32 * 9) {
        pg_prefetch_map(&p.kmap);
        pg_prefetch_map(&p.vmap);
        pg_prefetch_map(&p.qmap);
    }
    pt_fence_before();
    __syncthreads();
    pt_fence_after();
    pdl_trigger();
    pdl_wait();
    const int rt = pt_tile_rows(p.group), ru = 2 * rt;
    uint32_t longest;
    const uint32_t total = attn_plan_build<PT_THREADS>(sh.plan, p, ru, PT_BK_SHIFT, longest);
    constexpr uint32_t tmem = 0;  // all 512 columns
    if (sh.tmem != tmem && tid == 0) *p.status = PG_BAD_SM;
    const int n_cta = attn_ctas(p, total, longest), cta = blockIdx.x;
    if (tid == 0) sh.n_cta = n_cta;

    // 384 threads at 168 registers: the softmax warpgroups take 224 each, the third keeps 56
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (cta < n_cta && warp == 10) {
            // ---- scheduler
            const uint32_t x0 = attn_share(total, n_cta, cta), x1 = attn_share(total, n_cta, cta + 1);
            AttnUnit u;
            attn_unit_find(u, sh.plan, p, ru, PT_BK_SHIFT, x0);
            bool end = false;
            for (uint32_t i = 0;;) {
                const int b = u.u0 < x0 ? attn_step_at(u, p, x0) : 0, e = u.u0 + u.cost > x1 ? attn_step_at(u, p, x1) : u.steps;
                const int kt0 = u.lo >> PT_BK_SHIFT;
                if (!end && b >= e) {  // none of this unit's steps
                    end = u.u0 + u.cost >= x1;
                    if (!end) attn_unit_next(u, sh.plan, p, ru, PT_BK_SHIFT);
                    continue;
                }
                bool ok = i < 2 || pg_wait(&sh.wfree[i & 1], ((i >> 1) - 1) & 1, &sh.fail, p.wait_limit);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                PtWork &w = sh.work[i & 1];
                if (lane < 2 && !end) {  // lane t: tile t
                    const int rows = lane == 0 ? min(rt, u.rows) : max(0, u.rows - rt);
                    int lo = 0, hi = 0, ab = 0, ae = 0;
                    if (rows > 0 && u.hi > u.lo) attn_span(u.nq, u.kv, p, u.row0 + lane * rt, rows, lo, hi);
                    if (hi > lo) {
                        ab = max(2 * b, (lo >> 6) - 2 * kt0);
                        ae = max(ab, min(2 * e, ((hi + 63) >> 6) - 2 * kt0));
                    }
                    w.rows[lane] = rows;
                    w.ab[lane] = ab;
                    w.ae[lane] = ae;
                }
                if (lane == 0) {
                    w.mode = end ? PT_END : (b == 0 && e == u.steps ? PT_WHOLE : PT_PIECE);
                    if (!end) {
                        w.q0 = u.q0;
                        w.slot = u.slot;
                        w.g = u.g;
                        w.p0 = u.kv - u.nq;
                        w.row0 = u.row0;
                        w.lo = u.lo;
                        w.hi = u.hi;
                        w.kt0 = kt0;
                        w.b = b;
                        w.e = e;
                        w.slot_of = 2 * cta + (b > 0 ? 0 : 1);
                        w.ca = attn_owner(total, n_cta, attn_place(u, p, 0));
                        w.cb = attn_owner(total, n_cta, attn_place(u, p, u.steps - 1));
                    }
                }
                __syncwarp();
                if (lane == 0) pg_arrive(&sh.wfull[i & 1]);
                if (end) break;
                i++;
                end = u.u0 + u.cost >= x1;
                if (!end) attn_unit_next(u, sh.plan, p, ru, PT_BK_SHIFT);
            }
        } else if (cta < n_cta && warp == 9) {
            // ---- producer: lane b issues box b of a K or V tile
            const int box_rows = min(1 << p.kv.page_shift, PT_BK), nrb = PT_BK / box_rows;
            const int half = lane / nrb, rb = lane % nrb, mask = (1 << p.kv.page_shift) - 1;
            const bool boxed = lane < HALVES * nrb;
            const uint32_t dst0 = half * (128 * 128) + rb * box_rows * 128;
            uint32_t it = 0, nq = 0;  // K / V tiles and Q pairs issued
            for (uint32_t i = 0;; i++) {
                bool ok = pg_wait(&sh.wfull[i & 1], (i >> 1) & 1, &sh.fail, p.wait_limit);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const PtWork &w = sh.work[i & 1];
                if (w.mode == PT_END) break;
                if (w.ae[0] > w.ab[0] || w.ae[1] > w.ab[1]) {
                    const int32_t *tab = p.kv.table + (long long)w.slot * p.kv.max_pages;
                    const int used = (w.hi + mask) >> p.kv.page_shift, e = w.e, g = w.g;
                    for (int k = w.b; k < e; k++) {
                        const int key = ((w.kt0 + k) << PT_BK_SHIFT) + rb * box_rows, lp = key >> p.kv.page_shift;
                        int page = p.kv.n_pages;  // outside the tensor: reads as zeros
                        if (boxed && lp < used) page = tab[lp];
#pragma unroll
                        for (int v = 0; v < 2; v++, it++) {
                            const int st = it % NST;
                            if (it >= NST) ok = pg_wait(&sh.kvfree[st], (it / NST - 1) & 1, &sh.fail, p.wait_limit);
                            ok = __all_sync(0xffffffffu, ok);
                            if (!ok) break;
                            if (lane == 0) pg_expect_tx(&sh.kvfull[st], TB);
                            __syncwarp();
                            if (boxed)
                                pg_tma4(pg_saddr(ring + st * TB) + dst0, v ? &p.vmap : &p.kmap, half * 64, key & mask, g, page,
                                        &sh.kvfull[st]);
                        }
                        if (!ok) break;
                        if (k == w.b) {  // the queries' buffer is free last: K and V of the first step go before
                            if (nq > 0) ok = pg_wait(&sh.qfree, (nq - 1) & 1, &sh.fail, p.wait_limit);
                            ok = __all_sync(0xffffffffu, ok);
                            if (!ok) break;
                            if (lane == 0) {
                                const int nt = w.rows[1] > 0 ? 2 : 1;
                                pg_expect_tx(&sh.qfull, (uint32_t)(nt * HALVES * rt * 128));
                                for (int t = 0; t < nt; t++)
                                    for (int h = 0; h < HALVES; h++)
                                        pg_tma3(pg_saddr(qbuf + t * TB) + h * (128 * 128), &p.qmap, 64 * h, g * p.group,
                                                w.q0 + fdiv(w.row0 + t * rt, p.by_group), &sh.qfull);
                            }
                            nq++;
                        }
                    }
                    if (!ok) break;
                }
                __syncwarp();
                if (lane == 0) pg_arrive(&sh.wfree[i & 1]);
            }
            if (lane == 0) {  // every copy has landed before the CTA exits
                for (uint32_t s = 0; s < NST && s < it; s++)
                    pg_drain(&sh.kvfull[s], (s + (it - 1 - s) / NST * NST) / NST & 1);
                if (nq > 0) pg_drain(&sh.qfull, (nq - 1) & 1);
            }
        } else if (cta < n_cta && (warp == 8 || warp == 11)) {
            // ---- MMA issuer of tile t
            constexpr uint32_t IS = pt_idesc<BF>(64, false), IO = pt_idesc<BF>(HD, true);
            const int t = warp == 8 ? 0 : 1;
            const uint32_t me = pt_elect();
            uint32_t nq = 0, np = 0;  // Q pairs used; parity of pready[t][h] in bit h
            int st = 0, ph = 0;       // ring stage and parity of the next K or V tile
            auto next = [&]() {
                if (++st == NST) {
                    st = 0;
                    ph ^= 1;
                }
            };
            auto scores = [&](int h) {  // S_t,h = Q_t K_h^T
                const uint64_t a = pt_desc(pg_saddr(qbuf) + t * TB, 16), b = pt_desc(pg_saddr(ring) + st * TB + h * 8192, 16);
#pragma unroll
                for (int k = 0; k < HD / 16; k++) {
                    const uint32_t o = ((k >> 2) * (128 * 128) + (k & 3) * 32) >> 4;
                    pt_mma_ss(me, tmem + t * 128 + h * 64, a + o, b + o, IS, k > 0);
                }
                pt_commit(me, &sh.sfull[t][h]);
            };
            auto values = [&](int h, int vst, bool first, bool last) {  // O_t += P_t,h V_h
                const uint64_t b = pt_desc(pg_saddr(ring) + vst * TB + h * 8192, 128 * 128);
#pragma unroll
                for (int k = 0; k < 4; k++)
                    pt_mma_ts(me, tmem + 256 + t * 128, tmem + t * 128 + h * 64 + 8 * k, b + k * (2048 >> 4), IO, !first || k > 0);
                pt_commit(me, &sh.pvdone[t]);
                if (last) pt_commit(me, &sh.odone[t]);
            };
            for (uint32_t i = 0;; i++) {
                bool ok = pg_wait(&sh.wfull[i & 1], (i >> 1) & 1, &sh.fail, p.wait_limit);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const PtWork &w = sh.work[i & 1];
                if (w.mode == PT_END) break;
                const int b = w.b, e = w.e, ab = w.ab[t], ae = w.ae[t];
                const bool run = w.ae[0] > w.ab[0] || w.ae[1] > w.ab[1];
                __syncwarp();
                if (lane == 0) pg_arrive(&sh.wfree[i & 1]);
                if (!run) continue;
                auto on = [&](int j) { return j >= ab && j < ae; };
                ok = pg_wait(&sh.qfull, nq & 1, &sh.fail, p.wait_limit) && pg_wait(&sh.kvfull[st], ph, &sh.fail, p.wait_limit);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                nq++;
                pt_fence_after();
#pragma unroll
                for (int h = 0; h < 2; h++)
                    if (on(2 * b + h)) scores(h);
                pt_commit(me, &sh.kvfree[st]);
                if (e - b == 1) pt_commit(me, &sh.qfree);
                next();
                for (int k = b; k < e; k++) {
                    const bool more = k + 1 < e;
                    const int vst = st;
                    ok = pg_wait(&sh.kvfull[st], ph, &sh.fail, p.wait_limit);
                    next();  // now the next step's K tile
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if (on(2 * k + h)) {
                            ok = ok && pg_wait(&sh.pready[t][h], np >> h & 1, &sh.fail, p.wait_limit);
                            ok = __all_sync(0xffffffffu, ok);
                            if (!ok) break;
                            np ^= 1u << h;
                            pt_fence_after();
                            values(h, vst, 2 * k + h == ab, 2 * k + h + 1 == ae);
                        }
                        if (h == 1) pt_commit(me, &sh.kvfree[vst]);
                        if (more && h == 0) ok = ok && pg_wait(&sh.kvfull[st], ph, &sh.fail, p.wait_limit);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (more && on(2 * k + 2 + h)) scores(h);
                    }
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (more) {
                        pt_commit(me, &sh.kvfree[st]);
                        if (k + 2 == e) pt_commit(me, &sh.qfree);
                        next();
                    }
                }
                if (!ok) break;
            }
            pt_commit(me, &sh.mdone);  // every product has finished before tensor memory is released
            pg_drain(&sh.mdone, 0);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ---- softmax: thread = row of tile t. After a timed-out wait these warps run through
        // (the status says so), so that every barrier is met.
        const int t = warp >> 2, row = tid & 127;
        const uint32_t sa = tmem + t * 128 + ((uint32_t)(32 * (warp & 3)) << 16), oa = sa + 256;
        const uint64_t scale2 = pt_two(p.scale_log2, p.scale_log2);
        uint32_t it = 0, ns = 0, npv = 0, no = 0, nj = 0;  // ns: parity of sfull[t][h] in bit h; npv: products of this tile
        for (uint32_t i = 0; cta < n_cta; i++) {
            if (!__all_sync(0xffffffffu, pg_wait(&sh.wfull[i & 1], (i >> 1) & 1, &sh.fail, p.wait_limit))) break;
            const PtWork &w = sh.work[i & 1];
            const int mode = w.mode;
            if (mode == PT_END) break;
            const int rows = w.rows[t], row0 = w.row0 + t * rt, ab = w.ab[t], ae = w.ae[t];
            int rlo, rhi, all_lo = 0, all_hi;  // positions this row sees; those every row of the tile sees
            {
                const int tok = fdiv(row0 + row, p.by_group);
                rhi = row < rows ? max(0, w.p0 + tok + 1) : 0;
                rlo = p.window > 0 ? max(0, w.p0 + tok - p.window + 1) : 0;
                all_hi = w.p0 + fdiv(row0, p.by_group) + 1;
                if (p.window > 0) all_lo = max(0, w.p0 + fdiv(row0 + rows - 1, p.by_group) - p.window + 1);
            }
            const bool idle = 32 * (warp & 3) >= rows;  // no row of this warp exists: it only keeps step
            float m = -INFINITY, l = 0.f;
            auto await = [&](int j) {  // the scores of half step j are there
                const int h = j & 1;
                pg_wait_warp(&sh.sfull[t][h], ns >> h & 1, &sh.fail, p.wait_limit);
                ns ^= 1u << h;
                pt_fence_after();
            };
            auto fetch = [&](int j, float (&v)[64]) {
                pt_ld32(v, sa + 64 * (j & 1));
                pt_ld32(v + 32, sa + 64 * (j & 1) + 32);
            };
            // they have arrived in v: mask them, and the row's maximum among them
            auto arrived = [&](int j, float (&v)[64]) -> float {
                pt_wait_ld(v);
                pt_tie16(v + 16);
                pt_tie16(v + 32);
                pt_tie16(v + 48);
                const int key0 = (w.kt0 << PT_BK_SHIFT) + 64 * j;
                if (key0 < all_lo || key0 + 64 > all_hi) {
                    const int ca = rlo - key0, cb = rhi - key0;  // columns [ca, cb) are seen
#pragma unroll
                    for (int c = 0; c < 64; c += 32) {
                        const uint32_t keep = pt_below(cb - c) & ~pt_below(ca - c);
#pragma unroll
                        for (int n = 0; n < 32; n++)
                            if (!(keep >> n & 1)) v[c + n] = -INFINITY;
                    }
                }
                float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                for (int c = 4; c < 60; c += 8)
#pragma unroll
                    for (int n = 0; n < 4; n++) mx[n] = fmaxf(fmaxf(mx[n], v[c + n]), v[c + 4 + n]);
                return fmaxf(fmaxf(fmaxf(mx[0], v[60]), fmaxf(mx[1], v[61])), fmaxf(fmaxf(mx[2], v[62]), fmaxf(mx[3], v[63]))) *
                       p.scale_log2;
            };
            // probabilities of half step j are written: hand them over
            auto hand_over = [&](int j) {
                const int h = j & 1, tile0 = (w.kt0 + (j >> 1)) << PT_BK_SHIFT;
                npv++;
                if ((h == 0 || j == ab) && (tile0 < w.lo || tile0 + PT_BK > w.hi)) {
                    // values no row of the unit sees may hold anything: weight 0 must meet 0 there.
                    // Each tile clears them before its own product: the tiles' products do not
                    // wait for one another (zeros over the other tile's zeros change nothing).
                    const uint32_t vi = it + 2 * ((j >> 1) - w.b) + 1;
                    pg_wait_warp(&sh.kvfull[vi % NST], vi / NST & 1, &sh.fail, p.wait_limit);
                    if (tile0 + row < w.lo || tile0 + row >= w.hi)
#pragma unroll 1
                        for (int c = 0; c < 8 * HALVES; c++)  // pieces rotated by the row: eight rows on eight banks
                            *reinterpret_cast<uint4 *>(ring + (vi % NST) * TB + (c >> 3) * (128 * 128) + row * 128 +
                                                       (((c & 7) ^ (row & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                    pg_proxy_fence();
                }
                pt_wait_st();
                pt_fence_before();
                __syncwarp();
                if (lane == 0) pg_arrive(&sh.pready[t][h]);
            };
            auto half_step = [&](int j) {
                float v[64];
                await(j);
                fetch(j, v);
                const float mt = arrived(j, v);
                const bool grow = mt > m + pt_growth<BF>() || (m == -INFINITY && mt > m);
                if (__any_sync(0xffffffffu, grow)) {
                    const float mn = grow ? mt : m;
                    const float f = grow ? pt_exp2(m - mn) : 1.f;
                    m = mn;
                    l *= f;
                    if (j > ab) {
                        // the half before is in O (the one before that had finished when v's scores did)
                        pg_wait_warp(&sh.pvdone[t], (npv - 1) & 1, &sh.fail, p.wait_limit);
                        pt_fence_after();
#pragma unroll
                        for (int c = 0; c < HD; c += 16) {
                            float o[16];
                            uint32_t x[16];
                            pt_ld16(o, oa + c);
                            pt_wait_ld(o);
#pragma unroll
                            for (int n = 0; n < 16; n++) x[n] = __float_as_uint(o[n] * f);
                            pt_st16(oa + c, x);
                        }
                    }
                }
                const float nb = pt_shift<BF>() - (m == -INFINITY ? 0.f : m);
                const uint64_t nb2 = pt_two(nb, nb);
                uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < 64; c += 32) {
                    uint32_t x[16];
#pragma unroll
                    for (int n = 0; n < 16; n++) {
                        float2 y = pt_both(pt_fma2(pt_two(v[c + 2 * n], v[c + 2 * n + 1]), scale2, nb2));
                        if ((n & 3) < 4 - PT_POLY) {
                            y.x = pt_exp2(y.x);
                            y.y = pt_exp2(y.y);
                        } else {
                            y = pt_exp2_poly(y.x, y.y);
                        }
                        sum[n & 1] = pt_add2(sum[n & 1], pt_two(y.x, y.y));
                        x[n] = pack2<BF>(y.x, y.y);
                    }
                    pt_st16(sa + 64 * (j & 1) + c / 2, x);
                }
                const float2 l2 = pt_both(pt_add2(sum[0], sum[1]));
                l += l2.x + l2.y;
                hand_over(j);
            };
            if (idle) {
                for (int j = ab; j < ae; j++) {
                    await(j);
                    hand_over(j);
                }
            } else {
                for (int j = ab; j < ae; j++) half_step(j);
            }
            // ---- the unit's (or piece's) output
            if (w.ae[0] > w.ab[0] || w.ae[1] > w.ab[1]) it += 2 * (w.e - w.b);
            const bool did = ae > ab;
            if (did) {
                pg_wait_warp(&sh.odone[t], no++ & 1, &sh.fail, p.wait_limit);
                pt_fence_after();
            }
            const int tok = fdiv(row0 + row, p.by_group), head = w.g * p.group + row0 + row - tok * p.group;
            uint16_t *dst = p.out + (long long)(w.q0 + tok) * p.ldo + (long long)head * HD;
            bool bad = false;
            auto store16 = [&](int c, const float *o) {  // 16 output values of this thread's row
#pragma unroll
                for (int j = 0; j < 16; j += 8) {
#pragma unroll
                    for (int i2 = 0; i2 < 8; i2++) bad |= attn_spoiled<BF>(o[j + i2]);
                    *reinterpret_cast<uint4 *>(dst + c + j) =
                        make_uint4(pack2<BF>(o[j], o[j + 1]), pack2<BF>(o[j + 2], o[j + 3]), pack2<BF>(o[j + 4], o[j + 5]),
                                   pack2<BF>(o[j + 6], o[j + 7]));
                }
            };
            if (mode == PT_WHOLE) {
                const float inv = 1.f / l;
                if (!idle)
#pragma unroll
                    for (int c = 0; c < HD; c += 32) {
                        float o[32];
                        if (did) {
                            pt_ld32(o, oa + c);
                            pt_wait_ld(o);
                            pt_tie16(o + 16);
                        }
#pragma unroll
                        for (int j = 0; j < 32; j++) o[j] = did && rhi > rlo ? o[j] * inv : 0.f;
                        if (row < rows) {
                            store16(c, o);
                            store16(c + 16, o + 16);
                        }
                    }
            } else {
                const int ps = 2 * w.slot_of + t;
                float4 *po = reinterpret_cast<float4 *>(p.part_o) + (long long)ps * (HD / 4) * 128 + row;
                float *pm = p.part_ml + ps * 256 + row;
                if (!idle) {
                    // scores all NaN leave no maximum but a sum: the join must not pass it over
                    pm[0] = !did ? -INFINITY : l != 0.f ? fmaxf(m, -3.4e38f) : m;
                    pm[128] = l;
                    if (did)
#pragma unroll
                        for (int c = 0; c < HD; c += 32) {
                            float o[32];
                            pt_ld32(o, oa + c);
                            pt_wait_ld(o);
                            pt_tie16(o + 16);
#pragma unroll
                            for (int j = 0; j < 32; j += 4) po[(c + j) / 4 * 128] = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                        }
                }
                __syncwarp();
                if (lane == 0) pg_arrive(&sh.join);
                pg_wait_warp(&sh.join, nj++ & 1, &sh.fail, p.wait_limit);
                if (tid == 0) {
                    sh.last = pg_ticket(&p.tickets[w.ca]) == (unsigned)(w.cb - w.ca);
                    if (sh.last) {
                        p.tickets[w.ca] = 0u;
                        sh.joined[w.slot_of & 1] = 1;
                    }
                }
                __syncwarp();
                if (lane == 0) pg_arrive(&sh.join);
                pg_wait_warp(&sh.join, nj++ & 1, &sh.fail, p.wait_limit);
                if (sh.last && !idle) {
                    const int c0 = w.ca, c1 = w.cb;
                    float M = -INFINITY, L = 0.f;
                    for (int c = c0; c <= c1; c++)
                        M = fmaxf(M, __ldcg(p.part_ml + (2 * (2 * c + (c == c0)) + t) * 256 + row));
                    float o[HD];
#pragma unroll
                    for (int j = 0; j < HD; j++) o[j] = 0.f;
#pragma unroll 1
                    for (int c = c0; c <= c1; c++) {
                        const int sl = 2 * (2 * c + (c == c0)) + t;
                        const float mc = __ldcg(p.part_ml + sl * 256 + row), lc = __ldcg(p.part_ml + sl * 256 + 128 + row);
                        const float4 *src = reinterpret_cast<const float4 *>(p.part_o) + (long long)sl * (HD / 4) * 128 + row;
                        const float f = pt_exp2(mc - M);
                        if (mc != -INFINITY) L = fmaf(f, lc, L);
#pragma unroll
                        for (int j0 = 0; j0 < HD / 4; j0 += 16) {
                            float4 v[16];
#pragma unroll
                            for (int j = 0; j < 16; j++) v[j] = __ldcg(src + (j0 + j) * 128);
                            if (mc != -INFINITY)  // else no key of its part seen
#pragma unroll
                                for (int j = 0; j < 16; j++) {
                                    float *a = o + 4 * (j0 + j);
                                    a[0] = fmaf(f, v[j].x, a[0]);
                                    a[1] = fmaf(f, v[j].y, a[1]);
                                    a[2] = fmaf(f, v[j].z, a[2]);
                                    a[3] = fmaf(f, v[j].w, a[3]);
                                }
                        }
                    }
                    const float inv = 1.f / L;
                    if (row < rows)
#pragma unroll
                        for (int c = 0; c < HD; c += 16) {
#pragma unroll
                            for (int j = 0; j < 16; j++) o[c + j] = rhi > rlo ? o[c + j] * inv : 0.f;
                            store16(c, o + c);
                        }
                }
            }
            if (bad) sh.bad = 1;
            __syncwarp();
            if (lane == 0) pg_arrive(&sh.wfree[i & 1]);
        }
        // not finite, so again: the other warps have no wait left but the CTA's last barrier
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (sh.bad && !sh.fail) attn_exact_rows<HD, BF>(p, sh.plan, sh.n_cta, sh.joined, 2 * pt_tile_rows(p.group), PT_BK_SHIFT, 8);
    }
    pt_fence_before();
    __syncthreads();
    if (tid == 0 && sh.fail) *p.status = PG_GAVE_UP;
    if (warp == 8) {
        pt_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(sh.tmem) : "memory");
    }
}

}  // namespace fiber
