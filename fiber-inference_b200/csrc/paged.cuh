// paged.cuh — what the operators over the paged cache share: the device-side view and
// batch, the lookup of a token's place, the division of a ragged batch's attention over
// the CTAs, TMA and mbarrier helpers, and the attention of one row from the definition.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include "quant.cuh"

#ifndef HDCE
#define HDCE __host__ __device__ constexpr
#endif

namespace fiber {

// Division by a number known on the host: n / d = (mulhi(n, mul) + n) >> shift for n < 2^31.
struct FastDiv {
    uint32_t mul;
    int shift;
    uint32_t d;
};
inline FastDiv make_div(uint32_t d) {
    FastDiv f;
    f.shift = 0;
    while ((1ull << f.shift) < d) f.shift++;
    f.mul = (uint32_t)(((1ull << 32) * ((1ull << f.shift) - d)) / d + 1);
    f.d = d;
    return f;
}
FDEV int fdiv(int n, const FastDiv &f) { return (int)((__umulhi((uint32_t)n, f.mul) + (uint32_t)n) >> f.shift); }

struct PagedView {
    uint16_t *k, *v;  // 16-bit elements: fp16 or bf16
    const int32_t *table;
    int n_kv, page_shift, n_pages, n_slots, max_pages;
    long long page_stride, head_stride, pos_stride;
};

struct RaggedDev {
    int n_seqs, n_tokens;
    int slot0;  // slot of sequence 0 when slot is null
    const int32_t *q_start, *kv_len, *slot;
};

// A sequence as both operators read it: first token row, tokens, cached positions, slot.
// A slot or length outside the table gives an empty cache (kv = 0).
struct SeqInfo {
    int q0, nq, kv, slot;
};

FDEV SeqInfo make_seq(const RaggedDev &b, const PagedView &kv, int start, int end, int len, int slot) {
    SeqInfo s;
    s.q0 = min(max(start, 0), b.n_tokens);
    s.nq = min(max(end, s.q0), b.n_tokens) - s.q0;
    const bool ok = slot >= 0 && slot < kv.n_slots && len >= 0 && len <= ((long long)kv.max_pages << kv.page_shift);
    s.kv = ok ? len : 0;
    s.slot = ok ? slot : 0;
    return s;
}

// Position and slot of token `t`, by one warp; false when no sequence holds it. A 32-way
// search over q_start down to 32 sequences, whose bounds, lengths and slots are then
// loaded together.
FDEV bool find_token(const RaggedDev &b, const PagedView &kv, int t, int lane, int &pos, int &slot) {
    int lo = 0, n = b.n_seqs;
    while (n > 32) {
        const int step = (n + 31) / 32, i = lane * step;
        const int v = i < n ? b.q_start[lo + i] : 0x7fffffff;
        const int c = __popc(__ballot_sync(0xffffffffu, v <= t));
        if (c == 0) return false;
        lo += (c - 1) * step;
        n = min(step, n - (c - 1) * step);
    }
    SeqInfo s = {0, 0, 0, 0};
    if (lane < n)
        s = make_seq(b, kv, b.q_start[lo + lane], b.q_start[lo + lane + 1], b.kv_len[lo + lane],
                     b.slot ? b.slot[lo + lane] : b.slot0 + lo + lane);
    const unsigned hit = __ballot_sync(0xffffffffu, lane < n && t >= s.q0 && t < s.q0 + s.nq);
    if (!hit) return false;
    const int src = __ffs(hit) - 1;
    pos = __shfl_sync(0xffffffffu, s.kv - s.nq - s.q0, src) + t;
    slot = __shfl_sync(0xffffffffu, s.slot, src);
    return true;
}

// ---- 16-bit types ------------------------------------------------------------------------

template <bool BF>
FDEV float2 unpack2(uint32_t w) {
    if constexpr (BF)
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else
        return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <bool BF>
FDEV uint32_t pack2(float a, float b) {  // a in the low half
    uint32_t r;
    if constexpr (BF)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

// ---- mbarriers and TMA -------------------------------------------------------------------

constexpr long long PG_WAIT_CYCLES = 4000000000ll;   // about 2 s
constexpr long long PG_DRILL_CYCLES = 1000000ll;      // about 0.5 ms: the limit in a drill

FDEV uint32_t pg_saddr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
FDEV void pg_init(uint64_t *bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(pg_saddr(bar)), "r"(count) : "memory");
}
FDEV bool pg_try(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(pg_saddr(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// Waits for the phase of that parity; gives up when another thread of the CTA has
// (*fail), or after `limit` cycles (then sets *fail). The clock is looked at once in 256 tries
// only: a timer read before the first retry delayed every hand-over that was not ready at once.
FDEV bool pg_wait(uint64_t *bar, uint32_t parity, volatile int *fail, long long limit) {
    long long t0 = 0;
    for (uint32_t n = 0; !pg_try(bar, parity); n++) {
        if (n & 255) continue;
        if (fail && *fail) return false;
        const long long now = clock64();
        if (n == 0) t0 = now;
        if (now - t0 > limit) {
            if (fail) *fail = 1;
            return false;
        }
    }
    return true;
}
// The same by a whole warp, whose lanes may give up at different tries: they meet again
// before the warp-wide instructions that follow.
FDEV void pg_wait_warp(uint64_t *bar, uint32_t parity, volatile int *fail, long long limit) {
    pg_wait(bar, parity, fail, limit);
    __syncwarp();
}
// Waits for copies or products of this CTA that are in flight when it gives up or ends: always
// with the full limit.
FDEV void pg_drain(uint64_t *bar, uint32_t parity) { pg_wait(bar, parity, nullptr, PG_WAIT_CYCLES); }
FDEV void pg_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(pg_saddr(bar)) : "memory");
}
FDEV void pg_expect_tx(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(pg_saddr(bar)), "r"(bytes) : "memory");
}
FDEV void pg_tma4(uint32_t dst, const CUtensorMap *map, int c0, int c1, int c2, int c3, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(pg_saddr(bar))
        : "memory");
}
FDEV void pg_tma3(uint32_t dst, const CUtensorMap *map, int c0, int c1, int c2, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(pg_saddr(bar))
        : "memory");
}
FDEV void pg_prefetch_map(const CUtensorMap *map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
FDEV unsigned pg_ticket(unsigned *t) {  // orders this CTA's writes before, the others' after it
    unsigned v;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(v) : "l"(t) : "memory");
    return v;
}
FDEV void pg_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- attention -----------------------------------------------------------------------------

// What the division of the work counts: a unit costs `unit` plus `half` (up to half of its
// rows in use) or `full` per tile of keys. A unit of up to `snap` steps is not cut. A CTA's
// share is at least `share`, and at least `root` times the root of the longest unit's cost
// where that is known: with shares of x a unit costs x steps in a row and then a join of
// cost / x states, which is least at x ~ sqrt(cost).
struct AttnCost {
    int unit, half, full, snap, share;
    float root;
};

struct AttnPagedParams {
    CUtensorMap kmap, vmap;  // (head_dim, page_size, n_kv, n_pages); 128-byte swizzle
    CUtensorMap qmap;        // tile kernel: (head_dim, n_heads, n_tokens)
    PagedView kv;
    RaggedDev b;
    const uint16_t *q;
    uint16_t *out;
    long long ldq, ldo;
    int n_heads, group;  // group = n_heads / n_kv
    FastDiv by_group, by_ru;  // by_ru: rows of a unit
    int window;
    float scale, scale_log2;  // scale * log2(e): scores in powers of two
    AttnCost cost;
    long long wait_limit;     // cycles after which a wait gives up
    int drill;                // 1: no ring stage is ever free again, so that waits run out; else 0
    int *status;              // workspace: PG_GAVE_UP, PG_BAD_SM or PG_BAD_BATCH once that happened
    unsigned int *tickets;    // one per CTA, zero between calls
    float *part_ml;           // [2 * n_cta][rows][2]: running maximum (powers of two) and sum
    float *part_o;            // [2 * n_cta] unnormalised outputs
};

enum : int { PG_GAVE_UP = 1, PG_BAD_SM = 2, PG_BAD_BATCH = 3 };

constexpr int PG_MAX_SEQS = 128;  // sequences of one launch; larger batches take several

// How a launch's work is divided. The rows (token, head of the group) of a sequence and KV
// head are cut into units of RU rows; a unit takes one step per tile of BK keys that any
// of its rows sees (at least one, so rows that see nothing are written too). The costs of
// all units in the order (sequence, KV head, unit) are laid end to end, 0 .. T, and CTA c
// of n takes the steps whose places lie in [c T / n, (c + 1) T / n): equal shares whatever
// the lengths. A unit that is cut between CTAs leaves one softmax state per CTA; the last
// CTA to finish (ticket) joins them in CTA order, so the result does not depend on the
// timing.
struct AttnPlan {
    uint32_t prefix[PG_MAX_SEQS + 1];
    int4 seq[PG_MAX_SEQS];  // q0, nq, kv, slot
};

struct AttnUnit {
    int s, g, i;           // sequence, KV head, unit of RU rows
    int q0, nq, kv, slot;  // of the sequence
    int row0, rows;        // rows of the unit: row0 .. row0 + rows - 1 of nq * group
    int lo, hi;            // positions any row of the unit sees
    uint32_t u0, cost;     // where it starts, and what it costs
    int steps, per;        // its steps, and what one costs (0: all of them lie where it starts)
};

// Positions that the rows [row0, row0 + rows) see together.
FDEV void attn_span(int nq, int kv, const AttnPagedParams &p, int row0, int rows, int &lo, int &hi) {
    const int p0 = kv - nq, t0 = fdiv(row0, p.by_group), t1 = fdiv(row0 + rows - 1, p.by_group);
    hi = max(0, p0 + t1 + 1);
    lo = p.window > 0 ? max(0, p0 + t0 - p.window + 1) : 0;
}

FDEV int attn_steps(int lo, int hi, int bk_shift) {
    return max(1, hi > lo ? ((hi + (1 << bk_shift) - 1) >> bk_shift) - (lo >> bk_shift) : 0);
}
FDEV int attn_per(const AttnPagedParams &p, int rows, int ru) { return 2 * rows > ru ? p.cost.full : p.cost.half; }

FDEV uint32_t attn_unit_cost(int nq, int kv, const AttnPagedParams &p, int ru, int bk_shift, int i) {
    const int row0 = i * ru, rows = min(ru, nq * p.group - row0);
    int lo, hi;
    attn_span(nq, kv, p, row0, rows, lo, hi);
    return (uint32_t)(p.cost.unit + attn_per(p, rows, ru) * attn_steps(lo, hi, bk_shift));
}

// What the units of a sequence cost together, per KV head; all lanes of a warp.
FDEV uint32_t attn_seq_cost(int nq, int kv, const AttnPagedParams &p, int ru, int bk_shift, int lane) {
    const int nu = fdiv(nq * p.group + ru - 1, p.by_ru);
    uint32_t sum = 0;
    for (int i = lane; i < nu; i += 32) sum += attn_unit_cost(nq, kv, p, ru, bk_shift, i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// Fill the plan and return T; `longest`: the largest unit's cost, or 0. Up to 32 sequences
// each warp does it for itself (all write the same), without a barrier: one round trip for the
// lengths. More are shared among the CTA's threads. Where q_start decreases, the sequences may
// overlap and their costs pass 32 bits: T is 0 then, nothing is done and the status says so.
template <int THREADS>
FDEV uint32_t attn_plan_build(AttnPlan &pl, const AttnPagedParams &p, int ru, int bk_shift, uint32_t &longest) {
    const int tid = threadIdx.x, lane = tid & 31, ns = p.b.n_seqs;
    constexpr int SHORT = 4;  // sequences of more units are summed by whole warps
    bool falls = false;
    auto load = [&](int s) {
        const int start = p.b.q_start[s], end = p.b.q_start[s + 1];
        falls |= end < start;
        return make_seq(p.b, p.kv, start, end, p.b.kv_len[s], p.b.slot ? p.b.slot[s] : p.b.slot0 + s);
    };
    auto refuse = [&] {
        if (tid == 0) *p.status = PG_BAD_BATCH;
        return 0u;
    };
    auto few = [&](const SeqInfo &q, int nu) {
        uint32_t sum = 0;
        for (int i = 0; i < nu; i++) sum += attn_unit_cost(q.nq, q.kv, p, ru, bk_shift, i);
        return sum;
    };
    auto scan = [&](uint32_t v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += t;
        }
        return v;
    };
    if (ns <= 32) {
        SeqInfo q = {0, 0, 0, 0};
        if (lane < ns) q = load(lane);
        longest = 0;
        if (__any_sync(0xffffffffu, falls)) return refuse();
        const int nu = fdiv(q.nq * p.group + ru - 1, p.by_ru);
        uint32_t sum = nu <= SHORT ? few(q, nu) : 0;
        for (unsigned big = __ballot_sync(0xffffffffu, nu > SHORT); big; big &= big - 1) {
            const int s = __ffs(big) - 1;
            const uint32_t v = attn_seq_cost(__shfl_sync(0xffffffffu, q.nq, s), __shfl_sync(0xffffffffu, q.kv, s), p, ru, bk_shift, lane);
            if (lane == s) sum = v;
        }
        longest = __reduce_max_sync(0xffffffffu, nu > 0 ? attn_unit_cost(q.nq, q.kv, p, ru, bk_shift, nu - 1) : 0u);
        sum = scan(sum * (uint32_t)p.kv.n_kv);
        if (lane < ns) {
            pl.seq[lane] = make_int4(q.q0, q.nq, q.kv, q.slot);
            pl.prefix[lane + 1] = sum;
        }
        if (lane == 0) pl.prefix[0] = 0;
        __syncwarp();
        return __shfl_sync(0xffffffffu, sum, 31);
    }
    longest = 0;
    for (int s = tid; s < ns; s += THREADS) {
        const SeqInfo q = load(s);
        pl.seq[s] = make_int4(q.q0, q.nq, q.kv, q.slot);
        const int nu = fdiv(q.nq * p.group + ru - 1, p.by_ru);
        pl.prefix[s + 1] = nu <= SHORT ? few(q, nu) : 0;
    }
    if (tid == 0) pl.prefix[0] = 0;
    if (__syncthreads_or(falls)) return refuse();
    for (int s = tid >> 5; s < ns; s += THREADS / 32) {
        const int4 q = pl.seq[s];
        if (fdiv(q.y * p.group + ru - 1, p.by_ru) <= SHORT) continue;
        const uint32_t sum = attn_seq_cost(q.y, q.z, p, ru, bk_shift, lane);
        if (lane == 0) pl.prefix[s + 1] = sum;
    }
    __syncthreads();
    if (tid < 32) {
        uint32_t base = 0;
        for (int s0 = 0; s0 < ns; s0 += 32) {
            const int s = s0 + lane;
            const uint32_t v = scan(s < ns ? pl.prefix[s + 1] * (uint32_t)p.kv.n_kv : 0);
            __syncwarp();
            if (s < ns) pl.prefix[s + 1] = base + v;
            base += __shfl_sync(0xffffffffu, v, 31);
        }
    }
    __syncthreads();
    return pl.prefix[ns];
}

FDEV void attn_unit_fill(AttnUnit &u, const AttnPlan &pl, const AttnPagedParams &p, int ru, int bk_shift) {
    const int4 q = pl.seq[u.s];
    u.q0 = q.x;
    u.nq = q.y;
    u.kv = q.z;
    u.slot = q.w;
    u.row0 = u.i * ru;
    u.rows = min(ru, u.nq * p.group - u.row0);
    attn_span(u.nq, u.kv, p, u.row0, u.rows, u.lo, u.hi);
    u.steps = attn_steps(u.lo, u.hi, bk_shift);
    u.per = attn_per(p, u.rows, ru);
    u.cost = (uint32_t)(p.cost.unit + u.per * u.steps);
    if (u.steps <= p.cost.snap) u.per = 0;
}

// The unit that holds place x; all lanes of a warp together.
FDEV void attn_unit_find(AttnUnit &u, const AttnPlan &pl, const AttnPagedParams &p, int ru, int bk_shift, uint32_t x) {
    const int lane = threadIdx.x & 31;
    int a = 0, b = p.b.n_seqs;  // prefix[a] <= x < prefix[b]
    while (b - a > 1) {
        const int step = (b - a + 31) / 32, i = a + lane * step;
        const int c = __popc(__ballot_sync(0xffffffffu, i < b && pl.prefix[min(i, b)] <= x));
        a += (c - 1) * step;
        b = min(a + step, b);
    }
    u.s = a;
    const uint32_t head = (pl.prefix[a + 1] - pl.prefix[a]) / (uint32_t)p.kv.n_kv;
    uint32_t rem = x - pl.prefix[a];
    u.g = (int)(rem / head);
    rem -= (uint32_t)u.g * head;
    const int4 q = pl.seq[a];
    const int nu = fdiv(q.y * p.group + ru - 1, p.by_ru);
    for (int i0 = 0;; i0 += 32) {
        uint32_t n = i0 + lane < nu ? attn_unit_cost(q.y, q.z, p, ru, bk_shift, i0 + lane) : 0, sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += t;
        }
        const unsigned past = __ballot_sync(0xffffffffu, sum > rem);
        if (past) {
            const int l = __ffs(past) - 1;
            rem -= __shfl_sync(0xffffffffu, sum - n, l);
            u.i = i0 + l;
            break;
        }
        rem -= __shfl_sync(0xffffffffu, sum, 31);
    }
    u.u0 = x - rem;
    attn_unit_fill(u, pl, p, ru, bk_shift);
}

// The unit after u (the caller knows there is one).
FDEV void attn_unit_next(AttnUnit &u, const AttnPlan &pl, const AttnPagedParams &p, int ru, int bk_shift) {
    u.u0 += u.cost;
    u.i++;
    if (u.i * ru >= u.nq * p.group) {
        u.i = 0;
        u.g++;
        if (u.g == p.kv.n_kv) {
            u.g = 0;
            do u.s++;
            while (pl.prefix[u.s + 1] == pl.prefix[u.s]);  // sequences without tokens
        }
    }
    attn_unit_fill(u, pl, p, ru, bk_shift);
}

// CTAs of a launch, the start of CTA c's share, and the CTA whose share holds place x.
FDEV int attn_ctas(const AttnPagedParams &p, uint32_t total, uint32_t longest) {
    const uint32_t share = max((uint32_t)p.cost.share, (uint32_t)(p.cost.root * sqrtf((float)longest)));
    return total == 0 ? 0 : (int)min(gridDim.x, max(1u, total / share));
}
FDEV uint32_t attn_share(uint32_t total, int n_cta, int c) { return (uint32_t)((unsigned long long)total * c / n_cta); }
FDEV int attn_owner(uint32_t total, int n_cta, uint32_t x) {
    return (int)((((unsigned long long)x + 1) * n_cta - 1) / total);
}
// Step k of a unit lies at the place u0 + unit + k per. A share spans at least one step's
// cost, so every CTA between a cut unit's first and last has a piece of it.
FDEV uint32_t attn_place(const AttnUnit &u, const AttnPagedParams &p, int k) {
    return u.u0 + (u.per ? (uint32_t)(p.cost.unit + k * u.per) : 0u);
}
// The first step of the unit at or after place x.
FDEV int attn_step_at(const AttnUnit &u, const AttnPagedParams &p, uint32_t x) {
    if (u.per == 0) return x > u.u0 ? u.steps : 0;
    const int d = (int)(x - u.u0) - p.cost.unit;
    return d <= 0 ? 0 : min(u.steps, u.per == 1 ? d : (d + u.per - 1) / u.per);
}

// Whether x is not finite once rounded to 16 bits (half a step above the largest value is not).
template <bool BF>
FDEV bool attn_spoiled(float x) {
    return !(fabsf(x) < (BF ? __uint_as_float(0x7f7f8000u) : 65520.f));
}

// One row from the definition, by one warp: only the positions the row sees are read, so
// nothing behind a mask can reach it. A score that is NaN or +inf, or none above -inf, makes
// every weight NaN: such a row ends at the first of them. Else about 0.2 us a key, the latency of
// one warp's instructions. Lane i takes the output's values (HD / 32) i and up.
template <int HD, bool BF>
static __device__ __noinline__ void attn_row_exact(const AttnPagedParams &p, const uint16_t *q, uint16_t *out, int slot,
                                                   int g, uint32_t lo, uint32_t hi, int lane) {
    constexpr int W = HD / 64;  // 32-bit words per lane
    const PagedView &c = p.kv;
    const uint32_t mask = (1u << c.page_shift) - 1;
    const int32_t *tab = c.table + (long long)slot * c.max_pages;
    auto at = [&](uint32_t j) -> long long {  // -1: a table entry outside the pool reads as zeros
        const int page = tab[j >> c.page_shift];
        if (page < 0 || page >= c.n_pages) return -1;
        return (long long)page * c.page_stride + (long long)g * c.head_stride + (long long)(j & mask) * c.pos_stride;
    };
    float qf[HD / 8];
#pragma unroll
    for (int d = 0; d < HD / 64; d++) {
        const uint4 x = *reinterpret_cast<const uint4 *>(q + 64 * d + 8 * (lane & 7));
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = unpack2<BF>(xs[i]);
            qf[8 * d + 2 * i] = f.x;
            qf[8 * d + 2 * i + 1] = f.y;
        }
    }
    // The scores of 32 keys, lane i's at place a, by eight lanes to a key: 32 lanes with a key
    // each touch 32 cache lines per load (0.28 us a key instead of 0.2).
    auto scores = [&](long long a) -> float {
        float mine = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const long long ak = __shfl_sync(0xffffffffu, a, 4 * i + (lane >> 3));
            float s = 0.f;
#pragma unroll
            for (int d = 0; d < HD / 64; d++) {
                uint4 y = make_uint4(0u, 0u, 0u, 0u);
                if (ak >= 0) y = *reinterpret_cast<const uint4 *>(c.k + ak + 64 * d + 8 * (lane & 7));
                const uint32_t ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const float2 h = unpack2<BF>(ys[n]);
                    s = fmaf(qf[8 * d + 2 * n + 1], h.y, fmaf(qf[8 * d + 2 * n], h.x, s));
                }
            }
            if (ak < 0) s = 0.f;
            s += __shfl_xor_sync(0xffffffffu, s, 1);
            s += __shfl_xor_sync(0xffffffffu, s, 2);
            s += __shfl_xor_sync(0xffffffffu, s, 4);
            s = __shfl_sync(0xffffffffu, s, 8 * (lane & 3));
            if (lane >> 2 == i) mine = s;
        }
        return mine * p.scale;
    };
    uint32_t *dst = reinterpret_cast<uint32_t *>(out) + W * lane;
    float m = -INFINITY;
    bool nan = false;
    for (uint32_t j0 = lo; j0 < hi && !nan; j0 += 32) {
        const bool in = j0 + lane < hi;
        float s = scores(in ? at(j0 + lane) : -1);
        if (!in) s = -INFINITY;
        nan = __any_sync(0xffffffffu, !(s < INFINITY));
        m = fmaxf(m, s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (nan || m == -INFINITY) {
#pragma unroll
        for (int k = 0; k < W; k++) dst[k] = 0x7fff7fffu;
        return;
    }
    float l = 0.f, o2[2 * W];
#pragma unroll
    for (int k = 0; k < 2 * W; k++) o2[k] = 0.f;
    for (uint32_t j0 = lo; j0 < hi; j0 += 32) {
        const bool in = j0 + lane < hi;
        const long long a = in ? at(j0 + lane) : -1;
        const float s = scores(a), e = in ? expf(s - m) : 0.f;
        l += e;
#pragma unroll 8
        for (int i = 0; i < 32; i++) {  // past the end: weight 0 and value 0
            const float w = __shfl_sync(0xffffffffu, e, i);
            const long long av = __shfl_sync(0xffffffffu, a, i);
            const uint32_t *src = reinterpret_cast<const uint32_t *>(c.v + av) + W * lane;
#pragma unroll
            for (int k = 0; k < W; k++) {
                const float2 v = unpack2<BF>(av < 0 ? 0u : src[k]);
                o2[2 * k] = fmaf(w, v.x, o2[2 * k]);
                o2[2 * k + 1] = fmaf(w, v.y, o2[2 * k + 1]);
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
    for (int k = 0; k < W; k++) dst[k] = pack2<BF>(o2[2 * k] / l, o2[2 * k + 1] / l);
}

// The rows that this CTA has written (whole units, and the cut ones it has joined) and whose
// stored result is not finite, again and exactly: on the tensor cores a masked position has
// weight 0, and 0 * inf or 0 * NaN is NaN. By the first `warps` warps after the CTA's other work,
// when nothing in the kernel waits any more, since how long it takes depends on the data: 64 tokens of
// 32 heads (dim 128) over 16,384 positions, 32 rows a warp, take 0.16 ms where the first key is NaN
// (0.08 without), 110 ms where a value is.
template <int HD, bool BF>
static __device__ __noinline__ void attn_exact_rows(const AttnPagedParams &p, const AttnPlan &pl, int n_cta,
                                                    const int *joined, int ru, int bk_shift, int warps) {
    constexpr uint32_t EXP = BF ? 0x7f80u : 0x7c00u;
    const int cta = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t total = pl.prefix[p.b.n_seqs], x0 = attn_share(total, n_cta, cta), x1 = attn_share(total, n_cta, cta + 1);
    AttnUnit u;
    attn_unit_find(u, pl, p, ru, bk_shift, x0);
    for (;;) {
        const int b = u.u0 < x0 ? attn_step_at(u, p, x0) : 0, e = u.u0 + u.cost > x1 ? attn_step_at(u, p, x1) : u.steps;
        if (u.hi > u.lo && b < e && ((b == 0 && e == u.steps) || joined[b > 0 ? 0 : 1]))
            for (int r = warp; r < u.rows; r += warps) {
                const int t = fdiv(u.row0 + r, p.by_group), head = u.g * p.group + u.row0 + r - t * p.group;
                const int pos = u.kv - u.nq + t;
                if (pos < 0) continue;
                uint16_t *out = p.out + (long long)(u.q0 + t) * p.ldo + (long long)head * HD;
                bool bad = false;
#pragma unroll
                for (int k = 0; k < HD / 64; k++) {
                    const uint32_t w = reinterpret_cast<const uint32_t *>(out)[32 * k + lane];
                    bad |= (w & EXP) == EXP || (w >> 16 & EXP) == EXP;
                }
                if (__any_sync(0xffffffffu, bad))
                    attn_row_exact<HD, BF>(p, p.q + (long long)(u.q0 + t) * p.ldq + (long long)head * HD, out, u.slot, u.g,
                                           p.window > 0 ? max(0, pos - p.window + 1) : 0, pos + 1, lane);
            }
        if (u.u0 + u.cost >= x1) break;
        attn_unit_next(u, pl, p, ru, bk_shift);
    }
}

}  // namespace fiber
