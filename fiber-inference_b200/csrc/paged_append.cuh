// paged_append.cuh — rotate the new tokens' queries and keys and store keys and values
// in the paged cache.
//
// For a pair (a, b) of a head and the token's position p: a' = a cos - b sin,
// b' = a sin + b cos with (cos, sin) from an fp32 table, in fp32 with separate products
// (the expressions of the layer pass's own append, so both leave the same bits in the
// cache), rounded once to the cache's type.
//
// Bound by bytes: every value is read and written once, 3 operations each. 17,055 tokens
// of 32 + 8 + 8 heads of 128 (bf16, 420 MB) take 74 us, 5.7 TB/s or 87% of a plain copy's
// rate; one token takes 2.8 us on the device, the latency of two dependent lookups, and 512
// tokens of 32 + 4 + 4 heads of 64 (fp32 in, 8 MB) 3.8 us.
#pragma once
#include "paged.cuh"

namespace fiber {

struct AppendParams {
    PagedView kv;
    RaggedDev b;
    const void *q, *k, *v;  // q null: keys and values only
    long long ldq, ldk, ldv, ldo;
    int n_heads;            // 0 when q is null
    const float2 *rope;     // [max_pos][rot / 2], or null
    int max_pos, rot, adjacent;
    uint16_t *q_out;
};

constexpr int APPEND_THREADS = 128;
constexpr int APPEND_HPT = 4;  // heads per thread

// Thread tasks of one token: 16 values (two 8-value pieces) of APPEND_HPT heads each.
HDCE int append_warps_per_token(int heads, int hd) {
    return ((heads + APPEND_HPT - 1) / APPEND_HPT * (hd / 16) + 31) / 32;
}

template <class TI>
struct Raw8;  // eight input values as loaded
template <>
struct Raw8<float> {
    float4 a, b;
    FDEV void load(const void *p, long long i) {
        const float4 *s = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + i);
        a = __ldcs(s);
        b = __ldcs(s + 1);
    }
    FDEV void get(float (&x)[8]) const {
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
};
template <bool BF>
struct Raw8x16 {
    uint4 a;
    FDEV void load(const void *p, long long i) {
        a = __ldcs(reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(p) + i));
    }
    FDEV void get(float (&x)[8]) const {
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 f = unpack2<BF>(w[j]);
            x[2 * j] = f.x;
            x[2 * j + 1] = f.y;
        }
    }
};
template <>
struct Raw8<__half> : Raw8x16<false> {};
template <>
struct Raw8<__nv_bfloat16> : Raw8x16<true> {};

template <bool BF>
FDEV void store8(uint16_t *dst, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(dst) = make_uint4(pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3]), pack2<BF>(x[4], x[5]),
                                                 pack2<BF>(x[6], x[7]));
}

// One warp per (token, 32 thread tasks). A thread takes the same 16 values of four heads
// (two: 84 us, eight: 98 us for the case above), so the table's pairs are loaded once for the
// four; all its input loads are issued
// before the token's place (sequence, position, page) is looked up, whose two dependent
// round trips are the latency of a small call.
template <class TI, bool BF, int HD>
__global__ void __launch_bounds__(APPEND_THREADS) kv_append_kernel(const AppendParams p) {
    pdl_trigger();
    pdl_wait();
    constexpr int U = HD / 16;
    const int heads = p.n_heads + 2 * p.kv.n_kv, hstep = (heads + APPEND_HPT - 1) / APPEND_HPT;
    const int wpt = append_warps_per_token(heads, HD), lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * (APPEND_THREADS / 32) + (threadIdx.x >> 5);
    const int token = (int)(w / wpt);
    if (token >= p.b.n_tokens) return;
    const int task = (int)(w % wpt) * 32 + lane, u = task % U, h0 = task / U;
    const bool turn = u * 16 < p.rot, halves = turn && !p.adjacent;
    const int o0 = halves ? 8 * u : 16 * u, o1 = halves ? p.rot / 2 + 8 * u : 16 * u + 8;

    Raw8<TI> x0[APPEND_HPT], x1[APPEND_HPT];
#pragma unroll
    for (int i = 0; i < APPEND_HPT; i++) {
        const int h = h0 + i * hstep;
        if (h0 >= hstep || h >= heads) continue;
        const void *src = h < p.n_heads ? p.q : (h < p.n_heads + p.kv.n_kv ? p.k : p.v);
        const long long at = h < p.n_heads                ? token * p.ldq + (long long)h * HD
                             : h < p.n_heads + p.kv.n_kv ? token * p.ldk + (long long)(h - p.n_heads) * HD
                                                          : token * p.ldv + (long long)(h - p.n_heads - p.kv.n_kv) * HD;
        x0[i].load(src, at + o0);
        x1[i].load(src, at + o1);
    }
    int pos, slot;
    if (!find_token(p.b, p.kv, token, lane, pos, slot)) return;  // in no sequence: left alone
    if (h0 >= hstep) return;
    const bool placed = pos >= 0 && (!p.rope || pos < p.max_pos);
    int page = -1;
    if (placed) page = p.kv.table[(long long)slot * p.kv.max_pages + (pos >> p.kv.page_shift)];
    float2 cs[8];
    if (placed && turn) {
        const float4 *t = reinterpret_cast<const float4 *>(p.rope + (long long)pos * (p.rot / 2) + 8 * u);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float4 f = __ldg(t + j);
            cs[2 * j] = make_float2(f.x, f.y);
            cs[2 * j + 1] = make_float2(f.z, f.w);
        }
    }
    const bool in_pool = page >= 0 && page < p.kv.n_pages;
    const long long row = (long long)page * p.kv.page_stride + (long long)(pos & ((1 << p.kv.page_shift) - 1)) * p.kv.pos_stride;
#pragma unroll
    for (int i = 0; i < APPEND_HPT; i++) {
        const int h = h0 + i * hstep;
        if (h >= heads) continue;
        const int g = h - p.n_heads;  // >= 0: a key head, then value heads
        float a[8], b[8];
        x0[i].get(a);
        x1[i].get(b);
        if (turn && g < p.kv.n_kv) {
            if (halves) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float xa = a[j], xb = b[j];
                    a[j] = __fsub_rn(__fmul_rn(xa, cs[j].x), __fmul_rn(xb, cs[j].y));
                    b[j] = __fadd_rn(__fmul_rn(xa, cs[j].y), __fmul_rn(xb, cs[j].x));
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float xa = a[2 * j], xb = a[2 * j + 1], ya = b[2 * j], yb = b[2 * j + 1];
                    a[2 * j] = __fsub_rn(__fmul_rn(xa, cs[j].x), __fmul_rn(xb, cs[j].y));
                    a[2 * j + 1] = __fadd_rn(__fmul_rn(xa, cs[j].y), __fmul_rn(xb, cs[j].x));
                    b[2 * j] = __fsub_rn(__fmul_rn(ya, cs[4 + j].x), __fmul_rn(yb, cs[4 + j].y));
                    b[2 * j + 1] = __fadd_rn(__fmul_rn(ya, cs[4 + j].y), __fmul_rn(yb, cs[4 + j].x));
                }
            }
        }
        uint16_t *dst;
        if (g < 0) {
            dst = p.q_out + (long long)token * p.ldo + (long long)h * HD;
            if (!placed)
#pragma unroll
                for (int j = 0; j < 8; j++) a[j] = b[j] = 0.f;
        } else {
            if (!in_pool) continue;
            dst = g < p.kv.n_kv ? p.kv.k + row + (long long)g * p.kv.head_stride
                                : p.kv.v + row + (long long)(g - p.kv.n_kv) * p.kv.head_stride;
        }
        store8<BF>(dst + o0, a);
        store8<BF>(dst + o1, b);
    }
}

}  // namespace fiber
