"""The operators over the paged cache against their definitions in 64 bits.

Tolerances, with u the unit roundoff of the 16-bit type (half its eps: 2^-11 fp16, 2^-8 bf16):
  append: two fp32 products and their sum, then one rounding: |err| <= u |y| + 3 * 2^-24 (|a| + |b|),
    plus half an fp16 subnormal step (2^-25);
  attend, for one output o = sum p_j v_j with w = sum p_j |v_j|: probabilities are rounded (u w), the
    output is rounded (u |o|); a score is an fp32 sum of up to 128 exact products, off by at most
    2^-17 A with A = max scale * sum |q||k|, which moves a probability by twice that; exp and the
    sums 2^-15; an fp16 probability below 2^-14 of the row's largest is off by up to 2^-25 (keys * max |v|).
"""
from __future__ import annotations

import math

import numpy as np
import pytest

import fiber_b200 as fb

pytestmark = pytest.mark.gpu

U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def torch_():
    import torch

    return torch


class Setup:
    """Pools, table and batch for sequences [(new tokens, cached positions)]."""

    def __init__(self, lens, heads, kv_heads, dim, dtype="f16", page=64, layout="heads", window=0, seed=0, spare=3,
                 row_pad=0, slots="shuffled", fill=None, scale=None, max_q=None):
        torch = torch_()
        self.lens, self.H, self.KV, self.D, self.P = lens, heads, kv_heads, dim, page
        self.dtype, self.layout, self.window = dtype, layout, window
        self.dt = {"f16": torch.float16, "bf16": torch.bfloat16}[dtype]
        self.scale = 1.0 / math.sqrt(dim) if scale is None else scale
        g = torch.Generator().manual_seed(seed)
        n_seqs = len(lens)
        used = [-(-kv // page) for _, kv in lens]
        self.max_pages = max(1, max(used))
        self.n_pages = sum(used) + spare
        perm = torch.randperm(self.n_pages, generator=g).tolist()
        self.order = torch.randperm(n_seqs, generator=g).tolist() if slots == "shuffled" else list(range(n_seqs))
        # entries beyond a sequence's pages are never to be read
        self.table = torch.full((n_seqs, self.max_pages), 0x7fffffff, dtype=torch.int32)
        for s, k in enumerate(used):
            self.table[self.order[s], :k] = torch.tensor([perm.pop() for _ in range(k)], dtype=torch.int32)
        shape = (self.n_pages, kv_heads, page, dim) if layout == "heads" else (self.n_pages, page, kv_heads, dim)
        self.k = torch.randn(shape, generator=g).to(self.dt)
        self.v = torch.randn(shape, generator=g).to(self.dt)
        if fill is not None:  # every position no sequence holds
            for pool in (self.k, self.v):
                keep = torch.zeros(self.n_pages, page, dtype=torch.bool)
                for s, (_, kv) in enumerate(lens):
                    for j in range(kv):
                        keep[int(self.table[self.order[s], j // page]), j % page] = True
                m = keep[:, None, :, None] if layout == "heads" else keep[:, :, None, None]
                pool.copy_(torch.where(m, pool, torch.full_like(pool, fill)))
        starts = np.cumsum([0] + [n for n, _ in lens]).tolist()
        self.n = starts[-1]
        self.starts = starts
        self.rows = self.n + 2  # rows past the last sequence must stay as they are
        self.ld = heads * dim + row_pad
        gain = torch.linspace(0.5, 3.0, heads)[None, :, None]
        self.q = torch.zeros(self.rows, self.ld, dtype=self.dt)
        self.q[:, :heads * dim] = (torch.randn(self.rows, heads, dim, generator=g) * gain).reshape(self.rows, -1).to(self.dt)
        self.dk, self.dv, self.dq, self.dtab = self.k.cuda(), self.v.cuda(), self.q.cuda(), self.table.cuda()
        self.dstart = torch.tensor(starts, dtype=torch.int32).cuda()
        self.dlen = torch.tensor([kv for _, kv in lens], dtype=torch.int32).cuda()
        self.dslot = torch.tensor(self.order, dtype=torch.int32).cuda() if slots == "shuffled" else None
        self.view = self.make_view()
        self.batch = fb.RaggedBatch(self.dstart.data_ptr(), self.dlen.data_ptr(), n_seqs=n_seqs, n_tokens=self.rows,
                                    max_q=max(1, max(n for n, _ in lens)) if max_q is None else max_q,
                                    slot=self.dslot.data_ptr() if self.dslot is not None else None)
        self.out = torch.full((self.rows, self.ld), 7.0, dtype=self.dt, device="cuda")
        self.ws = torch.zeros(fb.attn_paged_workspace(self.view, self.batch, heads), dtype=torch.uint8, device="cuda")

    def make_view(self):
        hs, ps = (self.P * self.D, self.D) if self.layout == "heads" else (self.D, self.KV * self.D)
        return fb.PagedKV(self.dk.data_ptr(), self.dv.data_ptr(), self.dtab.data_ptr(), n_slots=len(self.lens),
                          max_pages=self.max_pages, n_pages=self.n_pages, page_size=self.P, n_kv_heads=self.KV,
                          head_dim=self.D, dtype={"f16": 1, "bf16": 30}[self.dtype],
                          page_stride=self.KV * self.P * self.D, head_stride=hs, pos_stride=ps)

    def attend(self, stream=None):
        fb.attn_paged(self.view, self.batch, self.dq.data_ptr(), self.out.data_ptr(), n_heads=self.H, ldq=self.ld,
                      ldo=self.ld, scale=self.scale, window=self.window, ws=self.ws.data_ptr(),
                      ws_bytes=self.ws.numel(), stream=stream)

    def cached(self, pool, s):
        """Positions 0 .. kv - 1 of sequence s, [kv, KV, D] in 64 bits."""
        torch = torch_()
        kv = self.lens[s][1]
        p = pool if self.layout == "positions" else pool.transpose(1, 2)
        pages = self.table[self.order[s], :-(-kv // self.P)].long()
        return p[pages].reshape(-1, self.KV, self.D)[:kv].to(torch.float64)

    def reference(self):
        """(out, tolerance), [rows, H, D] in 64 bits."""
        torch = torch_()
        G, u = self.H // self.KV, U[self.dtype]
        out = torch.zeros(self.n, self.H, self.D, dtype=torch.float64)
        tol = torch.zeros_like(out)
        for s, (n, kv) in enumerate(self.lens):
            if n == 0:
                continue
            k, v = self.cached(self.k, s), self.cached(self.v, s)
            q = self.q[self.starts[s]:self.starts[s] + n, :self.H * self.D].reshape(n, self.H, self.D).double()
            for i in range(n):
                pos = kv - n + i
                lo = max(0, pos - self.window + 1) if self.window else 0
                if pos < lo:
                    continue
                for h in range(self.H):
                    kk, vv = k[lo:pos + 1, h // G], v[lo:pos + 1, h // G]
                    x = (kk @ q[i, h]) * self.scale
                    p = torch.exp(x - x.max())
                    p = p / p.sum()
                    o, w = p @ vv, p @ vv.abs()
                    big = float((kk.abs() @ q[i, h].abs()).max()) * self.scale
                    out[self.starts[s] + i, h] = o
                    t = 1.05 * u * (o.abs() + w) + w * (2.0 ** -16 * big + 2.0 ** -15)
                    if self.dtype == "f16":
                        t = t + 2.0 ** -25 * (len(x) * float(vv.abs().max()) + 1)
                    tol[self.starts[s] + i, h] = t
        return out, tol

    def check(self):
        torch = torch_()
        fb.attn_paged_status(self.ws.data_ptr())
        got = self.out.cpu().double()
        assert torch.equal(got[self.n:], torch.full_like(got[self.n:], 7.0)), "rows of no sequence were written"
        assert torch.equal(got[:, self.H * self.D:], torch.full_like(got[:, self.H * self.D:], 7.0)), "row padding was written"
        want, tol = self.reference()
        got = got[:self.n, :self.H * self.D].reshape(self.n, self.H, self.D)
        assert torch.isfinite(got).all()
        bad = (got - want).abs() > tol
        assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / tol.clamp_min(1e-30)).max()),
                               torch.nonzero(bad)[:4].tolist())


SINGLES = [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 63), (1, 64), (1, 65), (1, 129), (1, 300)]
CHUNKS = [(1, 1), (2, 2), (5, 64), (16, 16), (17, 40), (33, 33), (64, 128), (130, 131), (7, 263)]
EMPTY = [(0, 5), (1, 0), (0, 0), (3, 0), (5, 2), (1, 1), (4, 4), (0, 70), (90, 70)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 1), (6, 2), (7, 1), (32, 2)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attn_single_tokens(dim, heads, kv_heads, dtype):
    s = Setup(SINGLES, heads, kv_heads, dim, dtype, seed=dim + heads)
    s.attend()
    s.check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 1), (3, 1), (14, 2), (20, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attn_chunks(dim, heads, kv_heads, dtype):
    s = Setup(CHUNKS, heads, kv_heads, dim, dtype, seed=dim + heads)
    s.attend()
    s.check()


@pytest.mark.parametrize("heads,kv_heads", [(33, 1), (64, 1), (128, 1), (127, 1), (96, 2)])
def test_attn_wide_groups(heads, kv_heads):
    """Up to 128 query heads per KV head: tiles of one to three tokens."""
    s = Setup([(1, 70), (5, 40), (3, 2), (4, 130)], heads, kv_heads, 64, "f16", 32, seed=heads)
    s.attend()
    s.check()


@pytest.mark.parametrize("nq", [1, 30])
def test_attn_window_beyond_the_cache(nq):
    """The widest window there is, with rows that see nothing: as without a window."""
    s = Setup([(nq, 20), (nq, 100)], 2, 1, 64, window=2 ** 31 - 1, seed=nq)
    s.attend()
    s.window = 0
    s.check()


@pytest.mark.parametrize("layout", ["heads", "positions"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("lens", [SINGLES, CHUNKS], ids=["singles", "chunks"])
def test_attn_pages_and_layouts(lens, page, layout):
    s = Setup(lens, 4, 2, 64, "f16", page, layout, row_pad=8, seed=page)
    s.attend()
    s.check()


@pytest.mark.parametrize("window", [1, 2, 15, 64, 65, 100, 1000])
@pytest.mark.parametrize("lens", [SINGLES, CHUNKS, EMPTY], ids=["singles", "chunks", "empty"])
def test_attn_window(lens, window):
    s = Setup(lens, 4, 2, 64, "bf16", 16, window=window, seed=window)
    s.attend()
    s.check()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("max_q", [None, 1, 4096])
def test_attn_empty_rows_and_lengths(dim, max_q):
    """Sequences without tokens, caches without positions, more tokens than positions; max_q is a hint."""
    s = Setup(EMPTY, 4, 2, dim, slots="own", seed=dim, max_q=max_q)
    s.ws = torch_().zeros(64 << 20, dtype=torch_().uint8, device="cuda")
    s.attend()
    s.check()
    got = s.out.cpu()[:, :4 * dim]
    assert (got[s.starts[1]] == 0).all() and (got[s.starts[3]:s.starts[3] + 3] == 0).all()
    assert (got[s.starts[4]:s.starts[4] + 3] == 0).all() and not (got[s.starts[4] + 3] == 0).all()


@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -65504.0])
@pytest.mark.parametrize("lens,window", [(SINGLES, 0), (CHUNKS, 0), (SINGLES, 20), (CHUNKS, 20)])
def test_attn_positions_of_no_sequence_do_not_matter(lens, window, fill):
    s = Setup(lens, 4, 2, 64, "f16", 64, window=window, fill=fill, seed=3)
    s.attend()
    s.check()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 1)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_attn_positions_behind_the_mask_do_not_matter(dim, heads, kv_heads, bad):
    """K and V of positions later tokens append, or that left the window, are not finite: only rows
    that see them may notice."""
    torch = torch_()
    lens, window = [(40, 150), (1, 90)], 48
    s = Setup(lens, heads, kv_heads, dim, "f16", 16, window=window, seed=9)
    hit = {0: [5, 60, 130, 149], 1: [10, 41]}  # poisoned positions; the second sequence's row sees 42 .. 89
    for q, js in hit.items():
        for j in js:
            page, at = int(s.table[s.order[q], j // 16]), j % 16
            s.k[page, :, at] = bad
            s.v[page, :, at] = bad
    s.dk.copy_(s.k)
    s.dv.copy_(s.v)
    s.attend()
    fb.attn_paged_status(s.ws.data_ptr())
    want, tol = s.reference()
    got = s.out.cpu().double()[:s.n, :heads * dim].reshape(s.n, heads, dim)
    clean = torch.tensor([not any(max(0, kv - n + i - window + 1) <= j <= kv - n + i for j in hit[q])
                          for q, (n, kv) in enumerate(lens) for i in range(n)])
    assert clean.sum() > 5 and (~clean).sum() > 5
    assert ((got - want).abs() <= tol)[clean].all()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])


@pytest.mark.parametrize("at", range(8))
@pytest.mark.parametrize("dim", [64, 128])
def test_attn_largest_values_behind_the_mask_do_not_matter(dim, at):
    """A weight behind the mask is exactly zero: values near bf16's largest there add nothing."""
    torch = torch_()
    lens, window = [(150, 200), (1, 90)], 30
    s = Setup(lens, 8, 2, dim, "bf16", 16, window=window, seed=21)
    j = 104 + at  # the first rows are before it, the last have it behind their window
    page = int(s.table[s.order[0], j // 16])
    s.v[page, :, j % 16] = 3e38
    s.dv.copy_(s.v)
    s.attend()
    fb.attn_paged_status(s.ws.data_ptr())
    want, tol = s.reference()
    got = s.out.cpu().double()[:s.n, :8 * dim].reshape(s.n, 8, dim)
    clean = torch.tensor([not i - window + 1 <= j <= i for i in range(50, 200)] + [True])
    assert clean.sum() == 151 - window
    assert ((got - want).abs() <= tol)[clean].all()


@pytest.mark.parametrize("at", range(8))
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attn_keys_that_are_not_finite_are_seen(bad, dtype, at):
    """One element of one key is not finite and every value is: the rows that see the key, and no
    others, get what the formula gives."""
    torch = torch_()
    lens = [(60, 130), (1, 90)]
    s = Setup(lens, 8, 2, 64, dtype, 16, seed=22)
    for q, j in ((0, 96 + at), (1, 40 + at)):
        s.k[int(s.table[s.order[q], j // 16]), :, j % 16, 5] = bad
    s.dk.copy_(s.k)
    s.attend()
    fb.attn_paged_status(s.ws.data_ptr())
    want, tol = s.reference()
    got = s.out.cpu().double()[:s.n, :8 * 64].reshape(s.n, 8, 64)
    nan = torch.isnan(want)
    assert nan.any() and not nan.all()
    assert torch.equal(torch.isnan(got), nan)
    clean = torch.tensor([i < 96 + at for i in range(70, 130)] + [False])
    assert ((got - want).abs() <= tol)[clean].all()


@pytest.mark.parametrize("lens", [(1, 3000), (40, 3000)], ids=["single", "chunk"])
@pytest.mark.parametrize("lo,hi", [(0, 128), (512, 1024), (0, 2950), (0, 3000)])
def test_attn_parts_whose_keys_are_all_nan_are_joined(lo, hi, lens):
    """Every row sees a NaN, also where a part of a divided unit holds nothing else."""
    torch = torch_()
    s = Setup([lens], 8, 1, 64, "f16", 16, seed=24)
    for j in range(lo, hi):
        s.k[int(s.table[s.order[0], j // 16]), :, j % 16] = float("nan")
    s.dk.copy_(s.k)
    s.attend()
    fb.attn_paged_status(s.ws.data_ptr())
    assert torch.isnan(s.out[:s.n, :8 * 64]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("window", [0, 25])
def test_attn_same_bits_again(window, dtype):
    """Two tiles of queries share each unit's K and V, whose first and last rows neither sees."""
    torch = torch_()
    lens = [(700, 1500), (333, 333), (90, 2000), (1, 3000)] * 3
    s = Setup(lens, 64, 4, 64, dtype, 32, window=window, seed=23, fill=float("nan"))
    s.attend()
    first = s.out.clone()
    assert torch.isfinite(first).all()
    for _ in range(60):
        s.attend()
        assert torch.equal(s.out, first)
    fb.attn_paged_status(s.ws.data_ptr())


@pytest.mark.parametrize("bad", [-1, 1 << 30])
def test_attn_table_entries_outside_the_pool_read_as_zeros(bad):
    torch = torch_()
    s = Setup([(1, 200), (70, 200)], 4, 2, 64, "f16", 64, seed=4, slots="own")
    for q in range(2):
        page = int(s.table[q, 1])
        s.k[page] = 0
        s.v[page] = 0
    s.dtab[:, 1] = bad
    s.attend()
    torch.cuda.synchronize()
    s.check()


def test_attn_slot_or_length_outside_the_table_gives_zeros():
    torch = torch_()
    s = Setup([(1, 10), (3, 30), (2, 20), (1, 12)], 2, 2, 64, seed=6)
    s.dslot[0] = 99
    s.dslot[1] = -1
    s.dlen[2] = 64 * s.max_pages + 1
    s.attend()
    torch.cuda.synchronize()
    got = s.out.cpu()[:, :128]
    assert (got[:6] == 0).all() and not (got[6] == 0).any()


@pytest.mark.parametrize("lens", [[(1, 4000)], [(1, 37), (1, 9001)], [(3, 2500)] * 2, [(40, 3000)], [(700, 1500), (1, 3000)],
                                  [(300, 300)]], ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 1, 128), (4, 4, 64)])
def test_attn_long_contexts_are_split_and_joined(lens, heads, kv_heads, dim):
    torch = torch_()
    s = Setup(lens, heads, kv_heads, dim, "f16", 32, seed=len(lens))
    s.attend()
    torch.cuda.synchronize()
    first = s.out.clone()
    for _ in range(3):  # the workspace is ready for the next call, and the bits do not change
        s.out.fill_(7.0)
        s.attend()
    torch.cuda.synchronize()
    assert torch.equal(first, s.out)
    big_reference(s)


def big_reference(s):
    """reference() in batched products, for longer contexts."""
    torch = torch_()
    fb.attn_paged_status(s.ws.data_ptr())
    G, u = s.H // s.KV, U[s.dtype]
    got = s.out.double()
    for q, (n, kv) in enumerate(s.lens):
        k, v = s.cached(s.k, q).cuda(), s.cached(s.v, q).cuda()
        pos = torch.arange(n, device="cuda")[:, None] + kv - n
        key = torch.arange(kv, device="cuda")[None]
        seen = (key <= pos) & ((key > pos - s.window) if s.window else True)
        for h in range(s.H):
            x = s.dq[s.starts[q]:s.starts[q] + n, h * s.D:(h + 1) * s.D].double()
            big = float((x.abs() @ k[:, h // G].abs().T).max()) * s.scale
            sc = torch.where(seen, x @ k[:, h // G].T * s.scale, -math.inf)
            p = torch.softmax(sc, 1)
            o, w = p @ v[:, h // G], p @ v[:, h // G].abs()
            tol = 1.05 * u * (o.abs() + w) + w * (2.0 ** -16 * big + 2.0 ** -15) + 2.0 ** -25 * (kv * float(v.abs().max()) + 1)
            err = (got[s.starts[q]:s.starts[q] + n, h * s.D:(h + 1) * s.D] - o).abs()
            assert (err <= tol).all(), (q, h, float((err / tol).max()))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("nq", [1, 50])
def test_attn_rising_and_falling_scores(nq, dtype):
    """Row maxima that keep rising along the keys (every tile rescales) and that come first."""
    torch = torch_()
    for sign in (1.0, -1.0):
        s = Setup([(nq, 900)], 2, 1, 64, dtype, seed=1)
        ramp = torch.linspace(0.0, 30.0 * sign, 900)
        pages = s.table[s.order[0], :-(-900 // 64)].long()
        for j in range(900):
            s.k[pages[j // 64], 0, j % 64, 0] = ramp[j]
        s.q[:, 0] = 6.0
        s.q[:, 64] = 9.0
        s.dk.copy_(s.k)
        s.dq.copy_(s.q)
        s.attend()
        big_reference(s)


def test_attn_many_sequences():
    """More sequences than one launch takes."""
    rng = np.random.default_rng(0)
    lens = [(int(rng.integers(0, 4)), int(rng.integers(0, 90))) for _ in range(300)]
    s = Setup(lens, 2, 1, 64, "f16", 16, seed=5)
    s.attend()
    s.check()


def test_attn_offsets_beyond_32_bits():
    """Pages far apart: element offsets above 2^32 in both pools."""
    torch = torch_()
    P, KV, D, pages = 64, 2, 64, 3
    stride = (1 << 31) + 64  # page 2 starts beyond 2^32 elements
    pool = torch.empty(2 * stride + KV * P * D, dtype=torch.float16, device="cuda")
    s = Setup([(1, 150), (20, 150)], 4, KV, D, "f16", P, seed=2, spare=0, slots="own")
    assert s.n_pages == 6
    # both sequences share the three far pages
    k, v = s.k[:3].clone(), s.v[:3].clone()
    for i in range(pages):
        pool[i * stride:i * stride + KV * P * D] = k[i].reshape(-1).cuda()
    vpool = torch.empty_like(pool)
    for i in range(pages):
        vpool[i * stride:i * stride + KV * P * D] = v[i].reshape(-1).cuda()
    s.table[:, :3] = torch.tensor([2, 0, 1], dtype=torch.int32)
    s.dtab.copy_(s.table)
    s.view = fb.PagedKV(pool.data_ptr(), vpool.data_ptr(), s.dtab.data_ptr(), n_slots=2, max_pages=3, n_pages=3, page_size=P,
                        n_kv_heads=KV, head_dim=D, page_stride=stride)
    s.attend()
    torch.cuda.synchronize()
    s.check()
    # and the append stores there
    b = fb.RaggedBatch(s.dstart.data_ptr(), s.dlen.data_ptr(), n_seqs=2, n_tokens=21, max_q=20)
    kv = torch.randn(21, 2 * KV * D, dtype=torch.float16, device="cuda")
    fb.kv_append(s.view, b, 1, None, kv.data_ptr(), kv.data_ptr() + 2 * KV * D, ld=2 * KV * D)
    torch.cuda.synchronize()
    for i in range(19):  # sequence 1, positions 130 .. 148 (149 is sequence 0's too)
        for far, part in ((pool, kv[1 + i, :KV * D]), (vpool, kv[1 + i, KV * D:])):
            row = far[stride:stride + KV * P * D].reshape(KV, P, D)[:, 130 - 128 + i]
            assert torch.equal(row, part.reshape(KV, D))


def test_attn_on_another_stream_and_in_a_graph():
    """A captured call follows lengths that change on the device."""
    torch = torch_()
    s = Setup([(1, 40), (1, 130)], 4, 2, 64, seed=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.attend(stream=side)
    side.synchronize()
    s.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.attend(stream=torch.cuda.current_stream())
    for lens in ([(1, 33), (1, 129)], [(1, 1), (1, 64)], [(1, 40), (1, 128)]):
        s.lens = lens
        s.dlen.copy_(torch.tensor([kv for _, kv in lens], dtype=torch.int32))
        s.out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        s.check()


# ---- append ------------------------------------------------------------------------------


def rope_table(max_pos, dim):
    torch = torch_()
    ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * torch.arange(dim // 2) / dim)
    return torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()


def turned(x, table, rot, adjacent):
    """[n, heads, D] in 64 bits -> (rotated, |a| + |b| of each value's pair)."""
    torch = torch_()
    y, mag = x.clone(), x.abs()
    c, s = table[:, None, :, 0], table[:, None, :, 1]
    i0, i1 = (slice(0, rot, 2), slice(1, rot, 2)) if adjacent else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, a * s + b * c
    mag[..., i0] = mag[..., i1] = a.abs() + b.abs()
    return y, mag


@pytest.mark.parametrize("lens", [SINGLES, CHUNKS, EMPTY, [(1, 30)] * 70], ids=["singles", "chunks", "empty", "many"])
@pytest.mark.parametrize("in_type,dtype,dim,rot,adjacent,page,layout,heads,kv_heads", [
    ("f32", "f16", 64, 64, False, 64, "heads", 8, 2), ("f32", "bf16", 128, 64, True, 16, "positions", 3, 3),
    ("same", "f16", 128, 128, True, 32, "heads", 5, 1), ("same", "bf16", 64, 16, False, 256, "positions", 32, 4),
    ("f32", "f16", 128, 0, False, 128, "positions", 4, 2), ("same", "f16", 64, 64, False, 64, "heads", 0, 2)])
def test_append(lens, in_type, dtype, dim, rot, adjacent, page, layout, heads, kv_heads):
    torch = torch_()
    s = Setup(lens, max(heads, 1) * kv_heads, kv_heads, dim, dtype, page, layout, seed=rot + page)
    it = torch.float32 if in_type == "f32" else s.dt
    width = (heads + 2 * kv_heads) * dim + 8
    x = torch.randn(s.rows, width, generator=torch.Generator().manual_seed(1)).to(it)
    dx = x.cuda()
    table = rope_table(max(2, max(kv for _, kv in lens)), rot or 16)
    dt = table.cuda()
    q_out = torch.full((s.rows, heads * dim + 8), 7.0, dtype=s.dt, device="cuda")
    size = x.element_size()
    fb.kv_append(s.view, s.batch, 0 if in_type == "f32" else {"f16": 1, "bf16": 30}[dtype],
                 dx.data_ptr() if heads else None, dx.data_ptr() + heads * dim * size,
                 dx.data_ptr() + (heads + kv_heads) * dim * size, ld=width, n_heads=heads,
                 q_out=q_out.data_ptr() if heads else None, ld_out=heads * dim + 8,
                 rope=fb.Rope(dt.data_ptr(), max_pos=len(table), dim=rot, adjacent=adjacent) if rot else None)
    torch.cuda.synchronize()
    u, tiny = U[dtype], 2.0 ** -25
    want_k, want_v = s.k.double(), s.v.double()
    tol_k = torch.zeros_like(want_k)
    tol_v = torch.zeros_like(want_v)
    want_q = torch.zeros(s.n, heads, dim, dtype=torch.float64)
    tol_q = torch.zeros_like(want_q)
    for q, (n, kv) in enumerate(lens):
        for i in range(n):
            pos, row = kv - n + i, x[s.starts[q] + i].double()
            if pos < 0:
                continue
            parts = row[:(heads + 2 * kv_heads) * dim].reshape(1, -1, dim)
            y, mag = turned(parts[:, :heads + kv_heads], table[pos:pos + 1].double(), rot, adjacent) if rot else \
                (parts[:, :heads + kv_heads], parts[:, :heads + kv_heads].abs())
            t = u * y.abs() + 3 * 2.0 ** -24 * mag + tiny
            want_q[s.starts[q] + i], tol_q[s.starts[q] + i] = y[0, :heads], t[0, :heads]
            page_, at = int(s.table[s.order[q], pos // page]), pos % page
            where = (page_, slice(None), at) if layout == "heads" else (page_, at)
            want_k[where], tol_k[where] = y[0, heads:], t[0, heads:]
            v = parts[0, heads + kv_heads:]
            want_v[where], tol_v[where] = v, u * v.abs() + tiny
    assert ((s.dk.cpu().double() - want_k).abs() <= tol_k).all()
    assert ((s.dv.cpu().double() - want_v).abs() <= tol_v).all()
    got = q_out.cpu().double()
    if heads:
        assert ((got[:s.n, :heads * dim].reshape(s.n, heads, dim) - want_q).abs() <= tol_q).all()
    assert (got[s.n:] == 7.0).all() and (got[:, heads * dim:] == 7.0).all()


def test_append_leaves_bad_places_alone():
    """Slots, lengths, table entries and rotary positions outside their ranges: nothing stored, queries zero."""
    torch = torch_()
    s = Setup([(1, 10), (1, 20), (1, 30), (1, 40), (2, 60)], 2, 2, 64, seed=6)
    s.dslot[0] = 99
    s.dlen[1] = 64 * s.max_pages + 1
    s.dtab[s.order[2], 0] = s.n_pages
    s.dtab[s.order[3], 0] = -7
    table = rope_table(59, 64).cuda()  # position 59, the last sequence's second token, lies beyond
    x = torch.randn(s.rows, 6 * 64, device="cuda")
    q = torch.full((s.rows, 128), 7.0, dtype=torch.float16, device="cuda")
    fb.kv_append(s.view, s.batch, 0, x.data_ptr(), x.data_ptr() + 512, x.data_ptr() + 1024, ld=6 * 64, n_heads=2,
                 q_out=q.data_ptr(), ld_out=128, rope=fb.Rope(table.data_ptr(), max_pos=59, dim=64))
    torch.cuda.synchronize()
    diff = (s.dk.cpu() != s.k).any(-1).any(1)
    page = int(s.table[s.order[4], 0])
    assert diff.sum() == 1 and diff[page, 58]
    z = (q.cpu() == 0).all(1).tolist()
    assert z[:6] == [True, True, False, False, False, True] and (q.cpu()[6:] == 7.0).all()


def test_append_in_place_queries():
    torch = torch_()
    s = Setup([(3, 30), (1, 5)], 4, 2, 64, seed=2)
    x = torch.randn(s.rows, 8 * 64, device="cuda").half()
    table = rope_table(64, 64).cuda()
    rope = fb.Rope(table.data_ptr(), max_pos=64, dim=64)
    out = torch.zeros(s.rows, 256, dtype=torch.float16, device="cuda")
    args = dict(ld=512, n_heads=4, rope=rope)
    fb.kv_append(s.view, s.batch, 1, x.data_ptr(), x.data_ptr() + 512, x.data_ptr() + 768, q_out=out.data_ptr(), ld_out=256,
                 **args)
    fb.kv_append(s.view, s.batch, 1, x.data_ptr(), x.data_ptr() + 512, x.data_ptr() + 768, q_out=x.data_ptr(), ld_out=512,
                 **args)
    torch.cuda.synchronize()
    assert torch.equal(x[:s.n, :256], out[:s.n])


def test_append_then_attend_equals_the_cache_class():
    """Through a KVCache's layer view: what kv_append stores is what KVCache.read returns and attn_paged sees."""
    torch = torch_()
    cache = fb.KVCache(0, 3, 2, 64, 200, max_batch=4)
    view = fb.kv_view(cache, 1)
    assert (view.page_size, view.n_slots, view.head_dim, view.n_kv_heads) == (64, 4, 64, 2)
    lens, slots = [(70, 70), (1, 1), (100, 100)], [3, 0, 2]
    start = torch.tensor([0, 70, 71, 171], dtype=torch.int32, device="cuda")
    klen = torch.tensor([70, 1, 100], dtype=torch.int32, device="cuda")
    slot = torch.tensor(slots, dtype=torch.int32, device="cuda")
    batch = fb.RaggedBatch(start.data_ptr(), klen.data_ptr(), n_seqs=3, n_tokens=171, max_q=100, slot=slot.data_ptr())
    x = torch.randn(171, (4 + 2 + 2) * 64, device="cuda")
    q = torch.empty(171, 256, dtype=torch.float16, device="cuda")
    fb.kv_append(view, batch, 0, x.data_ptr(), x.data_ptr() + 1024, x.data_ptr() + 1536, ld=512, n_heads=4, q_out=q.data_ptr(),
                 ld_out=256)
    torch.cuda.synchronize()
    for (n, _), sl, at in zip(lens, slots, [0, 70, 71]):
        k, v = cache.read(1, 0, n, slot=sl)
        assert np.array_equal(k, x[at:at + n, 256:384].half().float().cpu().numpy())
        assert np.array_equal(v, x[at:at + n, 384:].half().float().cpu().numpy())
        assert not cache.read(0, 0, n, slot=sl)[0].any() and not cache.read(2, 0, n, slot=sl)[1].any()
    ws = torch.zeros(fb.attn_paged_workspace(view, batch, 4), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    fb.attn_paged(view, batch, q.data_ptr(), out.data_ptr(), n_heads=4, ldq=256, ldo=256, scale=0.125, ws=ws.data_ptr(),
                  ws_bytes=ws.numel())
    torch.cuda.synchronize()
    for (n, _), at in zip(lens, [0, 70, 71]):
        h = x[at:at + n].half().double().reshape(n, 8, 64)
        for head in range(4):
            sc = h[:, head] @ h[:, 4 + head // 2].T * 0.125
            sc = sc.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf)
            v = h[:, 6 + head // 2]
            p = torch.softmax(sc, 1)
            tol = 1.05 * U["f16"] * ((p @ v).abs() + p @ v.abs()) + (p @ v.abs()) * (2.0 ** -16 * 40 + 2.0 ** -15) + 2.0 ** -25 * (6 * n + 1)
            assert ((out[at:at + n, head * 64:(head + 1) * 64].double() - p @ v).abs() <= tol).all()


# ---- rows that are computed again ------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,lens,window", [
    (4, 1, [(3, 3000)], 0), (8, 1, [(40, 3000)], 0), (4, 1, [(3, 3000), (2, 700)], 500),
    (8, 2, [(300, 2500), (1, 60), (20, 900)], 0), (6, 6, [(2, 40)] * 90, 0)], ids=str)
def test_attn_rows_computed_again_in_cut_and_whole_units(heads, kv_heads, lens, window, dim, dtype):
    """The last token's value is infinite: every earlier row of its tile is computed again, by whichever
    CTA wrote it, and only the last token's row sees it."""
    torch = torch_()
    s = Setup(lens, heads, kv_heads, dim, dtype, 16, window=window, seed=31)
    last = []
    for q, (n, kv) in enumerate(lens):
        s.v[int(s.table[s.order[q], (kv - 1) // 16]), :, (kv - 1) % 16] = float("inf")
        last.append(s.starts[q] + n - 1)
    s.dv.copy_(s.v)
    s.attend()
    fb.attn_paged_status(s.ws.data_ptr())
    first = s.out.clone()
    for _ in range(3):
        s.out.fill_(7.0)
        s.attend()
        assert torch.equal(s.out, first)
    got = first[:s.n, :heads * dim].double().reshape(s.n, heads, dim)
    assert (got[last] == float("inf")).all()
    G, u = heads // kv_heads, U[dtype]
    for q, (n, kv) in enumerate(lens):
        k, v = s.cached(s.k, q).cuda(), s.cached(s.v, q).cuda()
        v[kv - 1] = 0.0
        pos = torch.arange(n - 1, device="cuda")[:, None] + kv - n
        key = torch.arange(kv, device="cuda")[None]
        seen = (key <= pos) & ((key > pos - window) if window else True)
        for h in range(heads):
            x = s.dq[s.starts[q]:s.starts[q] + n - 1, h * dim:(h + 1) * dim].double()
            if n == 1:
                continue
            big = float((x.abs() @ k[:, h // G].abs().T).max()) * s.scale
            p = torch.softmax(torch.where(seen, x @ k[:, h // G].T * s.scale, -math.inf), 1)
            o, w = p @ v[:, h // G], p @ v[:, h // G].abs()
            tol = 1.05 * u * (o.abs() + w) + w * (2.0 ** -16 * big + 2.0 ** -15) + 2.0 ** -25 * (kv * float(v.abs().max()) + 1)
            err = (got[s.starts[q]:s.starts[q] + n - 1, h] - o).abs()
            assert (err <= tol).all(), (q, h, float((err / tol).max()))


def test_attn_long_rows_computed_again_hold_nobody_up():
    """256 rows over 160,000 positions of which the first holds a NaN value that they see, in front of clean
    units of the same CTA: the clean rows keep their bits and no wait gives up."""
    torch = torch_()
    P, KV, G, D, kv, n = 256, 8, 16, 64, 160_000, 16  # a unit is 16 tokens of 16 heads
    H, pages = KV * G, -(-kv // P)
    n_seqs = -(-2 * torch.cuda.get_device_properties(0).multi_processor_count // KV)  # two units a CTA
    gen = torch.Generator(device="cuda")
    gen.manual_seed(17)
    # every sequence reads the same pages, the first one with a first page of its own
    pools = [torch.randn(pages + 1, KV, P, D, generator=gen, device="cuda").bfloat16() for _ in range(2)]
    for p in pools:
        p[pages] = p[0]
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(n_seqs, 1)
    table[0, 0] = pages
    q = torch.randn(n_seqs * n, H * D, generator=gen, device="cuda").bfloat16()
    out = torch.zeros_like(q)
    start = torch.arange(n_seqs + 1, dtype=torch.int32, device="cuda") * n
    lens = torch.full((n_seqs,), kv, dtype=torch.int32, device="cuda")
    view = fb.PagedKV(pools[0].data_ptr(), pools[1].data_ptr(), table.data_ptr(), n_slots=n_seqs, max_pages=pages,
                      n_pages=pages + 1, page_size=P, n_kv_heads=KV, head_dim=D, dtype=30)
    batch = fb.RaggedBatch(start.data_ptr(), lens.data_ptr(), n_seqs=n_seqs, n_tokens=n_seqs * n, max_q=n)
    ws = torch.zeros(fb.attn_paged_workspace(view, batch, H), dtype=torch.uint8, device="cuda")

    def attend():
        fb.attn_paged(view, batch, q.data_ptr(), out.data_ptr(), n_heads=H, ldq=H * D, ldo=H * D, scale=0.125,
                      ws=ws.data_ptr(), ws_bytes=ws.numel())
        fb.attn_paged_status(ws.data_ptr())
        return out.clone()

    clean = attend()
    assert torch.isfinite(clean).all()
    pools[1][pages, 0, 0, 3] = float("nan")  # KV head 0 of the first sequence
    got = attend()
    hit = torch.zeros(n_seqs * n, H, dtype=torch.bool, device="cuda")
    hit[:n, :G] = True
    got, clean = got.reshape(-1, H, D), clean.reshape(-1, H, D)
    assert torch.equal(got[~hit], clean[~hit])
    assert torch.isnan(got[:n, :G, 3]).all()
    others = [d for d in range(D) if d != 3]
    k, v = (p[table[0].long(), 0].reshape(-1, D)[:kv].double() for p in pools)
    v[0, 3] = 0.0
    seen = torch.arange(kv, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] + kv - n
    for h in range(G):
        x = q[:n, h * D:(h + 1) * D].double()
        big = float((x.abs() @ k.abs().T).max()) * 0.125
        p = torch.softmax(torch.where(seen, x @ k.T * 0.125, -math.inf), 1)
        o, w = p @ v, p @ v.abs()
        tol = 1.05 * U["bf16"] * (o.abs() + w) + w * (2.0 ** -16 * big + 2.0 ** -15)
        assert ((got[:n, h].double() - o).abs() <= tol)[:, others].all()
    # a key that is NaN: the rows that see it are NaN at once
    pools[1][pages, 0, 0, 3] = 0.0
    pools[0][pages, 0, 0, 3] = float("nan")
    got = attend().reshape(-1, H, D)
    assert torch.isnan(got[:n, :G]).all() and torch.equal(got[~hit], clean[~hit])


# ---- waits that give up ----------------------------------------------------------------------


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nq", [1, 40], ids=["rows", "tile"])
def test_attn_waits_that_give_up_are_reported_and_the_workspace_serves_again(nq, dim):
    torch = torch_()
    lens = [(nq, 3000)] * 64 + [(1, 70)]  # some 2,000 positions and more per SM, one head each
    s = Setup(lens, 8, 2, dim, "f16", 64, seed=41)
    s.attend()
    fb.attn_paged_status(s.ws.data_ptr())
    first = s.out.clone()
    assert torch.isfinite(first).all()
    fb.attn_paged_drill(True)
    try:
        s.attend()
        with pytest.raises(fb.FiberError, match="gave up"):
            fb.attn_paged_status(s.ws.data_ptr())
        with pytest.raises(fb.FiberError, match="status -5"):  # it stays until the workspace is cleared
            fb.attn_paged_status(s.ws.data_ptr())
    finally:
        fb.attn_paged_drill(False)
    s.ws.zero_()
    for _ in range(2):
        s.out.fill_(7.0)
        s.attend()
        fb.attn_paged_status(s.ws.data_ptr())
        assert torch.equal(s.out, first)


# ---- many small weights ------------------------------------------------------------------------


@pytest.mark.parametrize("group", [1, 24], ids=["rows", "tile"])
@pytest.mark.parametrize("at", [0, 70_001, 131_071])
@pytest.mark.parametrize("below", [17.5, 18.75])
def test_attn_small_weights_of_many_keys_are_not_lost(below, at, group):
    """One key, of value 0, `below` nats above 131,071 others, of value 1: each weighs less than 2^-25 of it,
    together 0.1 to 0.3 percent. Beyond the general bound's terms a weight may be off by 2^-31 of the largest.
    128 sequences of 3 KV heads share the pages: more units than CTAs, so that most are not cut."""
    torch = torch_()
    kv, P, D, KV, S = 131_072, 256, 64, 3, 128
    H = KV * group
    k = torch.zeros(kv // P, KV, P, D, dtype=torch.float16, device="cuda")
    v = torch.ones_like(k)
    k[at // P, :, at % P, 0] = 16.0
    v[at // P, :, at % P] = 0.0
    q = torch.zeros(S, H * D, dtype=torch.float16, device="cuda")
    q[:, ::D] = below / 2  # scores 16 * below / 2 * 0.125 = below, and 0: exact
    out = torch.zeros_like(q)
    start = torch.arange(S + 1, dtype=torch.int32, device="cuda")
    lens = torch.full((S,), kv, dtype=torch.int32, device="cuda")
    table = torch.arange(kv // P, dtype=torch.int32, device="cuda").repeat(S, 1)
    view = fb.PagedKV(k.data_ptr(), v.data_ptr(), table.data_ptr(), n_slots=S, max_pages=kv // P, n_pages=kv // P,
                      page_size=P, n_kv_heads=KV, head_dim=D)
    batch = fb.RaggedBatch(start.data_ptr(), lens.data_ptr(), n_seqs=S, n_tokens=S, max_q=1)
    ws = torch.zeros(fb.attn_paged_workspace(view, batch, H), dtype=torch.uint8, device="cuda")
    fb.attn_paged(view, batch, q.data_ptr(), out.data_ptr(), n_heads=H, ldq=H * D, ldo=H * D, scale=0.125,
                  ws=ws.data_ptr(), ws_bytes=ws.numel())
    fb.attn_paged_status(ws.data_ptr())
    small = (kv - 1) * math.exp(-below)
    want = small / (1.0 + small)
    tol = 1.05 * U["f16"] * 2 * want + want * (2.0 ** -16 * below + 2.0 ** -15) + 2.0 ** -31 * kv
    assert float((out.double() - want).abs().max()) <= tol


# ---- large batches -----------------------------------------------------------------------------


def test_attn_131072_tokens_over_their_own_positions():
    """Eight query heads over one KV head, whose table has room for 2^20 positions."""
    torch = torch_()
    n, P, D, H = 131_072, 64, 64, 8
    g = torch.Generator(device="cuda")
    g.manual_seed(51)
    pools = [torch.randn(n // P, 1, P, D, generator=g, device="cuda").bfloat16() for _ in range(2)]
    table = torch.full(((1 << 20) // P,), -1, dtype=torch.int32, device="cuda")
    table[:n // P] = torch.randperm(n // P, generator=torch.Generator().manual_seed(1)).int().cuda()
    q = torch.randn(n, H * D, generator=g, device="cuda").bfloat16()
    out = torch.zeros_like(q)
    start = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    view = fb.PagedKV(pools[0].data_ptr(), pools[1].data_ptr(), table.data_ptr(), n_slots=1, max_pages=(1 << 20) // P,
                      n_pages=n // P, page_size=P, n_kv_heads=1, head_dim=D, dtype=30)
    batch = fb.RaggedBatch(start.data_ptr(), start.data_ptr() + 4, n_seqs=1, n_tokens=n, max_q=n)
    ws = torch.zeros(fb.attn_paged_workspace(view, batch, H), dtype=torch.uint8, device="cuda")
    fb.attn_paged(view, batch, q.data_ptr(), out.data_ptr(), n_heads=H, ldq=H * D, ldo=H * D, scale=0.125, ws=ws.data_ptr(),
                  ws_bytes=ws.numel())
    fb.attn_paged_status(ws.data_ptr())
    k, v = (p[table[:n // P].long()].reshape(-1, D).double() for p in pools)
    rows = torch.tensor([0, 1, 31, 32, 127, 128, 4095, 65_535, 65_536, 100_000, 131_040, 131_071], device="cuda")
    seen = torch.arange(n, device="cuda")[None] <= rows[:, None]
    for h in range(H):
        x = q[rows, h * D:(h + 1) * D].double()
        big = float((x.abs() @ k.abs().T).max()) * 0.125
        p = torch.softmax(torch.where(seen, x @ k.T * 0.125, -math.inf), 1)
        o, w = p @ v, p @ v.abs()
        tol = 1.05 * U["bf16"] * (o.abs() + w) + w * (2.0 ** -16 * big + 2.0 ** -15)
        assert ((out[rows, h * D:(h + 1) * D].double() - o).abs() <= tol).all()


# ---- sequences that overlap ------------------------------------------------------------------


@pytest.mark.parametrize("n_seqs", [3, 40, 140])
@pytest.mark.parametrize("nq", [2, 30], ids=["rows", "tile"])
def test_attn_decreasing_q_start_is_reported_and_nothing_is_written(nq, n_seqs):
    torch = torch_()
    s = Setup([(nq, 50)] * n_seqs, 2, 1, 64, "f16", 16, seed=61)
    s.attend()
    s.check()
    good = s.out.clone()
    start = s.dstart.clone()
    s.dstart[2] = 1
    s.out.fill_(7.0)
    s.attend()
    with pytest.raises(fb.FiberError, match="q_start decreases"):
        fb.attn_paged_status(s.ws.data_ptr())
    last = s.starts[128] if n_seqs > 128 else s.n  # a launch takes 128 sequences
    assert (s.out[:last] == 7.0).all() and torch.equal(s.out[last:], good[last:])
    s.ws.zero_()
    s.dstart.copy_(start)
    s.attend()
    s.check()


# ---- many sequences in the tile kernel ---------------------------------------------------------


@pytest.mark.parametrize("window", [0, 37])
@pytest.mark.parametrize("dim,dtype,n_seqs", [(64, "f16", 40), (128, "bf16", 40), (64, "bf16", 150), (128, "f16", 150)])
def test_attn_chunks_of_many_sequences(n_seqs, dim, dtype, window):
    """More sequences than a warp has lanes, and than a launch takes: chunks, single tokens and absences, a few
    sequences of many units."""
    rng = np.random.default_rng(n_seqs + window)
    lens = []
    for i in range(n_seqs):
        n = int(rng.choice([0, 1, 1, 5, 17, 40]))
        lens.append((n, n + int(rng.integers(0, 120))))
    lens[3], lens[n_seqs - 2] = (300, 420), (0, 0)
    s = Setup(lens, 6, 2, dim, dtype, 16, window=window, seed=n_seqs)
    for _ in range(2):  # the launches of a call share the workspace
        s.out.fill_(7.0)
        s.attend()
    s.check()
