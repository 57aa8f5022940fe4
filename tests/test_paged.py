"""Argument checks of the operators over the paged cache (no GPU work is reached)."""
from __future__ import annotations

import ctypes as C

import pytest

import fiber_b200 as fb

A = 1 << 20  # an address that is never used


def view(**kw):
    a = dict(k_pool=A, v_pool=A, page_table=A, n_slots=2, max_pages=4, n_pages=8, page_size=64, n_kv_heads=2, head_dim=64,
             dtype=1)
    a.update(kw)
    return fb.PagedKV(a.pop("k_pool"), a.pop("v_pool"), a.pop("page_table"), **a)


def batch(**kw):
    a = dict(n_seqs=1, n_tokens=4, max_q=4)
    a.update(kw)
    return fb.RaggedBatch(a.pop("q_start", A), a.pop("kv_len", A), **a)


def attend(kv=None, b=None, **kw):
    a = dict(q=A, out=A, n_heads=4, ldq=256, ldo=256, scale=0.125, ws=A, ws_bytes=1 << 40)
    a.update(kw)
    fb.attn_paged(kv or view(), b or batch(), a.pop("q"), a.pop("out"), **a)


def append(kv=None, b=None, in_type=0, **kw):
    a = dict(q=A, k=A, v=A, ld=512, n_heads=4, q_out=A, ld_out=256)
    a.update(kw)
    fb.kv_append(kv or view(), b or batch(), in_type, a.pop("q"), a.pop("k"), a.pop("v"), **a)


BAD_VIEWS = [dict(dtype=0), dict(dtype=12), dict(head_dim=96), dict(head_dim=32), dict(page_size=8), dict(page_size=48),
             dict(page_size=512), dict(n_pages=0), dict(n_slots=0), dict(max_pages=0), dict(n_kv_heads=0),
             dict(k_pool=A + 2), dict(v_pool=A + 8), dict(k_pool=0), dict(page_table=0), dict(pos_stride=63),
             dict(pos_stride=68), dict(head_stride=60), dict(page_stride=-64), dict(page_stride=1 << 40),
             dict(max_pages=1 << 26, page_size=64)]


@pytest.mark.parametrize("bad", BAD_VIEWS)
def test_both_refuse_a_bad_view(bad):
    for f in (attend, append):
        with pytest.raises(fb.FiberError, match="status -1"):
            f(kv=view(**bad))


@pytest.mark.parametrize("bad", [dict(n_seqs=-1), dict(n_tokens=-1), dict(q_start=0), dict(kv_len=0)])
def test_both_refuse_a_bad_batch(bad):
    for f in (attend, append):
        with pytest.raises(fb.FiberError, match="status -1"):
            f(b=batch(**bad))


@pytest.mark.parametrize("bad", [dict(n_heads=3), dict(n_heads=0), dict(n_heads=2 * 129, ldq=1 << 15, ldo=1 << 15),
                                 dict(q=0), dict(q=A + 4), dict(out=0), dict(out=A + 8), dict(ldq=248), dict(ldq=260),
                                 dict(ldo=255), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
                                 dict(scale=float("nan")), dict(window=-1), dict(ws=0), dict(ws=A + 4), dict(ws_bytes=0)])
def test_attn_refusals(bad):
    with pytest.raises(fb.FiberError, match="status -1"):
        attend(**bad)


def test_attn_refuses_max_q_below_one_and_counts_beyond_32_bits():
    with pytest.raises(fb.FiberError, match="max_q"):
        attend(b=batch(max_q=0))
    with pytest.raises(fb.FiberError, match="too large"):
        attend(kv=view(max_pages=1 << 24, n_kv_heads=8), b=batch(n_tokens=1 << 20), n_heads=64, ldq=4096, ldo=4096)


@pytest.mark.parametrize("bad", [dict(in_type=30), dict(in_type=12), dict(q=None), dict(q_out=None), dict(n_heads=0),
                                 dict(k=0), dict(v=0), dict(q=A + 8), dict(k=A + 4), dict(ld=120), dict(ld=514),
                                 dict(ld_out=128), dict(ld_out=260)])
def test_append_refusals(bad):
    with pytest.raises(fb.FiberError, match="status -1"):
        append(**bad)


@pytest.mark.parametrize("bad", [dict(table=0), dict(table=A + 8), dict(max_pos=0), dict(dim=0), dict(dim=24), dict(dim=128)])
def test_append_refuses_a_bad_rope(bad):
    a = dict(table=A, max_pos=16, dim=64)
    a.update(bad)
    with pytest.raises(fb.FiberError, match="rope"):
        append(rope=fb.Rope(a.pop("table"), **a))


def test_null_structs_and_empty_batches():
    L = fb.cuda_lib()
    append(b=batch(n_seqs=0))  # nothing to do: no launch
    attend(b=batch(n_tokens=0))
    assert L.fiber_attn_paged_status(None, None) == -1
    assert L.fiber_kv_view(None, 0, None) == -1
    assert L.fiber_kv_append(None, None, 0, None, 0, None, 0, None, 0, 0, None, None, 0, None) == -1
    assert L.fiber_attn_paged(None, None, None, 0, None, 0, 0, C.c_float(1.0), 0, None, 0, None) == -1
    with pytest.raises(fb.FiberError):
        fb.attn_paged_workspace(view(head_dim=96), batch(), 4)


@pytest.mark.parametrize("positions,tokens,seqs,max_q", [
    (131_072, 131_072, 1, 131_072), (1 << 20, 16_384, 32, 512), (1 << 20, 131_072, 1, 131_072), (1 << 20, 4096, 4096, 1)])
def test_large_batches_that_the_count_has_room_for_are_taken(positions, tokens, seqs, max_q):
    """Of 64 query and 8 KV heads."""
    kv = view(page_size=64, max_pages=positions // 64, n_kv_heads=8)
    assert fb.attn_paged_workspace(kv, batch(n_seqs=seqs, n_tokens=tokens, max_q=max_q), 64) > 0


@pytest.mark.parametrize("positions,tokens,heads,kv_heads", [
    (1 << 24, 1 << 20, 64, 8), (1 << 20, 1 << 20, 64, 8), (16, 1 << 24, 128, 1), (64, 2 ** 31 - 1, 1, 1)])
def test_larger_ones_are_refused(positions, tokens, heads, kv_heads):
    kv = view(page_size=16, max_pages=positions // 16, n_kv_heads=kv_heads)
    for max_q in (1, tokens):
        with pytest.raises(fb.FiberError, match="too large"):
            fb.attn_paged_workspace(kv, batch(n_tokens=tokens, max_q=max_q), heads)


def test_attn_refuses_its_output_over_its_queries():
    with pytest.raises(fb.FiberError, match="same buffer"):
        attend(q=A, out=A)


@pytest.mark.parametrize("bad", [dict(in_type=0, ld_out=512), dict(in_type=1, ld_out=256), dict(in_type=1, ld_out=1024)])
def test_append_in_place_takes_one_type_and_one_stride(bad):
    with pytest.raises(fb.FiberError, match="in place"):
        append(**bad)


def test_slots_of_almost_2_to_the_31_positions():
    for f in (attend, append):
        with pytest.raises(fb.FiberError, match="2\\^31"):
            f(kv=view(page_size=16, max_pages=(1 << 27) - 15, n_kv_heads=1))
    assert fb.attn_paged_workspace(view(page_size=16, max_pages=(1 << 27) - 16, n_kv_heads=1), batch(), 4) > 0
