"""Prompt chunks and single tokens of several sequences in one pass (fiber_forward_ragged).

The pass appends and attends with the operators over the paged cache, whose queries,
probabilities and outputs are fp16: three roundings of 2^-11 in each of the 2 or 3 layers,
independent of one another, are sqrt(9) * 2^-11 = 1.5e-3 of the logits' size; the bar is twice
that (relative RMS), against the oracle with fp16 K/V. Greedy tokens are the oracle's wherever its
two best logits lie further apart than the pass may move them.
"""
from __future__ import annotations

import numpy as np
import pytest

import fiber_b200 as fb
from oracle import oracle as orc

pytestmark = pytest.mark.gpu

REL_RMS = 3e-3


def _oracle_logits(path, tokens):
    st = orc.Model(path).state(512, kv_fp16=True)
    out = None
    for i, t in enumerate(tokens):
        out = st.forward(int(t), i)
    return np.array(out, np.float64)


def _check(am, lg, i, want):
    err = lg[i].astype(np.float64) - want
    scale = np.sqrt(np.mean(want ** 2))
    assert np.sqrt(np.mean(err ** 2)) < REL_RMS * scale
    top = np.sort(want)[-2:]
    if top[1] - top[0] > 8 * REL_RMS * scale:
        assert int(am[i]) == int(np.argmax(want))


@pytest.mark.parametrize("name", ["q4km", "q5km", "f16", "gqa8", "hd128"])
def test_chunks_and_single_tokens_match_the_oracle(tiny_model, name):
    path = tiny_model(name)
    hm = fb.HostModel(path)
    ctx = fb.Context(hm, max_seq=400, max_batch=6)
    kv = ctx.kv(400, max_batch=6)
    rng = np.random.default_rng(5)
    seqs = [rng.integers(1, hm.params.vocab_size, n).astype(np.int32) for n in (150, 1, 33, 70, 260)]
    slots = [3, 0, 5, 1, 2]
    # one pass takes every sequence's first part; then chunks, single tokens and absences mix
    cuts = [[64, 1, 32, 17, 130], [65, 1, 33, 18, 200], [150, 1, 33, 70, 201], [150, 1, 33, 70, 260]]
    done = [0] * len(seqs)
    for cut in cuts:
        which = [i for i in range(len(seqs)) if cut[i] > done[i]]
        am, lg = ctx.forward_ragged(kv, [slots[i] for i in which], [done[i] for i in which],
                                    [seqs[i][done[i]:cut[i]] for i in which])
        for k, i in enumerate(which):
            _check(am, lg, k, _oracle_logits(path, seqs[i][:cut[i]]))
            done[i] = cut[i]


def test_cache_is_the_one_the_other_paths_read(tiny_model):
    """A prompt taken in through ragged passes decodes on as one prefilled in its slot."""
    path = tiny_model("q4km")
    hm = fb.HostModel(path)
    ctx = fb.Context(hm, max_seq=256, max_batch=2)
    kv, kv2 = ctx.kv(256, max_batch=2), ctx.kv(256, max_batch=2)
    prompt = np.random.default_rng(7).integers(1, hm.params.vocab_size, 90).astype(np.int32)
    first = ctx.prefill(kv, prompt, slot=0)
    ctx.prefill(kv, prompt, slot=1)
    ctx.forward_ragged(kv2, [1, 0], [0, 0], [prompt[:50], prompt[:89]], want_logits=False)
    am, _ = ctx.forward_ragged(kv2, [0, 1], [89, 50], [prompt[89:], prompt[50:]])
    k, v = kv.read(0, 0, 90, slot=0)
    for s in (0, 1):
        k2, v2 = kv2.read(0, 0, 90, slot=s)
        # layer 0: the same inputs; products summed in another order may move a rounding by one fp16 step
        assert (np.abs(k - k2) <= 2.0 ** -10 * np.abs(k) + 2.0 ** -20).all()
        assert (np.abs(v - v2) <= 2.0 ** -10 * np.abs(v) + 2.0 ** -20).all()
    assert am.tolist() == [first, first]
    a, _ = ctx.decode_greedy_batch(kv, [first, first], [90, 90], 8)
    b, _ = ctx.decode_greedy_batch(kv2, [first, first], [90, 90], 8)
    assert a[:, 0].tolist() == b[:, 0].tolist() == b[:, 1].tolist()


def test_refusals(tiny_model):
    hm = fb.HostModel(tiny_model("q4km"))
    ctx = fb.Context(hm, max_seq=128, max_batch=2)
    kv = ctx.kv(128, max_batch=2)
    V = hm.params.vocab_size
    for slots, start, chunks, why in [([0, 1, 0], [0, 0, 0], [[1], [1], [1]], "max_batch"), ([2], [0], [[1]], "no slot"),
                                      ([-1], [0], [[1]], "no slot"), ([1, 1], [0, 4], [[1], [1]], "twice"),
                                      ([0], [0], [[]], "tokens"), ([0], [-1], [[1]], "positions"),
                                      ([0], [100], [[1] * 29], "positions"), ([0], [0], [[1, V]], "out of range"),
                                      ([0], [0], [[1] * 513], "tokens")]:
        with pytest.raises(fb.FiberError, match=why):
            ctx.forward_ragged(kv, slots, start, chunks)
    am, _ = ctx.forward_ragged(kv, [1], [0], [[5, 6, 7]])
    assert 0 <= am[0] < V


def test_first_pass_does_not_depend_on_the_legacy_stream(tiny_model):
    """Work queued on the default stream, which the context's stream does not wait for, may run beside the
    first pass and after it: the pass's workspace is zeroed on the context's own stream."""
    import torch

    path = tiny_model("q4km")
    hm = fb.HostModel(path)
    rng = np.random.default_rng(11)
    chunks = [rng.integers(1, hm.params.vocab_size, n).astype(np.int32) for n in (200, 1, 90)]
    want = [_oracle_logits(path, c) for c in chunks]
    a = torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16)
    for _ in range(3):
        ctx = fb.Context(hm, max_seq=256, max_batch=3)
        kv = ctx.kv(256, max_batch=3)
        torch.cuda.synchronize()
        b = a
        for _ in range(40):
            b = a @ b
        for _ in range(2):
            am, lg = ctx.forward_ragged(kv, [2, 0, 1], [0, 0, 0], chunks)
            for i in range(3):
                _check(am, lg, i, want[i])
        torch.cuda.synchronize()
        ctx.close()


def test_a_pass_whose_waits_give_up_says_so_and_the_next_one_is_right(tiny_model):
    """64 single tokens at position 1,990 of a zero cache: long enough for the drill to end the attention."""
    hm = fb.HostModel(tiny_model("q4km"))
    ctx = fb.Context(hm, max_seq=2048, max_batch=64)
    kv = ctx.kv(2048, max_batch=64)
    prompt = np.random.default_rng(3).integers(1, hm.params.vocab_size, 40).astype(np.int32)
    greedy = ctx.prefill(kv, prompt, slot=0)
    toks = np.random.default_rng(2).integers(1, hm.params.vocab_size, 64).astype(np.int32)

    def step():
        return ctx.forward_ragged(kv, list(range(64)), [1990] * 64, [[t] for t in toks])

    am, lg = step()
    assert np.isfinite(lg).all()
    fb.attn_paged_drill(True)
    try:
        with pytest.raises(fb.FiberError, match="status -5"):
            step()
    finally:
        fb.attn_paged_drill(False)
    for _ in range(2):
        am2, lg2 = step()
        assert np.array_equal(am2, am) and np.array_equal(lg2, lg)
    assert ctx.prefill(kv, prompt, slot=0) == greedy


def _tp_worker(rank, world, nid, path, seqs, cuts, q):
    try:
        ctx = fb.Context(fb.HostModel(path), device=rank, max_seq=256, tp=(rank, world, nid), max_batch=3)
        kv = ctx.kv(256, max_batch=3)
        out, done = [], [0] * len(seqs)
        for cut in cuts:
            which = [i for i in range(len(seqs)) if cut[i] > done[i]]
            am, lg = ctx.forward_ragged(kv, which, [done[i] for i in which], [seqs[i][done[i]:cut[i]] for i in which])
            out.append((am, lg))
            done = list(cut)
        q.put((rank, out, None))
        ctx.close()
    except Exception as e:  # report instead of hanging the parent
        q.put((rank, None, repr(e)))


def test_two_ranks_match_the_oracle(tiny_model):
    import torch
    import torch.multiprocessing as mp

    if not torch.cuda.is_available() or torch.cuda.device_count() < 2:
        pytest.skip("needs 2 GPUs")
    path = tiny_model("tp")
    rng = np.random.default_rng(6)
    seqs = [rng.integers(1, fb.HostModel(path).params.vocab_size, n).astype(np.int32) for n in (60, 1, 33)]
    cuts = [[40, 1, 30], [41, 1, 33], [60, 1, 33]]
    nid = fb.tp_unique_id()
    c = mp.get_context("spawn")
    q = c.Queue()
    procs = [c.Process(target=_tp_worker, args=(r, 2, nid, path, seqs, cuts, q)) for r in range(2)]
    for pr in procs:
        pr.start()
    res = {}
    try:
        for _ in procs:
            rank, out, err = q.get(timeout=300)
            res[rank] = (out, err)
    finally:
        for pr in procs:
            pr.join(timeout=60)
            if pr.is_alive():
                pr.kill()
    done = [0] * len(seqs)
    for step, cut in enumerate(cuts):
        which = [i for i in range(len(seqs)) if cut[i] > done[i]]
        want = {i: _oracle_logits(path, seqs[i][:cut[i]]) for i in which}
        for rank in range(2):
            out, err = res[rank]
            assert err is None, err
            for k, i in enumerate(which):
                _check(*out[step], k, want[i])
        done = list(cut)
