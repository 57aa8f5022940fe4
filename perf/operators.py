"""Operators over the paged KV cache: their cases, inputs, plain forms and exact values.

Two operators of one attention layer that serves many sequences at once:

  append   rotate the new tokens' queries and keys by their positions and store keys and
           values in the paged cache (out: the rotated queries, both pools)
  attend   softmax attention of every sequence's new tokens, a chunk or a single token,
           over that sequence's pages, causal, with an optional sliding window (out: one
           row of heads x dim per token)

A batch is ragged: sequence s brings the tokens q_start[s] .. q_start[s + 1] - 1 and has
kv_len[s] positions in the cache once they are appended, so its token i sits at position
kv_len[s] - (q_start[s + 1] - q_start[s]) + i.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}


def _case(name, op, heads, kv_heads, dim, dtype, page, layout, chunks, new, ctx, singles, single_ctx, mix, window=0,
          in_dtype="", rotary=0, pairs="halves"):
    """chunks sequences with new[0] .. new[1] new tokens after ctx[0] .. ctx[1] cached ones, then
    singles sequences with one new token after single_ctx[0] .. single_ctx[1]; `mix` draws the lengths."""
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page, "layout": layout,
         "chunks": chunks, "new_lo": new[0], "new_hi": new[1], "ctx_lo": ctx[0], "ctx_hi": ctx[1], "singles": singles,
         "sctx_lo": single_ctx[0], "sctx_hi": single_ctx[1], "mix": mix}
    if op == "append":
        c.update(in_dtype=in_dtype or dtype, rotary=rotary or dim, pairs=pairs)
    else:
        c.update(window=window)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the single-token step of the 1.1B configuration: one fp32 row of q|k|v
        _case("append-token", "append", 32, 4, 64, "f16", 64, "heads", 0, (0, 0), (0, 0), 1, (700, 700), 1,
              in_dtype="f32"),
        # one step of the 7B configuration with every slot of a batch of 64 in use
        _case("append-step64", "append", 32, 32, 128, "f16", 64, "heads", 0, (0, 0), (0, 0), 64, (20, 4000), 2),
        # one prompt chunk of the 1.1B configuration, fp32 rows as its projections leave them
        _case("append-chunk512", "append", 32, 4, 64, "f16", 64, "heads", 1, (512, 512), (0, 0), 0, (0, 0), 3,
              in_dtype="f32"),
        # prompts of many users taken in at once: ragged, short pages, half of each head rotated in adjacent pairs
        _case("append-ragged", "append", 32, 8, 128, "bf16", 16, "positions", 29, (1, 1201), (0, 900), 11, (1, 3000), 4,
              rotary=64, pairs="adjacent"),
        # single-token step of one short conversation (1.1B configuration): latency
        _case("token-short", "attend", 32, 4, 64, "f16", 64, "heads", 0, (0, 0), (0, 0), 1, (383, 383), 5),
        # single-token step over two long documents: the cache's bytes, few rows
        _case("token-long", "attend", 32, 8, 128, "bf16", 64, "heads", 0, (0, 0), (0, 0), 2, (99001, 131000), 6),
        # single-token step of 64 users whose conversations differ in length
        _case("token-step64", "attend", 32, 8, 128, "f16", 16, "positions", 0, (0, 0), (0, 0), 64, (200, 7900), 7),
        # five drafted tokens of 24 users checked in one pass (7B configuration)
        _case("draft-check", "attend", 32, 32, 128, "f16", 64, "heads", 24, (5, 5), (1000, 4000), 0, (0, 0), 8),
        # first prompt chunk of the 1.1B configuration
        _case("chunk-first", "attend", 32, 4, 64, "f16", 64, "heads", 1, (512, 512), (0, 0), 0, (0, 0), 9),
        # a late chunk of a long prompt
        _case("chunk-late", "attend", 32, 8, 128, "bf16", 64, "heads", 1, (2048, 2048), (14005, 14005), 0, (0, 0), 10),
        # prompt chunks of two users beside the single tokens of forty
        _case("mixed-step", "attend", 32, 8, 128, "f16", 16, "positions", 2, (700, 1100), (900, 3000), 40, (50, 6000), 11),
        # whole prompts under a sliding window
        _case("window-prompts", "attend", 32, 32, 64, "bf16", 32, "heads", 3, (1500, 3500), (0, 700), 0, (0, 0), 12,
              window=1000),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _range(rng, lo, hi):
    a, b = sorted((_log(rng, lo, hi), _log(rng, lo, hi)))
    return a, b


def draw(rng):
    """A case of the same ranges: every type, head layout, page size and cache layout, lengths from one token up."""
    most = {op: max((work(c) for c in listed() if c["op"] == op), key=lambda w: w["bytes"])["bytes"] for op in ("append", "attend")}
    most_flops = max(work(c)["flops"] for c in listed())
    while True:
        heads, kv_heads = rng.choice([(32, 4), (32, 32), (32, 8), (12, 12), (8, 1), (16, 2), (24, 8), (28, 4), (64, 4)])
        dim, dtype = rng.choice([64, 128]), rng.choice(["f16", "bf16"])
        page, layout = rng.choice([16, 32, 64, 128, 256]), rng.choice(["heads", "positions"])
        mix = rng.randrange(1 << 30)
        kind = rng.choice(["chunks", "singles", "both"])
        if rng.random() < 0.3:
            chunks = 0 if kind == "singles" else _log(rng, 1, 40)
            singles = 0 if kind == "chunks" else _log(rng, 1, 200)
            c = _case("", "append", heads, kv_heads, dim, dtype, page, layout, chunks, _range(rng, 1, 4096),
                      _range(rng, 1, 4000), singles, _range(rng, 1, 8000), mix,
                      in_dtype=rng.choice(["f32", dtype]), rotary=rng.choice([dim, dim // 2]),
                      pairs=rng.choice(["halves", "adjacent"]))
        else:
            chunks = 0 if kind == "singles" else _log(rng, 1, 24)
            singles = 0 if kind == "chunks" else _log(rng, 1, 128)
            new = _range(rng, 2, 64) if rng.random() < 0.4 else _range(rng, 16, 4096)
            c = _case("", "attend", heads, kv_heads, dim, dtype, page, layout, chunks, new, _range(rng, 1, 32000), singles,
                      _range(rng, 1, 130000), mix, window=rng.choice([0, 0, 0, _log(rng, 16, 8000)]))
        w = work(c)
        pool = sum(kv for _, kv in _lengths(c)) * kv_heads * dim * 4
        if w["bytes"] <= most[c["op"]] and w["flops"] <= most_flops and pool <= 1.5e9:
            return c


def _lengths(case):
    """[(new tokens, cache length with them)] of the case's sequences, in a shuffled order."""
    rng = random.Random(case["mix"])
    out = []
    for _ in range(case["chunks"]):
        n = rng.randint(case["new_lo"], case["new_hi"])
        out.append((n, n + rng.randint(case["ctx_lo"], case["ctx_hi"])))
    for _ in range(case["singles"]):
        out.append((1, 1 + rng.randint(case["sctx_lo"], case["sctx_hi"])))
    rng.shuffle(out)
    return out


def _rope_table(max_pos, rotary, device):
    """(cos, sin) of position * 10000^(-2i / rotary), fp32 [max_pos][rotary / 2][2]."""
    i = torch.arange(rotary // 2, dtype=torch.float64, device=device)
    angle = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * 10000.0 ** (-2.0 * i / rotary)
    return torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    lens = _lengths(case)
    H, KV, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    dt = TYPES[case["dtype"]]
    n = sum(a for a, _ in lens)
    pages = [-(-b // P) for _, b in lens]
    max_pages, n_pages = max(pages), sum(pages) + 3
    # slots in another order than the sequences, pages scattered over the pool
    order = torch.randperm(len(lens), generator=torch.Generator().manual_seed(seed))
    perm = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed + 1)).to(torch.int32)
    table = torch.zeros(len(lens), max_pages, dtype=torch.int32)
    at = 0
    for s, k in enumerate(pages):
        table[order[s], :k] = perm[at:at + k]
        at += k
    starts = [0]
    for a, _ in lens:
        starts.append(starts[-1] + a)
    shape = (n_pages, KV, P, D) if case["layout"] == "heads" else (n_pages, P, KV, D)
    st = {"case": case, "lens": lens, "table": table.to(dev), "slot": order.to(torch.int32).to(dev),
          "q_start": torch.tensor(starts, dtype=torch.int32, device=dev),
          "kv_len": torch.tensor([b for _, b in lens], dtype=torch.int32, device=dev),
          "k_pool": torch.randn(shape, generator=gen, device=dev, dtype=dt),
          "v_pool": torch.randn(shape, generator=gen, device=dev, dtype=dt)}
    if case["op"] == "append":
        it = TYPES[case["in_dtype"]]
        # one fused row of q|k|v per token, as the projections leave it
        st["qkv"] = torch.randn(n, (H + 2 * KV) * D, generator=gen, device=dev, dtype=torch.float32).to(it)
        st["rope"] = _rope_table(max(b for _, b in lens), case["rotary"], dev)
        st["q_out"] = torch.empty(n, H * D, device=dev, dtype=dt)
    else:
        # heads differ in how sharp their attention is
        gain = torch.linspace(0.5, 3.5, H, device=dev)[None, :, None]
        st["q"] = (torch.randn(n, H, D, generator=gen, device=dev) * gain).to(dt).reshape(n, H * D)
        st["out"] = torch.empty(n, H * D, device=dev, dtype=dt)
    if own:
        path = os.path.join(os.getcwd(), "fiber-inference_b200")
        if path not in sys.path:
            sys.path.insert(1, path)
        import fiber_b200 as fb

        ps = KV * P * D
        hs, rs = (P * D, D) if case["layout"] == "heads" else (D, KV * D)
        st["fb"] = fb
        st["view"] = fb.PagedKV(st["k_pool"].data_ptr(), st["v_pool"].data_ptr(), st["table"].data_ptr(), n_slots=len(lens),
                                max_pages=max_pages, n_pages=n_pages, page_size=P, n_kv_heads=KV, head_dim=D,
                                dtype=GGML[case["dtype"]], page_stride=ps, head_stride=hs, pos_stride=rs)
        st["batch"] = fb.RaggedBatch(st["q_start"].data_ptr(), st["kv_len"].data_ptr(), n_seqs=len(lens), n_tokens=n,
                                     max_q=max(a for a, _ in lens), slot=st["slot"].data_ptr())
        if case["op"] == "append":
            st["rotation"] = fb.Rope(st["rope"].data_ptr(), max_pos=st["rope"].shape[0], dim=case["rotary"],
                                     adjacent=case["pairs"] == "adjacent")
        else:
            st["ws"] = torch.zeros(fb.attn_paged_workspace(st["view"], st["batch"], H), dtype=torch.uint8, device=dev)
    return st


def run(st):
    case = st["case"]
    if own:
        return _own_append(st, case) if case["op"] == "append" else _own_attend(st, case)
    return _plain_append(st, case) if case["op"] == "append" else _plain_attend(st, case)


def _own_append(st, case):
    fb, qkv = st["fb"], st["qkv"]
    H, KV, D = case["heads"], case["kv_heads"], case["dim"]
    at, size = qkv.data_ptr(), qkv.element_size()
    fb.kv_append(st["view"], st["batch"], GGML[case["in_dtype"]], at, at + H * D * size, at + (H + KV) * D * size,
                 ld=qkv.shape[1], n_heads=H, q_out=st["q_out"].data_ptr(), ld_out=H * D, rope=st["rotation"],
                 stream=torch.cuda.current_stream().cuda_stream)
    return [st["q_out"], st["k_pool"], st["v_pool"]]


def _own_attend(st, case):
    H, D = case["heads"], case["dim"]
    st["fb"].attn_paged(st["view"], st["batch"], st["q"].data_ptr(), st["out"].data_ptr(), n_heads=H, ldq=H * D, ldo=H * D,
                        scale=1.0 / math.sqrt(D), window=case["window"], ws=st["ws"].data_ptr(), ws_bytes=st["ws"].numel(),
                        stream=torch.cuda.current_stream().cuda_stream)
    return [st["out"]]


def _rotate(x, table, rotary, pairs):
    """x [n, heads, dim] fp32, table [n, rotary / 2, 2]: the first `rotary` values of each head rotated."""
    cos, sin = table[:, None, :, 0], table[:, None, :, 1]
    y = x.clone()
    if pairs == "halves":
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        y[..., :rotary // 2] = a * cos - b * sin
        y[..., rotary // 2:rotary] = a * sin + b * cos
    else:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        y[..., 0:rotary:2] = a * cos - b * sin
        y[..., 1:rotary:2] = a * sin + b * cos
    return y


def _plain_append(st, case):
    H, KV, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    qkv, dt = st["qkv"].float(), st["q_out"].dtype
    n = qkv.shape[0]
    token = torch.arange(n, device=qkv.device, dtype=torch.int32)
    seq = (token[:, None] >= st["q_start"][None, 1:]).sum(1)
    pos = (st["kv_len"][seq] - st["q_start"][seq + 1] + token).long()
    table = st["rope"][pos]
    q = _rotate(qkv[:, :H * D].reshape(n, H, D), table, case["rotary"], case["pairs"])
    k = _rotate(qkv[:, H * D:(H + KV) * D].reshape(n, KV, D), table, case["rotary"], case["pairs"])
    v = qkv[:, (H + KV) * D:].reshape(n, KV, D)
    page = st["table"][st["slot"][seq].long(), pos // P].long()
    kp, vp = st["k_pool"], st["v_pool"]
    if case["layout"] == "heads":
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    kp[page, pos % P] = k.to(dt)
    vp[page, pos % P] = v.to(dt)
    st["q_out"].copy_(q.reshape(n, H * D).to(dt))
    return [st["q_out"], st["k_pool"], st["v_pool"]]


def _plain_attend(st, case):
    H, KV, D, P, window = case["heads"], case["kv_heads"], case["dim"], case["page"], case["window"]
    G, dev = H // KV, st["q"].device
    kp, vp = st["k_pool"], st["v_pool"]
    if case["layout"] == "heads":
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    at = 0
    for s, (n, kv) in enumerate(st["lens"]):
        pages = st["table"][st["slot"][s:s + 1].long()][0, :-(-kv // P)].long()
        k = kp[pages].reshape(-1, KV, D)[:kv].float().transpose(0, 1)
        v = vp[pages].reshape(-1, KV, D)[:kv].float().transpose(0, 1)
        step = max(1, int(4e8 / (H * kv)))  # rows of scores held at a time
        for i in range(0, n, step):
            m = min(step, n - i)
            q = st["q"][at + i:at + i + m].float().reshape(m, KV, G, D).permute(1, 0, 2, 3).reshape(KV, m * G, D)
            pos = (torch.arange(m, device=dev) + (kv - n + i)).repeat_interleave(G)[:, None]
            key = torch.arange(kv, device=dev)[None, :]
            hide = key > pos
            if window:
                hide = hide | (key <= pos - window)
            x = (q @ k.transpose(1, 2)) * (1.0 / math.sqrt(D))
            x.masked_fill_(hide, float("-inf"))
            x = torch.exp(x - x.amax(2, keepdim=True))
            o = (x @ v) / x.sum(2, keepdim=True)
            st["out"][at + i:at + i + m] = o.reshape(KV, m, G, D).permute(1, 0, 2, 3).reshape(m, H * D).to(st["out"].dtype)
        at += n
    return [st["out"]]


def work(case):
    """Each input read once, each output written once; 2 operations to a multiply-add."""
    H, KV, D = case["heads"], case["kv_heads"], case["dim"]
    lens = _lengths(case)
    n = sum(a for a, _ in lens)
    if case["op"] == "append":
        size = 4 if case["in_dtype"] == "f32" else 2
        positions = set()
        for a, b in lens:
            positions.update(range(b - a, b))
        rot = case["rotary"] / D
        return {"bytes": n * (H + 2 * KV) * D * (size + 2) + len(positions) * case["rotary"] * 4,
                "flops": 3 * n * (H + KV) * D * rot}
    rows = pairs = 0
    for a, b in lens:
        first = b - a + 1  # keys the first new token sees
        w = case["window"]
        if w:
            full = max(0, min(a, w - first + 1))  # tokens whose window reaches the start
            pairs += full * first + full * (full - 1) // 2 + (a - full) * w
            rows += min(b, a - 1 + w)
        else:
            pairs += a * first + a * (a - 1) // 2
            rows += b
    return {"bytes": 4 * n * H * D + 4 * rows * KV * D, "flops": 4 * D * H * pairs}


def exact(case, seed):
    """The outputs in 64 bits, from the definitions, token by token places and head by head sums."""
    st = prepare(dict(case), seed)
    H, KV, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    lens, table, slot = st["lens"], st["table"].cpu(), st["slot"].cpu()
    heads_first = case["layout"] == "heads"
    if case["op"] == "append":
        x = st["qkv"].double()
        where = [(s, b - a + i) for s, (a, b) in enumerate(lens) for i in range(a)]
        pos = torch.tensor([p for _, p in where], device=x.device)
        angle = st["rope"].double()[pos]
        turn = torch.complex(angle[..., 0], angle[..., 1])[:, None, :]
        R = case["rotary"]

        def rotated(y):
            y = y.clone()
            if case["pairs"] == "halves":
                z = torch.complex(y[..., :R // 2], y[..., R // 2:R]) * turn
                y[..., :R] = torch.cat([z.real, z.imag], -1)
            else:
                z = torch.complex(y[..., 0:R:2], y[..., 1:R:2]) * turn
                y[..., :R] = torch.stack([z.real, z.imag], -1).flatten(-2)
            return y

        n = x.shape[0]
        q, k, v = x.split([H * D, KV * D, KV * D], 1)
        k, v = rotated(k.reshape(n, KV, D)), v.reshape(n, KV, D)
        row = torch.tensor([int(table[slot[s], p // P]) * P + p % P for s, p in where], device=x.device)
        pools = []
        for pool, new in ((st["k_pool"], k), (st["v_pool"], v)):
            flat = pool.double()
            flat = (flat.transpose(1, 2) if heads_first else flat).reshape(-1, KV, D).clone()
            flat[row] = new
            flat = flat.reshape(-1, P, KV, D)
            pools.append((flat.transpose(1, 2) if heads_first else flat).contiguous())
        return [rotated(q.reshape(n, H, D)).reshape(n, H * D)] + pools
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device=st["out"].device)
    at = 0
    for s, (n, kv) in enumerate(lens):
        rows = torch.cat([torch.arange(P) + int(p) * P for p in table[slot[s], :-(-kv // P)]])[:kv].to(out.device)
        page, inside = rows // P, rows % P
        t = torch.arange(n, device=out.device) + (kv - n)
        j = torch.arange(kv, device=out.device)
        seen = j[None, :] <= t[:, None]
        if case["window"]:
            seen &= j[None, :] > t[:, None] - case["window"]
        for g in range(KV):
            k = (st["k_pool"][page, g, inside] if heads_first else st["k_pool"][page, inside, g]).double()
            v = (st["v_pool"][page, g, inside] if heads_first else st["v_pool"][page, inside, g]).double()
            for h in range(g * (H // KV), (g + 1) * (H // KV)):
                x = st["q"][at:at + n, h * D:(h + 1) * D].double() @ k.T / math.sqrt(D)
                x = torch.where(seen, x, torch.full_like(x, -math.inf))
                out[at:at + n, h * D:(h + 1) * D] = torch.exp(x - torch.logsumexp(x, 1, keepdim=True)) @ v
        at += n
    return [out]
