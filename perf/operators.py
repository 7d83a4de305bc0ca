"""The operators of a decoding step over a 4-bit cache, as cases that can be timed and checked.

append   rows of keys and values are rotated to their positions, quantised to 4 bits and written into the pages of
         their sequences; the queries of the same rows are rotated on the way.  The rows are then read back.
attend   the queries of every sequence of a batch over its pages: single tokens, verify rows, trees, prompts.
sample   tokens drawn from rows of logits with temperature, top-k, top-p and min-p, from given random numbers.

A group of 32 channels of one row and KV head shares one step d: with A the group's largest magnitude,
|d| = fp16(fp32(A / 8)), negative where the largest magnitude is a positive number's alone, so that it stands on -8;
a channel x has the code c = clamp(round(x / d), -8, 7) and stands for fp16(d c).

`own` false computes these in plain torch operations, `own` true through the library's entry points.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

HEADS = {  # query heads, KV heads, head size, rotation of neighbouring channels or of halves, rotation base
    "llama8b": (32, 8, 128, True, 500000.0),
    "qwen7b": (28, 4, 128, False, 1e6),
    "small": (8, 8, 64, True, 10000.0),
}
GROUP = 32
MAX_POS = 1 << 17


def listed():
    return [
        # the cache write of one decoded token: latency only
        dict(name="append1", op="append", heads="small", dtype="f32", lengths="1", start=100, page=64),
        # one token for each sequence of a serving batch, two of the rows padding
        dict(name="append_batch37", op="append", heads="qwen7b", dtype="f16", lengths="1*37", start=90000, page=64, pad=2),
        # a ragged prompt batch as the decoder hands it over: fp32 rows of the Q/K/V product
        dict(name="append_prompt2501", op="append", heads="llama8b", dtype="f32", lengths="1301,7,1193", start=77, page=128),
        # long prompts filled in at once
        dict(name="append_prompt16384", op="append", heads="llama8b", dtype="f16", lengths="8192,8192", start=0, page=64),
        # the small decoder's step
        dict(name="attend1_small", op="attend", heads="small", rows=1, lengths="101", mask="causal", page=64),
        # the verify step of four drafts at a long context
        dict(name="attend5_long", op="attend", heads="llama8b", rows=5, lengths="32768", mask="causal", page=64),
        # one token of each sequence of a ragged batch
        dict(name="attend_batch", op="attend", heads="qwen7b", rows=1,
             lengths="9001,33,4096,700,1,2222,64,5113,1500,31,8192,257,6000,12,3001,450", mask="causal", page=64),
        # a draft tree at a long context
        dict(name="attend_tree60", op="attend", heads="llama8b", rows=60, lengths="8192", mask="tree", page=32),
        # a chunk of a long prompt over what came before
        dict(name="attend_prompt2048", op="attend", heads="llama8b", rows=2048, lengths="8191", mask="causal", page=128),
        # the next token of one sequence, with the usual filters
        dict(name="sample1", op="sample", rows=1, vocab=128256, temperature=0.7, top_k=40, top_p=0.95, min_p=0.0, probs=False),
        # every row of a tree's logits, by probability mass
        dict(name="sample60", op="sample", rows=60, vocab=152064, temperature=1.0, top_k=0, top_p=0.9, min_p=0.01, probs=False),
        # draft tokens with the distributions they were drawn from, for rejection sampling against them
        dict(name="sample9_rows", op="sample", rows=9, vocab=32000, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, probs=True),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sample"])
    heads = rng.choice(sorted(HEADS))
    page = rng.choice([32, 64, 128, 256])
    if op == "append":
        total = _log(rng, 1, 12000)
        seqs = min(total, rng.choice([1, 1, 2, 5, 31]))
        cuts = sorted(rng.sample(range(1, total), seqs - 1)) if seqs > 1 else []
        lengths = [b - a for a, b in zip([0] + cuts, cuts + [total])]
        return dict(op=op, heads=heads, dtype=rng.choice(["f16", "f32"]), lengths=",".join(map(str, lengths)),
                    start=rng.choice([0, _log(rng, 1, 100000)]), page=page, pad=rng.choice([0, 0, 3]))
    if op == "attend":
        kind = rng.choice(["step", "batch", "verify", "tree", "prompt"])
        rows, mask = 1, "causal"
        lengths = [_log(rng, 1, 40000)]
        if kind == "batch":
            lengths = [_log(rng, 1, 12000) for _ in range(rng.randint(2, 24))]
        elif kind == "verify":
            rows = rng.randint(2, 16)
            lengths = [n + rows for n in lengths]
        elif kind == "tree":
            rows, mask = _log(rng, 3, 128), "tree"
            lengths = [_log(rng, 1, 16000) + rows]
        elif kind == "prompt":
            rows = _log(rng, 17, 2048)
            lengths = [_log(rng, 1, 6000) + rows for _ in range(rng.choice([1, 1, 2]) if rows < 900 else 1)]
        return dict(op=op, heads=heads, rows=rows, lengths=",".join(map(str, lengths)), mask=mask, page=page)
    vocab = rng.choice([32000, 128256, 152064, rng.randint(1000, 152064)])
    return dict(op=op, rows=max(1, min(_log(rng, 1, 128), 60 * 152064 // vocab)), vocab=vocab,
                temperature=round(rng.uniform(0.2, 1.5), 3), top_k=rng.choice([0, 0, _log(rng, 1, 2000)]),
                top_p=rng.choice([1.0, round(rng.uniform(0.4, 0.999), 4)]),
                min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 4)]), probs=rng.choice([False, False, True]))


# ---- inputs ----------------------------------------------------------------------
def _gen(seed, tag):
    return torch.Generator("cuda").manual_seed(int(seed) * 1000003 + tag)


def _lengths(case):
    text = case["lengths"]
    if "*" in text:
        one, times = text.split("*")
        return [int(one)] * int(times)
    return [int(v) for v in text.split(",")]


def _rows_of(seed, tag, rows, heads, hd):
    """Rows as a projection leaves them: about normal, a few channels an order of magnitude larger."""
    x = torch.randn((rows, heads, hd), generator=_gen(seed, tag), device="cuda")
    big = 1.0 + 6.0 * (torch.rand((1, heads, hd), generator=_gen(seed, tag + 50), device="cuda") > 0.97)
    return x * big


def _pages(case, seed, lengths):
    """(table [sequences][pages], pages of the pool): a sequence's pages lie anywhere."""
    need = [max(1, -(-n // case["page"])) for n in lengths]
    pool = sum(need) + 3
    ids = torch.randperm(pool, generator=torch.Generator().manual_seed(int(seed) + 5))[:sum(need)].tolist()
    table = torch.zeros((len(lengths), max(need)), dtype=torch.int32)
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
    return table.cuda(), pool


def _append_inputs(case, seed):
    H, KV, hd, _, _ = HEADS[case["heads"]]
    lengths, pad = _lengths(case), case.get("pad", 0)
    n = sum(lengths) + pad
    jitter = torch.randint(0, 1 + case["start"] // 2, (len(lengths),), generator=torch.Generator().manual_seed(int(seed))).tolist()
    starts = [case["start"] - j for j in jitter]
    seq = [s for s, m in enumerate(lengths) for _ in range(m)] + [-1] * pad
    slot = [starts[s] + i for s, m in enumerate(lengths) for i in range(m)] + [0] * pad
    dt = torch.float16 if case["dtype"] == "f16" else torch.float32
    q, k, v = (_rows_of(seed, t, n, h, hd).to(dt) for t, h in ((1, H), (2, KV), (3, KV)))
    return dict(q=q, k=k, v=v, seq=torch.tensor(seq, dtype=torch.int32, device="cuda"),
                slot=torch.tensor(slot, dtype=torch.int32, device="cuda"), ends=[a + m for a, m in zip(starts, lengths)])


def _tree_mask(seed, n):
    """Ancestor bits of a random tree in breadth-first order: [n][words] as int64."""
    rng = np.random.default_rng(int(seed) + 11)
    parents = [0] + [0] * (n - 1)
    for i in range(1, n):
        parents[i] = int(rng.integers(max(0, (i - 1) // 4), (i - 1) // 2 + 1))
    words = -(-n // 64)
    bits = np.zeros((n, words), np.uint64)
    for i in range(n):
        if i:
            bits[i] = bits[parents[i]]
        bits[i, i // 64] |= np.uint64(1) << np.uint64(i % 64)
    return torch.from_numpy(bits.view(np.int64)).cuda()


def _attend_inputs(case, seed):
    H, KV, hd, _, _ = HEADS[case["heads"]]
    lengths, rows = _lengths(case), case["rows"]
    n = rows * len(lengths)
    total = sum(lengths)
    return dict(q=_rows_of(seed, 1, n, H, hd).half(), k=_rows_of(seed, 2, total, KV, hd).half(),
                v=_rows_of(seed, 3, total, KV, hd).half(),
                row_start=torch.arange(0, n + 1, rows, dtype=torch.int32, device="cuda"),
                kv_len=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                seq=torch.tensor([s for s, m in enumerate(lengths) for _ in range(m)], dtype=torch.int32, device="cuda"),
                slot=torch.tensor([i for m in lengths for i in range(m)], dtype=torch.int32, device="cuda"),
                mask=_tree_mask(seed, rows) if case["mask"] == "tree" else None)


def _sample_inputs(case, seed):
    """Logits as a language model's: about normal, some tokens well above, each row of another sharpness; a few masked."""
    n, V = case["rows"], case["vocab"]
    x = torch.randn((n, V), generator=_gen(seed, 1), device="cuda")
    sharp = 0.8 + 2.4 * torch.rand((n, 1), generator=_gen(seed, 2), device="cuda")
    x = x * sharp
    top = torch.randint(0, V, (n, 24), generator=_gen(seed, 3), device="cuda")
    x.scatter_(1, top, sharp * (4.0 + 2.5 * torch.rand((n, 24), generator=_gen(seed, 4), device="cuda")))
    x[:, 7::997] = -math.inf
    u = torch.rand((n,), generator=_gen(seed, 5), device="cuda")
    return dict(logits=x, u=u)


# ---- the plain form ----------------------------------------------------------------
def _tables(hd, base):
    """cos and sin of position x base^(-2i/hd), from 64-bit angles, [positions][hd / 2] fp32"""
    inv = base ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    a = torch.arange(MAX_POS, dtype=torch.float64, device="cuda")[:, None] * inv
    return a.cos().float(), a.sin().float()


def _rotate(x, cos, sin, pairs):
    """x [rows][heads][hd] by cos, sin [rows][hd / 2]"""
    c, s = cos[:, None], sin[:, None]
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if pairs else (x[..., :half], x[..., half:])
    ra, rb = a * c - b * s, b * c + a * s
    return torch.stack((ra, rb), -1).flatten(-2) if pairs else torch.cat((ra, rb), -1)


def _quantise(x):
    """x [rows][heads][hd] in 64 bits -> (codes [rows][heads][hd] int8, steps [rows][heads][hd / 32] fp16)"""
    g = x.unflatten(-1, (-1, GROUP))
    low, high = -g.amin(-1), g.amax(-1)
    big = torch.maximum(low, high)
    d = (big / 8).float().half()
    d = torch.where(high > low, -d, d)
    bad = ~(big <= 65504.0)  # a NaN or what 16 bits do not hold
    d = torch.where(bad, torch.nan, d)
    step = d.double()[..., None]
    c = torch.where((step == 0) | bad[..., None], 0.0, (g / step).round()).clamp(-8, 7)
    return c.to(torch.int8).flatten(-2), d


def _values(codes, steps):
    return (codes.unflatten(-1, (-1, GROUP)).float() * steps.float()[..., None]).half().flatten(-2)


def _plain_append(st):
    inp, (H, KV, hd, pairs, _) = st["inp"], HEADS[st["case"]["heads"]]
    real = inp["seq"] >= 0
    pos = inp["slot"][real].long()
    cos, sin = st["cos"][pos], st["sin"][pos]
    q, k, v = st["q_out"], st["k_out"], st["v_out"]
    q[real] = _rotate(inp["q"][real].float(), cos, sin, pairs).half()
    k[real] = _values(*_quantise(_rotate(inp["k"][real].double(), cos.double(), sin.double(), pairs)))
    v[real] = _values(*_quantise(inp["v"][real].double()))
    return q, k, v


def _plain_cache(case, inp, table, n_pages):
    """The cache of an attend case: codes and steps by page."""
    H, KV, hd, pairs, base = HEADS[case["heads"]]
    cos, sin = _tables(hd, base)
    pos = inp["slot"].long()
    page = table[inp["seq"].long(), pos // case["page"]].long()
    at = page * case["page"] + pos % case["page"]
    out = {}
    for name in ("k", "v"):
        codes = torch.zeros((n_pages * case["page"], KV, hd), dtype=torch.int8, device="cuda")
        steps = torch.zeros((n_pages * case["page"], KV, hd // GROUP), dtype=torch.float16, device="cuda")
        for a in range(0, len(pos), 16384):
            x = inp[name][a:a + 16384].double()
            if name == "k":
                p = pos[a:a + 16384]
                x = _rotate(x, cos[p].double(), sin[p].double(), pairs)
            codes[at[a:a + 16384]], steps[at[a:a + 16384]] = _quantise(x)
        out[name] = (codes, steps)
    return out


def _visible(case, rows, T, mask, dev):
    """[rows][T] of the last `rows` of T positions: causal, or a tree's ancestors"""
    i, j = torch.arange(rows, device=dev)[:, None], torch.arange(T, device=dev)[None]
    if mask is None:
        return j <= i + (T - rows)
    b = (j - (T - rows)).clamp(min=0)
    bits = (mask[:, (b[0] // 64).clamp(max=mask.shape[1] - 1)] >> (b % 64)) & 1
    return (j < T - rows) | (bits == 1)


def _plain_attend(st):
    case, inp = st["case"], st["inp"]
    H, KV, hd, _, _ = HEADS[case["heads"]]
    rows, out = case["rows"], st["out"]
    scale = 1.0 / math.sqrt(hd)
    for s, T in enumerate(_lengths(case)):
        j = torch.arange(T, device="cuda")
        at = st["table"][s, j // case["page"]].long() * case["page"] + j % case["page"]
        k, v = (_values(c[at], d[at]).float() for c, d in (st["cache"]["k"], st["cache"]["v"]))
        seen = _visible(case, rows, T, inp["mask"], "cuda")
        q = inp["q"][s * rows:(s + 1) * rows].float().unflatten(1, (KV, H // KV))
        for h in range(KV):
            score = (q[:, h].reshape(-1, hd) @ k[:, h].T * scale).view(rows, H // KV, T)
            score = score.masked_fill(~seen[:, None], -math.inf)
            top = score.amax(-1, keepdim=True)
            w = (score - torch.where(top == -math.inf, 0.0, top)).exp()
            total = w.sum(-1, keepdim=True)
            o = (w.view(-1, T) @ v[:, h]).view(rows, H // KV, hd)
            out[s * rows:(s + 1) * rows, h * (H // KV):(h + 1) * (H // KV)] = torch.where(total > 0, o / total, 0.0).half()
    return out


def _plain_sample(st):
    case, (x, u) = st["case"], (st["inp"]["logits"], st["inp"]["u"])
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1]
    w = ((x.double() - x.amax(-1, keepdim=True).double()) / case["temperature"]).exp()
    by_rank = w.gather(1, order)
    if 0 < case["top_k"] < x.shape[1]:
        by_rank[:, case["top_k"]:] = 0.0
    if case["top_p"] < 1.0:
        mass = by_rank.cumsum(-1)
        before = mass - by_rank
        before[:, 1:] = mass[:, :-1]
        top_p = float(np.float32(case["top_p"]))
        by_rank = torch.where((before < top_p * mass[:, -1:]) | (torch.arange(x.shape[1], device="cuda") == 0), by_rank, 0.0)
    by_rank = torch.where(by_rank >= float(np.float32(case["min_p"])), by_rank, 0.0)
    kept = torch.zeros_like(w).scatter_(1, order, by_rank)
    mass = kept.cumsum(-1)
    total = mass[:, -1:]
    token = torch.searchsorted(mass, u.double()[:, None] * total, right=True)[:, 0].int()
    return (token, (kept / total).float()) if case["probs"] else token


# ---- one pass ----------------------------------------------------------------------
def _library():
    path = os.path.join(os.getcwd(), "abyo-speculate_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import speculate_hip
    return speculate_hip


def _pool(case, n_pages):
    H, KV, hd, pairs, base = HEADS[case["heads"]]
    return _library().HipKvPool(n_layers=1, n_heads=H, n_kv_heads=KV, head_dim=hd, n_pages=n_pages, page_tokens=case["page"],
                                max_pos=MAX_POS, rope_theta=base, interleaved=pairs)


def prepare(case, seed):
    st = dict(case=case)
    if case["op"] == "sample":
        st["inp"] = _sample_inputs(case, seed)
        if own:
            st["sampler"] = _library().HipSampler(case["vocab"], case["rows"])
            st["tokens"] = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
            st["probs"] = torch.empty((case["rows"], case["vocab"]), device="cuda") if case["probs"] else None
        return st
    H, KV, hd, pairs, base = HEADS[case["heads"]]
    if case["op"] == "append":
        st["inp"] = inp = _append_inputs(case, seed)
        st["table"], n_pages = _pages(case, seed, inp["ends"])
        n = len(inp["seq"])
        st["q_out"] = torch.zeros((n, H, hd), dtype=torch.float16, device="cuda")
        st["k_out"], st["v_out"] = (torch.zeros((n, KV, hd), dtype=torch.float16, device="cuda") for _ in range(2))
        if own:
            st["pool"] = _pool(case, n_pages)
        else:
            st["cos"], st["sin"] = _tables(hd, base)
        return st
    st["inp"] = inp = _attend_inputs(case, seed)
    lengths = _lengths(case)
    st["table"], n_pages = _pages(case, seed, lengths)
    n = case["rows"] * len(lengths)
    st["out"] = torch.zeros((n, H, hd), dtype=torch.float16, device="cuda")
    if own:
        S, table = _library(), st["table"]
        st["pool"] = pool = _pool(case, n_pages)
        pool.append(0, len(inp["seq"]), inp["k"].data_ptr(), inp["v"].data_ptr(), inp["slot"].data_ptr(), table.data_ptr(),
                    table.shape[0], table.shape[1], dtype=S.F16, seqs=inp["seq"].data_ptr(),
                    stream=torch.cuda.current_stream().cuda_stream)
        st["ws"] = torch.zeros(pool.attend_workspace(n, len(lengths), case["rows"], max(lengths)), dtype=torch.uint8, device="cuda")
    else:
        st["cache"] = _plain_cache(case, inp, st["table"], n_pages)
    for name in ("k", "v", "seq", "slot"):
        del inp[name]
    return st


def run(state):
    case, inp = state["case"], state["inp"]
    op = case["op"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[op](state)
    stream = torch.cuda.current_stream().cuda_stream
    if op == "sample":
        probs = state["probs"]
        state["sampler"].sample(inp["logits"].data_ptr(), case["rows"], inp["u"].data_ptr(), state["tokens"].data_ptr(),
                                temperature=case["temperature"], top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"],
                                probs=0 if probs is None else probs.data_ptr(), stream=stream)
        return state["tokens"] if probs is None else (state["tokens"], probs)
    pool, table = state["pool"], state["table"]
    if op == "append":
        S, n = _library(), len(inp["seq"])
        pool.append(0, n, inp["k"].data_ptr(), inp["v"].data_ptr(), inp["slot"].data_ptr(), table.data_ptr(), table.shape[0],
                    table.shape[1], dtype=S.F16 if case["dtype"] == "f16" else S.F32, seqs=inp["seq"].data_ptr(),
                    q=inp["q"].data_ptr(), q_out=state["q_out"].data_ptr(), stream=stream)
        pool.read(0, n, inp["slot"].data_ptr(), table.data_ptr(), table.shape[0], table.shape[1], state["k_out"].data_ptr(),
                  state["v_out"].data_ptr(), seqs=inp["seq"].data_ptr(), stream=stream)
        return state["q_out"], state["k_out"], state["v_out"]
    mask, ws = inp["mask"], state["ws"]
    pool.attend(0, inp["q"].data_ptr(), state["out"].data_ptr(), inp["row_start"].data_ptr(), inp["kv_len"].data_ptr(),
                table.data_ptr(), table.shape[0], table.shape[1], rows=len(inp["q"]), max_rows=case["rows"],
                max_len=max(_lengths(case)), ws=ws.data_ptr(), ws_bytes=ws.numel(),
                mask=0 if mask is None else mask.data_ptr(), mask_words=0 if mask is None else mask.shape[1], stream=stream)
    return state["out"]


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (8 if case["probs"] else 4), "flops": 4 * n}
    H, KV, hd, _, _ = HEADS[case["heads"]]
    lengths = _lengths(case)
    row4 = KV * (hd // 2 + hd // GROUP * 2)  # one position's keys or values in 4 bits
    if case["op"] == "append":
        n = sum(lengths)
        size = 2 if case["dtype"] == "f16" else 4
        # rows in, queries out, codes out and in again, values out
        return {"bytes": n * ((H + 2 * KV) * hd * size + H * hd * 2 + 4 * row4 + 2 * KV * hd * 2),
                "flops": n * (H + 3 * KV) * hd * 3}
    rows, seen = case["rows"], 0
    for T in lengths:
        seen += rows * (T - rows) + (rows * (rows + 1) // 2 if case["mask"] == "causal" else 8 * rows)
    return {"bytes": 2 * sum(lengths) * row4 + 2 * rows * len(lengths) * H * hd * 2, "flops": 4 * seen * H * hd}


# ---- the same in 64 bits -------------------------------------------------------------
def _turned(x, pos, base, pairs):
    """Row by row as complex numbers times e^(i angle), the angle's cos and sin held in 32 bits"""
    hd = x.shape[-1]
    angle = torch.outer(pos.double(), torch.tensor([base ** (-2.0 * i / hd) for i in range(hd // 2)], dtype=torch.float64,
                                                   device=x.device))
    turn = torch.complex(angle.cos().float().double(), angle.sin().float().double())[:, None]
    x = x.double()
    if pairs:
        return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], hd // 2, 2).contiguous()) * turn).flatten(-2)
    z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * turn
    return torch.cat((z.real, z.imag), -1)


def _stored(x):
    """What x stands for after 4 bits: the group's extreme of largest magnitude (the negative one if both) is -8 steps"""
    shape = x.shape
    x = x.reshape(-1, GROUP)
    small, large = x.min(1)[0], x.max(1)[0]
    extreme = torch.where(-small >= large, small, large)
    step = (extreme / -8.0).to(torch.float32).to(torch.float16).to(torch.float64)[:, None]
    code = torch.where(step == 0, torch.zeros_like(x), torch.round(x / step)).clamp(-8.0, 7.0)
    return (code * step).to(torch.float32).to(torch.float16).to(torch.float64).reshape(shape)


def exact(case, seed):
    if case["op"] == "sample":
        return _exact_sample(case, _sample_inputs(case, seed))
    H, KV, hd, pairs, base = HEADS[case["heads"]]
    if case["op"] == "append":
        inp = _append_inputs(case, seed)
        real, pos = inp["seq"] >= 0, inp["slot"]
        q = torch.where(real[:, None, None], _turned(inp["q"], pos, base, pairs), 0.0)
        k = torch.where(real[:, None, None], _stored(_turned(inp["k"], pos, base, pairs)), 0.0)
        v = torch.where(real[:, None, None], _stored(inp["v"].double()), 0.0)
        return q, k, v
    inp = _attend_inputs(case, seed)
    outs, at, rows = [], 0, case["rows"]
    for s, T in enumerate(_lengths(case)):
        k = _stored(_turned(inp["k"][at:at + T], torch.arange(T, device="cuda"), base, pairs))
        v = _stored(inp["v"][at:at + T].double())
        at += T
        q = inp["q"][s * rows:(s + 1) * rows].double()
        prefix = T - rows
        seen = torch.ones((rows, T), dtype=torch.bool)
        if inp["mask"] is None:
            seen[:, prefix:] = torch.tril(torch.ones((rows, rows), dtype=torch.bool))
        else:
            words = inp["mask"].cpu().numpy().view(np.uint64)
            for i in range(rows):
                whole = sum(int(w) << (64 * n) for n, w in enumerate(words[i]))
                seen[i, prefix:] = torch.tensor([bool(whole >> j & 1) for j in range(rows)])
        seen = seen.cuda()
        out = torch.empty((rows, H, hd), dtype=torch.float64, device="cuda")
        for h in range(H):
            score = q[:, h] @ k[:, h * KV // H].T / math.sqrt(hd)
            score[~seen] = -math.inf
            out[:, h] = torch.softmax(score, -1) @ v[:, h * KV // H]
        outs.append(out)
    return torch.cat(outs)


def _exact_sample(case, inp):
    x, u = inp["logits"].cpu().numpy().astype(np.float64), inp["u"].cpu().numpy().astype(np.float64)
    n, V = x.shape
    tokens, probs = np.empty(n, np.int32), np.zeros((n, V))
    for r in range(n):
        rank = np.lexsort((np.arange(V), -x[r]))
        w = np.exp((x[r][rank] - x[r][rank[0]]) / case["temperature"])
        keep = min(V, case["top_k"] or V)
        if case["top_p"] < 1.0:
            mass = np.cumsum(w[:keep])
            keep = int(np.searchsorted(mass, float(np.float32(case["top_p"])) * mass[-1], side="left")) + 1
        if case["min_p"] > 0.0:
            keep = min(keep, int(np.count_nonzero(w >= float(np.float32(case["min_p"])))))
        probs[r, rank[:keep]] = w[:keep] / w[:keep].sum()
        cdf = np.cumsum(probs[r])
        tokens[r] = int(np.searchsorted(cdf, u[r] * cdf[-1], side="right"))
    return (tokens, probs) if case["probs"] else tokens
