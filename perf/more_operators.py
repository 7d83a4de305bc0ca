"""The operators of a decoding step over an 8-bit cache that is kept short, as cases that can be timed and checked.

append   the last rows of every sequence of a batch are rotated to their positions, quantised to 8 bits with one scale for
         each block of 32 positions and KV head, and written into the pages; the queries of the same rows are rotated on
         the way.  The blocks written to are then read back.
attend   the queries of the sequences over their pages: single tokens, verify rows, trees, prompts, also through a sliding
         window with first positions that stay visible, and with each row's log-sum-exp.
weights  the attention weight that every cached position gets from the rows, added to what it had.
evict    of every sequence and KV head the positions with the most weight stay, up to a budget, and are moved together.

A block is 32 positions of one KV head, keys and values apart.  With A the largest magnitude of what it holds (earlier
positions as they are stored, the call's rows as they come) its scale is the smallest 2^E, E in [-15, 8], with
A <= 448 2^E; a value x is held as the 8-bit float (4 exponent bits, 3 of mantissa) nearest to x / 2^E, halves to even.

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
BLOCK = 32
MAX_POS = 1 << 17


def listed():
    ragged = "9001,33,4096,700,1,2222,64,5113,1500,31,8192,257,6000,12,3001,450"
    return [
        # one token for each sequence of a serving batch, two of the rows padding; most blocks hold positions already
        dict(name="append_batch37", op="append", heads="qwen7b", dtype="f16", lengths="1*37", start=9000, page=64, pad=2),
        # long prompts filled in behind what their sequences have
        dict(name="append_prompt16384", op="append", heads="llama8b", dtype="f16", lengths="9001,7383", start=77, page=64, pad=0),
        # one token of each sequence of a ragged batch
        dict(name="attend_batch", op="attend", heads="qwen7b", rows=1, lengths=ragged, mask="causal", page=64, window=0, sinks=0,
             lse=False),
        # the verify step of four drafts at a long context
        dict(name="attend5_long", op="attend", heads="llama8b", rows=5, lengths="32768", mask="causal", page=64, window=0, sinks=0,
             lse=False),
        # a draft tree at a long context
        dict(name="attend_tree60", op="attend", heads="llama8b", rows=60, lengths="8192", mask="tree", page=32, window=0, sinks=0,
             lse=False),
        # a chunk of a long prompt over what came before, with the statistics that scoring its positions needs
        dict(name="attend_prompt2048", op="attend", heads="llama8b", rows=2048, lengths="8191", mask="causal", page=128, window=0,
             sinks=0, lse=True),
        # single tokens of long sequences that look back a fixed distance
        dict(name="window_step", op="attend", heads="llama8b", rows=1, lengths="60000,120001,4097,31007", mask="causal", page=64,
             window=4096, sinks=4, lse=False),
        # a chunk of a prompt that looks back a fixed distance
        dict(name="window_prompt2048", op="attend", heads="small", rows=2048, lengths="16001", mask="causal", page=64, window=1024,
             sinks=64, lse=False),
        # after a decoding step of a small batch: its weights go to the running sums
        dict(name="weights_step", op="weights", heads="qwen7b", rows=1, lengths="5000,8191,33,2049", mask="causal", page=64, window=0,
             sinks=0),
        # the last rows of a prompt score its positions
        dict(name="weights_prompt512", op="weights", heads="llama8b", rows=512, lengths="16384", mask="causal", page=64, window=0,
             sinks=0),
        # a serving batch whose sequences passed their budget, some of them not yet
        dict(name="evict_batch", op="evict", heads="qwen7b", lengths="2176,2177,2300,2048,2500,1000,4095,2176", budget=2048, sinks=4,
             recent=256, page=64),
        # a long prompt cut down before decoding
        dict(name="evict_prompt32768", op="evict", heads="llama8b", lengths="32768", budget=4096, sinks=4, recent=512, page=64),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "weights", "evict"])
    heads = rng.choice(sorted(HEADS))
    page = rng.choice([32, 64, 128, 256])
    if op == "append":
        total = _log(rng, 1, 12000)
        seqs = min(total, rng.choice([1, 1, 2, 5, 31]))
        cuts = sorted(rng.sample(range(1, total), seqs - 1)) if seqs > 1 else []
        lengths = [b - a for a, b in zip([0] + cuts, cuts + [total])]
        return dict(op=op, heads=heads, dtype=rng.choice(["f16", "f32"]), lengths=",".join(map(str, lengths)),
                    start=rng.choice([0, _log(rng, 1, 20000)]), page=page, pad=rng.choice([0, 0, 3]))
    if op == "evict":
        seqs = rng.choice([1, 1, 2, 6])
        lengths = [_log(rng, 1, 32000 // seqs) for _ in range(seqs)]
        budget = _log(rng, 1, 4096)
        sinks = min(budget, rng.choice([0, 4, 33]))
        return dict(op=op, heads=heads, lengths=",".join(map(str, lengths)), budget=budget, sinks=sinks,
                    recent=min(budget - sinks, rng.choice([0, _log(rng, 1, 1000)])), page=page)
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
    window = rng.choice([0, _log(rng, 1, 8192)])
    case = dict(op=op, heads=heads, rows=rows, lengths=",".join(map(str, lengths)), mask=mask, page=page, window=window,
                sinks=rng.choice([0, 4, 50]) if window else 0)
    if op == "attend":
        case["lse"] = rng.choice([False, True])
    return case


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


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(case, seed, lengths, tag=5):
    """(table [sequences][pages], pages given out): a sequence's pages lie anywhere."""
    need = [max(1, -(-n // case["page"])) for n in lengths]
    ids = torch.randperm(sum(need) + 3, generator=torch.Generator().manual_seed(int(seed) + tag))[:sum(need)].tolist()
    table = torch.full((len(lengths), max(need)), -1, dtype=torch.int32)
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
    return table, sum(need) + 3


def _append_inputs(case, seed):
    """The call's rows, and those that the first block of each sequence's range holds already."""
    H, KV, hd, _, _ = HEADS[case["heads"]]
    lengths, pad = _lengths(case), case["pad"]
    # the sequences begin at different places, whatever the seed
    jitter = torch.randint(0, 1 + case["start"] // 2, (len(lengths),), generator=torch.Generator().manual_seed(7)).tolist()
    starts = [case["start"] - j for j in jitter]
    held = [a % BLOCK for a in starts]
    dt = torch.float16 if case["dtype"] == "f16" else torch.float32
    n = sum(lengths) + pad
    q, k, v = (_rows_of(seed, t, n, h, hd).to(dt) for t, h in ((1, H), (2, KV), (3, KV)))
    hk, hv = (_rows_of(seed, t, max(1, sum(held)), KV, hd).to(dt) for t in (4, 5))
    # earlier positions of one sequence in eight are far larger than what comes, or far smaller
    for s in range(0, len(held), 8):
        a = sum(held[:s])
        hv[a:a + held[s]] *= 30.0 if s % 16 else 0.01
    ends = [a + m for a, m in zip(starts, lengths)]
    return dict(q=q, k=k, v=v, hk=hk, hv=hv, starts=starts, held=held, ends=ends)


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
    total = sum(lengths)
    return dict(q=_rows_of(seed, 1, rows * len(lengths), H, hd).half(), k=_rows_of(seed, 2, total, KV, hd).half(),
                v=_rows_of(seed, 3, total, KV, hd).half(), mask=_tree_mask(seed, rows) if case["mask"] == "tree" else None)


def _previous(case, seed):
    """Running sums: a few positions have most of the weight, some none."""
    KV, T = HEADS[case["heads"]][1], max(_lengths(case))
    x = torch.randn((len(_lengths(case)), KV, T), generator=_gen(seed, 6), device="cuda").mul(2.0).exp()
    return torch.where(torch.rand(x.shape, generator=_gen(seed, 7), device="cuda") < 0.2, 0.0, x)


def _evict_inputs(case, seed):
    KV, hd = HEADS[case["heads"]][1:3]
    total = sum(_lengths(case))
    return dict(k=_rows_of(seed, 2, total, KV, hd).half(), v=_rows_of(seed, 3, total, KV, hd).half(), scores=_previous(case, seed))


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


def _two_to(e):
    """2^e exactly, in 64 bits"""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _blocks(x, block, n_blocks):
    """x [rows][heads][hd] in 64 bits, row r in block[r] -> (codes as 8-bit floats in bytes, exponents [n_blocks][heads])"""
    top = torch.zeros((n_blocks, x.shape[1]), dtype=torch.float64, device=x.device)
    top.scatter_reduce_(0, block[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    m, e = torch.frexp(top / 448.0)  # top / 448 = m 2^e, m in [1/2, 1)
    e = torch.where(top == 0, -15, e - (m == 0.5).int()).clamp(-15, 8)
    y = x * _two_to(-e[block][..., None])
    # the spacing of 8-bit floats at y: 2^-9 up to 2^-6, above it an eighth of the power of two below y
    spacing = _two_to((torch.frexp(y)[1] - 4).clamp(min=-9))
    y = (y / spacing).round() * spacing
    return y.float().to(torch.float8_e4m3fn).view(torch.uint8), e


def _values(codes, exps):
    """codes [rows][heads][hd] with exponents [rows][heads] -> fp32"""
    return codes.view(torch.float8_e4m3fn).float() * _two_to(exps[..., None]).float()


def _append_blocks(inp):
    """(of every row of the blocks written to, in order: its block, its place among the call's rows, or -1 - its place among
    those held; blocks in all)"""
    block, at, base, new, old = [], [], 0, 0, 0
    for a, end, held in zip(inp["starts"], inp["ends"], inp["held"]):
        first = a - held
        block += [base + (p - first) // BLOCK for p in range(first, end)]
        at += [-1 - (old + i) for i in range(held)] + [new + i for i in range(end - a)]
        base, new, old = base + -(-(end - first) // BLOCK), new + end - a, old + held
    return torch.tensor(block, device="cuda"), torch.tensor(at, device="cuda"), base


def _positions(starts, ends):
    return torch.tensor([p for a, b in zip(starts, ends) for p in range(a, b)], dtype=torch.int64, device="cuda")


def _plain_held(inp, cos, sin, pairs):
    """What the first blocks hold before the call, as stored."""
    pos = _positions([a - h for a, h in zip(inp["starts"], inp["held"])], inp["starts"])
    seq = torch.tensor([s for s, h in enumerate(inp["held"]) for _ in range(h)], dtype=torch.int64, device="cuda")
    out = []
    for name in ("hk", "hv"):
        x = inp[name][:len(pos)].double()
        if name == "hk":
            x = _rotate(x, cos[pos].double(), sin[pos].double(), pairs)
        codes, e = _blocks(x, seq, len(inp["held"]))
        out.append((codes, e[seq]))
    return out


def _plain_append(st):
    inp, (H, KV, hd, pairs, _) = st["inp"], HEADS[st["case"]["heads"]]
    pos, n = st["pos"], len(st["pos"])
    cos, sin = st["cos"][pos], st["sin"][pos]
    q = torch.zeros((len(inp["q"]), H, hd), dtype=torch.float16, device="cuda")
    q[:n] = _rotate(inp["q"][:n].float(), cos, sin, pairs).half()
    outs = [q]
    for name, held in zip(("k", "v"), st["held"]):
        x = inp[name][:n].double()
        if name == "k":
            x = _rotate(x, cos.double(), sin.double(), pairs)
        new = st["at"] >= 0
        rows = torch.empty((len(new), KV, hd), dtype=torch.float64, device="cuda")
        rows[new] = x[st["at"][new]]
        rows[~new] = _values(*held).double()
        codes, e = _blocks(rows, st["block"], st["n_blocks"])
        outs.append(_values(codes, e[st["block"]]).half())
    return outs


def _plain_cache(case, inp, table, n_pages):
    """The cache of whole sequences: codes by position and exponents by block, page after page."""
    H, KV, hd, pairs, base = HEADS[case["heads"]]
    cos, sin = _tables(hd, base)
    page, out = case["page"], {}
    for name in ("k", "v"):
        codes = torch.zeros((n_pages * page, KV, hd), dtype=torch.uint8, device="cuda")
        exps = torch.zeros((n_pages * page // BLOCK, KV), dtype=torch.int32, device="cuda")
        first = 0
        for s, T in enumerate(_lengths(case)):
            for a in range(0, T, 16384):
                p = torch.arange(a, min(T, a + 16384), device="cuda")
                x = inp[name][first + p].double()
                if name == "k":
                    x = _rotate(x, cos[p].double(), sin[p].double(), pairs)
                c, e = _blocks(x, (p - a) // BLOCK, -(-len(p) // BLOCK))
                at = table[s].cuda()[p // page].long() * page + p % page
                codes[at] = c
                exps[at[::BLOCK] // BLOCK] = e
            first += T
        out[name] = (codes, exps)
    return out


def _held_rows(cache, table, page, s, p):
    """(keys, values) at positions p of sequence s, fp32"""
    at = table[s, p // page].long() * page + p % page
    return tuple(_values(c[at], e[at // BLOCK]) for c, e in (cache["k"], cache["v"]))


def _visible(case, T, mask, dev):
    """[rows][T]: what the last rows of T positions see"""
    rows = case["rows"]
    i, j = torch.arange(rows, device=dev)[:, None] + (T - rows), torch.arange(T, device=dev)[None]
    seen = j <= i
    if mask is not None:
        b = (j - (T - rows)).clamp(min=0)
        bits = (mask[:, (b[0] // 64).clamp(max=mask.shape[1] - 1)] >> (b % 64)) & 1
        seen = (j < T - rows) | (bits == 1)
    if case["window"]:
        seen = seen & ((j < case["sinks"]) | (j > i - case["window"]))
    return seen


def _plain_scores(st, s, T):
    """Per KV head: scores [rows x heads][T] of sequence s with -inf where nothing is seen, and the head's values"""
    case, inp, (H, KV, hd, _, _) = st["case"], st["inp"], HEADS[st["case"]["heads"]]
    rows, rep = case["rows"], H // KV
    k, v = _held_rows(st["cache"], st["table"], case["page"], s, torch.arange(T, device="cuda"))
    seen = _visible(case, T, inp["mask"], "cuda")
    q = inp["q"][s * rows:(s + 1) * rows].float().unflatten(1, (KV, rep))
    for h in range(KV):
        x = (q[:, h].reshape(-1, hd) @ k[:, h].T * (1.0 / math.sqrt(hd))).view(rows, rep, T)
        yield x.masked_fill(~seen[:, None], -math.inf).view(-1, T), v[:, h]


def _plain_attend(st):
    case, (H, KV, hd, _, _) = st["case"], HEADS[st["case"]["heads"]]
    rows, rep, n = case["rows"], H // KV, case["rows"] * len(_lengths(case))
    out = torch.empty((n, H, hd), dtype=torch.float16, device="cuda")
    lse = torch.empty((n, H), device="cuda")
    for s, T in enumerate(_lengths(case)):
        for h, (x, v) in enumerate(_plain_scores(st, s, T)):
            top = x.amax(-1, keepdim=True)
            top = torch.where(top == -math.inf, 0.0, top)
            w = (x - top).exp()
            total = w.sum(-1, keepdim=True)
            o = torch.where(total > 0, (w @ v) / total, 0.0)
            out[s * rows:(s + 1) * rows, h * rep:(h + 1) * rep] = o.view(rows, rep, hd).half()
            lse[s * rows:(s + 1) * rows, h * rep:(h + 1) * rep] = (top + total.log()).view(rows, rep)
    return (out, lse) if case.get("lse") or case["op"] == "weights" else out


def _plain_weights(st):
    case, (H, KV, hd, _, _) = st["case"], HEADS[st["case"]["heads"]]
    rows, rep = case["rows"], H // KV
    out = st["previous"].clone()
    for s, T in enumerate(_lengths(case)):
        for h, (x, _) in enumerate(_plain_scores(st, s, T)):
            lse = st["lse"][s * rows:(s + 1) * rows, h * rep:(h + 1) * rep].reshape(-1, 1)
            out[s, h, :T] += torch.where(lse == -math.inf, 0.0, (x - lse).exp()).sum(0)
    return out


def _plain_evict(st):
    case, inp, KV = st["case"], st["inp"], HEADS[st["case"]["heads"]][1]
    B, first, last, lengths = case["budget"], case["sinks"], case["recent"], _lengths(case)
    kept = torch.full((len(lengths), KV, B), -1, dtype=torch.int32, device="cuda")
    scores = torch.zeros((len(lengths), KV, B), device="cuda")
    keys, values = [], []
    for s, T in enumerate(lengths):
        n, x = min(T, B), inp["scores"][s, :, :T]
        if T > B:
            middle = first + torch.sort(x[:, first:T - last], dim=-1, descending=True, stable=True)[1][:, :B - first - last]
            ends = [torch.arange(a, b, device="cuda").expand(KV, -1) for a, b in ((0, first), (T - last, T))]
            at = torch.cat((ends[0], middle, ends[1]), 1).sort(-1)[0]
        else:
            at = torch.arange(T, device="cuda").expand(KV, -1)
        kept[s, :, :n] = at.int()
        scores[s, :, :n] = x.gather(1, at)
        for x, out in zip(_held_rows(st["cache"], st["table"], case["page"], s, torch.arange(T, device="cuda")), (keys, values)):
            x = x.transpose(0, 1).gather(1, at[..., None].expand(-1, -1, x.shape[-1])).transpose(0, 1)
            block = torch.arange(n, device="cuda") // BLOCK
            codes, e = _blocks(x.double(), block, -(-n // BLOCK))
            out.append(_values(codes, e[block]).half())
    return kept, torch.minimum(st["kv_len"], torch.full_like(st["kv_len"], B)), scores, torch.cat(keys), torch.cat(values)


# ---- one pass ----------------------------------------------------------------------
def _library():
    path = os.path.join(os.getcwd(), "abyo-speculate_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import speculate_hip
    return speculate_hip


def _pool(case, n_pages):
    H, KV, hd, pairs, base = HEADS[case["heads"]]
    return _library().HipKv8Pool(n_layers=1, n_heads=H, n_kv_heads=KV, head_dim=hd, n_pages=n_pages, page_tokens=case["page"],
                                 max_pos=MAX_POS, rope_theta=base, interleaved=pairs)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _starts(counts):
    return _i32([sum(counts[:i]) for i in range(len(counts) + 1)])


def _append(pool, table, row_start, kv_len, max_rows, k, v, q=0, q_out=0):
    S = _library()
    pool.append(0, len(k), row_start.data_ptr(), kv_len.data_ptr(), table.data_ptr(), table.shape[0], table.shape[1],
                max_rows=max_rows, k=k.data_ptr(), v=v.data_ptr(), dtype=S.F32 if k.dtype == torch.float32 else S.F16, q=q,
                q_out=q_out, stream=_stream())


def _read(pool, st, k_out, v_out):
    table = st["read_table"]
    pool.read(0, len(k_out), st["read_slot"].data_ptr(), table.data_ptr(), table.shape[0], table.shape[1], k_out.data_ptr(),
              v_out.data_ptr(), seqs=st["read_seq"].data_ptr(), stream=_stream())


def _rows_to_read(st, starts, ends, KV, hd):
    st["read_slot"] = _positions(starts, ends).int()
    st["read_seq"] = _i32([s for s, (a, b) in enumerate(zip(starts, ends)) for _ in range(a, b)])
    st["k_out"], st["v_out"] = (torch.zeros((len(st["read_slot"]), KV, hd), dtype=torch.float16, device="cuda") for _ in range(2))


def prepare(case, seed):
    st = dict(case=case)
    H, KV, hd, pairs, base = HEADS[case["heads"]]
    if case["op"] == "append":
        st["inp"] = inp = _append_inputs(case, seed)
        starts, ends, held = inp["starts"], inp["ends"], inp["held"]
        table, n_pages = _pages(case, seed, ends)
        if own:
            st["pool"], st["table"] = _pool(case, n_pages), table.cuda()
            st["read_table"], st["kv_len"] = st["table"], _i32(ends)
            counts = _lengths(case)
            st["starts"], st["max_rows"] = _starts(counts), max(counts)
            if sum(held):
                _append(st["pool"], st["table"], _starts(held), _i32(starts), max(held), inp["hk"], inp["hv"])
            _rows_to_read(st, [a - h for a, h in zip(starts, held)], ends, KV, hd)
            st["q_out"] = torch.zeros((len(inp["q"]), H, hd), dtype=torch.float16, device="cuda")
        else:
            st["cos"], st["sin"] = _tables(hd, base)
            st["held"] = _plain_held(inp, st["cos"], st["sin"], pairs)
            st["block"], st["at"], st["n_blocks"] = _append_blocks(inp)
            st["pos"] = _positions(starts, ends)
        return st
    st["inp"] = inp = (_evict_inputs if case["op"] == "evict" else _attend_inputs)(case, seed)
    lengths = _lengths(case)
    table, n_pages = _pages(case, seed, lengths)
    st["table"], st["kv_len"] = table.cuda(), _i32(lengths)
    if case["op"] == "weights":
        # the statistics of the step that is scored, the same for both forms
        st["cache"] = _plain_cache(case, inp, table, n_pages)
        st["lse"], st["previous"] = _plain_attend(st)[1], _previous(case, seed)
        if own:
            del st["cache"]
    if own:
        n_new = 0
        if case["op"] == "evict":
            B = case["budget"]
            new_table, n_new = _pages(case, seed, [min(T, B) for T in lengths], tag=6)
            st["read_table"] = torch.where(new_table < 0, new_table, new_table + n_pages).cuda()
            _rows_to_read(st, [0] * len(lengths), [min(T, B) for T in lengths], KV, hd)
            st["kept"] = torch.empty((len(lengths), KV, B), dtype=torch.int32, device="cuda")
            st["new_len"], st["scores"] = torch.empty_like(st["kv_len"]), torch.zeros((len(lengths), KV, B), device="cuda")
        st["pool"] = pool = _pool(case, n_pages + n_new)
        _append(pool, st["table"], _starts(lengths), st["kv_len"], max(lengths), inp["k"], inp["v"])
        if case["op"] != "evict":
            rows = case["rows"]
            n = rows * len(lengths)
            st["starts"] = _starts([rows] * len(lengths))
            st["out"] = torch.zeros((n, H, hd), dtype=torch.float16, device="cuda")
            if case["op"] == "weights":
                st["sums"] = st["previous"].clone()
            else:
                st["lse"] = torch.zeros((n, H), device="cuda") if case["lse"] else None
                st["ws"] = torch.zeros(pool.attend_workspace(n, len(lengths), rows, max(lengths), window=case["window"],
                                                             sinks=case["sinks"]), dtype=torch.uint8, device="cuda")
    elif "cache" not in st:
        st["cache"] = _plain_cache(case, inp, table, n_pages)
    del inp["k"], inp["v"]
    return st


def run(state):
    case, inp = state["case"], state["inp"]
    op = case["op"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "weights": _plain_weights, "evict": _plain_evict}[op](state)
    pool, table = state["pool"], state["table"]
    if op == "append":
        _append(pool, table, state["starts"], state["kv_len"], state["max_rows"], inp["k"], inp["v"], inp["q"].data_ptr(),
                state["q_out"].data_ptr())
        _read(pool, state, state["k_out"], state["v_out"])
        return state["q_out"], state["k_out"], state["v_out"]
    if op == "evict":
        pool.evict(0, state["kv_len"].data_ptr(), table.data_ptr(), table.shape[0], table.shape[1], scores=inp["scores"].data_ptr(),
                   scores_ld=inp["scores"].shape[2], budget=case["budget"], sinks=case["sinks"], recent=case["recent"],
                   kept=state["kept"].data_ptr(), new_len=state["new_len"].data_ptr(), scores_out=state["scores"].data_ptr(),
                   new_table=state["read_table"].data_ptr(), new_table_ld=state["read_table"].shape[1], stream=_stream())
        _read(pool, state, state["k_out"], state["v_out"])
        return state["kept"], state["new_len"], state["scores"], state["k_out"], state["v_out"]
    mask, lengths = inp["mask"], _lengths(case)
    common = dict(row_start=state["starts"].data_ptr(), kv_len=state["kv_len"].data_ptr(), table=table.data_ptr(), n_seqs=table.shape[0],
                  table_ld=table.shape[1], rows=len(inp["q"]), max_rows=case["rows"], max_len=max(lengths),
                  mask=0 if mask is None else mask.data_ptr(), mask_words=0 if mask is None else mask.shape[1], window=case["window"],
                  sinks=case["sinks"], stream=_stream())
    if op == "weights":
        pool.weights(0, inp["q"].data_ptr(), state["lse"].data_ptr(), state["sums"].data_ptr(), state["sums"].shape[2],
                     previous=state["previous"].data_ptr(), **common)
        return state["sums"]
    lse, ws = state["lse"], state["ws"]
    pool.attend(0, inp["q"].data_ptr(), state["out"].data_ptr(), lse=0 if lse is None else lse.data_ptr(), ws=ws.data_ptr(),
                ws_bytes=ws.numel(), **common)
    return state["out"] if lse is None else (state["out"], lse)


def _pairs(case):
    """(pairs of a row and a position that it sees, positions that some row sees)"""
    pairs = union = 0
    rows, W, S = case["rows"], case["window"], case["sinks"]
    for T in _lengths(case):
        for i in range(rows):
            end = T - rows + (i + 1 if case["mask"] == "causal" else 1)
            pairs += end if not W else min(end, W) + min(S, max(0, end - W))
        union += T if not W else min(T, W + rows - 1) + min(S, max(0, T - W - rows + 1))
    return pairs, union


def work(case):
    H, KV, hd, _, _ = HEADS[case["heads"]]
    lengths = _lengths(case)
    row8 = KV * hd  # one position's keys or values
    if case["op"] == "append":
        n, size = sum(lengths), 2 if case["dtype"] == "f16" else 4
        # rows in, queries out, codes out and in again, values out
        return {"bytes": n * ((H + 2 * KV) * hd * size + H * hd * 2 + 4 * row8 + 4 * row8), "flops": n * (H + 3 * KV) * hd * 3}
    if case["op"] == "evict":
        kept = sum(min(T, case["budget"]) for T in lengths)
        # scores in, kept positions' rows in, out and read back, indexes and scores out
        return {"bytes": 4 * KV * sum(lengths) + kept * (3 * 2 * row8 + 4 * row8 + 8 * KV), "flops": KV * sum(lengths)}
    pairs, union = _pairs(case)
    rows = case["rows"] * len(lengths)
    if case["op"] == "weights":
        return {"bytes": union * row8 + rows * H * (2 * hd + 4) + 8 * KV * sum(lengths), "flops": 2 * pairs * H * hd}
    return {"bytes": 2 * union * row8 + 4 * rows * H * hd, "flops": 4 * pairs * H * hd}


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


def _nearest8(y):
    """The nearest of the finite 8-bit floats, by search among all of them; a half goes to the even code"""
    grid = torch.tensor([math.ldexp(c, -9) if c < 8 else math.ldexp(8 + c % 8, c // 8 - 10) for c in range(127)],
                        dtype=torch.float64, device=y.device)
    a = y.abs()
    hi = torch.searchsorted(grid, a).clamp(1, 126)
    lo = hi - 1
    down, up = a - grid[lo], grid[hi] - a
    pick = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    return torch.where(y < 0, -grid[pick], grid[pick])


def _stored(x):
    """What consecutive rows x [rows][heads][hd] stand for, from the first position of a block"""
    out = torch.empty_like(x)
    for a in range(0, len(x), 8192):
        part = x[a:a + 8192]
        pad = -len(part) % BLOCK
        b = torch.cat((part, part.new_zeros((pad,) + part.shape[1:]))).unflatten(0, (-1, BLOCK))
        top = b.abs().amax((1, 3))
        scale = torch.full_like(top, 2.0 ** 8)
        for e in range(7, -16, -1):
            scale = torch.where(top <= 448.0 * 2.0 ** e, 2.0 ** e, scale)
        scale = scale[:, None, :, None]
        out[a:a + 8192] = (_nearest8(b / scale) * scale).flatten(0, 1)[:len(part)]
    return out


def _exact_append(case, seed):
    H, KV, hd, pairs, base = HEADS[case["heads"]]
    inp = _append_inputs(case, seed)
    q = torch.zeros((len(inp["q"]), H, hd), dtype=torch.float64, device="cuda")
    keys, values, new, old = [], [], 0, 0
    for a, end, held in zip(inp["starts"], inp["ends"], inp["held"]):
        pos = torch.arange(a - held, end, device="cuda")
        q[new:new + end - a] = _turned(inp["q"][new:new + end - a], pos[held:], base, pairs)
        was = [_stored(_turned(inp["hk"][old:old + held], pos[:held], base, pairs)), _stored(inp["hv"][old:old + held].double())]
        now = [_turned(inp["k"][new:new + end - a], pos[held:], base, pairs), inp["v"][new:new + end - a].double()]
        for out, x, y in zip((keys, values), was, now):
            out.append(_stored(torch.cat((x, y))))
        new, old = new + end - a, old + held
    return [q, torch.cat(keys), torch.cat(values)]


def _exact_seen(case, T, mask):
    rows, W = case["rows"], case["window"]
    seen = torch.ones((rows, T), dtype=torch.bool)
    seen[:, T - rows:] = torch.tril(torch.ones((rows, rows), dtype=torch.bool))
    if mask is not None:
        words = mask.cpu().numpy().view(np.uint64)
        for i in range(rows):
            whole = sum(int(w) << (64 * n) for n, w in enumerate(words[i]))
            seen[i, T - rows:] = torch.tensor([bool(whole >> j & 1) for j in range(rows)])
    if W:
        for i in range(rows):
            seen[i, min(case["sinks"], T):max(min(case["sinks"], T), T - rows + i - W + 1)] = False
    return seen.cuda()


def exact(case, seed):
    if case["op"] == "append":
        return _exact_append(case, seed)
    H, KV, hd, pairs, base = HEADS[case["heads"]]
    if case["op"] == "evict":
        return _exact_evict(case, _evict_inputs(case, seed))
    inp = _attend_inputs(case, seed)
    rows, at, outs, stats = case["rows"], 0, [], []
    sums = _previous(case, seed).double() if case["op"] == "weights" else None
    for s, T in enumerate(_lengths(case)):
        k = _stored(_turned(inp["k"][at:at + T], torch.arange(T, device="cuda"), base, pairs))
        v = _stored(inp["v"][at:at + T].double())
        at += T
        q = inp["q"][s * rows:(s + 1) * rows].double()
        seen = _exact_seen(case, T, inp["mask"])
        out = torch.empty((rows, H, hd), dtype=torch.float64, device="cuda")
        lse = torch.empty((rows, H), dtype=torch.float64, device="cuda")
        for h in range(H):
            score = q[:, h] @ k[:, h * KV // H].T / math.sqrt(hd)
            score[~seen] = -math.inf
            lse[:, h] = torch.logsumexp(score, -1)
            p = torch.softmax(score, -1)
            if sums is None:
                out[:, h] = p @ v[:, h * KV // H]
            else:
                sums[s, h * KV // H, :T] += p.sum(0)
        outs.append(out)
        stats.append(lse)
    if sums is not None:
        return sums
    return (torch.cat(outs), torch.cat(stats)) if case["lse"] else torch.cat(outs)


def _exact_evict(case, inp):
    H, KV, hd, pairs, base = HEADS[case["heads"]]
    B, lengths, score = case["budget"], _lengths(case), inp["scores"].cpu().numpy()
    kept = np.full((len(lengths), KV, B), -1, np.int32)
    moved = np.zeros((len(lengths), KV, B))
    keys, values, at = [], [], 0
    for s, T in enumerate(lengths):
        n = min(T, B)
        k = _stored(_turned(inp["k"][at:at + T], torch.arange(T, device="cuda"), base, pairs))
        v = _stored(inp["v"][at:at + T].double())
        at += T
        for h in range(KV):
            rank = score[s, h, :T].astype(np.float64).copy()
            rank[:case["sinks"]] = np.inf
            rank[T - min(T, case["recent"]):] = np.inf
            stay = np.sort(np.lexsort((np.arange(T), -rank))[:n])
            kept[s, h, :n] = stay
            moved[s, h, :n] = score[s, h, stay]
        at_h = torch.from_numpy(kept[s, :, :n].astype(np.int64)).cuda()
        for x, out in ((k, keys), (v, values)):
            out.append(_stored(torch.stack([x[at_h[h], h] for h in range(KV)], 1)))
    return kept, np.minimum(np.array(lengths, np.int32), B), moved, torch.cat(keys), torch.cat(values)
